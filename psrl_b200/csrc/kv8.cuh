// Shared pieces of the kernels that read the 8-bit paged KV cache (kv_fp8.cu
// documents its format): argument checks, the TMA map over its pages and the
// code conversions.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "driver_api.h"

namespace psrl {
namespace kv8 {

// Two e4m3 codes (low byte first) as two f16, exactly; codes 0x7f and 0xff are NaN.
__device__ __forceinline__ uint32_t f16_of2(uint32_t codes) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(r) : "r"(codes));
  return r;
}
// The same for the high half of a word.
__device__ __forceinline__ uint32_t f16_of2_hi(uint32_t codes) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %1;\n cvt.rn.f16x2.e4m3x2 %0, hi;\n}" : "=r"(r) : "r"(codes));
  return r;
}

// Programmatic dependent launch: the joining kernel is put on the SMs while the
// kernel before it still runs (launch_dependents there), computes what needs no
// partials, and waits for that kernel's end and its writes (wait_prior).
__device__ __forceinline__ void launch_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }
__device__ __forceinline__ void wait_prior() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <typename... P, typename... A>
inline void launch_after(void (*kern)(P...), unsigned grid, unsigned block, A... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(grid);
  c.blockDim = dim3(block);
  c.stream = stream();
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at;
  c.numAttrs = 1;
  PSRL_CHECK_CUDA(cudaLaunchKernelEx(&c, kern, static_cast<P>(args)...));
}

// Tensor map over the codes: rows of 128 bytes (one vector each), boxes of
// min(tile, block_size) rows.
inline CUtensorMap map_codes(const at::Tensor& t, int tile, CUtensorMapSwizzle swizzle) {
  CUtensorMap m;
  const cuuint64_t rows = (cuuint64_t)(t.size(0) * t.size(1) * t.size(2));
  TORCH_CHECK(rows < (1ull << 31), "cache of more than 2^31 vectors");
  cuuint64_t dims[2] = {128, rows};
  cuuint64_t strides[1] = {128};
  cuuint32_t box[2] = {128u, (cuuint32_t)std::min<int64_t>(tile, t.size(2))};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = PSRL_DRV(cuTensorMapEncodeTiled)(&m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, t.data_ptr(), dims, strides, box,
                                                estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (", (int)r, ")");
  return m;
}

// Checks shared by the attention entry points over a paged cache; k_scale and
// v_scale undefined: a bf16 cache.
inline void check_paged(const at::Tensor& q, const at::Tensor& k_cache, const at::Tensor& v_cache,
                        const at::Tensor& k_scale, const at::Tensor& v_scale, const at::Tensor& block_table,
                        const at::Tensor& kv_lens, int64_t B) {
  const bool fp8 = k_scale.defined();
  TORCH_CHECK(k_cache.dim() == 4 && k_cache.sizes() == v_cache.sizes() && k_cache.size(3) == 128 &&
                  k_cache.size(1) > 0 && k_cache.size(2) > 0,
              "k_cache and v_cache must both be [blocks, nkv, block_size, 128]");
  for (const at::Tensor* t : {&k_cache, &v_cache})
    TORCH_CHECK(t->scalar_type() == (fp8 ? at::kFloat8_e4m3fn : at::kBFloat16) && t->is_contiguous() &&
                    t->device() == q.device() && reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                "caches must be contiguous ", fp8 ? "float8_e4m3fn" : "bf16", " on q's device, 16-byte aligned");
  if (fp8) {
    for (const at::Tensor* t : {&k_scale, &v_scale})
      TORCH_CHECK(t->scalar_type() == at::kByte && t->is_contiguous() && t->dim() == 3 &&
                      t->size(0) == k_cache.size(0) && t->size(1) == k_cache.size(1) &&
                      t->size(2) == k_cache.size(2) && t->device() == q.device() &&
                      reinterpret_cast<uintptr_t>(t->data_ptr()) % 16 == 0,
                  "exponents must be contiguous uint8 [blocks, nkv, block_size] on q's device, 16-byte aligned");
  }
  const int64_t bs = k_cache.size(2);
  TORCH_CHECK(bs >= 16 && (bs & (bs - 1)) == 0, "block_size must be a power of two >= 16");
  TORCH_CHECK(block_table.scalar_type() == at::kInt && block_table.dim() == 2 && block_table.size(0) == B &&
                  (block_table.size(1) == 0 || block_table.stride(1) == 1) && block_table.device() == q.device(),
              "block_table must be int32 [B, max_blocks] on q's device with unit inner stride");
  TORCH_CHECK(kv_lens.scalar_type() == at::kInt && kv_lens.dim() == 1 && kv_lens.size(0) == B &&
                  kv_lens.is_contiguous() && kv_lens.device() == q.device(),
              "kv_lens must be int32 [B] on q's device");
}

}  // namespace kv8
}  // namespace psrl
