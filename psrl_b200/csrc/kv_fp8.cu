// 8-bit paged KV cache: rotary embedding fused with the quantised write of new
// keys and values, and pages read back as bf16.
//
// A vector x (one token's key or value of one kv head, d = 64 or 128) is held
// as d float8 e4m3 codes and one exponent byte:
//   e    = min { e in [-63, 120] : max|x| <= 448 * 2^e }     (-63 for a zero vector)
//   code = e4m3(x * 2^-e), round to nearest even;  byte = e + 127
//   value = code * 2^(byte - 127)
// A power-of-two scale costs a float code no precision, makes x * 2^-e and the
// value exact (the value is exact in bf16 too), and needs no division.  A
// vector with a NaN or an infinity gets byte 255 and reads as NaN.
//
// rope_quant_kernel: eight lanes per (token, head), 16 values each (8 of the
// lower half, their 8 rotary partners): two 16-byte loads per lane, the rotation
// in fp32 without contraction (every product and difference rounded once, so
// the codes do not depend on how the compiler fuses), keys rounded to bf16
// before they are quantised (the numbers a bf16 cache would hold), max|x| as an
// integer maximum over the eight lanes.  cos / sin stay in registers for the HV
// heads a lane group handles.  Bound by HBM bytes: (nq + 2 nkv) * 2d in,
// nq * 2d + 2 nkv (d + 1) out per token.  Measured on a B200: 10240 tokens at random
// slots, 32 q / 8 kv heads, 50 us (4.7 TB/s); HV 1, 2 and 6 gave 54, 51 and 58.
// read_kv_kernel: 3001 pages of 8 heads x 64 tokens 104 us (5.7 TB/s).
#include <cuda_fp8.h>

#include "common.cuh"

namespace psrl {

namespace {

struct RopeQuantArgs {
  const bf16* qkv;
  int64_t row;
  const int* pos;
  const float* cos_t;
  const float* sin_t;
  int table_rows;
  bf16* q_out;
  uint8_t *k, *v, *ks, *vs;
  const int* slots;
  int64_t num_slots;
  int T, nq, nkv, block_size;
};

// largest |x| of eight packed bf16 pairs as the bf16 bit pattern (infinities and
// NaNs order above every finite value)
__device__ __forceinline__ uint32_t absmax_bits(const uint32_t* w, int n) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < n; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

// exponent byte of a vector whose largest |x| has these bf16 bits
__device__ __forceinline__ uint32_t exponent_byte(uint32_t bits) {
  if (bits >= 0x7f80u) return 255u;
  const int e = (int)(bits >> 7) - 135 + ((bits & 127u) > 96u ? 1 : 0);  // 448 = 1.75 * 2^8, 1.75 = 1 + 96 / 128
  return (uint32_t)(min(max(e, -63), 120) + 127);
}

__device__ __forceinline__ uint2 codes8(const uint32_t* w, float inv) {
  uint16_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const bf162*>(w + i));
    c[i] = __nv_cvt_float2_to_fp8x2(make_float2(f.x * inv, f.y * inv), __NV_SATFINITE, __NV_E4M3);
  }
  return make_uint2(c[0] | ((uint32_t)c[1] << 16), c[2] | ((uint32_t)c[3] << 16));
}

template <int D, int HV>
__global__ void __launch_bounds__(256) rope_quant_kernel(RopeQuantArgs a) {
  constexpr int HALF = D / 2;
  constexpr int L = HALF / 8;         // lanes per head
  constexpr int PER_WARP = 32 / L;    // heads a warp handles at once
  const int heads = a.nq + 2 * a.nkv;
  const int groups = (heads + PER_WARP * HV - 1) / (PER_WARP * HV);
  const int64_t warp = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, sub = lane / L, j = lane % L;
  const int t = (int)(warp / groups);
  if (t >= a.T) return;
  const int h0 = (int)(warp % groups) * PER_WARP * HV + sub;
  const bf16* row = a.qkv + (int64_t)t * a.row;
  uint4 lo[HV], hi[HV];
#pragma unroll
  for (int i = 0; i < HV; ++i) {
    const int h = h0 + i * PER_WARP;
    if (h < heads) {
      lo[i] = *reinterpret_cast<const uint4*>(row + (int64_t)h * D + j * 8);
      hi[i] = *reinterpret_cast<const uint4*>(row + (int64_t)h * D + HALF + j * 8);
    }
  }
  const int ps = a.pos[t];
  const int slot = a.slots[t];
  const bool in_table = ps >= 0 && ps < a.table_rows;
  float c[8], s[8];
  if (h0 < a.nq + a.nkv) {
#pragma unroll
    for (int k = 0; k < 8; k += 4) {
      // a position outside the table has no angle: its rows become NaN
      float4 cv = make_float4(NAN, NAN, NAN, NAN), sv = cv;
      if (in_table) {
        cv = *reinterpret_cast<const float4*>(a.cos_t + (int64_t)ps * HALF + j * 8 + k);
        sv = *reinterpret_cast<const float4*>(a.sin_t + (int64_t)ps * HALF + j * 8 + k);
      }
      c[k] = cv.x; c[k + 1] = cv.y; c[k + 2] = cv.z; c[k + 3] = cv.w;
      s[k] = sv.x; s[k + 1] = sv.y; s[k + 2] = sv.z; s[k + 3] = sv.w;
    }
  }
  const bool store = slot >= 0 && slot < a.num_slots;
  const int64_t blk = store ? slot / a.block_size : 0;
  const int off = store ? slot % a.block_size : 0;
#pragma unroll
  for (int i = 0; i < HV; ++i) {
    const int h = h0 + i * PER_WARP;
    const bool live = h < heads;
    uint32_t w[8];
    if (live) {
      *reinterpret_cast<uint4*>(w) = lo[i];
      *reinterpret_cast<uint4*>(w + 4) = hi[i];
      if (h < a.nq + a.nkv) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<const bf162*>(w + k));
          const float2 y = __bfloat1622float2(*reinterpret_cast<const bf162*>(w + 4 + k));
          const float c0 = c[2 * k], c1 = c[2 * k + 1], s0 = s[2 * k], s1 = s[2 * k + 1];
          const bf162 ra = __floats2bfloat162_rn(__fsub_rn(__fmul_rn(x.x, c0), __fmul_rn(y.x, s0)),
                                                 __fsub_rn(__fmul_rn(x.y, c1), __fmul_rn(y.y, s1)));
          const bf162 rb = __floats2bfloat162_rn(__fadd_rn(__fmul_rn(y.x, c0), __fmul_rn(x.x, s0)),
                                                 __fadd_rn(__fmul_rn(y.y, c1), __fmul_rn(x.y, s1)));
          w[k] = *reinterpret_cast<const uint32_t*>(&ra);
          w[4 + k] = *reinterpret_cast<const uint32_t*>(&rb);
        }
      }
      if (h < a.nq) {
        bf16* dst = a.q_out + (int64_t)t * a.nq * D + (int64_t)h * D + j * 8;
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(w);
        *reinterpret_cast<uint4*>(dst + HALF) = *reinterpret_cast<const uint4*>(w + 4);
      }
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) w[k] = 0;
    }
    uint32_t m = absmax_bits(w, 8);
#pragma unroll
    for (int o = 1; o < L; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (live && h >= a.nq && store) {
      const bool is_k = h < a.nq + a.nkv;
      const int hk = is_k ? h - a.nq : h - a.nq - a.nkv;
      const int64_t vec = (blk * a.nkv + hk) * a.block_size + off;
      const uint32_t byte = exponent_byte(m);
      const float inv = byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);  // 2^-(byte - 127)
      if (byte == 255u) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k] = 0;
      }
      uint8_t* dst = (is_k ? a.k : a.v) + vec * D + j * 8;
      *reinterpret_cast<uint2*>(dst) = codes8(w, inv);
      *reinterpret_cast<uint2*>(dst + HALF) = codes8(w + 4, inv);
      if (j == 0) (is_k ? a.ks : a.vs)[vec] = (uint8_t)byte;
    }
  }
}

// One thread per 16 codes: 16 bytes in, 32 out.
template <int D>
__global__ void __launch_bounds__(256)
    read_kv_kernel(const uint8_t* __restrict__ cache, const uint8_t* __restrict__ scale,
                   const int* __restrict__ blocks, int64_t n, int64_t num_blocks, int rows, bf16* __restrict__ out,
                   const int* __restrict__ out_blocks, int64_t out_num) {
  constexpr int C = D / 16;
  const int64_t per_block = (int64_t)rows * C;
  const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= n * per_block) return;
  const int64_t p = i / per_block;
  const int rest = (int)(i - p * per_block), r = rest / C, c = rest % C;
  const int64_t src = blocks[p], dst = out_blocks ? out_blocks[p] : p;
  if (src < 0 || src >= num_blocks || dst < 0 || dst >= out_num) return;
  const uint4 w = *reinterpret_cast<const uint4*>(cache + ((src * rows + r) * C + c) * 16);
  const uint32_t byte = scale[src * rows + r];
  const float f = byte == 255u ? NAN : (byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23));
  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
  uint32_t o[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(ws[k >> 1] >> (16 * (k & 1))), __NV_E4M3);
    const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&h));
    const bf162 b = __floats2bfloat162_rn(x.x * f, x.y * f);
    o[k] = *reinterpret_cast<const uint32_t*>(&b);
  }
  uint4* d = reinterpret_cast<uint4*>(out + ((dst * rows + r) * C + c) * 16);
  d[0] = make_uint4(o[0], o[1], o[2], o[3]);
  d[1] = make_uint4(o[4], o[5], o[6], o[7]);
}

}  // namespace

// Shared checks of an 8-bit cache and its exponent bytes.
static void check_cache(const at::Tensor& cache, const at::Tensor& scale, const char* name) {
  TORCH_CHECK(cache.is_cuda() && cache.scalar_type() == at::kFloat8_e4m3fn && cache.dim() == 4 &&
                  cache.is_contiguous() && reinterpret_cast<uintptr_t>(cache.data_ptr()) % 16 == 0,
              name, " must be a contiguous float8_e4m3fn CUDA tensor [blocks, nkv, block_size, d]");
  TORCH_CHECK(scale.is_cuda() && scale.scalar_type() == at::kByte && scale.is_contiguous() && scale.dim() == 3 &&
                  scale.size(0) == cache.size(0) && scale.size(1) == cache.size(1) && scale.size(2) == cache.size(2) &&
                  scale.device() == cache.device(),
              name, "'s exponents must be contiguous uint8 [blocks, nkv, block_size] on its device");
}

// qkv [T, (nq + 2 nkv) * d] bf16 (rows may be strided) is left as it is; returns
// the rotated queries [T, nq * d] and writes the rotated keys and the values of
// every token with a slot in [0, blocks * block_size) into the 8-bit caches.
at::Tensor rope_quant_kv(at::Tensor qkv, at::Tensor positions, at::Tensor cos_t, at::Tensor sin_t, int64_t nq,
                         int64_t nkv, int64_t d, at::Tensor k_cache, at::Tensor v_cache, at::Tensor k_scale,
                         at::Tensor v_scale, at::Tensor slots) {
  CHECK_CUDA_TENSOR(qkv);
  CHECK_DTYPE(qkv, at::kBFloat16);
  TORCH_CHECK(d == 128 || d == 64, "head_dim must be 64 or 128");
  TORCH_CHECK(nq > 0 && nkv > 0 && qkv.dim() == 2 && qkv.size(1) == (nq + 2 * nkv) * d,
              "qkv must be [T, (nq + 2 nkv) * d]");
  TORCH_CHECK(qkv.stride(1) == 1 && qkv.stride(0) % 8 == 0 && reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
              "qkv rows must start on 16-byte boundaries with unit inner stride");
  check_cache(k_cache, k_scale, "k_cache");
  check_cache(v_cache, v_scale, "v_cache");
  TORCH_CHECK(k_cache.sizes() == v_cache.sizes() && k_cache.size(1) == nkv && k_cache.size(3) == d,
              "k_cache and v_cache must both be [blocks, nkv, block_size, d]");
  const int64_t T = qkv.size(0);
  for (const at::Tensor* t : {&positions, &slots})
    TORCH_CHECK(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == T && t->is_contiguous() &&
                    t->device() == qkv.device(),
                "positions and slots must be int32 [T] on qkv's device");
  for (const at::Tensor* t : {&cos_t, &sin_t})
    TORCH_CHECK(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == d / 2 && t->is_contiguous() &&
                    t->device() == qkv.device() && t->size(0) == cos_t.size(0),
                "rotary tables must be fp32 [positions, d / 2] on qkv's device");
  TORCH_CHECK(k_cache.device() == qkv.device() && v_cache.device() == qkv.device(), "caches must be on qkv's device");
  at::cuda::CUDAGuard g(qkv.device());
  auto q_out = at::empty({T, nq * d}, qkv.options());
  if (T == 0) return q_out;
  RopeQuantArgs a{};
  a.qkv = reinterpret_cast<const bf16*>(qkv.data_ptr());
  a.row = qkv.stride(0);
  a.pos = positions.data_ptr<int>();
  a.cos_t = cos_t.data_ptr<float>();
  a.sin_t = sin_t.data_ptr<float>();
  a.table_rows = (int)std::min<int64_t>(cos_t.size(0), 0x7fffffff);
  a.q_out = reinterpret_cast<bf16*>(q_out.data_ptr());
  a.k = reinterpret_cast<uint8_t*>(k_cache.data_ptr());
  a.v = reinterpret_cast<uint8_t*>(v_cache.data_ptr());
  a.ks = k_scale.data_ptr<uint8_t>();
  a.vs = v_scale.data_ptr<uint8_t>();
  a.slots = slots.data_ptr<int>();
  a.num_slots = k_cache.size(0) * k_cache.size(2);
  a.T = (int)T;
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.block_size = (int)k_cache.size(2);
  const int per_warp = 32 / ((int)d / 16);
  const int64_t heads = nq + 2 * nkv;
  auto blocks = [&](int hv) {
    const int64_t warps = T * ((heads + per_warp * hv - 1) / (per_warp * hv));
    return (unsigned)((warps + 7) / 8);
  };
  // Heads per lane group: one while the launch would leave SMs without a block,
  // else four (their loads in flight together, cos / sin read once for them).
  if (T * heads < (int64_t)num_sms() * 8 * per_warp * 4) {
    if (d == 128) rope_quant_kernel<128, 1><<<blocks(1), 256, 0, stream()>>>(a);
    else rope_quant_kernel<64, 1><<<blocks(1), 256, 0, stream()>>>(a);
  } else {
    if (d == 128) rope_quant_kernel<128, 4><<<blocks(4), 256, 0, stream()>>>(a);
    else rope_quant_kernel<64, 4><<<blocks(4), 256, 0, stream()>>>(a);
  }
  PSRL_CHECK_LAUNCH();
  return q_out;
}

// out[out_blocks[i]] = values of cache[blocks[i]] (bf16); out_blocks empty: out[i].
// Pairs with an id outside their tensor are skipped.
void read_kv_cache(at::Tensor cache, at::Tensor scale, at::Tensor blocks, at::Tensor out,
                   c10::optional<at::Tensor> out_blocks) {
  check_cache(cache, scale, "cache");
  const int64_t d = cache.size(3), n = blocks.numel();
  TORCH_CHECK(d == 128 || d == 64, "head_dim must be 64 or 128");
  TORCH_CHECK(blocks.scalar_type() == at::kInt && blocks.dim() == 1 && blocks.is_contiguous() &&
                  blocks.device() == cache.device(),
              "blocks must be int32 [n] on the cache's device");
  TORCH_CHECK(out.scalar_type() == at::kBFloat16 && out.dim() == 4 && out.is_contiguous() &&
                  out.device() == cache.device() && out.size(1) == cache.size(1) && out.size(2) == cache.size(2) &&
                  out.size(3) == d && reinterpret_cast<uintptr_t>(out.data_ptr()) % 16 == 0,
              "out must be contiguous bf16 [m, nkv, block_size, d] on the cache's device");
  const int* ob = nullptr;
  if (out_blocks.has_value()) {
    TORCH_CHECK(out_blocks->scalar_type() == at::kInt && out_blocks->numel() == n && out_blocks->is_contiguous() &&
                    out_blocks->device() == cache.device(),
                "out_blocks must be int32 [n] on the cache's device");
    ob = out_blocks->data_ptr<int>();
  } else {
    TORCH_CHECK(out.size(0) >= n, "out holds fewer than n pages");
  }
  const int64_t rows = cache.size(1) * cache.size(2);
  const int64_t threads = n * rows * (d / 16);
  if (threads == 0) return;
  at::cuda::CUDAGuard g(cache.device());
  const unsigned grid = (unsigned)((threads + 255) / 256);
  auto run = [&](auto kern) {
    kern<<<grid, 256, 0, stream()>>>(reinterpret_cast<const uint8_t*>(cache.data_ptr()), scale.data_ptr<uint8_t>(),
                                     blocks.data_ptr<int>(), n, cache.size(0), (int)rows,
                                     reinterpret_cast<bf16*>(out.data_ptr()), ob, out.size(0));
  };
  if (d == 128) run(read_kv_kernel<128>);
  else run(read_kv_kernel<64>);
  PSRL_CHECK_LAUNCH();
}

}  // namespace psrl
