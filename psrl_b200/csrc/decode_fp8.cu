// Paged decode attention over the 8-bit KV cache (head_dim 128): one query token
// per sequence, optional sliding window and sinks.
//
//   o = softmax(scale * q K^T over the visible keys) V
//
// Bound by the cache bytes: 2 * 129 per (key, kv head).  What the design does
// about it:
//
//  * Equal shares.  The 64-key tiles of all (sequence, kv head) pairs form one
//    list; every resident CTA takes an equal contiguous share of it, whatever
//    the lengths, so ragged batches leave no SM waiting.  A CTA whose share
//    cuts a pair writes a partial (normalised fp32 row, base-2 log-sum); a
//    second small launch joins the partials in tile order.  The shares are
//    computed on the device from kv_lens, so one captured graph serves all lengths.
//  * A producer warp keeps NS tiles (K, V: TMA boxes with the 128-byte swizzle;
//    exponent bytes: 4-byte cp.async) in flight over an mbarrier ring, across
//    pair boundaries.
//  * Four consumer warps take 16 keys of each tile.  The products are taken
//    transposed, S^T = K Q^T and O^T += V^T P^T, so that the 16 rows of an
//    m16n8k16 are keys (columns of V) and its 8 columns the query heads of the
//    group: groups of up to 8 heads waste nothing (NT = 1), 9 to 16 take two
//    column tiles.  P^T gets from accumulator to operand layout with movmatrix.
//  * Fragments come straight out of the swizzled tile with conflict-free 16-byte
//    loads: the contraction order over d and the output order over d are permuted
//    so that a thread's fragment is the 32 consecutive codes 32t.. of keys g and
//    g+8 (K) and the 16 consecutive codes 16g.. of keys 2t, 2t+1, 2t+8, 2t+9 (V).
//  * e4m3 -> f16 is one conversion per pair, exact; f16 products with fp32
//    accumulation.  A query row is scaled by a power of two so that its largest
//    value is in [2^14, 2^15) (its bf16 values are then exact in f16 down to 2^-31
//    of the largest), and the probabilities keep f16's 11 bits.
//  * The exponents cost nothing per element: 2^ek scales a row of S^T, and
//    P 2^ev is the second product's operand, with the running maximum taken over
//    log2(p) + ev so that it stays within f16's range.
//
// Measured on a B200: 48 sequences up to 32768 tokens, 32 q / 8 kv heads, 336 us
// (6.3 TB/s, 97% of copy bandwidth); 64 sequences up to 9216, 16 / 2 heads, 50 us
// (4.1 TB/s: 28 tiles per CTA, so start, merge and join show); one of 517 tokens 10.8
// us in a graph.  With the heads as rows (16 of them, half of them empty) and codes
// converted by masks it was 555 us: 620 instructions per warp and tile against 400.
#include "checks.cuh"
#include "common.cuh"
#include "driver_api.h"
#include "kv8.cuh"
#include "tcgen05.cuh"

namespace psrl {
namespace dec8 {

using namespace tc5;

constexpr int D = 128;
constexpr int TK = 64;                        // keys per tile
constexpr int NS = 3;                         // ring depth
constexpr int TILE = TK * D;                  // 8 KB of codes
constexpr int STAGE = 2 * TILE;               // K, V
constexpr int OFF_EXP = NS * STAGE;           // per stage: 64 K exponents, 64 V exponents
constexpr int OFF_MERGE = OFF_EXP + NS * 2 * TK;
constexpr int MROW = 132;                     // merge row pitch in floats (conflict-free float2 stores)
constexpr int NTHREADS = 160;                 // 4 consumer warps + producer
constexpr float GROW = 8.0f;                  // rescale O when the running maximum grows by more than 2^8

struct Args {
  const bf16* q;
  int64_t q_row;
  const uint8_t *ks, *vs;
  int64_t num_blocks;
  const int* block_table;
  int64_t bt_row;
  const int* kv_lens;
  int B, nq, nkv, max_blocks, block_size, window, sinks;
  int workers;
  float scale_log2;
  bf16* o;
  float* part_o;    // [2 * workers][16][D]
  float* part_lse;  // [2 * workers][16], base 2
  int* err;
};

// Visible 64-key tiles of a sequence: tiles [0, ns) hold the sinks, then tiles
// w0 .. end of the window.
struct Tiles {
  int len, lo, ns, w0, n;
  __device__ __forceinline__ int key0(int i) const { return (i < ns ? i : i - ns + w0) * TK; }
};
__device__ __forceinline__ Tiles tiles_of(const Args& a, int b) {
  Tiles t;
  t.len = max(0, min(a.kv_lens[b], a.max_blocks * a.block_size));
  t.lo = a.window > 0 ? max(0, t.len - a.window) : 0;
  t.w0 = t.lo / TK;
  t.ns = min((min(a.sinks, t.lo) + TK - 1) / TK, t.w0);
  t.n = t.ns + (t.len + TK - 1) / TK - t.w0;
  return t;
}

__device__ __forceinline__ void mma_f16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// an 8 x 8 matrix of 16-bit values, a row per four lanes, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// Block-wide scan over the sequences: returns the number of items (tiles of all
// pairs); thread i has sequences [lo, hi), the first of which starts at item `before`.
template <int NT>
__device__ __forceinline__ int64_t scan_items(const Args& a, int64_t* sh, int64_t* before, int* lo, int* hi) {
  const int per = (a.B + NT - 1) / NT;
  *lo = min(a.B, (int)threadIdx.x * per);
  *hi = min(a.B, *lo + per);
  int64_t mine = 0;
  for (int b = *lo; b < *hi; ++b) mine += tiles_of(a, b).n;
  mine *= a.nkv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) sh[warp] = inc;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NT / 32; ++w) {
    if (w < warp) base += sh[w];
    total += sh[w];
  }
  *before = base + inc - mine;
  return total;
}
__device__ __forceinline__ int64_t share_of(int64_t total, int workers) {
  return max((int64_t)1, (total + workers - 1) / workers);
}

constexpr int smem_bytes(int nt) { return OFF_MERGE + 4 * 8 * nt * MROW * 4 + 1024; }
constexpr int resident(int nt) { return nt == 1 ? 3 : 2; }  // CTAs per SM

template <int NT>
__global__ void __launch_bounds__(NTHREADS, resident(NT))
    decode8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, Args a) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t bars[2 * NS];
  __shared__ int64_t s_scan[NTHREADS / 32];
  __shared__ int64_t s_first;
  __shared__ int s_b;
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ volatile int s_abort;
  __shared__ volatile int s_fail;  // a consumer warp gave up (written by consumers only)
  const uint32_t full = smem_u32(bars), empty = full + 8 * NS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    s_abort = 0;
    s_fail = 0;
    s_b = a.B;
    for (int i = 0; i < NS; ++i) {
      mbar_init(full + 8 * i, 33);  // the TMA bytes' arrive and one per producer lane (exponent bytes)
      mbar_init(empty + 8 * i, 4);  // one arrive per consumer warp
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  int64_t before;
  int blo, bhi;
  const int64_t total = scan_items<NTHREADS>(a, s_scan, &before, &blo, &bhi);
  const int64_t per = share_of(total, a.workers);
  const int64_t start = (int64_t)blockIdx.x * per, stop = min(total, start + per);
  kv8::launch_dependents();
  if (start >= total) return;  // uniform
  for (int b = blo; b < bhi; ++b) {
    const int64_t n = (int64_t)tiles_of(a, b).n * a.nkv;
    if (start >= before && start < before + n) {
      s_b = b;
      s_first = before;
    }
    before += n;
  }
  __syncthreads();
  int b = s_b;
  Tiles tl = tiles_of(a, b);
  int hk = (int)((start - s_first) / tl.n);
  int i = (int)((start - s_first) - (int64_t)hk * tl.n);
  const int count = (int)(stop - start);

  if (warp == 4) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
    const int rows = min(TK, a.block_size);  // rows of one TMA box
    const int* bt = a.block_table + (int64_t)b * a.bt_row;
    for (int it = 0; it < count; ++it) {
      const int st = it % NS;
      bool ok = true;
      if (it >= NS) ok = mbar_wait(empty + 8 * st, ((it / NS) & 1) ^ 1);
      if (!__all_sync(0xffffffffu, ok) || s_abort) {
        if (lane == 0) {
          if (!s_abort && a.err) atomicCAS(a.err, 0, 41);
          s_abort = 1;
        }
        break;
      }
      const int key0 = tl.key0(i);
      const uint32_t sk = smem_u32(smem) + st * STAGE, sv = sk + TILE, fb = full + 8 * st;
      // exponent bytes: lanes 0..15 four keys of K each, lanes 16..31 of V;
      // pages past the end and ids outside the cache read as zeros
      {
        const int key = key0 + (lane & 15) * 4;
        const int page = key / a.block_size;
        const int blk = page < a.max_blocks && key < tl.len ? bt[page] : -1;
        const bool in = blk >= 0 && blk < a.num_blocks;
        const uint8_t* src = lane < 16 ? a.ks : a.vs;
        if (in) src += ((int64_t)blk * a.nkv + hk) * a.block_size + key % a.block_size;
        const uint32_t dst = smem_u32(smem) + OFF_EXP + st * 2 * TK + lane * 4;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(in ? 4 : 0) : "memory");
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(fb) : "memory");
      }
      if (lane == 0) {
        mbar_expect_tx(fb, STAGE);
        for (int r = 0; r < TK; r += rows) {
          const int key = key0 + r, page = key / a.block_size;
          // a box outside the tensor is filled with zeros
          int y = -TK;
          if (page < a.max_blocks && key < tl.len) {
            const int blk = bt[page];
            if (blk >= 0 && blk < a.num_blocks) y = (blk * a.nkv + hk) * a.block_size + key % a.block_size;
          }
          tma_load_2d(sk + r * D, &tmK, 0, y, fb);
          tma_load_2d(sv + r * D, &tmV, 0, y, fb);
        }
      }
      if (++i == tl.n) {
        i = 0;
        if (++hk == a.nkv && it + 1 < count) {
          hk = 0;
          do tl = tiles_of(a, ++b);
          while (tl.n == 0);
          bt = a.block_table + (int64_t)b * a.bt_row;
        }
      }
    }
    return;
  }

  // ---------------------------------------------------------------- consumers
  const int g = lane >> 2, t = lane & 3;
  const int grp = a.nq / a.nkv;
  float* merge = reinterpret_cast<float*>(smem + OFF_MERGE);
  const int base = warp * 16;  // this warp's keys of a tile
  // offsets within a tile of this thread's K rows g, g+8 (16-byte chunks 2t, 2t+1) and
  // V rows 2t, 2t+1, 2t+8, 2t+9 (chunk g); row & 7 does not depend on the warp
  const int ko = (base + g) * D + (((2 * t) ^ g) << 4);
  const int v0o = (base + 2 * t) * D + ((g ^ (2 * t)) << 4), v1o = (base + 2 * t + 1) * D + ((g ^ (2 * t + 1)) << 4);
  int it = 0;
  bool ok = true;
  while (it < count) {
    const int seg0 = i, seg = min(tl.n - i, count - it);  // tiles of this pair in this share
    // queries: head 8u + g, the fragment words of step k hold d = 32t + 4k + {0, 1} and {2, 3}
    uint32_t qf[NT][8][2];
    float fr[NT][2];  // heads 8u + 2t, +1: scale * log2(e) and the f16 scaling of the head's query
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      const int head = 8 * u + g;
      uint4 w[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        w[c] = make_uint4(0, 0, 0, 0);
        if (head < grp)
          w[c] = *reinterpret_cast<const uint4*>(a.q + (int64_t)b * a.q_row + (int64_t)(hk * grp + head) * D + 32 * t +
                                                 8 * c);
      }
      const uint32_t* x = reinterpret_cast<const uint32_t*>(w);
      uint32_t m = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = __vmaxu2(m, x[k] & 0x7fff7fffu);
      m = max(m & 0xffffu, m >> 16);
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
      // 2^(14 - E) for a largest value in [2^E, 2^(E+1)); both it and its inverse stay finite
      const int up = min(max(14 - ((int)(m >> 7) - 127), -113), 126);
      const float f = __uint_as_float((uint32_t)(up + 127) << 23);
      const float back = a.scale_log2 * __uint_as_float((uint32_t)(127 - up) << 23);
      fr[u][0] = __shfl_sync(0xffffffffu, back, 8 * t);      // from the lanes of head 2t
      fr[u][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);  // and 2t + 1
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const float2 y = __bfloat1622float2(*reinterpret_cast<const bf162*>(x + 2 * k + c));
          const half2 h = __floats2half2_rn(y.x * f, y.y * f);
          qf[u][k][c] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    float o[NT][8][4];  // rows d = 16g + 2k, + 1; columns heads 8u + 2t, + 1
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int k = 0; k < 8; ++k) o[u][k][0] = o[u][k][1] = o[u][k][2] = o[u][k][3] = 0.f;
    float m_r[NT][2], l_r[NT][2];
#pragma unroll
    for (int u = 0; u < NT; ++u) {
      m_r[u][0] = m_r[u][1] = -INFINITY;
      l_r[u][0] = l_r[u][1] = 0.f;
    }

    for (int e = 0; e < seg; ++e, ++it, ++i) {
      const int st = it % NS;
      ok = mbar_wait(full + 8 * st, (it / NS) & 1) && !s_abort;
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      const uint8_t* kt = smem + st * STAGE;
      const uint8_t* vt = kt + TILE;
      const uint8_t* ex = smem + OFF_EXP + st * 2 * TK + base;
      uint32_t ka[8], kb[8];  // codes of keys g and g + 8
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        *reinterpret_cast<uint4*>(ka + 4 * c) = *reinterpret_cast<const uint4*>(kt + (ko ^ (c << 4)));
        *reinterpret_cast<uint4*>(kb + 4 * c) = *reinterpret_cast<const uint4*>(kt + 8 * D + (ko ^ (c << 4)));
      }
      const uint32_t ek0 = ex[g], ek1 = ex[g + 8], ev0 = ex[TK + g], ev1 = ex[TK + g + 8];
      uint32_t v[4][4];
      *reinterpret_cast<uint4*>(v[0]) = *reinterpret_cast<const uint4*>(vt + v0o);
      *reinterpret_cast<uint4*>(v[1]) = *reinterpret_cast<const uint4*>(vt + v1o);
      *reinterpret_cast<uint4*>(v[2]) = *reinterpret_cast<const uint4*>(vt + 8 * D + v0o);
      *reinterpret_cast<uint4*>(v[3]) = *reinterpret_cast<const uint4*>(vt + 8 * D + v1o);
      float s[NT][4];
#pragma unroll
      for (int u = 0; u < NT; ++u) s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t f[4] = {kv8::f16_of2(ka[k]), kv8::f16_of2(kb[k]), kv8::f16_of2_hi(ka[k]), kv8::f16_of2_hi(kb[k])};
#pragma unroll
        for (int u = 0; u < NT; ++u) mma_f16(s[u], f, qf[u][k][0], qf[u][k][1]);
      }
      float kf[2] = {__uint_as_float(ek0 << 23), __uint_as_float(ek1 << 23)};         // 2^ek
      float vf[2] = {(float)((int)ev0 - 127), (float)((int)ev1 - 127)};               // ev
      // keys outside the context or the window, and exponents of 255: rare tiles
      const int tile0 = tl.key0(i) + base;
      const bool edge = tile0 + 16 > tl.len || (tile0 < tl.lo && tile0 + 16 > a.sinks);
      if (__any_sync(0xffffffffu, edge || max(max(ek0, ek1), max(ev0, ev1)) == 255u)) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int key = tile0 + g + 8 * c;
          if (!(key < tl.len && (key >= tl.lo || key < a.sinks))) {
            kf[c] = 1.f;
            vf[c] = 0.f;
#pragma unroll
            for (int u = 0; u < NT; ++u) s[u][2 * c] = s[u][2 * c + 1] = -INFINITY;
          } else if ((c ? ek1 : ek0) == 255u || (c ? ev1 : ev0) == 255u) {
            kf[c] = vf[c] = NAN;
          }
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          // whatever the page holds in rows nobody sees: 0 * NaN would be one
          const int key = tile0 + 2 * t + (c & 1) + 8 * (c >> 1);
          if (!(key < tl.len && (key >= tl.lo || key < a.sinks))) v[c][0] = v[c][1] = v[c][2] = v[c][3] = 0;
        }
      }
      float y[NT][4], f[NT][4], top[NT][2];
      bool grow = false;
#pragma unroll
      for (int u = 0; u < NT; ++u) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[u][k] = fr[u][k & 1] * kf[k >> 1];
          y[u][k] = fmaf(s[u][k], f[u][k], vf[k >> 1]);
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float m = fmaxf(y[u][c], y[u][2 + c]);
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
          m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
          top[u][c] = m;
          grow |= m > m_r[u][c] + GROW || (m_r[u][c] == -INFINITY && m > m_r[u][c]);
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          float corr[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float mn = fmaxf(m_r[u][c], top[u][c]);
            corr[c] = m_r[u][c] == -INFINITY ? 0.f : ex2(m_r[u][c] - mn);
            m_r[u][c] = mn;
            l_r[u][c] *= corr[c];
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            o[u][k][0] *= corr[0];
            o[u][k][1] *= corr[1];
            o[u][k][2] *= corr[0];
            o[u][k][3] *= corr[1];
          }
        }
      }
      uint32_t pf[NT][2];
#pragma unroll
      for (int u = 0; u < NT; ++u) {
        const float r0 = m_r[u][0] == -INFINITY ? 0.f : m_r[u][0], r1 = m_r[u][1] == -INFINITY ? 0.f : m_r[u][1];
#pragma unroll
        for (int c = 0; c < 2; ++c) {  // keys g, g + 8
          const half2 h = __floats2half2_rn(ex2(y[u][2 * c] - r0), ex2(y[u][2 * c + 1] - r1));
          l_r[u][0] += ex2(fmaf(s[u][2 * c], f[u][2 * c], -r0));
          l_r[u][1] += ex2(fmaf(s[u][2 * c + 1], f[u][2 * c + 1], -r1));
          pf[u][c] = transpose8(*reinterpret_cast<const uint32_t*>(&h));
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        // codes of two keys side by side, for one column of V after the other
        const uint32_t a01 = __byte_perm(v[0][k], v[1][k], 0x5140), a23 = __byte_perm(v[0][k], v[1][k], 0x7362);
        const uint32_t b01 = __byte_perm(v[2][k], v[3][k], 0x5140), b23 = __byte_perm(v[2][k], v[3][k], 0x7362);
        const uint32_t f0[4] = {kv8::f16_of2(a01), kv8::f16_of2_hi(a01), kv8::f16_of2(b01), kv8::f16_of2_hi(b01)};
        const uint32_t f1[4] = {kv8::f16_of2(a23), kv8::f16_of2_hi(a23), kv8::f16_of2(b23), kv8::f16_of2_hi(b23)};
#pragma unroll
        for (int u = 0; u < NT; ++u) {
          mma_f16(o[u][2 * k], f0, pf[u][0], pf[u][1]);
          mma_f16(o[u][2 * k + 1], f1, pf[u][0], pf[u][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty + 8 * st);
    }
    if (!ok && lane == 0) {
      if (!s_abort && a.err) atomicCAS(a.err, 0, 42);
      s_abort = 1;
      s_fail = 1;
    }
    // ------------------------------------------------- join the four warps
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l_r[u][c] += __shfl_xor_sync(0xffffffffu, l_r[u][c], x);
        if (g == 0) {
          s_m[warp][8 * u + 2 * t + c] = m_r[u][c];
          s_l[warp][8 * u + 2 * t + c] = l_r[u][c];
        }
      }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (s_fail) return;  // uniform: not written between this barrier and the next
    // columns d = 16g + 2k, + 1 of a head's output sit at 16k + 2g
#pragma unroll
    for (int u = 0; u < NT; ++u)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int row = 8 * u + 2 * t + c;
        const float mg = fmaxf(fmaxf(s_m[0][row], s_m[1][row]), fmaxf(s_m[2][row], s_m[3][row]));
        const float cw = m_r[u][c] == -INFINITY ? 0.f : ex2(m_r[u][c] - mg);
        if (row < grp) {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            *reinterpret_cast<float2*>(merge + (warp * 8 * NT + row) * MROW + 16 * k + 2 * g) =
                make_float2(o[u][k][c] * cw, o[u][k][2 + c] * cw);
        }
      }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    const bool whole = seg0 == 0 && seg == tl.n;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (it == seg ? 0 : 1);  // the share's first pair, or its last
    for (int idx = threadIdx.x; idx < grp * D; idx += 128) {
      const int row = idx / D, d = idx % D, p = 16 * ((d >> 1) & 7) + 2 * (d >> 4) + (d & 1);
      float m = s_m[0][row];
#pragma unroll
      for (int w = 1; w < 4; ++w) m = fmaxf(m, s_m[w][row]);
      float l = 0.f, acc = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        l += s_m[w][row] == -INFINITY ? s_l[w][row] : s_l[w][row] * ex2(s_m[w][row] - m);
        acc += merge[(w * 8 * NT + row) * MROW + p];
      }
      // a NaN anywhere in the row's sums stays a NaN; nothing visible gives zeros
      const float val = l == 0.f ? 0.f : acc / l;
      if (whole) {
        a.o[((int64_t)b * a.nq + hk * grp + row) * D + d] = __float2bfloat16(val);
      } else {
        a.part_o[(slot * 16 + row) * D + d] = val;
        if (d == 0) a.part_lse[slot * 16 + row] = l == 0.f ? -INFINITY : m + log2f(l);
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // merge area and s_m are free again
    if (i == tl.n) {
      i = 0;
      if (++hk == a.nkv && it < count) {
        hk = 0;
        do tl = tiles_of(a, ++b);
        while (tl.n == 0);
      }
    }
  }
}

// One CTA per (sequence, query head): joins the partials of a pair that several
// CTAs shared, in tile order, and writes the rows of empty sequences.
__global__ void __launch_bounds__(128) decode8_join(Args a) {
  __shared__ int64_t s_scan[4];
  __shared__ int64_t s_first;
  __shared__ float s_m[4], s_l[4];
  __shared__ __align__(16) float s_o[4][D];
  const int b = blockIdx.x / a.nq, h = blockIdx.x % a.nq;
  const int grp = a.nq / a.nkv, hk = h / grp, row = h % grp;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t before;
  int blo, bhi;
  const int64_t total = scan_items<128>(a, s_scan, &before, &blo, &bhi);
  for (int k = blo; k < bhi; ++k) {
    if (k == b) s_first = before;
    before += (int64_t)tiles_of(a, k).n * a.nkv;
  }
  __syncthreads();
  const int64_t per = share_of(total, a.workers);
  const int n = tiles_of(a, b).n;
  kv8::wait_prior();  // every block: this kernel must not end before the one it follows
  bf16* out = a.o + ((int64_t)b * a.nq + h) * D;
  if (n == 0) {
    out[threadIdx.x] = __float2bfloat16(0.f);
    return;
  }
  const int64_t first = s_first + (int64_t)hk * n, last = first + n - 1;
  const int64_t w0 = first / per, w1 = last / per;
  if (w0 == w1) return;  // one CTA had the whole pair and wrote it
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int64_t w = w0 + warp; w <= w1; w += 4) {
    const int64_t slot = (2 * w + (w * per < first ? 1 : 0)) * 16 + row;
    const float lse = a.part_lse[slot];
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + slot * D + lane * 4);
    if (lse == -INFINITY) continue;
    const float mn = fmaxf(m, lse);  // a NaN lse makes c1 a NaN, which stays in the sums
    const float c0 = m == -INFINITY ? 0.f : ex2(m - mn), c1 = ex2(lse - mn);
    m = mn;
    l = l * c0 + c1;
    acc.x = acc.x * c0 + v.x * c1;
    acc.y = acc.y * c0 + v.y * c1;
    acc.z = acc.z * c0 + v.z * c1;
    acc.w = acc.w * c0 + v.w * c1;
  }
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  *reinterpret_cast<float4*>(&s_o[warp][lane * 4]) = acc;
  __syncthreads();
  float mg = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; ++w) mg = fmaxf(mg, s_m[w]);
  float den = 0.f, num = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (s_m[w] == -INFINITY && s_l[w] == 0.f) continue;
    const float c = ex2(s_m[w] - mg);
    den += s_l[w] * c;
    num += s_o[w][threadIdx.x] * c;
  }
  out[threadIdx.x] = __float2bfloat16(den == 0.f ? 0.f : num / den);
}

}  // namespace dec8

using namespace dec8;

// Paged decode over the 8-bit cache.  q [B, nq, 128] bf16 (rows may be strided),
// caches float8_e4m3fn [blocks, nkv, block_size, 128] with exponent bytes
// [blocks, nkv, block_size]; window 0 = none.
at::Tensor attn_decode_fp8(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, at::Tensor k_scale, at::Tensor v_scale,
                           at::Tensor block_table, at::Tensor kv_lens, double scale, int64_t window, int64_t sinks,
                           at::Tensor err) {
  CHECK_CUDA_TENSOR(q);
  CHECK_DTYPE(q, at::kBFloat16);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == D, "q must be [B, heads, 128]");
  TORCH_CHECK(q.stride(2) == 1 && q.stride(1) == D && q.stride(0) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "q rows must hold contiguous heads and start 16-byte aligned");
  const int64_t B = q.size(0), nq = q.size(1);
  kv8::check_paged(q, k_cache, v_cache, k_scale, v_scale, block_table, kv_lens, B);
  const int64_t nkv = k_cache.size(1);
  TORCH_CHECK(nq % nkv == 0 && nq / nkv <= 16, "GQA group must be <= 16");
  TORCH_CHECK(window >= 0 && sinks >= 0 && window < (1 << 30) && sinks < (1 << 30), "window and sinks must not be negative");
  at::cuda::CUDAGuard g(q.device());
  auto o = at::empty({B, nq, D}, q.options());
  if (B == 0) return o;
  const int64_t cap = block_table.size(1) * k_cache.size(2);
  TORCH_CHECK(cap < (1ll << 31) && B * nq < (1ll << 31), "block table too wide");
  if (cap == 0 || k_cache.size(0) == 0) return o.zero_();
  const CUtensorMap tk = kv8::map_codes(k_cache, TK, CU_TENSOR_MAP_SWIZZLE_128B),
                    tv = kv8::map_codes(v_cache, TK, CU_TENSOR_MAP_SWIZZLE_128B);
  Args a{};
  a.q = reinterpret_cast<const bf16*>(q.data_ptr());
  a.q_row = q.stride(0);
  a.ks = k_scale.data_ptr<uint8_t>();
  a.vs = v_scale.data_ptr<uint8_t>();
  a.num_blocks = k_cache.size(0);
  a.block_table = block_table.data_ptr<int>();
  a.bt_row = block_table.stride(0);
  a.kv_lens = kv_lens.data_ptr<int>();
  a.B = (int)B;
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.max_blocks = (int)block_table.size(1);
  a.block_size = (int)k_cache.size(2);
  a.window = (int)window;
  a.sinks = window > 0 ? (int)sinks : 0;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.o = reinterpret_cast<bf16*>(o.data_ptr());
  a.err = err.data_ptr<int>();
  // one column tile of up to 8 heads leaves room for three CTAs on an SM; never
  // more of them than tiles there can be
  const int nt = nq / nkv <= 8 ? 1 : 2;
  const int64_t most = B * nkv * ((cap + TK - 1) / TK);
  a.workers = (int)std::min<int64_t>(resident(nt) * num_sms(), most);
  auto part = at::empty({2 * a.workers * 16 * (D + 1)}, q.options().dtype(at::kFloat));
  a.part_o = part.data_ptr<float>();
  a.part_lse = a.part_o + 2ll * a.workers * 16 * D;
  static_assert(3 * (smem_bytes(1) + 2048) <= 228 * 1024 && 2 * (smem_bytes(2) + 2048) <= 228 * 1024, "resident CTAs");
  auto* kern = nt == 1 ? decode8_kernel<1> : decode8_kernel<2>;
  ensure_smem_attr(kern, smem_bytes(nt));
  kern<<<a.workers, NTHREADS, smem_bytes(nt), stream()>>>(tk, tv, a);
  PSRL_CHECK_LAUNCH();
  kv8::launch_after(decode8_join, (unsigned)(B * nq), 128u, a);
  return o;
}

}  // namespace psrl
