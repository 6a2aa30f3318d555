// Attention of a chunk of new tokens per sequence over its paged context
// (head_dim 128), for an 8-bit cache (kv_fp8.cu documents its format) or a bf16
// one, with an optional sliding window and sinks, on tcgen05 / TMEM.
//
// The chunk's own keys are in the cache already: sequence b's n queries are the
// last n of its len positions, query p sees the keys j <= p with p - j < window
// or j < sinks.
//
//  * Packed heads.  A 128-row query tile holds 128 / g tokens x the g query heads
//    of one kv head (one 3-D TMA box per 64 columns), so a K/V tile is fetched and
//    converted once for all of them, and a few new tokens fill a tile.
//  * One CTA per (kv head, sequence, two query tiles A and B, part of the keys).
//    The tiles share every 128-key K/V tile, and the tensor core alternates
//    between them: S_g = Q_g K^T, softmax of the other tile meanwhile, O_g += P_g V
//    with P written back to tensor memory over S.
//      warp 0       TMA: Q, then K/V pages, found through the block table: bf16 ones
//                   straight into the MMA's tiles (128-byte swizzle); codes, with
//                   their exponent bytes, into a ring of raw half tiles
//      warp 1       MMA issuer
//      warps 4..11  softmax, one thread per row, tiles A and B
//      warps 12..19 8-bit cache: codes to bf16, exactly (bits moved into place, times
//                   a power of two), from the raw ring into the MMA's tiles; four
//                   warps for K, four for V, so that neither waits for the other's
//                   tile to become free
//    Values at or past len count as zeros, whatever their page holds.
//    With an 8-bit cache, registers are moved from the other warpgroups to the softmax.
//  * Few query tiles: the key tiles of a block are split over CTAs, whose partial
//    rows (fp32, with a base-2 log-sum) a second kernel joins in key order.
//  * A vector with exponent 255 reads as NaN.  A value vector's NaN is carried by
//    its key's scores and its own codes are read as zeros, so a row that does not
//    see the key is not touched by it (0 * NaN).
//
// Measured on a B200: 8192 new tokens over 24576, 32 q / 8 kv heads, bf16 pages 2.3 ms
// (1180 TFLOP/s), 8-bit 3.3 ms (835).  Both are bound by the chain softmax -> P V -> next
// S of a tile (two tiles in flight fill tensor memory); the 8-bit one also by shared
// memory, which the conversion's loads and stores share with the MMA's operands.  One
// warpgroup for K and V took 3.9 ms; K's codes as an e4m3 operand (Q as the sum of two
// e4m3 rows, nothing converted but V) 3.9 ms too: there every softmax thread has to
// fetch 128 key factors a tile.  Short chunks are bound by the number of key tiles of
// one CTA and its start and end: 9 sequences of up to 61 tokens over up to 8191, 16 q /
// 2 kv heads, 72 us.
#include "common.cuh"
#include "driver_api.h"
#include "kv8.cuh"
#include "tcgen05.cuh"

namespace psrl {
namespace chunk {

using namespace tc5;

constexpr int D = 128;
constexpr int BQ = 128, BKV = 128;
constexpr int ATOM = 128 * 64 * 2;  // 128 rows x 64 bf16 (one 128-byte swizzle atom column)
constexpr int TILE = 2 * ATOM;      // 32 KB
constexpr int OFF_K = 2 * TILE, OFF_V = OFF_K + 2 * TILE, OFF_BAR = OFF_V + 2 * TILE;
// 8-bit cache: ring of raw half tiles (64 keys): their codes, and per half 64 exponent
// bytes of K and 64 of V
constexpr int RK = BKV / 2, RAW = RK * D, NRAW = 4;
constexpr int OFF_RAW = OFF_BAR + 256, OFF_EXP = OFF_RAW + NRAW * RAW;
constexpr int smem_bytes(bool fp8) { return (fp8 ? OFF_EXP + NRAW * 2 * RK : OFF_BAR + 256) + 1024; }
static_assert(smem_bytes(true) <= 227 * 1024, "shared memory of a block");
constexpr int threads_of(bool fp8) { return fp8 ? 640 : 384; }
constexpr float RESCALE_LOG2 = 8.0f;

struct Args {
  const int* cu_q;
  const int* kv_lens;
  const int* block_table;
  int64_t bt_row;
  const uint8_t *ks, *vs;  // exponent bytes (8-bit cache)
  int64_t num_blocks;
  int T, nq, nkv, group, tok;  // tok: tokens per query tile
  int max_blocks, block_shift;
  int window, sinks, splits, blocks_z;
  int B, sms;
  float scale_log2;
  bf16* o;          // [T, nq, D]
  float* part_o;    // [splits][T][nq][D]
  float* part_lse;  // [splits][T][nq], base 2
  int* err;
};

__device__ __forceinline__ void set_err(int* err, int code, int it = -1) {
  if (err && atomicCAS(err, 0, code) == 0) {
    err[1] = blockIdx.x;
    err[2] = blockIdx.y;
    err[3] = blockIdx.z;
    err[4] = threadIdx.x >> 5;
    err[5] = it;
  }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(mbar)
      : "memory");
}

// Four e4m3 codes as two bf16 pairs holding value * 2^-120 (sign, exponent and
// mantissa bits moved into place; subnormal codes become subnormal bf16 numbers),
// times m (a power of two or NaN, in both halves).
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ void bf16_of4(uint32_t w, uint32_t m, uint32_t* out) {
  const uint32_t a = __byte_perm(w, 0, 0x1404), b = __byte_perm(w, 0, 0x3424);
  out[0] = mul_bf16x2((a & 0x80008000u) | ((a >> 4) & 0x07f007f0u), m);
  out[1] = mul_bf16x2((b & 0x80008000u) | ((b >> 4) & 0x07f007f0u), m);
}

template <bool FP8>
__global__ void __launch_bounds__(threads_of(FP8), 1)
    chunk_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                 const __grid_constant__ CUtensorMap tmV, Args a) {
  constexpr int NTHREADS = threads_of(FP8);
  const int hk = blockIdx.x, b = blockIdx.y;
  const int blk = a.blocks_z - 1 - (int)blockIdx.z / a.splits, part = (int)blockIdx.z % a.splits;
  const int s0 = max(0, min(a.cu_q[b], a.T)), n = min(a.cu_q[b + 1], a.T) - s0;
  if (b == (int)gridDim.y - 1 && blockIdx.z == 0) {
    // rows behind the last sequence are zeros (this kv head's query heads)
    const int64_t end = max(0, min(a.cu_q[b + 1], a.T)), per = a.group * (D / 8);
    for (int64_t i = end * per + threadIdx.x; i < (int64_t)a.T * per; i += NTHREADS)
      *reinterpret_cast<uint4*>(a.o + (i / per) * a.nq * D + (int64_t)hk * a.group * D + (i % per) * 8) =
          make_uint4(0, 0, 0, 0);
  }
  const int i0 = blk * 2 * a.tok;  // first token of the block
  if (i0 >= n) return;             // uniform, before any barrier
  const int len = max(0, min(a.kv_lens[b], a.max_blocks << a.block_shift));
  const int off = len - n;  // token i sits at position i + off
  const int iB = i0 + a.tok, iE = min(n, i0 + 2 * a.tok);
  // list of key tiles: entry j is tile j below ns, tile j + gap from there on
  const int w0 = a.window > 0 ? max(0, i0 + off - a.window + 1) / BKV : 0;
  const int ns = a.window > 0 ? min((a.sinks + BKV - 1) / BKV, w0) : 0;
  const int gap = w0 - ns;
  auto entries = [&](int last) { return last + off < 0 ? 0 : (last + off) / BKV + 1 - gap; };
  const int lA = entries(min(iB, n) - 1), lB = iB < n ? entries(iE - 1) : 0;
  const int all = max(lA, lB);
  // This part's share.  The parts of all blocks are equally long (at least two tiles), so that
  // together they are about one per SM whatever the lengths; a block has as many as it needs
  int per = all;
  __shared__ int s_tiles, s_blocks;
  if (a.splits > 1) {
    if (threadIdx.x == 0) s_tiles = s_blocks = 0;
    __syncthreads();
    int tiles = 0, blocks = 0;
    for (int i = threadIdx.x; i < a.B; i += NTHREADS) {
      const int ni = max(0, min(a.cu_q[i + 1], a.T) - max(0, min(a.cu_q[i], a.T)));
      const int li = max(0, min(a.kv_lens[i], a.max_blocks << a.block_shift));
      const int nb = (ni + 2 * a.tok - 1) / (2 * a.tok);
      int t = (li + BKV - 1) / BKV;
      if (a.window > 0) t = min(t, (min(a.window, 1 << 24) + min(a.sinks, 1 << 24) + 2 * a.tok + BKV - 1) / BKV + 1);
      tiles += nb * t;
      blocks += nb;
    }
    if (tiles) {
      atomicAdd(&s_tiles, tiles);
      atomicAdd(&s_blocks, blocks);
    }
    __syncthreads();
    const int spare = a.sms / a.nkv - s_blocks;
    if (spare > 0) per = (s_tiles + spare - 1) / spare;
    per = max(max(2, per), (all + a.splits - 1) / a.splits);
  }
  const int j0 = part * per, j1 = min(all, j0 + per);
  const int nA = max(0, min(lA, j1) - j0), nB = max(0, min(lB, j1) - j0), nK = max(nA, nB);
  auto key_tile = [&](int j) { return j + j0 < ns ? j + j0 : j + j0 + gap; };
  kv8::launch_dependents();
  if (part > 0 && nK == 0) {
    // nothing left for this part: its rows count for nothing in the join
    for (int i = threadIdx.x; i < (iE - i0) * a.group; i += NTHREADS)
      a.part_lse[(int64_t)part * a.T * a.nq + (int64_t)(s0 + i0 + i / a.group) * a.nq + hk * a.group + i % a.group] =
          -INFINITY;
    return;
  }

  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + OFF_BAR);
  const uint32_t bq = smem_u32(bars), bkf = bq + 8, bke = bkf + 16, bvf = bke + 16, bve = bvf + 16, bsf = bve + 16,
                 bpf = bsf + 16, bof = bpf + 16, brf = bof + 8, bre = brf + 8 * NRAW;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14 + 2 * NRAW);
  __shared__ volatile int s_abort;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = a.tok * a.group;  // rows of a query tile that hold queries
  if (threadIdx.x == 0) {
    s_abort = 0;
    mbar_init(bq, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bkf + 8 * i, FP8 ? 4 : 1);  // one arrive per converting warp, or the TMA bytes'
      mbar_init(bvf + 8 * i, FP8 ? 4 : 1);
      mbar_init(bke + 8 * i, 1);
      mbar_init(bve + 8 * i, 1);
      mbar_init(bsf + 8 * i, 1);
      mbar_init(bpf + 8 * i, 4);  // one arrive per softmax warp
    }
    for (int i = 0; i < NRAW; ++i) {
      mbar_init(brf + 8 * i, 33);  // the TMA bytes' arrive and one per lane (exponents)
      mbar_init(bre + 8 * i, 4);
    }
    mbar_init(bof, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  // rows past the last whole token
  for (int i = threadIdx.x; i < 2 * (BQ - rows) * 16; i += NTHREADS) {
    const int t = i / ((BQ - rows) * 16), k = i - t * (BQ - rows) * 16, r = rows + (k >> 4);
    *reinterpret_cast<uint4*>(smem + t * TILE + (k & 1) * ATOM + r * 128 + ((k >> 1) & 7) * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_async_smem();
  if (warp == 0) tmem_alloc_1cta(smem_u32(tmem_slot), 512);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  // TMEM columns: S_A 0..127, S_B 128..255, O_A 256..383, O_B 384..511
  auto tS = [&](int g) { return tmem + 128u * (uint32_t)g; };
  auto tO = [&](int g) { return tmem + 256u + 128u * (uint32_t)g; };

  if (warp < 4) {
    if constexpr (FP8) asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
    if (warp == 0 && nK > 0) {
      // ----------------------------------------------------------- producer
      if (lane == 0) {
        tma_prefetch_desc(&tmQ);
        tma_prefetch_desc(&tmK);
        tma_prefetch_desc(&tmV);
        mbar_expect_tx(bq, (nB ? 2 : 1) * (uint32_t)rows * 256);
        const uint32_t sq = smem_u32(smem);
        for (int t = 0; t < (nB ? 2 : 1); ++t) {
          tma_load_3d(sq + t * TILE, &tmQ, 0, hk * a.group, s0 + i0 + t * a.tok, bq);
          tma_load_3d(sq + t * TILE + ATOM, &tmQ, 64, hk * a.group, s0 + i0 + t * a.tok, bq);
        }
      }
      const int* bt = a.block_table + (int64_t)b * a.bt_row;
      const int bs = 1 << a.block_shift;
      // row of the page tensor that holds the key, or one outside it (TMA fills zeros)
      auto row_of = [&](int key) {
        const int p = key < len ? bt[key >> a.block_shift] : -1;
        return p >= 0 && p < a.num_blocks ? (p * a.nkv + hk) * bs + (key & (bs - 1)) : -BKV;
      };
      bool ok = true;
      if constexpr (FP8) {
        const int box = min(RK, bs);
        // step h: half h & 1 of K (h & 2 = 0) or V of entry h / 4
        for (int h = 0; h < 4 * nK; ++h) {
          const int st = h % NRAW, key0 = key_tile(h >> 2) * BKV + (h & 1) * RK;
          if (h >= NRAW) ok = mbar_wait(bre + 8 * st, ((h / NRAW) & 1) ^ 1);
          if (!__all_sync(0xffffffffu, ok) || s_abort) break;
          {
            // exponents: lanes 0..15 four keys of K each, lanes 16..31 of V
            const int row = row_of(key0 + (lane & 15) * 4);
            const uint8_t* e = lane < 16 ? a.ks : a.vs;
            if (row >= 0) e += row;
            const uint32_t dst = smem_u32(smem) + OFF_EXP + st * 2 * RK + lane * 4;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(e), "r"(row >= 0 ? 4 : 0) : "memory");
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(brf + 8 * st) : "memory");
          }
          if (lane == 0) {
            mbar_expect_tx(brf + 8 * st, RAW);
            const uint32_t dst = smem_u32(smem) + OFF_RAW + st * RAW;
            for (int r = 0; r < RK; r += box)
              tma_load_2d(dst + r * D, (h & 2) ? &tmV : &tmK, 0, row_of(key0 + r), brf + 8 * st);
          }
        }
      } else if (lane == 0) {
        const int box = min(BKV, bs);
        for (int u = 0; u < 2 * nK && ok && !s_abort; ++u) {
          const int j = u >> 1, st = j & 1, key0 = key_tile(j) * BKV;
          const bool is_v = u & 1;
          if (j >= 2) ok = mbar_wait((is_v ? bve : bke) + 8 * st, ((j >> 1) & 1) ^ 1);
          if (!ok) break;
          const uint32_t fb = (is_v ? bvf : bkf) + 8 * st;
          mbar_expect_tx(fb, TILE);
          const uint32_t dst = smem_u32(smem) + (is_v ? OFF_V : OFF_K) + st * TILE;
          for (int r = 0; r < BKV; r += box) {
            const int y = row_of(key0 + r);
            tma_load_2d(dst + r * 128, is_v ? &tmV : &tmK, 0, y, fb);
            tma_load_2d(dst + ATOM + r * 128, is_v ? &tmV : &tmK, 64, y, fb);
          }
        }
      }
      if (!ok && lane == 0) {
        if (!s_abort) set_err(a.err, 55);
        s_abort = 1;
      }
    } else if (warp == 1 && elect_one()) {
      // --------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_qk = idesc_bf16_f32(BQ, BKV, false, false);
      constexpr uint32_t idesc_pv = idesc_bf16_f32(BQ, D, false, true);
      bool ok = nK == 0 || mbar_wait(bq, 0);
      int k_ready = -1, v_ready = -1;
      auto wait_k = [&](int j) {
        if (j > k_ready) ok = ok && mbar_wait(bkf + 8 * (j & 1), (j >> 1) & 1);
        k_ready = j;
      };
      auto wait_v = [&](int j) {
        if (j > v_ready) ok = ok && mbar_wait(bvf + 8 * (j & 1), (j >> 1) & 1);
        v_ready = j;
      };
      // descriptors: a base per operand, constants added per product
      constexpr uint64_t T16 = TILE >> 4;
      const uint64_t dQ = desc_sw128(smem_u32(smem), 16, 1024), dK = desc_sw128(smem_u32(smem + OFF_K), 16, 1024);
      const uint64_t dV = desc_sw128(smem_u32(smem + OFF_V), ATOM, 1024);
      auto issue_s = [&](int g, int j) {
        fence_after();
        const uint64_t q = dQ + g * T16, kk = dK + (j & 1) * T16;
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint64_t o = ((k >> 2) * ATOM + (k & 3) * 32) >> 4;
          mma_1cta(tS(g), q + o, kk + o, idesc_qk, k > 0);
        }
        commit_1cta(bsf + 8 * g);
      };
      auto issue_pv = [&](int g, int j) {
        fence_after();
        const uint64_t v = dV + (j & 1) * T16;
#pragma unroll
        for (int k = 0; k < BKV / 16; ++k) mma_1cta_ts(tO(g), tS(g) + k * 8, v + (k * 2048 >> 4), idesc_pv, (j > 0 || k > 0));
      };
      if (nK > 0 && ok) {
        wait_k(0);
        if (ok && nA) issue_s(0, 0);
        if (ok && nB) issue_s(1, 0);
        commit_1cta(bke);
      }
      for (int j = 0; j < nK && ok && !s_abort; ++j) {
        wait_v(j);
        if (ok && j < nA) {
          ok = mbar_wait(bpf, j & 1);
          if (ok) issue_pv(0, j);
        }
        if (ok && j + 1 < nA) {
          wait_k(j + 1);
          if (ok) issue_s(0, j + 1);
        }
        if (ok && j < nB) {
          ok = mbar_wait(bpf + 8, j & 1);
          if (ok) issue_pv(1, j);
        }
        commit_1cta(bve + 8 * (j & 1));  // V_j no longer read
        if (ok && j + 1 < nB) {
          wait_k(j + 1);
          if (ok) issue_s(1, j + 1);
        }
        if (j + 1 < nK) commit_1cta(bke + 8 * ((j + 1) & 1));  // K_{j+1} no longer read
        if (!ok) {
          set_err(a.err, 52, j);
          s_abort = 1;
        }
      }
      commit_1cta(bof);
    }
  } else if (warp >= 12) {
    // ------------------------------------------------- codes to bf16 tiles
    if constexpr (FP8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 48;");
      // warps 12..15 convert K, 16..19 V; a thread codes 16c.. of rows sub + 16 i of a half
      const bool is_v = warp >= 16;
      const int ct = (threadIdx.x - 384) & 127, sub = ct >> 3, c = ct & 7;
      // the two 16-byte halves in an order that spreads a row's threads over all banks
      const int first = c >> 2, c0 = 2 * (c & 3);
      const int to0 = sub * 128 + (((c0 + first) ^ (sub & 7)) << 4), to1 = sub * 128 + (((c0 + 1 - first) ^ (sub & 7)) << 4);
      // RARE: an exponent that does not fit one bf16 factor (values of 2^16 and more), or keys past len
      auto convert = [&](auto rare, int h) {
        constexpr bool RARE = decltype(rare)::value;
        const int j = h >> 2, st = h % NRAW;
        const uint8_t* from = smem + OFF_RAW + st * RAW + sub * D + c * 16;
        const uint8_t* ex = smem + OFF_EXP + st * 2 * RK + sub;
        uint8_t* tile = smem + (is_v ? OFF_V : OFF_K) + (j & 1) * TILE + (c >> 2) * ATOM + (h & 1) * RK * 128;
        const int left = len - key_tile(j) * BKV - (h & 1) * RK;  // rows of the half below len
#pragma unroll 2
        for (int i = 0; i < 4; ++i) {
          uint4 w = *reinterpret_cast<const uint4*>(from + i * 16 * D);
          if (RARE && i * 16 + sub >= left) w = make_uint4(0, 0, 0, 0);
          const uint32_t ek = ex[i * 16], ev = ex[RK + i * 16];
          const uint32_t e = is_v ? ev : ek;
          // 2^(e - 127 + 120) where bf16 holds it, else in two factors.  A NaN of either vector
          // goes through the key; the value's codes then count as zeros
          uint32_t m = min(e + 120u, 254u) << 7;
          if (max(ek, ev) == 255u) m = is_v ? (ev == 255u ? 0u : m) : 0x7fc0u;
          m |= m << 16;
          uint32_t out[8];
          bf16_of4(w.x, m, out);
          bf16_of4(w.y, m, out + 2);
          bf16_of4(w.z, m, out + 4);
          bf16_of4(w.w, m, out + 6);
          if constexpr (RARE) {
            uint32_t m2 = e > 134u && e < 255u ? (e - 7u) << 7 : 0x3f80u;
            m2 |= m2 << 16;
#pragma unroll
            for (int k = 0; k < 8; ++k) out[k] = mul_bf16x2(out[k], m2);
          }
          const uint4 lo = make_uint4(out[0], out[1], out[2], out[3]), hi = make_uint4(out[4], out[5], out[6], out[7]);
          *reinterpret_cast<uint4*>(tile + to0 + i * 16 * 128) = first ? hi : lo;
          *reinterpret_cast<uint4*>(tile + to1 + i * 16 * 128) = first ? lo : hi;
        }
      };
      bool ok = true;
      for (int n2 = 0; n2 < 2 * nK; ++n2) {
        const int h = 4 * (n2 >> 1) + (is_v ? 2 : 0) + (n2 & 1);
        const int j = h >> 2, st = h % NRAW;
        ok = mbar_wait(brf + 8 * st, (h / NRAW) & 1);
        if (j >= 2 && !(h & 1)) ok = ok && mbar_wait((is_v ? bve : bke) + 8 * (j & 1), ((j >> 1) & 1) ^ 1);
        if (!__all_sync(0xffffffffu, ok) || s_abort) {
          if (lane == 0 && !s_abort) set_err(a.err, 51, h);
          s_abort = 1;
          break;
        }
        const uint32_t e4 = *reinterpret_cast<const uint32_t*>(smem + OFF_EXP + st * 2 * RK + lane * 4);
        const bool rare = __vcmpgtu4(e4, 0x86868686u) != 0 || key_tile(j) * BKV + (h & 1) * RK + RK > len;  // 134
        if (__any_sync(0xffffffffu, rare)) convert(std::true_type{}, h);
        else convert(std::false_type{}, h);
        if (h & 1) fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bre + 8 * st);
          if (h & 1) mbar_arrive((is_v ? bvf : bkf) + 8 * (j & 1));
        }
      }
    }
  } else {
    // -------------------------------------------------------------- softmax
    if constexpr (FP8) asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const int g = (warp - 4) >> 2;  // 0: tile A (warps 4..7), 1: tile B (warps 8..11)
    const int nt = g == 0 ? nA : nB;
    const int quad = warp & 3;
    const int r = quad * 32 + lane;  // row within the tile
    const int tr = r / a.group;
    const int tok = i0 + g * a.tok + tr;  // token within the chunk
    const bool valid = r < rows && tok < n;
    const int pos = tok + off;
    const uint32_t ts = tS(g) + ((uint32_t)(quad * 32) << 16), to = tO(g) + ((uint32_t)(quad * 32) << 16);
    float m = -INFINITY, l = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      if (!mbar_wait(bsf + 8 * g, j & 1) || s_abort) {
        if (!s_abort) set_err(a.err, 53, j);
        ok = false;
        break;
      }
      fence_after();
      const int key0 = key_tile(j) * BKV;
      if (!FP8 && key0 + BKV > len) {
        // bf16 pages came as they are: values past len must be zeros before P V reads them
        if (!mbar_wait(bvf + 8 * (j & 1), (j >> 1) & 1)) {
          if (!s_abort) set_err(a.err, 56, j);
          s_abort = 1;
          ok = false;
          break;
        }
        uint8_t* tile = smem + OFF_V + (j & 1) * TILE;
        for (int i = r; i < (key0 + BKV - len) * 16; i += BQ)
          *reinterpret_cast<uint4*>(tile + (i & 1) * ATOM + (len - key0 + (i >> 4)) * 128 + ((i >> 1) & 7) * 16) =
              make_uint4(0, 0, 0, 0);
        fence_async_smem();
      }
      const int lim = pos - key0;                                   // last key column this row sees
      const int lo = a.window > 0 ? lim - a.window + 1 : 0, sk = a.sinks - key0;  // from lo on, and those before sk
      const bool masked_tile = __any_sync(0xffffffffu, lim < BKV - 1 || (lo > 0 && sk < BKV));
      uint32_t v[128];
      tmem_ld32(ts, v);
      tmem_ld32(ts + 32, v + 32);
      tmem_ld32(ts + 64, v + 64);
      tmem_ld32(ts + 96, v + 96);
      tmem_wait_ld();
      if (masked_tile) {
#pragma unroll
        for (int i = 0; i < 128; ++i)
          if (i > lim || (i < lo && i >= sk)) v[i] = 0xff800000u;  // -inf: a key this row does not see
      }
      float mq[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < 128; ++i) mq[i & 3] = fmaxf(mq[i & 3], __uint_as_float(v[i]));
      const float mx = fmaxf(fmaxf(mq[0], mq[1]), fmaxf(mq[2], mq[3]));
      const float m_new = fmaxf(m, mx * a.scale_log2);
      // the decision to rescale O is taken for the whole warp (tcgen05.ld / st are collective)
      const bool grow = __any_sync(0xffffffffu, j > 0 && m != -INFINITY && m_new > m + RESCALE_LOG2);
      float alpha = 1.f;
      if (j == 0 || (!grow && m == -INFINITY)) {
        m = m_new;
      } else if (grow) {
        alpha = (m == -INFINITY) ? 0.f : ex2(m - m_new);
        m = m_new;
      }
      const float ref = (m == -INFINITY) ? 0.f : m;
      float ls0 = 0.f, ls1 = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c0 = c * 32 + 2 * i;
          const float p0 = ex2(fmaf(__uint_as_float(v[c0]), a.scale_log2, -ref));
          const float p1 = ex2(fmaf(__uint_as_float(v[c0 + 1]), a.scale_log2, -ref));
          ls0 += p0;
          ls1 += p1;
          // bf16 probabilities: what the MMA takes beside bf16 values; l keeps the fp32 ones
          const bf162 pp = __floats2bfloat162_rn(p0, p1);
          pk[i] = *reinterpret_cast<const uint32_t*>(&pp);
        }
        tmem_st16(ts + c * 16, pk);
      }
      if (grow) {
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          uint32_t ov[32];
          tmem_ld32(to + c * 32, ov);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) ov[i] = __float_as_uint(__uint_as_float(ov[i]) * alpha);
          tmem_st32(to + c * 32, ov);
        }
      }
      l = l * alpha + (ls0 + ls1);
      tmem_wait_st();
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bpf + 8 * g);
    }
    if (!mbar_wait(bof, 0)) ok = false;
    fence_after();
    if (ok && !s_abort) {
      const int64_t orow = (int64_t)(s0 + tok) * a.nq + hk * a.group + (r - tr * a.group);
      // l == 0: no key seen; a NaN stays one
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        uint32_t v[32];
        if (nt > 0) {
          tmem_ld32(to + c * 32, v);
          tmem_wait_ld();
        }
        if (valid && (a.splits == 1 || nt > 0)) {
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) f[i] = nt > 0 ? __uint_as_float(v[i]) * inv : 0.f;
          if (a.splits == 1) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) *reinterpret_cast<bf16x8*>(a.o + orow * D + c * 32 + i) = pack8(f + i);
          } else {
            float* dst = a.part_o + ((int64_t)part * a.T * a.nq + orow) * D + c * 32;
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(dst + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
          }
        }
      }
      if (valid && a.splits > 1)
        a.part_lse[(int64_t)part * a.T * a.nq + orow] = l == 0.f ? -INFINITY : m + log2f(l);
    } else if (!s_abort) {
      set_err(a.err, 54);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 0) {
    fence_after();
    tmem_free_1cta(tmem, 512);
  }
}

// One warp per (token, query head) of the sequences: joins the parts in key order.
__global__ void __launch_bounds__(256) chunk_join(Args a, int B) {
  const int64_t w = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)max(0, min(a.cu_q[B], a.T)) * a.nq;
  kv8::wait_prior();  // every block: this kernel must not end before the one it follows
  if (w >= rows) return;
  const int64_t stride = (int64_t)a.T * a.nq;
  float m = -INFINITY;
  for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_lse[s * stride + w]);
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s = 0; s < a.splits; ++s) {
    const float lse = a.part_lse[s * stride + w];
    if (lse == -INFINITY) continue;
    const float c = ex2(lse - (m == -INFINITY ? 0.f : m));  // a NaN lse makes the row NaN
    const float4 v = *reinterpret_cast<const float4*>(a.part_o + (s * stride + w) * D + lane * 4);
    l += c;
    acc.x += v.x * c;
    acc.y += v.y * c;
    acc.z += v.z * c;
    acc.w += v.w * c;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  bf162 o[2] = {__floats2bfloat162_rn(acc.x * inv, acc.y * inv), __floats2bfloat162_rn(acc.z * inv, acc.w * inv)};
  *reinterpret_cast<uint2*>(a.o + w * D + lane * 4) = *reinterpret_cast<const uint2*>(o);
}

static CUtensorMap map_q(const at::Tensor& q, int group, int tok) {
  CUtensorMap m;
  cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)q.size(1), (cuuint64_t)q.size(0)};
  cuuint64_t strides[2] = {(cuuint64_t)q.stride(1) * 2, (cuuint64_t)q.stride(0) * 2};
  cuuint32_t box[3] = {64u, (cuuint32_t)group, (cuuint32_t)tok};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = PSRL_DRV(cuTensorMapEncodeTiled)(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q.data_ptr(), dims, strides,
                                                box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (", (int)r, ")");
  return m;
}

// bf16 pages as rows of 128: boxes of 64 columns x min(128, block_size) rows.
static CUtensorMap map_pages(const at::Tensor& t) {
  CUtensorMap m;
  const cuuint64_t rows = (cuuint64_t)(t.size(0) * t.size(1) * t.size(2));
  TORCH_CHECK(rows < (1ull << 31), "cache of more than 2^31 vectors");
  cuuint64_t dims[2] = {(cuuint64_t)D, rows};
  cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  cuuint32_t box[2] = {64u, (cuuint32_t)std::min<int64_t>(BKV, t.size(2))};
  cuuint32_t estr[2] = {1, 1};
  CUresult r = PSRL_DRV(cuTensorMapEncodeTiled)(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, t.data_ptr(), dims, strides,
                                                box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (", (int)r, ")");
  return m;
}

}  // namespace chunk

using namespace chunk;

// q [T, nq, 128] bf16; sequence b's queries [cu_q[b], cu_q[b+1]) are the last of
// its kv_lens[b] positions.  k_scale / v_scale absent: a bf16 cache.  window 0: none.
at::Tensor attn_paged_chunk(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, c10::optional<at::Tensor> k_scale,
                            c10::optional<at::Tensor> v_scale, at::Tensor cu_q, at::Tensor kv_lens,
                            at::Tensor block_table, int64_t max_q_len, double scale, int64_t window, int64_t sinks,
                            at::Tensor err) {
  CHECK_CUDA_TENSOR(q);
  CHECK_DTYPE(q, at::kBFloat16);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == D && q.stride(2) == 1 && q.stride(0) % 8 == 0 && q.stride(1) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0,
              "q must be [T, heads, 128], rows and heads on 16-byte boundaries");
  TORCH_CHECK(cu_q.scalar_type() == at::kInt && cu_q.dim() == 1 && cu_q.numel() >= 1 && cu_q.is_contiguous() &&
                  cu_q.device() == q.device(),
              "cu_q must be int32 [B + 1] on q's device");
  const int64_t T = q.size(0), nq = q.size(1), B = cu_q.numel() - 1;
  const bool fp8 = k_scale.has_value();
  TORCH_CHECK(fp8 == v_scale.has_value(), "an 8-bit cache needs both k_scale and v_scale");
  kv8::check_paged(q, k_cache, v_cache, fp8 ? *k_scale : at::Tensor(), fp8 ? *v_scale : at::Tensor(), block_table,
                   kv_lens, B);
  const int64_t nkv = k_cache.size(1);
  TORCH_CHECK(nq % nkv == 0 && nq / nkv <= BQ, "query heads must be a multiple of the kv heads, at most 128 times");
  TORCH_CHECK(window >= 0 && sinks >= 0 && window < (1 << 30) && sinks < (1 << 30), "window and sinks must not be negative");
  at::cuda::CUDAGuard g(q.device());
  auto o = at::empty({T, nq, D}, q.options());
  const int64_t cap = block_table.size(1) * k_cache.size(2);
  TORCH_CHECK(cap < (1ll << 31), "block table too wide");
  if (T == 0) return o;
  if (B == 0 || max_q_len <= 0 || cap == 0 || k_cache.size(0) == 0) return o.zero_();
  TORCH_CHECK(T < (1ll << 31) && B < 65536, "too many rows or sequences");
  Args a{};
  a.cu_q = cu_q.data_ptr<int>();
  a.kv_lens = kv_lens.data_ptr<int>();
  a.block_table = block_table.data_ptr<int>();
  a.bt_row = block_table.stride(0);
  a.ks = fp8 ? k_scale->data_ptr<uint8_t>() : nullptr;
  a.vs = fp8 ? v_scale->data_ptr<uint8_t>() : nullptr;
  a.num_blocks = k_cache.size(0);
  a.T = (int)T;
  a.nq = (int)nq;
  a.nkv = (int)nkv;
  a.group = (int)(nq / nkv);
  a.tok = BQ / a.group;
  a.max_blocks = (int)block_table.size(1);
  a.block_shift = __builtin_ctzll((unsigned long long)k_cache.size(2));
  a.window = (int)window;
  a.sinks = window > 0 ? (int)sinks : 0;
  a.scale_log2 = (float)(scale * 1.4426950408889634);
  a.o = reinterpret_cast<bf16*>(o.data_ptr());
  a.err = err.data_ptr<int>();
  const int64_t per_block = 2 * a.tok;
  a.blocks_z = (int)((std::min(max_q_len, T) + per_block - 1) / per_block);
  // Split the keys while there are fewer blocks (at most one CTA each) than SMs.  How
  // long a part is, the kernel finds from the lengths; here only the most parts that
  // a block may get: four times its share of the SMs, none under two key tiles.
  const int64_t ctas = nkv * std::min<int64_t>(B * a.blocks_z, T / per_block + B);
  const int64_t span = window > 0 ? std::min(cap, window + a.sinks + per_block) : cap;
  int64_t splits = 1;
  if (2 * ctas <= num_sms())
    splits = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(4 * num_sms() / ctas, 64),
                                                    (span + 2 * BKV - 1) / (2 * BKV)));
  a.B = (int)B;
  a.sms = num_sms();
  TORCH_CHECK(a.blocks_z * splits < 65536, "too many query blocks");
  a.splits = (int)splits;
  at::Tensor part;
  if (splits > 1) {
    part = at::empty({splits * T * nq * (D + 1)}, q.options().dtype(at::kFloat));
    a.part_o = part.data_ptr<float>();
    a.part_lse = a.part_o + splits * T * nq * D;
  }
  const CUtensorMap tq = map_q(q, a.group, a.tok);
  const CUtensorMap tk = fp8 ? kv8::map_codes(k_cache, RK, CU_TENSOR_MAP_SWIZZLE_NONE) : map_pages(k_cache);
  const CUtensorMap tv = fp8 ? kv8::map_codes(v_cache, RK, CU_TENSOR_MAP_SWIZZLE_NONE) : map_pages(v_cache);
  auto* kern = fp8 ? chunk_kernel<true> : chunk_kernel<false>;
  ensure_smem_attr(kern, smem_bytes(fp8));
  kern<<<dim3((unsigned)nkv, (unsigned)B, (unsigned)(a.blocks_z * splits)), threads_of(fp8), smem_bytes(fp8), stream()>>>(tq, tk, tv,
                                                                                                                        a);
  PSRL_CHECK_LAUNCH();
  if (splits > 1) {
    kv8::launch_after(chunk_join, (unsigned)((T * nq * 32 + 255) / 256), 256u, a, (int)B);
  }
  return o;
}

}  // namespace psrl
