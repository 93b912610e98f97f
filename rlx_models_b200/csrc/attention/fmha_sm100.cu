// Flash attention forward on the 5th-generation tensor cores (head_dim 128).
//
// One CTA per (sequence, one or two tiles of 128 query rows, kv head); rows are
// (token, query head) pairs of one GQA group (row = token * G + g), so every
// K/V page is read once per kv head. Warp roles:
//   warps 0, 3    TMA producers: the Q tiles once (3-D boxes [16 tokens][G
//                 heads][64 dims]), then tiles of 128 keys (eight 16-key pages),
//                 K the one and V the other: a tile in scattered pages is 16
//                 copies, and one thread issuing both was the pace of the kernel;
//   warp 1 (, 2)  MMA issuer, one thread per query tile: S_j = Q K_j^T into
//                 TMEM, then O += P_j V_j with P_j read from TMEM (A operand)
//                 and V_j from shared memory as an MN-major B operand;
//   4 warps       per query tile: softmax, one query row per thread (TMEM lane
//                 quadrant = warp % 4): row max over the masked S tile, P =
//                 exp2(S*scale - m) to TMEM as bf16, row sums in fp32. The
//                 running max is rescaled lazily: O (in TMEM) is corrected only
//                 when the max grows by more than 2^8, so most tiles never touch
//                 O. At the end they normalise O (learned sink logits join the
//                 denominator) and store the rows.
// A tile of scores costs the tensor cores (S and P V) and the exponential units
// about 1024 cycles each, so they have to work at the same time:
//   two query tiles   the softmax of one runs beside that of the other and the
//                     products of both, on the same K and V. Both use one S
//                     buffer in turn: it is free again when the scores are in
//                     registers, so S_{j+1} is there when the softmax of tile j
//                     ends. TMEM: S, P of each (64 columns), O of each. The
//                     softmax warps take registers over from the other four.
//   one query tile    S_{j+1} is computed beside the softmax of tile j in a
//                     second buffer, P_j lies over S_j. TMEM: S0, S1, O. Four
//                     warps, one a scheduler, leave the exponential units idle
//                     through each tile's loads, maximum and stores, but where
//                     every tile finds an SM of its own this is the shorter way.
// Either way a row sees its tiles in the same order with the same arithmetic.
// 2 x 1024 tokens over 8192, 32 / 8 heads: 397 us with one tile a CTA, 220 with
// two (1170 TFLOP/s, in 256 CTAs on 148 SMs, tensor pipes and exponential units 65%
// busy); 4 x 2048 from the start: 273 and 166.
// A key tile then takes about 3200 cycles for both: each softmax warp works through
// 360 (scores to registers), 400 (maximum), 400 (the wait for the last product)
// and 1500 cycles (exponentials, whose units it shares with the other tile).
//
// Masks: causal over absolute positions (queries are the last q_len of ctx
// positions), sliding window, context length; the DiT joint attention runs
// non-causally with query rows placed through the key block table.
//
// Reference behaviour: the fused SDPA of rlx-models-core
// src/standard_decoder.rs:11946-12079 (sinks, sliding window) and rlx-flux1
// src/transformer.rs:327-340 (joint, unmasked attention).
#include <cuda_bf16.h>

#include <algorithm>
#include <cstdlib>
#include <stdexcept>
#include <type_traits>

#include "../common/b200.cuh"
#include "../common/launch.h"
#include "../common/pdl_launch.h"
#include "../common/tma_host.h"

namespace b200 {
namespace fmha {

constexpr int kD = 128;
constexpr int kBN = 128;                   // keys per tile
constexpr uint32_t kHalf = 128 * 64 * 2;   // [128 rows][64 dims] bf16, 128B-swizzled
constexpr uint32_t kQ = 2 * kHalf;         // one Q tile
constexpr uint32_t kKV = 2 * kHalf;        // one K (or V) tile: a slot of the ring
template <int TILES>
struct Cfg {
  static constexpr int KS = TILES == 2 ? 2 : 3, VS = 3;  // Q tiles and the rings fill the shared memory
  static constexpr uint32_t SMEM = 1024 + TILES * kQ + (KS + VS) * kKV + 256;
  static constexpr int THREADS = 128 + 128 * TILES;
};
constexpr uint32_t kTmemCols = 512;
constexpr uint32_t kPCol = 128;            // two tiles: P of each, 64 columns
constexpr uint32_t kOCol = 256;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;            // lazy rescale threshold (log2 units)

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// x * s + b of two numbers, each rounded as by fmaf, in one instruction
__device__ __forceinline__ void fma2(float& y0, float& y1, uint32_t x0, uint32_t x1, float s, float b) {
  asm("{\n\t.reg .b64 x, s, b, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\tmov.b64 b, {%5, %5};\n\t"
      "fma.rn.f32x2 y, x, s, b;\n\tmov.b64 {%0, %1}, y;\n\t}"
      : "=f"(y0), "=f"(y1)
      : "r"(x0), "r"(x1), "f"(s), "f"(b));
}

__device__ __forceinline__ void tma_load_3d_q(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y, int z) {
  tma_load_3d(dst, m, bar, x, y, z);
}

__device__ __forceinline__ void tmem_st_32x32b_x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
      "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
      "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
      "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

// Key tiles [begin, begin + n) that the query tile at token tok0 sees; no tokens: none.
struct TileRange {
  int ntok, begin, n;
};

__device__ __forceinline__ TileRange tile_range(const AttnArgs& a, int ctx, int q_len, int tok0, int rows_tok) {
  TileRange r;
  r.ntok = min(rows_tok, q_len - tok0);
  const int pos_lo = ctx - q_len + tok0, pos_hi = pos_lo + r.ntok - 1;
  int k_begin = 0;
  if (a.causal != 0 && a.window > 0) k_begin = max(0, pos_lo - a.window + 1);
  const int k_end = a.causal != 0 ? min(ctx, pos_hi + 1) : ctx;
  r.begin = k_begin / kBN;
  r.n = r.ntok > 0 ? max(1, (k_end - r.begin * kBN + kBN - 1) / kBN) : 0;
  return r;
}

template <int TILES>
__global__ void __launch_bounds__(Cfg<TILES>::THREADS, 1)
    fmha_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                    const __grid_constant__ CUtensorMap tmV, const AttnArgs a, int q_blocks, int rows_tok) {
  constexpr int KS = Cfg<TILES>::KS, VS = Cfg<TILES>::VS;
  extern __shared__ uint8_t smem_dyn[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_dyn) + 1023) & ~uintptr_t(1023));
  uint8_t* Qs = smem;
  uint8_t* Ks = smem + TILES * kQ;
  uint8_t* Vs = Ks + KS * kKV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(Vs + VS * kKV);
  uint64_t* q_full = bars;
  uint64_t* k_full = bars + 1;
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + VS;
  uint64_t* s_full = v_empty + VS;  // one tile: of its two S buffers; two tiles: of each, as those that follow
  uint64_t* p_full = s_full + 2;
  uint64_t* o_done = p_full + 2;
  uint64_t* s_free = o_done + 2;    // two tiles: the S buffer has been read by this one
  uint64_t* join = s_free + 2;      // two tiles: the second may take its first turn
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(join + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  pdl_wait();
  pdl_trigger();
  const int G = a.Hq / a.Hkv;
  // last query tiles first: under a causal mask they are the longest, and the short ones fill the tail
  const int b = blockIdx.x % a.B, qb = q_blocks - 1 - blockIdx.x / a.B, hkv = blockIdx.y;
  const int q0 = a.cu_q[b];
  const int q_len = a.cu_q[b + 1] - q0;
  const int tok0 = qb * TILES * rows_tok;
  if (tok0 >= q_len) return;  // uniform for the CTA, before any barrier or TMEM use
  const int ctx = a.ctx_lens[b];
  const bool causal = a.causal != 0;
  // the key tiles of each query tile, and those of the CTA: [first, last)
  TileRange own[TILES];
  int first = INT32_MAX, last = 0;
#pragma unroll
  for (int t = 0; t < TILES; ++t) {
    own[t] = tile_range(a, ctx, q_len, tok0 + t * rows_tok, rows_tok);
    if (own[t].n > 0) {
      first = min(first, own[t].begin);
      last = max(last, own[t].begin + own[t].n);
    }
  }
  const int32_t* btab = a.block_tables + (int64_t)b * a.max_blocks;
  const int max_page = max(1, (ctx + 15) >> 4);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    for (int s = 0; s < KS; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], TILES);
    }
    for (int s = 0; s < VS; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], TILES);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&o_done[i], 1);
      mbar_init(&s_free[i], 4);
    }
    mbar_init(join, 1);
    fence_mbarrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // (two tiles: 128 * 72 + 256 * 216 registers, the 384 * 168 of the launch)
  if (warp == 0 || warp == 3) {
    if constexpr (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (elect_one_sync()) {
      const bool is_v = warp == 3;
      const CUtensorMap* tm = is_v ? &tmV : &tmK;
      tma_prefetch_desc(tm);
      if (!is_v) {
        tma_prefetch_desc(&tmQ);
        const int tiles = TILES == 2 && own[TILES - 1].n > 0 ? 2 : 1;
        mbar_arrive_expect_tx(q_full, tiles * kQ);
        for (int c = 0; c < tiles * (rows_tok / 16); ++c) {
          const int t = tok0 + 16 * c;
          const int row = a.q_paged ? btab[min(t >> 4, max_page - 1)] * 16 : q0 + t;
          const int to = c / (rows_tok / 16) * kQ + c % (rows_tok / 16) * (16 * G * 128);
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tma_load_3d_q(Qs + h * kHalf + to, &tmQ, q_full, h * 64, hkv * G, row);
        }
      }
      uint8_t* ring = is_v ? Vs : Ks;
      uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
      const int slots = is_v ? VS : KS;
      int s = 0;
      uint32_t ph = 0;
      int next[kBN / 16];  // block ids, asked for one tile ahead
      auto ask = [&](int j) {
        if (a.kv_contig) return;
#pragma unroll
        for (int pg = 0; pg < kBN / 16; ++pg)  // pages past the context are masked
          next[pg] = btab[min(j * (kBN / 16) + pg, max_page - 1)];
      };
      ask(first);
      for (int j = first; j < last; ++j) {
        int id[kBN / 16];
#pragma unroll
        for (int pg = 0; pg < kBN / 16; ++pg) id[pg] = next[pg];
        ask(j + 1);
        if (!mbar_wait(&empty[s], ph ^ 1, a.status, kErrTimeoutEmpty)) break;
        uint8_t* st = ring + s * kKV;
        uint64_t* bar = &full[s];
        mbar_arrive_expect_tx(bar, kKV);
        if (a.kv_contig) {  // the tile's 8 pages are one box (pages past the context hold zeros and are masked)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tma_load_4d(st + h * kHalf, tm, bar, h * 64, 0, hkv, b * a.max_blocks + j * (kBN / 16));
        } else {
#pragma unroll
          for (int pg = 0; pg < kBN / 16; ++pg) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if (a.kv_dense)
                tma_load_3d(st + h * kHalf + pg * 2048, tm, bar, h * 64, hkv, id[pg] * 16);
              else
                tma_load_2d(st + h * kHalf + pg * 2048, tm, bar, h * 64, (id[pg] * a.Hkv + hkv) * 16);
            }
          }
        }
        if (++s == slots) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1 || (TILES == 2 && warp == 2)) {
    if constexpr (TILES == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (elect_one_sync()) {
      constexpr uint32_t idS = umma_idesc_bf16(128, kBN, false, false);
      constexpr uint32_t idO = umma_idesc_bf16(128, kD, false, true);  // V: MN-major B
      const int t = warp - 1, n = last - first;  // query tile; j counts key tiles from `first`
      auto wait_k = [&](int j) {
        return mbar_wait(&k_full[j % KS], (uint32_t)(j / KS) & 1, a.status, kErrTimeoutFull);
      };
      auto wait_v = [&](int j) {
        return mbar_wait(&v_full[j % VS], (uint32_t)(j / VS) & 1, a.status, kErrTimeoutFull);
      };
      auto mma_s = [&](int buf, int j, bool alone) {
        const uint32_t qa = smem_u32(Qs) + t * kQ, kb = smem_u32(Ks) + j % KS * kKV;
        const uint32_t d = tmem + (TILES == 2 ? 0 : buf * kBN);
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kD / 16; ++kk) {
          const uint32_t off = (kk >> 2) * kHalf + (kk & 3) * 32;
          umma_f16(d, umma_desc_sw128(qa + off, 16, 1024), umma_desc_sw128(kb + off, 16, 1024), idS, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[buf]);
        umma_commit(&k_empty[j % KS]);
        if (TILES == 2 && alone) umma_commit(&k_empty[j % KS]);  // for the tile that takes no part
      };
      auto mma_o = [&](int buf, int j, bool more, bool alone) {
        const uint32_t pa = tmem + (TILES == 2 ? kPCol + t * (kBN / 2) : buf * kBN);
        const uint32_t vb = smem_u32(Vs) + j % VS * kKV;
        tc_fence_after();
#pragma unroll
        for (int kk = 0; kk < kBN / 16; ++kk)
          umma_f16_ts(tmem + kOCol + t * kD, pa + kk * 8, umma_desc_sw128(vb + kk * 2048, kHalf, 1024), idO,
                      (more || kk > 0) ? 1u : 0u);
        umma_commit(&o_done[buf]);
        umma_commit(&v_empty[j % VS]);
        if (TILES == 2 && alone) umma_commit(&v_empty[j % VS]);
      };
      bool ok = mbar_wait(q_full, 0, a.status, kErrTimeoutFull);
      if constexpr (TILES == 1) {
        ok = ok && wait_k(0);
        if (ok) mma_s(0, 0, false);
        for (int j = 0; ok && j < n; ++j) {
          if (j + 1 < n) {
            // S buffer (j+1)&1 held P_{j-1}: wait until P_{j-1} V_{j-1} has completed
            if (j >= 1 && !mbar_wait(&o_done[(j - 1) & 1], ((j - 1) >> 1) & 1, a.status, kErrTimeoutAccEmpty)) break;
            if (!wait_k(j + 1)) break;
            mma_s((j + 1) & 1, j + 1, false);
          }
          if (!mbar_wait(&p_full[j & 1], (j >> 1) & 1, a.status, kErrTimeoutFull)) break;
          if (!wait_v(j)) break;
          mma_o(j & 1, j, j > 0, false);
        }
      } else {
        // Tile t sees key tiles [lo[t], hi[t]); tile 0 begins and ends no later than tile 1. One thread issues the
        // products of each tile. They take turns with the S buffer, S_j of tile 0, S_j of tile 1, S_{j+1} of tile 0 ...,
        // each as soon as the one before is in its warps' registers, so that scores are ready when a softmax ends.
        int lo[2], hi[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          lo[i] = own[TILES == 2 ? i : 0].n > 0 ? own[TILES == 2 ? i : 0].begin - first : n;
          hi[i] = own[TILES == 2 ? i : 0].n > 0 ? lo[i] + own[TILES == 2 ? i : 0].n : n;
        }
        auto sees = [&](int i, int j) { return j >= lo[i] && j < hi[i]; };
        auto read = [&](int i, int j) {  // tile i has read its S_j
          return mbar_wait(&s_free[i], (uint32_t)(j - lo[i]) & 1, a.status, kErrTimeoutAccEmpty);
        };
        // Parities tell a turn from the next one, not from the one after: whoever waits for a turn knows that the one
        // before it is over. Tile 0 has waited for each turn of its own until tile 1 takes its first (`meet`), and then
        // for each of tile 1, as tile 1 for each of tile 0. What tile 1 has not followed until then it is told by `join`.
        const int meet = min(lo[1], hi[0] - 1);
        auto turn = [&](int j) {
          if (t == 0) {
            if (sees(1, j - 1) ? !read(1, j - 1) : sees(0, j - 1) && !read(0, j - 1)) return false;
            if (j == meet) mbar_arrive(join);
            return true;
          }
          if (j == lo[1]) return mbar_wait(join, 0, a.status, kErrTimeoutAccEmpty) && read(0, meet);
          return sees(0, j) ? read(0, j) : read(1, j - 1);
        };
        auto next_s = [&](int j) {
          if (!sees(t, j)) return true;
          if (!turn(j) || !wait_k(j)) return false;
          mma_s(t, j, !sees(1 - t, j));
          return true;
        };
        auto next_o = [&](int j) {
          if (!sees(t, j)) return true;
          if (!mbar_wait(&p_full[t], (uint32_t)(j - lo[t]) & 1, a.status, kErrTimeoutFull) || !wait_v(j)) return false;
          mma_o(t, j, j > lo[t], !sees(1 - t, j));
          return true;
        };
        ok = ok && next_s(lo[t]);
        for (int j = lo[t]; ok && j < hi[t]; ++j) ok = next_s(j + 1) && next_o(j);
      }
    }
  } else if (warp >= 4) {
    if constexpr (TILES == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    // softmax / correction / epilogue: one query row per thread
    const int q = warp & 3, qt = TILES == 2 ? (warp >> 2) - 1 : 0;
    const TileRange mine = qt == 0 ? own[0] : own[TILES - 1];
    const int my_tok0 = tok0 + qt * rows_tok, ntok = mine.ntok, begin = mine.begin, n_tiles = mine.n;
    // buffer of the j-th tile, parity of its turn
    auto buf = [&](int j) { return TILES == 2 ? qt : j & 1; };
    auto par = [&](int j) { return (uint32_t)(TILES == 2 ? j : j >> 1) & 1; };
    const int row = q * 32 + lane;
    const int tok = row / G, g = row % G;
    const bool row_ok = tok < ntok;
    const int qpos = ctx - q_len + my_tok0 + tok;
    const float sl2 = a.scale * kLog2e;
    const uint32_t lane_base = tmem + ((uint32_t)(q * 32) << 16);
    const uint32_t o_base = lane_base + kOCol + qt * kD;
    float m_used = -INFINITY, l = 0.f;
    bool ok = n_tiles > 0;
    // tcgen05.ld / st / wait are warp-collective (.sync.aligned): every branch
    // around them below is warp-uniform; per-row choices only pick values.
    for (int j = 0; j < n_tiles; ++j) {
      if (!__all_sync(0xffffffffu, mbar_wait(&s_full[buf(j)], par(j), a.status, kErrTimeoutAccFull))) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t sb = lane_base + (TILES == 2 ? 0 : buf(j) * kBN);
      const uint32_t pb = TILES == 2 ? lane_base + kPCol + qt * (kBN / 2) : sb;
      const int key0 = (begin + j) * kBN;
      // keys of this tile visible to the row: [lo, hi); a row of no query masks nothing, which costs more (its result
      // goes nowhere): one sequence of 24 new tokens in 16384, 4 heads a KV head, takes 167 us instead of 325
      int lo = 0, hi = kBN;
      if (row_ok) {
        int kmin = 0, kmax = ctx;  // absolute positions
        if (causal) {
          kmax = min(kmax, qpos + 1);
          if (a.window > 0) kmin = max(kmin, qpos - a.window + 1);
        }
        lo = max(0, kmin - key0);
        hi = min(kBN, kmax - key0);
      }
      // the row's scores, read once; most tiles lie inside every row's range and need no masks
      uint32_t sv[kBN / 32][32];
#pragma unroll
      for (int c = 0; c < kBN / 32; ++c) tmem_ld_32x32b_x32(sb + c * 32, sv[c]);
      tmem_wait_ld();
      if constexpr (TILES == 2) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&s_free[qt]);
      }
      const bool inside = __all_sync(0xffffffffu, lo == 0 && hi == kBN);
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};  // four chains: a maximum waits 4 cycles for the last
      if (inside) {
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c)
#pragma unroll
          for (int t = 0; t < 32; ++t) mx4[t & 3] = fmaxf(mx4[t & 3], __uint_as_float(sv[c][t]));
      } else {
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c)
#pragma unroll
          for (int t = 0; t < 32; ++t)
            if (c * 32 + t >= lo && c * 32 + t < hi) mx4[t & 3] = fmaxf(mx4[t & 3], __uint_as_float(sv[c][t]));
      }
      const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
      const float m_tile = mx * sl2;
      const bool grow = m_tile > m_used + kRescale;  // this row's max moved by more than 2^8
      const bool rescale = __any_sync(0xffffffffu, grow);
      if (j > 0 && (TILES == 2 || rescale)) {
        // O holds P V of earlier tiles, and P_{j-1} lies where P_j goes (two tiles): wait for the last product
        if (!__all_sync(0xffffffffu,
                        mbar_wait(&o_done[buf(j - 1)], par(j - 1), a.status, kErrTimeoutAccFull))) {
          ok = false;
          break;
        }
        tc_fence_after();
      }
      if (j > 0 && rescale) {  // rescale the rows that grew
        // rows whose max was still -inf have an all-zero O row: any factor works
        const float f = grow ? (m_used == -INFINITY ? 0.f : ex2(m_used - m_tile)) : 1.f;
#pragma unroll 1
        for (int c = 0; c < kD / 32; ++c) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(o_base + c * 32, v);
          tmem_wait_ld();
#pragma unroll
          for (int t = 0; t < 32; ++t) v[t] = __float_as_uint(__uint_as_float(v[t]) * f);
          tmem_st_32x32b_x32(o_base + c * 32, v);
        }
        tmem_wait_st();
        l *= f;
      }
      if (grow) m_used = m_tile;
      auto weights = [&](auto masked) {
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int t = 0; t < 32; t += 2) {
            float p0, p1;
            fma2(p0, p1, sv[c][t], sv[c][t + 1], sl2, -m_used);
            p0 = ex2(p0);
            p1 = ex2(p1);
            if constexpr (decltype(masked)::value) {
              const int k0 = c * 32 + t;
              if (k0 < lo || k0 >= hi) p0 = 0.f;
              if (k0 + 1 < lo || k0 + 1 >= hi) p1 = 0.f;
            }
            l += p0 + p1;
            pk[t / 2] = pack_bf16x2(p0, p1);
          }
          tmem_st_32x32b_x16(pb + c * 16, pk);
        }
      };
      if (inside) weights(std::false_type{});
      else weights(std::true_type{});
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[buf(j)]);
    }
    if (ok && __all_sync(0xffffffffu, mbar_wait(&o_done[buf(n_tiles - 1)], par(n_tiles - 1), a.status,
                                                kErrTimeoutAccFull))) {
      tc_fence_after();
      const int head = hkv * G + g;
      float L = l, f = 1.f;
      if (a.sinks != nullptr) {
        const float sk = a.sinks[head] * kLog2e;
        const float Mx = fmaxf(m_used, sk);
        f = (m_used == -INFINITY) ? 0.f : ex2(m_used - Mx);
        L = L * f + ex2(sk - Mx);
      }
      const float inv = L > 0.f ? f / L : 0.f;
      const int t = my_tok0 + tok;
      if (a.lse != nullptr && a.sinks == nullptr && row_ok && !a.q_paged)  // training: log2-sum-exp2 of the scaled row
        a.lse[(int64_t)(q0 + t) * a.Hq + head] = L > 0.f ? m_used + __log2f(L) : -INFINITY;
      const int64_t orow = a.q_paged ? (int64_t)btab[min(t >> 4, max_page - 1)] * 16 + (t & 15) : (int64_t)(q0 + t);
      __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.out) +
                           orow * (a.out_ld ? a.out_ld : (int64_t)a.Hq * kD) + (int64_t)head * kD;
#pragma unroll 1
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t v[32];
        tmem_ld_32x32b_x32(o_base + c * 32, v);
        tmem_wait_ld();
        if (row_ok) {
#pragma unroll
          for (int qd = 0; qd < 4; ++qd) {
            uint4 w;
            w.x = pack_bf16x2(__uint_as_float(v[qd * 8 + 0]) * inv, __uint_as_float(v[qd * 8 + 1]) * inv);
            w.y = pack_bf16x2(__uint_as_float(v[qd * 8 + 2]) * inv, __uint_as_float(v[qd * 8 + 3]) * inv);
            w.z = pack_bf16x2(__uint_as_float(v[qd * 8 + 4]) * inv, __uint_as_float(v[qd * 8 + 5]) * inv);
            w.w = pack_bf16x2(__uint_as_float(v[qd * 8 + 6]) * inv, __uint_as_float(v[qd * 8 + 7]) * inv);
            *reinterpret_cast<uint4*>(dst + c * 32 + qd * 8) = w;
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace fmha

bool fmha_supported(const AttnArgs& a) {
  static const bool legacy = [] {
    const char* e = std::getenv("B200_ATTN_LEGACY");
    return e != nullptr && e[0] == '1';
  }();
  const int G = a.Hq / a.Hkv;
  // logit softcapping runs on the mma.sync kernel, and so do scales below 0: row maxima are taken before the scale here
  return !legacy && a.D == 128 && a.softcap <= 0.f && a.scale >= 0.f && a.Hq % a.Hkv == 0 && G >= 1 && G <= 8 &&
         (G & (G - 1)) == 0 && a.q_rows > 0;
}

void fmha_launch(const AttnArgs& a, cudaStream_t st) {
  using namespace fmha;
  const int G = a.Hq / a.Hkv;
  const int rows_tok = 128 / G;
  CUtensorMap tq = make_tmap_3d(a.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kD, a.Hq, a.q_rows, kD,
                                (uint64_t)a.Hq * kD, 64, G, 16);
  CUtensorMap tk, tv;
  if (a.kv_contig) {  // [pages, Hkv, 16, D]: 8 pages of one head = box [8][1][16][64]
    tk = make_tmap_4d(a.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kD, 16, a.Hkv, a.num_blocks, 64, 16, 1, 8);
    tv = make_tmap_4d(a.v_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kD, 16, a.Hkv, a.num_blocks, 64, 16, 1, 8);
  } else if (a.kv_dense) {  // [rows, Hkv, D]: one 16-row page of one head = box [16][1][64]
    tk = make_tmap_3d(a.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kD, a.Hkv, a.kv_rows, kD,
                      (uint64_t)a.Hkv * kD, 64, 1, 16);
    tv = make_tmap_3d(a.v_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kD, a.Hkv, a.kv_rows, kD,
                      (uint64_t)a.Hkv * kD, 64, 1, 16);
  } else {
    const int64_t kv_rows = a.num_blocks * a.Hkv * 16;
    tk = make_tmap_2d(a.k_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kv_rows, kD, kD, 16, 64);
    tv = make_tmap_2d(a.v_cache, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, kv_rows, kD, kD, 16, 64);
  }
  const int q_tiles = (a.max_q_len + rows_tok - 1) / rows_tok;
  auto run = [&](auto kernel, int tiles, uint32_t smem, int threads) {
    const int q_blocks = (q_tiles + tiles - 1) / tiles;
    ensure_smem(kernel, smem);
    launch_pdl(kernel, dim3(a.B * q_blocks, a.Hkv), dim3(threads), smem, st, tq, tk, tv, a, q_blocks, rows_tok);
  };
  // Two query tiles a CTA where single ones would not find an SM each: one sequence over 8192 tokens with 148 tiles takes
  // 82 us in single ones, with 152 tiles 115 in pairs (two rounds of single ones would be 164).
  if (q_tiles > 1 && (int64_t)a.B * q_tiles * a.Hkv > num_sms(a.device))
    run(fmha_fwd_kernel<2>, 2, Cfg<2>::SMEM, Cfg<2>::THREADS);
  else
    run(fmha_fwd_kernel<1>, 1, Cfg<1>::SMEM, Cfg<1>::THREADS);
}

}  // namespace b200
