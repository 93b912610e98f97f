// Paged KV cache in 8 bits: int8 codes [NB, Hkv, 16, D] with one power-of-two
// scale per (block, KV head), value = code * scale. Three kernels write, widen
// and attend over such pages:
//
// * store: new rows are quantised into their blocks. For the rows x of a block
//   and head, s = 2^e with the smallest e >= -100 such that max|x| <= 127 s, and
//   code = rint(x / s). A block that is already partly filled keeps
//   s' = max(s_old, s) and its old codes become rint(code * s_old / s'). Because
//   scales are powers of two the quotients are exact, so the codes are those of
//   the definition in exact arithmetic, and because each growth at least doubles
//   s the errors of repeated requantisation add up to at most one step (a sum
//   1/2 + 1/4 + ... of the last scale). A scale amax / 127 would be
//   3.4 dB finer on average for a block written at once, but rounds the old codes
//   again at every new maximum of a block that grows token by token.
// * dequant: bf16 copies of the pages of a prefill batch (exact: 7-bit codes
//   times a power of two fit bf16's 8-bit significand).
// * attention: decode and short multi-token (draft verification) queries read
//   the codes directly, see attn_kernel.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>
#include <string>

#include "../common/b200.cuh"
#include "../common/launch.h"
#include "../common/pdl_launch.h"
#include "../common/tma_host.h"

namespace b200 {
namespace kv8 {

constexpr int kMinExp = -100;  // smallest scale 2^-100: an all-zero block still has a usable reciprocal

// ---------------------------------------------------------------------------
// store
// ---------------------------------------------------------------------------
constexpr int kStoreWarps = 8;

// One warp per (run of adjacent tokens of one block, KV head, K or V). Lane l
// owns 16 columns of the rows l / (D / 16) + i * (512 / D): 16-byte code loads
// and stores, 32-byte bf16 loads, all rows of the block in flight at once. The
// kernel moves 3 bytes per element and is bound by launch and load latency for
// a decode step, by HBM for a prefill.
template <int D>
__global__ void __launch_bounds__(kStoreWarps * 32) store_kernel(KvInt8StoreArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int CPR = D / 16;       // 16-column chunks per row
  constexpr int RPW = 32 / CPR;     // rows per warp pass
  constexpr int NI = 16 / RPW;      // passes over a block
  const int lane = threadIdx.x & 31;
  const int64_t task = (int64_t)blockIdx.x * kStoreWarps + (threadIdx.x >> 5);
  const int per_group = a.Hkv * 2;
  const int64_t grp = task / per_group;
  const int hk = (int)(task % per_group);
  const int h = hk >> 1;
  const bool is_v = (hk & 1) != 0;
  const int64_t t0 = grp * a.group, t1 = min(t0 + (int64_t)a.group, a.T);
  if (t0 >= a.T) return;
  const __nv_bfloat16* x = is_v ? a.v : a.k;
  const int64_t xt = is_v ? a.v_stride_t : a.k_stride_t, xh = is_v ? a.v_stride_h : a.k_stride_h;
  int8_t* codes = is_v ? a.v_cache : a.k_cache;
  float* scales = is_v ? a.v_scale : a.k_scale;

  for (int64_t t = t0; t < t1; ++t) {
    const int64_t slot = a.slots[t];
    if (slot < 0) continue;
    const int64_t blk = slot >> 4;
    if (t > 0) {  // only the first token of a run of one block works
      const int64_t prev = a.slots[t - 1];
      if (prev >= 0 && (prev >> 4) == blk) continue;
    }
    if (blk >= a.num_blocks) {
      if (lane == 0) report_error(a.status, kErrBounds, (int)min(blk, (int64_t)0x7fffffff));
      continue;
    }
    // lane o < 16: newest token of the run written at offset o (-1: none)
    int64_t src = -1;
    for (int64_t base = t;; base += 32) {
      const int64_t tt = base + lane;
      const int64_t s = tt < a.T ? a.slots[tt] : -1;
      const bool same = s >= 0 && (s >> 4) == blk;
      const unsigned in = __ballot_sync(0xffffffffu, same);
      const int len = in == 0xffffffffu ? 32 : __ffs(~in) - 1;  // tokens of the run in this chunk
      const int off = (int)(s & 15);
#pragma unroll
      for (int o = 0; o < 16; ++o) {
        const unsigned m = __ballot_sync(0xffffffffu, lane < len && off == o);
        if (lane == o && m != 0) src = base + (31 - __clz(m));
      }
      if (len < 32) break;
    }
    const bool fresh = __shfl_sync(0xffffffffu, src, 0) >= 0;
    const int64_t page = (blk * a.Hkv + h);
    const int c = (lane % CPR) * 16;
    uint4 lo[NI], hi[NI];
    bool given[NI];
    uint32_t amax = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = lane / CPR + i * RPW;
      const int64_t st = __shfl_sync(0xffffffffu, src, r);
      given[i] = st >= 0;
      if (given[i]) {
        const uint4* p = reinterpret_cast<const uint4*>(x + st * xt + h * xh + c);
        lo[i] = p[0];
        hi[i] = p[1];
      }
    }
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      if (given[i]) {
        const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {  // magnitudes of bf16 order like their bits; infinities and NaN do not count
          const uint32_t u = w[j] & 0x7fffu, v = (w[j] >> 16) & 0x7fffu;
          amax = max(amax, max(u < 0x7f80u ? u : 0u, v < 0x7f80u ? v : 0u));
        }
      }
    }
    amax = __reduce_max_sync(0xffffffffu, amax);
    // amax = (1 + m / 128) 2^E <= 127 * 2^e = (1 + 126 / 128) 2^(e + 6)
    const int e = max((int)(amax >> 7) - 127 - 6 + ((amax & 127u) == 127u ? 1 : 0), kMinExp);
    float s = __int_as_float((e + 127) << 23), ratio = 0.f;
    if (!fresh) {
      const float old = scales[page];
      s = fmaxf(s, old);
      ratio = old / s;
    }
    const float inv = 1.f / s;  // a power of two: exact
    int8_t* dst = codes + page * (16 * D);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = lane / CPR + i * RPW;
      uint4* p = reinterpret_cast<uint4*>(dst + r * D + c);
      uint32_t o[4];
      if (given[i]) {
        const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          // __float2int_rn: ties to even, NaN -> 0, infinities saturate (then clamp)
          const int q0 = max(-127, min(127, __float2int_rn(bf16_lo(w[2 * j]) * inv)));
          const int q1 = max(-127, min(127, __float2int_rn(bf16_hi(w[2 * j]) * inv)));
          const int q2 = max(-127, min(127, __float2int_rn(bf16_lo(w[2 * j + 1]) * inv)));
          const int q3 = max(-127, min(127, __float2int_rn(bf16_hi(w[2 * j + 1]) * inv)));
          o[j] = __byte_perm(__byte_perm(q0, q1, 0x0040), __byte_perm(q2, q3, 0x0040), 0x5410);
        }
      } else if (fresh) {
        o[0] = o[1] = o[2] = o[3] = 0;
      } else if (ratio != 1.f) {
        const uint4 old = *p;
        const uint32_t w[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t acc = 0;
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const int q = (int)(int8_t)(w[j] >> (8 * b));
            acc |= ((uint32_t)__float2int_rn((float)q * ratio) & 255u) << (8 * b);
          }
          o[j] = acc;
        }
      } else {
        continue;
      }
      *p = make_uint4(o[0], o[1], o[2], o[3]);
    }
    if (lane == 0) scales[page] = s;
  }
}

// ---------------------------------------------------------------------------
// bf16 copies of pages
// ---------------------------------------------------------------------------
// 4 codes -> 4 bf16 values code * s, exact: 2^23 + (code + 128) as a float is
// built by a byte permute, the offset subtracted, the product a power-of-two one.
__device__ __forceinline__ uint2 widen_bf16(uint32_t w, float s) {
  const uint32_t u = w ^ 0x80808080u;
  const float f0 = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7440)) - 8388736.f) * s;
  const float f1 = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7441)) - 8388736.f) * s;
  const float f2 = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7442)) - 8388736.f) * s;
  const float f3 = (__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7443)) - 8388736.f) * s;
  return make_uint2(pack_bf16x2(f0, f1), pack_bf16x2(f2, f3));
}

// One CTA per (sequence, page): every KV head, K and V. 1 byte read and 2
// written per element: bound by HBM.
__global__ void __launch_bounds__(256) dequant_kernel(KvInt8DequantArgs a) {
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / a.max_blocks, p = blockIdx.x % a.max_blocks;
  const int ctx = a.ctx_lens[b];
  if (p * 16 >= ctx && p > 0) return;
  const int64_t id = a.tables[(int64_t)b * a.max_blocks + p];
  const bool known = id >= 0 && id < a.num_blocks && ctx > 0;
  if (!known && ctx > 0 && threadIdx.x == 0) report_error(a.status, kErrBounds, (int)id);
  const int head = 16 * a.D, n = a.Hkv * head;
  const int64_t dst = (int64_t)blockIdx.x * n;
  if (!known) {  // the first page of an empty sequence, which attention may still load, and pages that do not exist
    for (int i = threadIdx.x * 8; i < n; i += 256 * 8) {
      *reinterpret_cast<uint4*>(a.k_out + dst + i) = make_uint4(0, 0, 0, 0);
      *reinterpret_cast<uint4*>(a.v_out + dst + i) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  for (int i = threadIdx.x * 16; i < 2 * n; i += 256 * 16) {
    const bool is_v = i >= n;
    const int j = is_v ? i - n : i;
    const int8_t* codes = is_v ? a.v_cache : a.k_cache;
    const float s = (is_v ? a.v_scale : a.k_scale)[id * a.Hkv + j / head];
    const uint4 w = *reinterpret_cast<const uint4*>(codes + id * n + j);
    __nv_bfloat16* out = (is_v ? a.v_out : a.k_out) + dst + j;
    const uint2 x = widen_bf16(w.x, s), y = widen_bf16(w.y, s), z = widen_bf16(w.z, s), u = widen_bf16(w.w, s);
    reinterpret_cast<uint4*>(out)[0] = make_uint4(x.x, x.y, y.x, y.y);
    reinterpret_cast<uint4*>(out)[1] = make_uint4(z.x, z.y, u.x, u.y);
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// Work is cut evenly over the grid, whatever the lengths: the pages of every
// (sequence, KV head, block of query rows) lie end to end in one line of units,
// CTA i takes units [i U / N, (i + 1) U / N). A segment that one CTA covers is
// written out by it, the parts of the others are joined by merge_kernel, which
// repeats the same arithmetic; so the workspace has two slots per CTA and does
// not grow with the contexts.
//
// Inside a CTA the four warps take pages in turn, each with its own TMA ring
// (no exchange between warps until a segment ends), running maximum, sum and
// accumulators. Both products run transposed, S^T = K Q^T and O^T = V^T P^T
// (mma m16n8k16, f16 operands, f32 sums): the 16 keys of a page and 16 of its
// columns fill the 16-row operand, and 8 query rows (the group of a KV head) the
// 8-column one, half the multiplies of the other orientation for a group of 4.
//   * K: ldmatrix hands a thread 4 consecutive codes of a key; a product does
//     not care in which order its terms come, so Q is held in that order.
//   * V: ldmatrix.trans moves pairs of bytes, a thread gets (d, d + 1) of two
//     keys: rows g and g + 8 of the operand are columns 2 g and 2 g + 1.
//   * codes widen exactly: the byte code + 128 under the exponent of 1024 is
//     1024 + 128 + code in f16; K subtracts 1152 and folds its scale into the
//     scores, V computes code * (s / s_ref) by one fma, with s_ref the largest
//     V scale of the warp's pages so far (powers of two: exact down to 2^-24).
//   * Q is scaled by a power of two per row to below 2, so that any bf16 row
//     keeps its 8 bits in f16. P is rounded to f16 (2^-12 of each weight).
//   * weights are 2^(score - m) with m 8 below the running maximum, so that f16
//     holds weights down to 2^-22 of the largest with all its bits and loses none
//     above 2^-33: long contexts have most of their mass in small weights. m moves
//     only when a score exceeds it by 15 (2^15 fits f16), so most pages need no
//     exchange between lanes and no rescaling.
template <int D_, int NT_>
struct Cfg {
  static constexpr int D = D_, NT = NT_, ROWS = 8 * NT_, STEPS = D_ / 16;
  static constexpr int PAGE = 16 * D_, STAGE = 2 * PAGE;
  static constexpr int CTAS = NT_ == 1 ? 4 : (NT_ == 2 ? 3 : 2);  // resident per SM (registers)
  static constexpr int NST = (NT_ <= 2 ? 3 : (NT_ == 3 ? 4 : 5)) * (D_ == 64 ? 2 : 1);
  static constexpr int RING = 4 * NST * STAGE;
  static constexpr int OLD = D_ + 4;  // padded row of the exchange buffer, in floats
  static constexpr int EXCH = 4 * ROWS * OLD * 4;
  static constexpr int MAIN = RING > EXCH ? RING : EXCH;
  static constexpr int QLD = D_ * 2 + 32;  // padded Q row in bytes (conflict-free 8-byte loads)
  static constexpr bool QS = NT_ > 2;      // Q in shared memory instead of registers
  static constexpr int QBYTES = QS ? ROWS * QLD : 0;
  static constexpr int STATS = 4 * ROWS * 3 * 4;
  static constexpr int FIXED = MAIN + QBYTES + STATS + 4 * NST * 8 + 64;
  static constexpr int smem(int B) { return 1024 + FIXED + (B + 1) * 8; }
};

struct SeqInfo {
  int ctx, n, q0, lo, pages, rb;
};

template <int ROWS>
__device__ __forceinline__ SeqInfo seq_info(const PagedInt8Args& a, int b) {
  SeqInfo s;
  s.ctx = min(max(a.ctx_lens[b], 0), a.max_blocks * 16);
  if (a.cu_q != nullptr) {
    const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
    s.q0 = min(max(lo, 0), a.T);
    s.n = min(max(hi - lo, 0), min(a.T - s.q0, a.max_q_len));
  } else {
    s.q0 = b;
    s.n = 1;
  }
  s.lo = 0;
  if (a.window > 0) s.lo = max(0, s.ctx - s.n - a.window + 1) / 16;
  s.pages = (s.ctx + 15) / 16 - s.lo;
  s.rb = (s.n * a.G + ROWS - 1) / ROWS;
  return s;
}

__device__ __forceinline__ int64_t cta_begin(int64_t i, int64_t U, int64_t N) { return i * U / N; }

// CTAs that work when there are U units: at least 4 units (one per warp) each.
__device__ __forceinline__ int64_t active_ctas(int64_t U, int grid) {
  const int64_t n = (U + 3) / 4;
  return n < grid ? n : grid;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2_add(uint32_t a, uint32_t b) {
  const __half2 r = __hadd2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<__half2*>(&a), *reinterpret_cast<__half2*>(&b),
                            *reinterpret_cast<__half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t dup_h2(float a) { return pack_h2(a, a); }

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kShift = 8.f;  // m: the running maximum minus this (log2), see above
constexpr float kLimit = 15.f;  // a score above m + kLimit moves m

// Byte offset of 16-byte chunk c of row r in a page written by TMA with the
// swizzle of its row width (128-byte rows: chunk ^ row; 64-byte rows: chunk ^ row / 2).
template <int D>
__device__ __forceinline__ uint32_t page_off(int r, int c) {
  return D == 128 ? (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)) : (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4));
}

template <int D, int NT>
__global__ void __launch_bounds__(128, Cfg<D, NT>::CTAS) attn_kernel(const __grid_constant__ CUtensorMap tmK,
                                                                     const __grid_constant__ CUtensorMap tmV,
                                                                     PagedInt8Args a) {
  using C = Cfg<D, NT>;
  constexpr int ROWS = C::ROWS, STEPS = C::STEPS, NST = C::NST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  uint8_t* qs = base + C::MAIN;
  float* st_m = reinterpret_cast<float*>(qs + C::QBYTES);  // [4][ROWS] per warp: maximum, sum, V reference scale
  float* st_l = st_m + 4 * ROWS;
  float* st_r = st_l + 4 * ROWS;
  uint64_t* bars = reinterpret_cast<uint64_t*>(st_r + 4 * ROWS);
  int64_t* wsum = reinterpret_cast<int64_t*>(bars + 4 * NST);  // [4] + failure flag
  int* s_fail = reinterpret_cast<int*>(wsum + 4);
  int64_t* pre = reinterpret_cast<int64_t*>(base + C::FIXED);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  uint64_t* full = bars + warp * NST;
  uint8_t* ring = base + warp * NST * C::STAGE;

  if (lane == 0)
    for (int i = 0; i < NST; ++i) mbar_init(&full[i], 1);
  if (tid == 0) {
    *s_fail = 0;
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  fence_mbarrier_init();
  pdl_wait();
  pdl_trigger();

  // prefix sums of the units of every sequence
  const int per = (a.B + 127) / 128;
  int64_t mine = 0;
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < a.B) {
      const SeqInfo s = seq_info<ROWS>(a, b);
      mine += (int64_t)a.Hkv * s.rb * s.pages;
    }
  }
  int64_t inc = mine;
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) wsum[warp] = inc;
  __syncthreads();
  int64_t run = inc - mine;
  for (int w = 0; w < warp; ++w) run += wsum[w];
  for (int i = 0; i < per; ++i) {
    const int b = tid * per + i;
    if (b < a.B) {
      pre[b] = run;
      const SeqInfo s = seq_info<ROWS>(a, b);
      run += (int64_t)a.Hkv * s.rb * s.pages;
    }
  }
  const int64_t U = wsum[0] + wsum[1] + wsum[2] + wsum[3];
  if (tid == 0) pre[a.B] = U;
  __syncthreads();
  const int64_t N = active_ctas(U, gridDim.x);
  if (blockIdx.x >= N) return;
  const int64_t u0 = cta_begin(blockIdx.x, U, N), u1 = cta_begin(blockIdx.x + 1, U, N);

  const uint32_t bias = 0xE480E480u;  // f16x2 of -1152
  uint32_t it = 0;                    // pages this warp has taken from its ring (stage and parity)
  int64_t u = u0;
  int b = 0;
  {  // last b with pre[b] <= u0 (empty sequences share a prefix: take the last)
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u0) lo = mid;
      else hi = mid;
    }
    b = lo;
  }

  while (u < u1) {
    while (pre[b + 1] <= u) ++b;
    const SeqInfo sq = seq_info<ROWS>(a, b);
    const int64_t rel = u - pre[b];
    const int hs = (int)(rel / sq.pages);
    const int h = hs / sq.rb, rb = hs % sq.rb;
    const int64_t seg0 = pre[b] + (int64_t)hs * sq.pages, seg1 = seg0 + sq.pages;
    const int64_t ue = seg1 < u1 ? seg1 : u1;
    const int pa = sq.lo + (int)(u - seg0), pb = sq.lo + (int)(ue - seg0);
    const int row0 = rb * ROWS, nrows = min(ROWS, sq.n * a.G - row0);
    const int pos0 = sq.ctx - sq.n;  // position of the first new token

    // ---- pages of this warp: pa + warp + 4 j, j < cnt; lane i holds the block of page j = 32 k + i ----
    const int cnt = pb - pa > warp ? (pb - pa - warp + 3) / 4 : 0;
    const int32_t* tab = a.tables + (int64_t)b * a.max_blocks + pa + warp;
    auto fetch = [&](int j0, int& id, float& sk, float& sv) {
      id = 0;
      sk = sv = 0.f;
      if (j0 + lane < cnt) {
        id = tab[4 * (j0 + lane)];
        if (id < 0 || id >= a.num_blocks) {
          report_error(a.status, kErrBounds, id);
          id = 0;
        } else {
          sk = a.k_scale[(int64_t)id * a.Hkv + h];
          sv = a.v_scale[(int64_t)id * a.Hkv + h];
        }
      }
    };
    int id0, id1;
    float sk0, sk1, sv0, sv1;
    fetch(0, id0, sk0, sv0);
    auto issue = [&](int id, uint32_t slot) {  // one lane
      uint8_t* dst = ring + slot * C::STAGE;
      mbar_arrive_expect_tx(&full[slot], C::STAGE);
      const int y = (id * a.Hkv + h) * 16;
      tma_load_2d(dst, &tmK, &full[slot], 0, y);
      tma_load_2d(dst + C::PAGE, &tmV, &full[slot], 0, y);
    };
#pragma unroll 1
    for (int j = 0; j < NST && j < cnt; ++j) {
      const int id = __shfl_sync(0xffffffffu, id0, j);
      if (lane == 0) issue(id, (it + j) % NST);
    }
    fetch(32, id1, sk1, sv1);

    // ---- Q: rows n = g of each tile in the order of the K fragments, scaled to below 2 ----
    uint32_t qf[C::QS ? 1 : NT][STEPS][2];
    float rs[NT][2];  // score factors of columns 2 t4 and 2 t4 + 1
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = row0 + nt * 8 + g;
      uint2 w[STEPS];
      uint32_t am = 0;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) w[s] = make_uint2(0, 0);
      if (nt * 8 + g < nrows) {
        const int tok = r / a.G, head = h * a.G + r % a.G;
        const __nv_bfloat16* qp = a.q + ((int64_t)(sq.q0 + tok) * a.Hq + head) * D + 4 * t4;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) w[s] = *reinterpret_cast<const uint2*>(qp + 16 * s);
      }
#pragma unroll
      for (int s = 0; s < STEPS; ++s)
        am = max(am, max(max(w[s].x & 0x7fffu, (w[s].x >> 16) & 0x7fffu),
                         max(w[s].y & 0x7fffu, (w[s].y >> 16) & 0x7fffu)));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
      const int e = min(max((int)(am >> 7) - 127, -100), 120);
      const float down = __int_as_float((127 - e) << 23), up = __int_as_float((127 + e) << 23);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint32_t x = pack_h2(bf16_lo(w[s].x) * down, bf16_hi(w[s].x) * down);
        const uint32_t y = pack_h2(bf16_lo(w[s].y) * down, bf16_hi(w[s].y) * down);
        if constexpr (C::QS) {
          if (warp == 0) *reinterpret_cast<uint2*>(qs + (nt * 8 + g) * C::QLD + 32 * s + 8 * t4) = make_uint2(x, y);
        } else {
          qf[nt][s][0] = x;
          qf[nt][s][1] = y;
        }
      }
      rs[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t4) * a.scale;
      rs[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t4 + 4) * a.scale;
    }
    if constexpr (C::QS) __syncthreads();

    float o[NT][STEPS][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) o[nt][s][0] = o[nt][s][1] = o[nt][s][2] = o[nt][s][3] = 0.f;
    }
    float sref = 0.f, iref = 0.f;
    // positions of this thread's columns (query rows 2 t4, 2 t4 + 1 of each tile)
    const int first_pos = pos0 + row0 / a.G, last_pos = pos0 + (row0 + max(nrows, 1) - 1) / a.G;

    int j = 0;
    bool dead = false;
#pragma unroll 1
    for (; j < cnt; ++j) {
      if ((j & 31) == 0 && j > 0) {
        id0 = id1;
        sk0 = sk1;
        sv0 = sv1;
        fetch(j + 32, id1, sk1, sv1);
      }
      const uint32_t n_it = it + j;
      const uint32_t slot = n_it % NST;
      const float sk = __shfl_sync(0xffffffffu, sk0, j & 31);
      const float sv = __shfl_sync(0xffffffffu, sv0, j & 31);
      const int jn = j + NST;
      const int idn = __shfl_sync(0xffffffffu, (jn >> 5) == (j >> 5) ? id0 : id1, jn & 31);
      if (!mbar_wait(&full[slot], (n_it / NST) & 1, a.status, kErrTimeoutFull)) {
        dead = true;
        break;
      }
      const uint32_t kb = smem_u32(ring + slot * C::STAGE), vb = kb + C::PAGE;
      // codes of the page into registers, then the slot is free for page j + NST
      uint32_t kw[STEPS][2], vw[STEPS][2];
#pragma unroll
      for (int s = 0; s < STEPS; s += 2) {
        const uint32_t off = page_off<D>((lane & 7) + ((lane >> 3) & 1) * 8, s + (lane >> 4));
        ldmatrix_x4(kb + off, kw[s][0], kw[s][1], kw[s + 1][0], kw[s + 1][1]);
        ldmatrix_x4_trans(vb + off, vw[s][0], vw[s][1], vw[s + 1][0], vw[s + 1][1]);
      }
      __syncwarp();
      if (lane == 0 && jn < cnt) issue(idn, slot);

      // S^T = K Q^T
      float sc[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint32_t x = kw[s][0] ^ 0x80808080u, y = kw[s][1] ^ 0x80808080u;
        const uint32_t a0 = h2_add(__byte_perm(x, 0x64646464u, 0x4140), bias);
        const uint32_t a1 = h2_add(__byte_perm(y, 0x64646464u, 0x4140), bias);
        const uint32_t a2 = h2_add(__byte_perm(x, 0x64646464u, 0x4342), bias);
        const uint32_t a3 = h2_add(__byte_perm(y, 0x64646464u, 0x4342), bias);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          if constexpr (C::QS) {
            const uint2 q2 = *reinterpret_cast<const uint2*>(qs + (nt * 8 + g) * C::QLD + 32 * s + 8 * t4);
            mma_f16(sc[nt], a0, a1, a2, a3, q2.x, q2.y);
          } else {
            mma_f16(sc[nt], a0, a1, a2, a3, qf[nt][s][0], qf[nt][s][1]);
          }
        }
      }

      // scores in units of log2, masks
      const int key0 = (pa + warp + 4 * j) * 16;
      const bool edge = key0 + 15 > first_pos || (a.window > 0 && key0 <= last_pos - a.window);
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float x = sc[nt][i] * (rs[nt][i & 1] * sk);
          if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
          x *= kLog2e;
          if (edge) {
            const int key = key0 + g + (i >> 1) * 8;
            const int pos = pos0 + (row0 + nt * 8 + 2 * t4 + (i & 1)) / a.G;
            if (key > pos || (a.window > 0 && key <= pos - a.window)) x = -INFINITY;
          }
          sc[nt][i] = x;
          grow |= x > m[nt][i & 1] + kLimit;
        }
      }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = fmaxf(m[nt][c], fmaxf(sc[nt][c], sc[nt][2 + c]) - kShift);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float f = mx == -INFINITY ? 1.f : ex2(m[nt][c] - mx);
            m[nt][c] = mx;
            l[nt][c] *= f;
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
              o[nt][s][c] *= f;
              o[nt][s][2 + c] *= f;
            }
          }
        }
      }
      // weights, transposed to the operand order
      uint32_t pf[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float m0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], m1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
        const float p0 = ex2(sc[nt][0] - m0), p1 = ex2(sc[nt][1] - m1);
        const float p2 = ex2(sc[nt][2] - m0), p3 = ex2(sc[nt][3] - m1);
        l[nt][0] += p0 + p2;
        l[nt][1] += p1 + p3;
        pf[nt][0] = transpose8x8(pack_h2(p0, p1));
        pf[nt][1] = transpose8x8(pack_h2(p2, p3));
      }
      // O^T += V^T P^T
      if (sv > sref) {  // a larger V scale: the sums are kept in units of the largest
        const float f = sref / sv;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[nt][s][i] *= f;
        sref = sv;
        iref = 1.f / sv;
      }
      const float c = sv * iref;
      const uint32_t c2 = dup_h2(c), n2 = dup_h2(-1152.f * c);
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint32_t x = vw[s][0] ^ 0x80808080u, y = vw[s][1] ^ 0x80808080u;
        const uint32_t a0 = h2_fma(__byte_perm(x, 0x64646464u, 0x4240), c2, n2);
        const uint32_t a1 = h2_fma(__byte_perm(x, 0x64646464u, 0x4341), c2, n2);
        const uint32_t a2 = h2_fma(__byte_perm(y, 0x64646464u, 0x4240), c2, n2);
        const uint32_t a3 = h2_fma(__byte_perm(y, 0x64646464u, 0x4341), c2, n2);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][s], a0, a1, a2, a3, pf[nt][0], pf[nt][1]);
      }
    }
    if (dead) {  // copies in flight land before the CTA leaves
      const int issued = min(cnt, j + NST);
      for (int k = j + 1; k < issued; ++k)
        if (!mbar_wait(&full[(it + k) % NST], ((it + k) / NST) & 1, a.status, kErrTimeoutDrain)) break;
      if (lane == 0) *s_fail = 1;
    }
    it += cnt;

    // ---- join the four warps ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float s = l[nt][c];
        s += __shfl_xor_sync(0xffffffffu, s, 4);
        s += __shfl_xor_sync(0xffffffffu, s, 8);
        s += __shfl_xor_sync(0xffffffffu, s, 16);
        if (g == 0) {
          const int r = nt * 8 + 2 * t4 + c;
          st_m[warp * ROWS + r] = m[nt][c];
          st_l[warp * ROWS + r] = s;
          st_r[warp * ROWS + r] = sref;
        }
      }
    }
    __syncthreads();  // every ring is drained: its memory becomes the exchange buffer
    if (*s_fail) return;
    float* exch = reinterpret_cast<float*>(base);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nt * 8 + 2 * t4 + c;
        if (r < nrows) {
          float* dst = exch + (warp * ROWS + r) * C::OLD + 2 * g;
#pragma unroll
          for (int s = 0; s < STEPS; ++s)
            *reinterpret_cast<float2*>(dst + 16 * s) = make_float2(o[nt][s][c], o[nt][s][2 + c]);
        }
      }
    }
    __syncthreads();
    const bool whole = seg0 >= u0 && seg1 <= u1;
    float* part = a.ws + ((int64_t)blockIdx.x * 2 + (seg0 < u0 ? 0 : 1)) * ROWS * (D + 2);
    for (int i = tid; i < nrows * (D / 4); i += 128) {
      const int r = i / (D / 4), d = (i % (D / 4)) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) mx = fmaxf(mx, st_m[w * ROWS + r]);
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float sum = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = st_m[w * ROWS + r];
        const float f = mw == -INFINITY ? 0.f : ex2(mw - mx), fr = f * st_r[w * ROWS + r];  // (0 * NaN stays NaN)
        const float4 v = *reinterpret_cast<const float4*>(exch + (w * ROWS + r) * C::OLD + d);
        sum += f * st_l[w * ROWS + r];
        acc.x += fr * v.x;
        acc.y += fr * v.y;
        acc.z += fr * v.z;
        acc.w += fr * v.w;
      }
      const int rr = row0 + r, tok = rr / a.G, head = h * a.G + rr % a.G;
      if (whole) {
        if (a.sinks != nullptr && mx != -INFINITY) {
          const float sk2 = a.sinks[head] * kLog2e, top = fmaxf(mx, sk2), f = ex2(mx - top);
          sum = sum * f + ex2(sk2 - top);
          acc.x *= f;
          acc.y *= f;
          acc.z *= f;
          acc.w *= f;
        }
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // no visible key: 0
        uint2* dst = reinterpret_cast<uint2*>(a.out + ((int64_t)(sq.q0 + tok) * a.Hq + head) * D + d);
        *dst = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
      } else {
        *reinterpret_cast<float4*>(part + r * D + d) = acc;
        if (d == 0) {
          part[ROWS * D + r] = mx;
          part[ROWS * D + ROWS + r] = sum;
        }
      }
    }
    fence_proxy_async_smem();  // the exchange buffer is written by TMA next
    __syncthreads();
    u = ue;
  }
}

// Joins the parts of the segments that several CTAs share and writes zeros for
// rows without keys. One CTA of D threads per (sequence, query row of a KV head).
template <int D, int NT>
__global__ void __launch_bounds__(D) merge_kernel(PagedInt8Args a, int grid) {
  using C = Cfg<D, NT>;
  constexpr int ROWS = C::ROWS, NW = D / 32;
  __shared__ int64_t s_sum[2][NW];
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x, h = blockIdx.y, rr = blockIdx.z, tid = threadIdx.x;
  const SeqInfo sq = seq_info<ROWS>(a, b);
  if (rr >= sq.n * a.G) return;
  const int tok = rr / a.G, head = h * a.G + rr % a.G;
  __nv_bfloat16* out = a.out + ((int64_t)(sq.q0 + tok) * a.Hq + head) * D + tid;
  if (sq.pages <= 0) {
    *out = __float2bfloat16(0.f);
    return;
  }
  int64_t before = 0, all = 0;
  for (int i = tid; i < a.B; i += D) {
    const SeqInfo s = seq_info<ROWS>(a, i);
    const int64_t n = (int64_t)a.Hkv * s.rb * s.pages;
    all += n;
    if (i < b) before += n;
  }
  for (int o = 16; o > 0; o >>= 1) {
    before += __shfl_xor_sync(0xffffffffu, before, o);
    all += __shfl_xor_sync(0xffffffffu, all, o);
  }
  if ((tid & 31) == 0) {
    s_sum[0][tid >> 5] = before;
    s_sum[1][tid >> 5] = all;
  }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    before += s_sum[0][w];
    all += s_sum[1][w];
  }
  const int64_t U = all, N = active_ctas(U, grid);
  const int rb = rr / ROWS, r = rr % ROWS;
  const int64_t s0 = before + ((int64_t)h * sq.rb + rb) * sq.pages, s1 = s0 + sq.pages;
  const int64_t i0 = ((s0 + 1) * N - 1) / U, i1 = (s1 * N - 1) / U;  // first and last CTA of the segment
  if (i0 == i1) return;
  auto part = [&](int64_t i) {
    return a.ws + (i * 2 + (s0 < cta_begin(i, U, N) ? 0 : 1)) * ROWS * (D + 2);
  };
  float mx = -INFINITY;
  for (int64_t i = i0 + (tid & 31); i <= i1; i += 32) mx = fmaxf(mx, part(i)[ROWS * D + r]);
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  const float sk2 = a.sinks != nullptr ? a.sinks[head] * kLog2e : -INFINITY;
  const float top = fmaxf(mx, sk2);
  float acc = 0.f, sum = sk2 == -INFINITY ? 0.f : ex2(sk2 - top);
#pragma unroll 4
  for (int64_t i = i0; i <= i1; ++i) {
    const float* p = part(i);
    const float mi = p[ROWS * D + r];
    const float f = mi == -INFINITY ? 0.f : ex2(mi - top);
    sum += f * p[ROWS * D + ROWS + r];
    acc += f * p[r * D + tid];
  }
  *out = __float2bfloat16(sum == 0.f ? 0.f : acc / sum);
}

}  // namespace kv8

void kv_int8_store_launch(const KvInt8StoreArgs& args, int D, cudaStream_t st) {
  using namespace kv8;
  if (args.T == 0 || args.Hkv == 0) return;
  KvInt8StoreArgs a = args;
  // one token per warp keeps every warp on its own block when blocks get one token each (a decode
  // step); longer batches are prefill, where 15 of 16 warps would find that they have nothing to do
  a.group = a.T <= 1024 ? 1 : 16;
  const int64_t tasks = (a.T + a.group - 1) / a.group * a.Hkv * 2;
  const unsigned grid = (unsigned)((tasks + kStoreWarps - 1) / kStoreWarps);
  if (D == 128)
    launch_pdl(store_kernel<128>, dim3(grid), dim3(kStoreWarps * 32), 0, st, a);
  else
    launch_pdl(store_kernel<64>, dim3(grid), dim3(kStoreWarps * 32), 0, st, a);
}

void kv_int8_dequant_launch(const KvInt8DequantArgs& a, cudaStream_t st) {
  if (a.B == 0 || a.max_blocks == 0) return;
  launch_pdl(kv8::dequant_kernel, dim3((unsigned)(a.B * a.max_blocks)), dim3(256), 0, st, a);
}

namespace kv8 {
// 8-row query tiles of a CTA: as few as hold every row of a sequence, at most 4
static int tiles(int G, int max_q_len) { return std::min(4, (G * max_q_len + 7) / 8); }

static int grid_ctas(int nt, int device, int B, int Hkv, int G, int max_q_len, int max_blocks) {
  const int per_sm = nt == 1 ? 4 : (nt == 2 ? 3 : 2);
  const int64_t rb = ((int64_t)G * max_q_len + 8 * nt - 1) / (8 * nt);
  const int64_t units = (int64_t)B * Hkv * rb * max_blocks;
  return (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)per_sm * num_sms(device), (units + 3) / 4));
}

template <int D, int NT>
static void run(const PagedInt8Args& a, int grid, cudaStream_t st) {
  const uint64_t rows = (uint64_t)a.num_blocks * a.Hkv * 16;
  const CUtensorMapSwizzle sw = D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B;
  const CUtensorMap tk = make_tmap_2d(a.k_cache, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, D, D, 16, D, sw);
  const CUtensorMap tv = make_tmap_2d(a.v_cache, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, D, D, 16, D, sw);
  const int smem = Cfg<D, NT>::smem(a.B);
  auto k = attn_kernel<D, NT>;
  ensure_smem(k, smem);
  launch_pdl(k, dim3(grid), dim3(128), smem, st, tk, tv, a);
  launch_pdl(merge_kernel<D, NT>, dim3(a.B, a.Hkv, a.G * a.max_q_len), dim3(D), 0, st, a, grid);
}
}  // namespace kv8

int64_t paged_int8_ws_floats(int device, int B, int Hkv, int G, int D, int max_q_len, int max_blocks) {
  const int nt = kv8::tiles(G, max_q_len);
  return (int64_t)kv8::grid_ctas(nt, device, B, Hkv, G, max_q_len, max_blocks) * 2 * 8 * nt * (D + 2);
}

void paged_int8_launch(const PagedInt8Args& a, cudaStream_t st) {
  using namespace kv8;
  if (a.B == 0 || a.T == 0 || a.max_q_len == 0) return;
  const int nt = tiles(a.G, a.max_q_len);
  const int grid = grid_ctas(nt, a.device, a.B, a.Hkv, a.G, a.max_q_len, a.max_blocks);
  if (a.D == 128) {
    if (nt == 1) run<128, 1>(a, grid, st);
    else if (nt == 2) run<128, 2>(a, grid, st);
    else if (nt == 3) run<128, 3>(a, grid, st);
    else run<128, 4>(a, grid, st);
  } else {
    if (nt == 1) run<64, 1>(a, grid, st);
    else if (nt == 2) run<64, 2>(a, grid, st);
    else if (nt == 3) run<64, 3>(a, grid, st);
    else run<64, 4>(a, grid, st);
  }
}

}  // namespace b200
