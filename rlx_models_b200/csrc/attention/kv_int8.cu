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
#include <cfloat>
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
constexpr int kStoreWarps = 4;

// One warp per (run of adjacent tokens of one block, KV head, K or V). Lane l
// owns 16 columns of the rows l / (D / 16) + i * (512 / D): 16-byte code loads
// and stores, 32-byte bf16 loads, all rows of the block in flight at once. The
// kernel moves 3 bytes per element and is bound by launch and load latency for
// a decode step, by HBM for a prefill.
//
// Two runs of one block would be two warps that write one block and its scale, so
// only one of them does and the other is reported. In batches of up to kScan tokens
// a warp looks at the slots before its run, asked for beside its own; longer ones
// have a launch in front in which every run writes its name to its block's owner
// (whichever comes last stays), with nothing to clear first. 64 tokens of 64
// requests 3.0 us without the look and 3.2 with it, 256 5.3 and 5.9; a prompt of 1000
// 6.9 and 7.8 with the launch, of 8192 10.7 and 12.1 (8 heads of 128).
constexpr int kScan = 256;

// The first token of a run: a slot whose block is not the one before it.
__device__ __forceinline__ bool run_begins(int64_t before, int64_t slot) {
  return slot >= 0 && (before < 0 || (before >> 4) != (slot >> 4));
}

__global__ void __launch_bounds__(256) owner_kernel(KvInt8StoreArgs a) {
  pdl_wait();
  pdl_trigger();
  const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.T) return;
  const int64_t slot = a.slots[t], before = t > 0 ? a.slots[t - 1] : -1;
  if (run_begins(before, slot) && (slot >> 4) < a.num_blocks) a.owner[slot >> 4] = (int32_t)t;
}

template <int D, bool kOwner>
__global__ void __launch_bounds__(kStoreWarps * 32, 6) store_kernel(KvInt8StoreArgs a) {
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

  // slots of the group and behind it (lane i: token t0 + i), and the first tokens of the runs in the group
  const int64_t near = t0 + lane < a.T ? a.slots[t0 + lane] : -1;
  int64_t ahead = __shfl_up_sync(0xffffffffu, near, 1);
  if (lane == 0) ahead = t0 > 0 ? a.slots[t0 - 1] : -1;
  constexpr int kPrior = kOwner ? 0 : kScan / 32;
  uint32_t prior[kPrior + 1];  // low words of the slots in front (lane i: tokens i, 32 + i ...)
#pragma unroll
  for (int i = 0; i < kPrior; ++i) {
    const int t = i * 32 + lane;
    prior[i] = t < t0 ? reinterpret_cast<const uint32_t*>(a.slots)[2 * t] : ~0u;
  }
  unsigned firsts = __ballot_sync(0xffffffffu, t0 + lane < t1 && run_begins(ahead, near));
  while (firsts != 0) {
    const int at = __ffs(firsts) - 1;
    firsts &= firsts - 1;
    const int64_t blk = __shfl_sync(0xffffffffu, near, at) >> 4;
    if (blk >= a.num_blocks) {
      if (lane == 0) report_error(a.status, kErrBounds, (int)min(blk, (int64_t)0x7fffffff));
      continue;
    }
    const int64_t page = blk * a.Hkv + h;
    const float old = scales[page];  // (asked for early; used when the block is not new)
    bool other = false;  // a run of this block elsewhere in the batch
    if constexpr (kOwner) other = a.owner[blk] != (int32_t)(t0 + at);
#pragma unroll
    for (int i = 0; i < kPrior; ++i)
      if ((prior[i] >> 4) == (uint32_t)blk) other |= (a.slots[i * 32 + lane] >> 4) == blk;
    if (__any_sync(0xffffffffu, other)) {
      if (lane == 0) report_error(a.status, kErrOrder, (int)min(blk, (int64_t)0x7fffffff));
      continue;
    }
    // lane o < 16: newest token of the run written at offset o, from t0 (-1: none)
    int src = -1;
    int64_t slot = __shfl_down_sync(0xffffffffu, near, at);
    int span = 32 - at;  // lanes with a slot of this piece of the run
    for (int base = at;;) {
      const unsigned in = __ballot_sync(0xffffffffu, lane < span && slot >= 0 && (slot >> 4) == blk);
      const int len = in == 0xffffffffu ? 32 : __ffs(~in) - 1;  // tokens of the run in this piece
      const int off = lane < len ? (int)(slot & 15) : 16 + lane, off0 = __shfl_sync(0xffffffffu, off, 0);
      if (__all_sync(0xffffffffu, lane >= len || off == off0 + lane)) {  // one behind the other
        if (lane >= off0 && lane < off0 + len) src = base + lane - off0;
      } else {
        const unsigned same = __match_any_sync(0xffffffffu, off);  // tokens of one offset: the last one counts
        for (unsigned todo = __ballot_sync(0xffffffffu, off < 16 && (same >> lane) == 1u); todo != 0; todo &= todo - 1) {
          const int from = __ffs(todo) - 1;
          if (lane == __shfl_sync(0xffffffffu, off, from)) src = base + from;
        }
      }
      if (len < span) break;
      base += span;
      span = 32;
      slot = t0 + base + lane < a.T ? a.slots[t0 + base + lane] : -1;
    }
    const bool fresh = __shfl_sync(0xffffffffu, src, 0) >= 0;
    const int c = (lane % CPR) * 16;
    uint4 lo[NI], hi[NI];
    bool given[NI];
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int r = lane / CPR + i * RPW;
      const int st = __shfl_sync(0xffffffffu, src, r);
      given[i] = st >= 0;
      lo[i] = hi[i] = make_uint4(0, 0, 0, 0);
      if (given[i]) {
        const uint4* p = reinterpret_cast<const uint4*>(x + (t0 + st) * xt + h * xh + c);
        lo[i] = p[0];
        hi[i] = p[1];
      }
    }
    // magnitudes of bf16 order like their bits
    uint32_t amax2 = 0;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) amax2 = __vmaxu2(amax2, w[j] & 0x7fff7fffu);
    }
    uint32_t amax = __reduce_max_sync(0xffffffffu, max(amax2 & 0xffffu, amax2 >> 16));
    const bool finite = amax < 0x7f80u;
    if (!finite) {  // infinities and NaN do not count
      amax = 0;
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint32_t w[8] = {lo[i].x, lo[i].y, lo[i].z, lo[i].w, hi[i].x, hi[i].y, hi[i].z, hi[i].w};
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t u = w[j] & 0x7fffu, v = (w[j] >> 16) & 0x7fffu;
          amax = max(amax, max(u < 0x7f80u ? u : 0u, v < 0x7f80u ? v : 0u));
        }
      }
      amax = __reduce_max_sync(0xffffffffu, amax);
    }
    // amax = (1 + m / 128) 2^E <= 127 * 2^e = (1 + 126 / 128) 2^(e + 6)
    const int e = max((int)(amax >> 7) - 127 - 6 + ((amax & 127u) == 127u ? 1 : 0), kMinExp);
    float s = __int_as_float((e + 127) << 23), ratio = 0.f;
    if (!fresh) {
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
          float f[4] = {bf16_lo(w[2 * j]), bf16_hi(w[2 * j]), bf16_lo(w[2 * j + 1]), bf16_hi(w[2 * j + 1])};
          // x / s is exact, so that adding 1.5 * 2^23 rounds it once, ties to even: the code is the low byte
          uint32_t q[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v = f[k] * inv;
            if (!finite) v = v != v ? 0.f : fminf(fmaxf(v, -127.f), 127.f);
            q[k] = __float_as_uint(v + 12582912.f);
          }
          o[j] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
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

// The queries lo .. hi of a sequence lie within q and are no more than announced.
__device__ __forceinline__ bool queries_fit(int lo, int hi, int rows, int most) {
  return lo >= 0 && lo <= hi && hi <= rows && hi - lo <= most;
}

// One CTA per (sequence, page, quarter of its heads' codes): 16 codes a thread
// and step, up to four steps' loads in flight. 1 byte read and 2 written per
// element: bound by HBM.
constexpr int kDequantThreads = 128, kDequantSteps = 4;

__global__ void __launch_bounds__(kDequantThreads) dequant_kernel(KvInt8DequantArgs a) {
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x / a.out_blocks, p = blockIdx.x % a.out_blocks;
  const int id = p < a.max_blocks ? a.tables[(int64_t)b * a.max_blocks + p] : -1;
  const int ctx = min(max(a.ctx_lens[b], 0), a.max_blocks * 16);
  if (p == 0 && blockIdx.y == 0 && threadIdx.x == 0) {
    if (a.ctx_out != nullptr) a.ctx_out[b] = ctx;
    bool fits = a.ctx_lens[b] <= ctx;  // within its block table
    if (a.cu_q != nullptr) {
      const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
      fits = fits && queries_fit(lo, hi, a.q_rows, a.max_q_len);
      a.cu_out[b] = min(max(lo, 0), a.q_rows);  // attention over the copies stays within q
      if (b == a.B - 1) a.cu_out[a.B] = min(max(hi, 0), a.q_rows);
    }
    if (!fits) report_error(a.status, kErrBounds, b);
  }
  if (a.table_out != nullptr && blockIdx.y == 0 && threadIdx.x == 0) a.table_out[blockIdx.x] = blockIdx.x;
  const int pages = (ctx + 15) / 16, filled = (max(pages, 1) + a.pad - 1) / a.pad * a.pad;
  if (p >= filled) return;
  const bool known = p < pages && id >= 0 && id < a.num_blocks;
  if (!known && p < pages && threadIdx.x == 0) report_error(a.status, kErrBounds, id);
  const int head = 16 * a.D, n = a.Hkv * head;
  const int64_t src = (int64_t)id * n, dst = (int64_t)blockIdx.x * n;
  const int j0 = (blockIdx.y * kDequantSteps * kDequantThreads + threadIdx.x) * 16;
  uint4 w[kDequantSteps];
  float s[kDequantSteps];
#pragma unroll
  for (int k = 0; k < kDequantSteps; ++k) {  // K codes, then V codes
    const int j = j0 + k * kDequantThreads * 16;
    w[k] = make_uint4(0, 0, 0, 0);
    s[k] = 0.f;  // unknown pages and those behind a context that attention may still load hold zeros
    if (known && j < 2 * n) {
      const bool is_v = j >= n;
      const int c = is_v ? j - n : j;
      w[k] = __ldcs(reinterpret_cast<const uint4*>((is_v ? a.v_cache : a.k_cache) + src + c));
      s[k] = (is_v ? a.v_scale : a.k_scale)[(int64_t)id * a.Hkv + c / head];
    }
  }
#pragma unroll
  for (int k = 0; k < kDequantSteps; ++k) {
    const int j = j0 + k * kDequantThreads * 16;
    if (j < 2 * n) {
      const bool is_v = j >= n;
      __nv_bfloat16* out = (is_v ? a.v_out : a.k_out) + dst + (is_v ? j - n : j);
      const uint2 x = widen_bf16(w[k].x, s[k]), y = widen_bf16(w[k].y, s[k]);
      const uint2 z = widen_bf16(w[k].z, s[k]), u = widen_bf16(w[k].w, s[k]);
      asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out), "r"(x.x), "r"(x.y), "r"(y.x),
                   "r"(y.y), "r"(z.x), "r"(z.y), "r"(u.x), "r"(u.y)
                   : "memory");
    }
  }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
// Work is cut evenly over the warps of the grid, whatever the lengths: the pages
// of every (sequence, KV head, block of query rows) lie end to end in one line of
// units, warp i takes units [i c, (i + 1) c). A segment that one warp covers is
// written out by it, the parts of the others are joined by merge_kernel; so the
// workspace has two slots per warp (the segment it begins inside, the one it ends
// inside) and does not grow with the contexts. Warps do not meet: no barrier
// stands in the way of the loads, and the ring of a warp runs on into its next
// segment (block ids, then pages, are asked for while the last one is worked on).
// Where the host knows that no segment has more than kWholePages pages (a sliding
// window, a narrow block table), warps take whole segments in turn instead: no
// prefix sums, no parts, no second launch (128 requests with a window of 128
// tokens: 11.2 us instead of 20).
//
// Each warp has its own TMA ring, running maximum, sum and accumulators. Both
// products run transposed, S^T = K Q^T and O^T = V^T P^T (mma m16n8k16, f16
// operands, f32 sums): the 16 keys of a page and 16 of its columns fill the 16-row
// operand, and 8 query rows (the group of a KV head) the 8-column one, half the
// multiplies of the other orientation for a group of 4.
//   * K: ldmatrix hands a thread 4 consecutive codes of a key; a product does
//     not care in which order its terms come, so Q is held in that order.
//   * V: ldmatrix.trans moves pairs of bytes, a thread gets (d, d + 1) of two
//     keys: rows g and g + 8 of the operand are columns 2 g and 2 g + 1.
//   * codes become f16 without arithmetic: the byte code + 128 in the low bits of
//     a half is the subnormal (code + 128) 2^-24, which the tensor cores multiply
//     exactly; 3 integer instructions for 4 codes, where converting costs 5 (the
//     loop is bound by instruction issue, not by HBM). The offset is taken out
//     exactly: S starts at -128 sum(q), and O gets one more product per tile with
//     the constant -128 (page by page, so that nothing accumulates to cancel).
//     2^24 and the block's K scale go into the factor of the scores, its V scale
//     relative to a unit of the segment (the largest of its first 32 pages) into the
//     weights.
//   * Q is scaled by a power of two per row to below 2, so that a bf16 row
//     (below 2^116) keeps its 8 bits in f16. P is rounded to f16 (2^-12 of each weight).
//   * weights are 2^(score - m) times the V scale, with m 8 below the running maximum
//     of both, score + log2 of the scale, so that f16 holds products down to 2^-22 of
//     the largest with all its bits and loses none above 2^-33: long contexts have most
//     of their mass in small weights, and a page whose scale is far above or below the
//     others' counts by what it adds to the result. Sums of weights are fp32 and may
//     lie as far from 1 as the scales lie apart: up to 2^80 nothing is lost. m moves
//     only when it is exceeded by 15 (2^15 fits f16), so most pages need no exchange
//     between lanes and no rescaling.
template <int D_, int NT_>
struct Cfg {
  static constexpr int D = D_, NT = NT_, ROWS = 8 * NT_, STEPS = D_ / 16;
  static constexpr int PAGE = 16 * D_, STAGE = 2 * PAGE;
  static constexpr int PP = NT_ <= 2 ? 2 : 1;  // pages a warp works on at once (more registers than that do not fit)
  static constexpr int CTAS = 2;               // resident per SM (registers)
  // Pages on their way per warp. Deeper rings are slower: 3 pages of 4 KB for each of 8 warps of an SM already fill
  // the memory system, and what is asked for beyond only delays block ids, scales and queries behind it (64 requests
  // of 512 to 2304 tokens, 12 warps an SM: 52.6 us with 4 pages, 47.6 with 3, 45.2 with 2; 8 warps with 3: 45.2).
  static constexpr int NST = 3 * (D_ == 64 ? 2 : 1);
  static constexpr int RING = 4 * NST * STAGE;
  static constexpr int QLD = D_ * 2 + 32;  // padded Q row in bytes (conflict-free 8-byte loads)
  static constexpr int QBYTES = ROWS * QLD;  // per warp
  static constexpr int FIXED = RING + 4 * QBYTES + 4 * NST * 8 + 16;
  static constexpr int smem(int B) { return 1024 + FIXED + (B + 1) * 4; }
};

// Most pages that `tokens` neighbouring queries see through a window.
__host__ __device__ inline int window_pages(int window, int tokens) {
  return (int)(((long long)window + tokens - 1 + 14) / 16 + 1);
}

struct SeqInfo {
  int ctx, n, q0, pages, rb;  // pages: units of each of the rb blocks of query rows, at least the pages it sees
};

template <int ROWS>
__device__ __forceinline__ SeqInfo seq_info(const PagedInt8Args& a, int b) {
  SeqInfo s;
  s.ctx = min(max(a.ctx_lens[b], 0), a.max_blocks * 16);
  if (a.cu_q != nullptr) {
    const int lo = a.cu_q[b], hi = a.cu_q[b + 1];
    s.q0 = min(max(lo, 0), a.T);
    s.n = hi > lo ? (int)min((int64_t)hi - lo, (int64_t)min(a.T - s.q0, a.max_q_len)) : 0;
  } else {
    s.q0 = b;
    s.n = 1;
  }
  s.pages = (s.ctx + 15) / 16;
  if (a.window > 0) s.pages = min(s.pages, window_pages(a.window, min(s.n, (ROWS - 1) / a.G + 2)));
  s.rb = (s.n * a.G + ROWS - 1) / ROWS;
  return s;
}

// Pages [lo, hi) that the rows of block rb see.
struct PageRange {
  int lo, hi;
};

template <int ROWS>
__device__ __forceinline__ PageRange page_range(const PagedInt8Args& a, const SeqInfo& s, int rb) {
  const int pos0 = s.ctx - s.n, first = pos0 + rb * ROWS / a.G;
  const int last = pos0 + min(s.n * a.G - 1, rb * ROWS + ROWS - 1) / a.G;
  PageRange r;
  r.lo = a.window > 0 ? max(0, first - a.window + 1) / 16 : 0;
  r.hi = max(r.lo, last < 0 ? 0 : last / 16 + 1);
  return r;
}

// A context longer than its block table, queries that do not fit: what is too much is left out, and reported.
__device__ __forceinline__ void check_seq(const PagedInt8Args& a, int b) {
  if (a.ctx_lens[b] > (int64_t)a.max_blocks * 16 ||
      (a.cu_q != nullptr && !queries_fit(a.cu_q[b], a.cu_q[b + 1], a.T, a.max_q_len)))
    report_error(a.status, kErrBounds, b);
}

constexpr int kWholePages = 16;

// Units per warp: at least 4, below which joining parts costs more than the pages.
__device__ __forceinline__ int warp_units(int U, int grid) { return max(4, (U + 4 * grid - 1) / (4 * grid)); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
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

__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
  const __half2 r = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&r);
}
// 4 codes -> (code + 128) 2^-24 as f16 subnormals, two to a register: `flip` first, then bytes 0 and 2, bytes 1 and 3.
__device__ __forceinline__ uint32_t flip(uint32_t w) { return w ^ 0x80808080u; }
__device__ __forceinline__ uint32_t codes_even(uint32_t u) { return __byte_perm(u, 0, 0x4240); }
__device__ __forceinline__ uint32_t codes_odd(uint32_t u) { return __byte_perm(u, 0, 0x4341); }
constexpr uint32_t kMinus128 = 0x80808080u;  // f16x2 of -128 * 2^-24

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kShift = 8.f;  // m: the running maximum minus this (log2), see above
constexpr float kLimit = 15.f;  // a score above m + kLimit moves m
constexpr int kUnitExp = 60;    // the segment's unit lies within 2^-60 and 2^60, where sums of weights have room
constexpr float kFarScale = 0x1p100f, kNearLog = -80.f;  // scales further from the unit than these count as these
constexpr float kNone = -1e30f; // m before the first visible key: finite, so that a masked score (-inf) has weight 0

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
  constexpr int ROWS = C::ROWS, STEPS = C::STEPS, NST = C::NST, PP = C::PP;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* base = smem_raw + ((1024 - (smem_u32(smem_raw) & 1023)) & 1023);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t4 = lane & 3;
  uint8_t* ring = base + warp * NST * C::STAGE;
  uint8_t* qs = base + C::RING + warp * C::QBYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(base + C::RING + 4 * C::QBYTES) + warp * NST;
  int* wsum = reinterpret_cast<int*>(base + C::RING + 4 * C::QBYTES + 4 * NST * 8);
  int* pre = reinterpret_cast<int*>(base + C::FIXED);  // [B + 1] units in front of each sequence

  if (lane == 0)
    for (int i = 0; i < NST; ++i) mbar_init(&full[i], 1);
  if (tid == 0) {
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  fence_mbarrier_init();
  __syncwarp();
  pdl_wait();
  pdl_trigger();

  const int worker = blockIdx.x * 4 + warp, workers = gridDim.x * 4;
  const int rb_max = (a.G * a.max_q_len + ROWS - 1) / ROWS, segments = a.B * a.Hkv * rb_max;
  int U = 0;
  if (!a.whole) {
    // prefix sums of the units of every sequence
    const int per = (a.B + 127) / 128;
    int mine = 0;
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b < a.B) {
        const SeqInfo s = seq_info<ROWS>(a, b);
        mine += a.Hkv * s.rb * s.pages;
        if (blockIdx.x == 0) check_seq(a, b);
      }
    }
    int inc = mine;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    int run = inc - mine;
    for (int w = 0; w < warp; ++w) run += wsum[w];
    U = wsum[0] + wsum[1] + wsum[2] + wsum[3];
    for (int i = 0; i < per; ++i) {
      const int b = tid * per + i;
      if (b < a.B) {
        pre[b] = run;
        if (blockIdx.x == 0) a.ws_pre[b] = run;  // for merge_kernel
        if (i + 1 < per) {
          const SeqInfo s = seq_info<ROWS>(a, b);
          run += a.Hkv * s.rb * s.pages;
        }
      }
    }
    if (tid == 0) {
      pre[a.B] = U;
      if (blockIdx.x == 0) a.ws_pre[a.B] = U;
    }
    __syncthreads();
  }
  int u0, u1;
  if (a.whole) {  // units count this warp's own pages, one segment behind the other
    if (worker >= segments) return;
    u0 = 0;
    u1 = INT32_MAX;
  } else {
    const int chunk = warp_units(U, gridDim.x);
    if ((int64_t)worker * chunk >= U) return;
    u0 = worker * chunk;
    u1 = min(u0 + chunk, U);
  }

  // ---- the part of a segment at hand: units [u, ue) of [seg0, seg1), of which cnt hold pages that its rows see ----
  int u = u0, ue, seg0, seg1, page, cnt;
  int at = 0;  // pages of this warp before this part
  int b, h, row0, nrows, pos0, first_pos, last_pos, q0;
  const int32_t* tab;
  int seg = worker;  // (whole) the segment at hand
  if (!a.whole) {  // last b with pre[b] <= u0 (empty sequences share a prefix: the last of them is not empty)
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pre[mid] <= u0) lo = mid;
      else hi = mid;
    }
    b = lo;
  }
  // Lane i holds page j = 32 k + i of the current 32 and of the next: its first row in the cache, its scales; and the
  // block id of the 32 after. They are loaded 16 pages and more before they are needed.
  int y0 = 0, y1 = 0, id = 0;
  float sk0 = 0.f, sk1 = 0.f, sv0 = 0.f, sv1 = 0.f;
  // the part that follows: its first block ids (lane i: page i < n_cnt), its KV head
  int n_id = 0, n_cnt = 0, n_h = 0;
  auto load_ids = [&](int j0) { id = j0 + lane < cnt ? tab[j0 + lane] : 0; };
  auto known = [&](int i) { return i >= 0 && i < a.num_blocks; };
  auto resolve = [&](int j0, int& y, float& sk, float& sv) {
    y = 0;
    sk = sv = 0.f;
    if (j0 + lane < cnt) {
      if (known(id)) {
        const int row = id * a.Hkv + h;
        y = row * 16;
        sk = a.k_scale[row];
        sv = a.v_scale[row];
      } else {
        report_error(a.status, kErrBounds, id);
      }
    }
  };
  int asked = 0;                                         // pages of this warp asked for so far
  uint32_t in_slot = 0, out_slot = 0, out_phase = 0;     // ring positions
  auto issue = [&](int y) {
    if (lane == 0) {
      uint8_t* dst = ring + in_slot * C::STAGE;
      mbar_arrive_expect_tx(&full[in_slot], C::STAGE);
      tma_load_2d(dst, &tmK, &full[in_slot], 0, y);
      tma_load_2d(dst + C::PAGE, &tmV, &full[in_slot], 0, y);
    }
    in_slot = in_slot + 1 == NST ? 0 : in_slot + 1;
    ++asked;
  };
  auto next_slot = [&]() {
    if (++out_slot == NST) {
      out_slot = 0;
      out_phase ^= 1;
    }
  };
  // (pages, rows and head of the segment that unit v lies in; b moves on to its sequence)
  auto segment_of = [&](int v, int& bb, SeqInfo& sq, int& hs) {
    while (pre[bb + 1] <= v) ++bb;
    sq = seq_info<ROWS>(a, bb);
    hs = (v - pre[bb]) / sq.pages;
  };
  auto locate = [&]() {
    SeqInfo sq;
    int hs, rb;
    if (a.whole) {
      b = seg / (a.Hkv * rb_max);
      hs = seg % (a.Hkv * rb_max);
      h = hs / rb_max;
      rb = hs % rb_max;
      sq = seq_info<ROWS>(a, b);
      if (lane == 0 && hs == 0) check_seq(a, b);
      seg0 = u;
      seg1 = ue = u + (rb < sq.rb ? sq.pages : 0);
    } else {
      segment_of(u, b, sq, hs);
      h = hs / sq.rb;
      rb = hs % sq.rb;
      seg0 = pre[b] + hs * sq.pages;
      seg1 = seg0 + sq.pages;
      ue = seg1 < u1 ? seg1 : u1;
    }
    const PageRange r = page_range<ROWS>(a, sq, rb);
    page = r.lo + u - seg0;
    cnt = max(0, min(ue - u, r.hi - page));
    tab = a.tables + (int64_t)b * a.max_blocks + page;
    row0 = rb * ROWS;
    nrows = min(ROWS, sq.n * a.G - row0);
    q0 = sq.q0;
    pos0 = sq.ctx - sq.n;
    first_pos = pos0 + row0 / a.G;
    last_pos = pos0 + (row0 + max(nrows, 1) - 1) / a.G;
  };
  auto peek = [&]() {  // at the part behind this one
    n_cnt = 0;
    if (a.whole ? seg + workers < segments : ue < u1) {
      int nb = b, hs, rb, units;
      SeqInfo sq;
      if (a.whole) {
        nb = (seg + workers) / (a.Hkv * rb_max);
        hs = (seg + workers) % (a.Hkv * rb_max);
        sq = seq_info<ROWS>(a, nb);
        n_h = hs / rb_max;
        rb = hs % rb_max;
        units = rb < sq.rb ? sq.pages : 0;
      } else {
        segment_of(ue, nb, sq, hs);
        n_h = hs / sq.rb;
        rb = hs % sq.rb;
        units = min(sq.pages, u1 - ue);
      }
      const PageRange r = page_range<ROWS>(a, sq, rb);
      n_cnt = max(0, min(units, r.hi - r.lo));
      n_id = lane < n_cnt ? a.tables[(int64_t)nb * a.max_blocks + r.lo + lane] : 0;
    }
  };
  // Q: rows n = g of each tile in the order of the K fragments, scaled to below 2. The rows are asked for as soon as
  // the segment is known (fetch_q) and put in place when they are there (place_q).
  uint2 qraw[NT][STEPS];
  float rs[NT][2], s_init[NT][2];  // score factors and starts (-128 sum q) of columns 2 t4 and 2 t4 + 1
  int posc[NT][2];                 // their positions
  auto fetch_q = [&]() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) qraw[nt][s] = make_uint2(0, 0);
      if (nt * 8 + g < nrows) {
        const int r = row0 + nt * 8 + g, tok = r / a.G, head = h * a.G + r % a.G;
        const __nv_bfloat16* qp = a.q + ((int64_t)(q0 + tok) * a.Hq + head) * D + 4 * t4;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) qraw[nt][s] = *reinterpret_cast<const uint2*>(qp + 16 * s);
      }
    }
  };
  auto place_q = [&]() {
    __syncwarp();  // every lane has read the rows of the last segment
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      uint32_t am = 0;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const uint2 w = qraw[nt][s];
        am = max(am, max(max(w.x & 0x7fffu, (w.x >> 16) & 0x7fffu), max(w.y & 0x7fffu, (w.y >> 16) & 0x7fffu)));
      }
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
      const int e = min(max((int)(am >> 7) - 127, -100), 100);
      // (the scale's sign goes with Q, so that factors are positive and one minimum bounds them)
      const float down = copysignf(__int_as_float((127 - e) << 23), a.scale), up = __int_as_float((127 + e) << 23);
      float sum = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        // codes (0, 2) and (1, 3) of a word meet in one operand register
        const uint2 w = qraw[nt][s];
        const uint32_t x = pack_h2(bf16_lo(w.x) * down, bf16_lo(w.y) * down);
        const uint32_t y = pack_h2(bf16_hi(w.x) * down, bf16_hi(w.y) * down);
        const float2 fx = __half22float2(*reinterpret_cast<const __half2*>(&x));
        const float2 fy = __half22float2(*reinterpret_cast<const __half2*>(&y));
        sum += (fx.x + fx.y) + (fy.x + fy.y);
        *reinterpret_cast<uint2*>(qs + (nt * 8 + g) * C::QLD + 32 * s + 8 * t4) = make_uint2(x, y);
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      sum *= -128.f / 16777216.f;
      const float f = fminf(up * fabsf(a.scale) * (16777216.f * (a.softcap > 0.f ? 1.f : kLog2e)), FLT_MAX);
      const int pos = pos0 + (row0 + nt * 8 + g) / a.G;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        rs[nt][c] = __shfl_sync(0xffffffffu, f, 8 * t4 + 4 * c);
        s_init[nt][c] = __shfl_sync(0xffffffffu, sum, 8 * t4 + 4 * c);
        posc[nt][c] = __shfl_sync(0xffffffffu, pos, 8 * t4 + 4 * c);
      }
    }
    __syncwarp();
  };

  locate();
  load_ids(0);
  fetch_q();

  while (true) {
    // ids of the first 32 pages are here or on their way; some of the pages may have been asked for already
    resolve(0, y0, sk0, sv0);
#pragma unroll 1
    while (asked - at < min(cnt, NST)) issue(__shfl_sync(0xffffffffu, y0, asked - at));
    load_ids(32);
    place_q();
    peek();

    float o[NT][STEPS][4], m[NT][2], l[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      m[nt][0] = m[nt][1] = kNone;
      l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
      for (int s = 0; s < STEPS; ++s) o[nt][s][0] = o[nt][s][1] = o[nt][s][2] = o[nt][s][3] = 0.f;
    }
    const int sv_exp = __reduce_max_sync(0xffffffffu, __float_as_int(sv0) >> 23);
    const int unit_exp = min(max(sv_exp, 127 - kUnitExp), 127 + kUnitExp);
    const float unit = __int_as_float(unit_exp << 23), per_unit = __int_as_float((254 - unit_exp) << 23);
    int key0 = page * 16;
#pragma unroll 1
    for (int j = 0; j < cnt; j += PP, key0 += 16 * PP) {
      if ((j & 15) == 0) {
        if ((j & 31) != 0) {
          resolve(j + 16, y1, sk1, sv1);
          load_ids(j + 48);
        } else if (j > 0) {
          y0 = y1;
          sk0 = sk1;
          sv0 = sv1;
        }
      }
      // codes of the pages into registers, then their slots are free for the pages NST further on
      uint32_t kw[PP][STEPS][2], vw[PP][STEPS][2];
      float sk[PP], sv[PP];
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        sk[p] = __shfl_sync(0xffffffffu, sk0, j + p);
        sv[p] = __shfl_sync(0xffffffffu, sv0, j + p);
        if (p == 0 || j + p < cnt) {
          if (!mbar_wait(&full[out_slot], out_phase, a.status, kErrTimeoutFull)) {
            // copies in flight land before the CTA leaves (those behind the one given up on)
            for (int k = at + j + p + 1; k < asked; ++k) {
              next_slot();
              if (!mbar_wait(&full[out_slot], out_phase, a.status, kErrTimeoutDrain)) break;
            }
            return;
          }
          const uint32_t kb = smem_u32(ring) + out_slot * C::STAGE, vb = kb + C::PAGE;
          next_slot();
#pragma unroll
          for (int s = 0; s < STEPS; s += 2) {
            const uint32_t off = page_off<D>((lane & 7) + ((lane >> 3) & 1) * 8, s + (lane >> 4));
            ldmatrix_x4(kb + off, kw[p][s][0], kw[p][s][1], kw[p][s + 1][0], kw[p][s + 1][1]);
            ldmatrix_x4_trans(vb + off, vw[p][s][0], vw[p][s][1], vw[p][s + 1][0], vw[p][s + 1][1]);
          }
        } else {  // an odd last page: the other half is masked below, and its weights are 0 times whatever is here
#pragma unroll
          for (int s = 0; s < STEPS; ++s) kw[p][s][0] = kw[p][s][1] = vw[p][s][0] = vw[p][s][1] = 0;
        }
      }
      // S^T = K Q^T
      float sc[PP][NT][4];
#pragma unroll
      for (int p = 0; p < PP; ++p)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[p][nt][0] = sc[p][nt][2] = s_init[nt][0];
          sc[p][nt][1] = sc[p][nt][3] = s_init[nt][1];
        }
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        uint2 q2[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          q2[nt] = *reinterpret_cast<const uint2*>(qs + (nt * 8 + g) * C::QLD + 32 * s + 8 * t4);
#pragma unroll
        for (int p = 0; p < PP; ++p) {
          const uint32_t x = flip(kw[p][s][0]), y = flip(kw[p][s][1]);
          const uint32_t a0 = codes_even(x), a1 = codes_even(y), a2 = codes_odd(x), a3 = codes_odd(y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(sc[p][nt], a0, a1, a2, a3, q2[nt].x, q2[nt].y);
        }
      }
      __syncwarp();
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const int i = asked - at;  // page of this part, or of the next one
        if (i < min(j + PP, cnt) + NST) {  // (an odd last page frees one slot only)
          if (i < cnt) {
            issue(__shfl_sync(0xffffffffu, (i ^ j) < 32 ? y0 : y1, i));
          } else if (i - cnt < n_cnt) {
            const int v = __shfl_sync(0xffffffffu, n_id, i - cnt);
            issue(known(v) ? (v * a.Hkv + n_h) * 16 : 0);
          }
        }
      }

      // scores in units of log2, masks
#pragma unroll
      for (int p = 0; p < PP; ++p)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          // (finite for the largest K scales too: a product of zero stays zero)
          const float f0 = fminf(rs[nt][0] * sk[p], FLT_MAX), f1 = fminf(rs[nt][1] * sk[p], FLT_MAX);
          sc[p][nt][0] *= f0;
          sc[p][nt][1] *= f1;
          sc[p][nt][2] *= f0;
          sc[p][nt][3] *= f1;
        }
      if (a.softcap > 0.f) {
        const float icap = 1.f / a.softcap, cap = a.softcap * kLog2e;
#pragma unroll
        for (int p = 0; p < PP; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[p][nt][i] = cap * tanhf(sc[p][nt][i] * icap);
      }
      const bool edge = key0 + 16 * PP - 1 > first_pos || (a.window > 0 && key0 <= last_pos - a.window) || j + PP > cnt;
      if (edge) {
#pragma unroll
        for (int p = 0; p < PP; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int key = key0 + 16 * p + g + (i >> 1) * 8;
              const int pos = posc[nt][i & 1];
              if (key > pos || (a.window > 0 && key <= pos - a.window) || j + p >= cnt) sc[p][nt][i] = -INFINITY;
            }
      }
      // V scales in units and their log2. Scores of 2^24 and more are further apart than the limits: the distance to m
      // is taken first, and m rounded up, so that no weight passes f16.
      float cv[PP], lv[PP];
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        cv[p] = fminf(sv[p] * per_unit, kFarScale);
        lv[p] = fmaxf(lg2(cv[p]), kNearLog);
      }
      auto top = [&](int p, int nt, int c) { return fmaxf(sc[p][nt][c], sc[p][nt][2 + c]); };
      bool grow = false;
#pragma unroll
      for (int p = 0; p < PP; ++p)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) grow |= top(p, nt, c) - m[nt][c] > kLimit - lv[p];
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float mx = m[nt][c];
#pragma unroll
            for (int p = 0; p < PP; ++p) {
              const float t = top(p, nt, c);
              mx = fmaxf(mx, fmaxf(t + (lv[p] - kShift), __fadd_ru(t, lv[p] - kLimit)));
            }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float f = ex2(m[nt][c] - mx);
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
      uint32_t pf[PP][NT][2];
#pragma unroll
      for (int p = 0; p < PP; ++p) {
        const float c = cv[p];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float p0 = ex2(sc[p][nt][0] - m[nt][0]), p1 = ex2(sc[p][nt][1] - m[nt][1]);
          const float p2 = ex2(sc[p][nt][2] - m[nt][0]), p3 = ex2(sc[p][nt][3] - m[nt][1]);
          l[nt][0] += p0 + p2;
          l[nt][1] += p1 + p3;
          pf[p][nt][0] = transpose8x8(pack_h2(p0 * c, p1 * c));
          pf[p][nt][1] = transpose8x8(pack_h2(p2 * c, p3 * c));
        }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int p = 0; p < PP; ++p)
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          const uint32_t x = flip(vw[p][s][0]), y = flip(vw[p][s][1]);
          const uint32_t a0 = codes_even(x), a1 = codes_odd(x), a2 = codes_even(y), a3 = codes_odd(y);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(o[nt][s], a0, a1, a2, a3, pf[p][nt][0], pf[p][nt][1]);
        }
#pragma unroll
      for (int p = 0; p < PP; ++p)
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            mma_f16(o[nt][s], kMinus128, kMinus128, kMinus128, kMinus128, pf[p][nt][0], pf[p][nt][1]);
    }

    // ---- the rows of this part: out, or to the workspace ----
    const bool whole = seg0 >= u0 && seg1 <= u1;
    float* part = a.ws + ((int64_t)worker * 2 + (seg0 < u0 ? 0 : 1)) * ROWS * (D + 2);
    // O 2^24 / sum is a mean of codes; the unit, up to 2^122, comes behind it, so that nothing passes fp32 on the way
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[nt][c];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = nt * 8 + 2 * t4 + c;
        if (r < nrows) {
          if (whole) {
            const int rr = row0 + r, head = h * a.G + rr % a.G;
            float f = 16777216.f;
            if (a.sinks != nullptr) {
              const float sk2 = a.sinks[head] * kLog2e, top = fmaxf(m[nt][c], sk2), fm = ex2(m[nt][c] - top);
              sum = sum * fm + ex2(sk2 - top);
              f *= fm;
            }
            f = sum == 0.f ? 0.f : f / sum;  // no visible key: 0
            __nv_bfloat16* dst = a.out + ((int64_t)(q0 + rr / a.G) * a.Hq + head) * D + 2 * g;
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
              *reinterpret_cast<uint32_t*>(dst + 16 * s) =
                  pack_bf16x2(o[nt][s][c] * f * unit, o[nt][s][2 + c] * f * unit);
          } else {
            const float f = sum == 0.f ? 0.f : 16777216.f / sum;
            float* dst = part + r * D + 2 * g;
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
              *reinterpret_cast<float2*>(dst + 16 * s) =
                  make_float2(o[nt][s][c] * f * unit, o[nt][s][2 + c] * f * unit);
            if (g == 0) {
              part[ROWS * D + r] = m[nt][c];
              part[ROWS * D + ROWS + r] = sum;
            }
          }
        }
      }
    }
    u = ue;
    at += cnt;
    seg += workers;
    if (a.whole ? seg >= segments : u >= u1) break;
    locate();
    id = n_id;
    fetch_q();
  }
}

// Joins the parts of the segments that several warps share and writes zeros for
// rows without keys. A part is the mean of its values, its maximum and its sum of
// weights: means are averaged, so that no value passes the largest one. D / 4 lanes
// hold a row; with few rows several such groups share a row's parts (a context that
// is cut over many CTAs has few rows next to it), with many a CTA takes as many rows
// as it has groups.
constexpr int kMergeThreads = 256;
constexpr float kNothing = 1e-36f;  // sums of weights next to a sink that outweighs them by 2^100

template <int D, int NT>
__global__ void __launch_bounds__(kMergeThreads) merge_kernel(PagedInt8Args a, int grid) {
  constexpr int ROWS = 8 * NT, LANES = D / 4, GROUPS = kMergeThreads / LANES;
  __shared__ float4 s_acc[kMergeThreads];
  __shared__ float2 s_ml[GROUPS];  // maximum and sum of each group
  pdl_wait();
  pdl_trigger();
  const int b = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
  const int before = a.ws_pre[b], U = a.ws_pre[a.B];
  const SeqInfo sq = seq_info<ROWS>(a, b);
  const int rows = sq.n * a.G;
  const int grp = tid / LANES, lane = tid % LANES, d = lane * 4;
  const int ways = rows < GROUPS ? GROUPS / max(rows, 1) : 1;  // groups that share a row
  const int rr = ways > 1 ? grp / ways : blockIdx.z * GROUPS + grp, way = ways > 1 ? grp % ways : 0;
  const bool on = rr < rows && (ways == 1 || blockIdx.z == 0);
  if (ways > 1 && blockIdx.z > 0) return;
  uint2* out = on ? reinterpret_cast<uint2*>(a.out + ((int64_t)(sq.q0 + rr / a.G) * a.Hq + h * a.G + rr % a.G) * D + d)
                  : nullptr;
  if (sq.pages <= 0) {
    if (on) *out = make_uint2(0, 0);
    return;
  }
  const int rb = rr / ROWS, r = rr % ROWS;
  const int s0 = before + (h * sq.rb + rb) * sq.pages, s1 = s0 + sq.pages;
  const int chunk = warp_units(U, grid);
  const int i0 = s0 / chunk, i1 = (s1 - 1) / chunk;  // first and last warp of the segment
  const bool join = on && i0 != i1;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f, sink = 0.f, m_own = kNone;
  if (join) {
    // the first warp ends inside the segment, the others begin inside it
    auto part = [&](int i) { return a.ws + ((int64_t)i * 2 + (i == i0 ? 1 : 0)) * ROWS * (D + 2); };
    float top = a.sinks != nullptr ? a.sinks[h * a.G + rr % a.G] * kLog2e : kNone;
    sink = a.sinks != nullptr ? 1.f : 0.f;  // the sink's weight, and the sums, relative to 2^top
    constexpr int BATCH = 4;                // parts loaded at once: few rounds of latency
    for (int i = i0 + way; i <= i1; i += BATCH * ways) {
      float pm[BATCH], pl[BATCH];
      float4 v[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const bool there = i + k * ways <= i1;
        const float* p = part(there ? i + k * ways : i);
        pm[k] = there ? p[ROWS * D + r] : kNone;
        pl[k] = there ? p[ROWS * D + ROWS + r] : 0.f;
        v[k] = *reinterpret_cast<const float4*>(p + r * D + d);
      }
      float mx = top;
#pragma unroll
      for (int k = 0; k < BATCH; ++k) mx = fmaxf(mx, pm[k]);
      const float f = ex2(top - mx), old = sum * f;
      sink *= f;
      top = mx;
      sum = old;
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        pl[k] *= ex2(pm[k] - top);
        sum += pl[k];
      }
      const float inv = sum < kNothing ? 0.f : 1.f / sum, keep = old * inv;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const float w = pl[k] * inv;
        acc.x += w * v[k].x;
        acc.y += w * v[k].y;
        acc.z += w * v[k].z;
        acc.w += w * v[k].w;
      }
    }
    m_own = top;
  }
  if (ways > 1) {
    s_acc[tid] = acc;
    if (lane == 0) s_ml[grp] = make_float2(m_own, sum);
    __syncthreads();
    if (join && way == 0) {  // (rows * ways <= GROUPS: the groups of a row lie inside the arrays)
      float top = m_own;
      for (int w = 1; w < ways; ++w) top = fmaxf(top, s_ml[grp + w].x);
      const float f0 = ex2(m_own - top), own = sum * f0;
      sink *= f0;
      sum = own;
      for (int w = 1; w < ways; ++w) sum += ex2(s_ml[grp + w].x - top) * s_ml[grp + w].y;
      const float inv = sum < kNothing ? 0.f : 1.f / sum, keep = own * inv;
      acc = make_float4(acc.x * keep, acc.y * keep, acc.z * keep, acc.w * keep);
      for (int w = 1; w < ways; ++w) {
        const float4 v = s_acc[tid + w * LANES];
        const float2 ml = s_ml[grp + w];
        const float f = ex2(ml.x - top) * ml.y * inv;
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
      }
    }
  }
  if (join && way == 0) {
    const float f = sum < kNothing ? 0.f : sum / (sum + sink);  // (the sink has no value)
    *out = make_uint2(pack_bf16x2(acc.x * f, acc.y * f), pack_bf16x2(acc.z * f, acc.w * f));
  }
}

}  // namespace kv8

int64_t kv_int8_store_scan() { return kv8::kScan; }

int kv_int8_store_launch(const KvInt8StoreArgs& args, int D, cudaStream_t st) {
  using namespace kv8;
  if (args.T == 0 || args.Hkv == 0) return 0;
  KvInt8StoreArgs a = args;
  // one token per warp keeps every warp on its own block when blocks get one token each (a decode
  // step); longer batches are prefill, where 15 of 16 warps would find that they have nothing to do
  a.group = a.T <= 1024 ? 1 : 16;
  const int64_t tasks = (a.T + a.group - 1) / a.group * a.Hkv * 2;
  const unsigned grid = (unsigned)((tasks + kStoreWarps - 1) / kStoreWarps);
  auto run = [&](auto kernel) { launch_pdl(kernel, dim3(grid), dim3(kStoreWarps * 32), 0, st, a); };
  if (a.owner != nullptr) {
    launch_pdl(owner_kernel, dim3((unsigned)((a.T + 255) / 256)), dim3(256), 0, st, a);
    D == 128 ? run(store_kernel<128, true>) : run(store_kernel<64, true>);
  } else {
    D == 128 ? run(store_kernel<128, false>) : run(store_kernel<64, false>);
  }
  return a.owner != nullptr ? 2 : 1;
}

void kv_int8_dequant_launch(const KvInt8DequantArgs& a, cudaStream_t st) {
  if (a.B == 0 || a.out_blocks == 0) return;
  const int per_cta = kv8::kDequantThreads * kv8::kDequantSteps * 16;
  const int parts = (2 * a.Hkv * 16 * a.D + per_cta - 1) / per_cta;
  launch_pdl(kv8::dequant_kernel, dim3((unsigned)(a.B * a.out_blocks), (unsigned)parts), dim3(kv8::kDequantThreads), 0,
             st, a);
}

namespace kv8 {
static int ctas_per_sm(int nt) {
  const int by_tiles[4] = {Cfg<128, 1>::CTAS, Cfg<128, 2>::CTAS, Cfg<128, 3>::CTAS, Cfg<128, 4>::CTAS};
  return by_tiles[nt - 1];
}

// 8-row query tiles of a warp: as few as hold every row of a sequence, at most 4
static int tiles(int G, int max_q_len) { return std::min(4, (G * max_q_len + 7) / 8); }

// pages of a segment that the host can rule out beyond, and whether warps take whole segments
static int most_pages(int nt, int G, int window, int max_q_len, int max_blocks) {
  return window > 0 ? std::min(max_blocks, window_pages(window, std::min(max_q_len, (8 * nt - 1) / G + 2))) : max_blocks;
}

static int grid_ctas(int nt, int device, int B, int Hkv, int G, int max_q_len, int pages, bool whole) {
  const int64_t per_sm = ctas_per_sm(nt);
  const int64_t segments = (int64_t)B * Hkv * (((int64_t)G * max_q_len + 8 * nt - 1) / (8 * nt));
  const int64_t work = whole ? (segments + 3) / 4 : (segments * pages + 15) / 16;
  return (int)std::max<int64_t>(1, std::min<int64_t>(per_sm * num_sms(device), work));
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
  if (a.whole) return;
  const int groups = kMergeThreads / (D / 4);
  launch_pdl(merge_kernel<D, NT>, dim3(a.B, a.Hkv, (a.G * a.max_q_len + groups - 1) / groups), dim3(kMergeThreads), 0,
             st, a, grid);
}
}  // namespace kv8

int64_t paged_int8_ws_floats(int device, int B, int Hkv, int G, int D, int max_q_len, int max_blocks, int window) {
  using namespace kv8;
  const int nt = tiles(G, max_q_len), pages = most_pages(nt, G, window, max_q_len, max_blocks);
  if (pages <= kWholePages) return 0;
  return (int64_t)grid_ctas(nt, device, B, Hkv, G, max_q_len, pages, false) * 4 * 2 * 8 * nt * (D + 2) + B + 1;
}

int paged_int8_launch(const PagedInt8Args& args, cudaStream_t st) {
  using namespace kv8;
  PagedInt8Args a = args;
  if (a.B == 0 || a.T == 0 || a.max_q_len == 0) return 0;
  const int nt = tiles(a.G, a.max_q_len);
  const int pages = most_pages(nt, a.G, a.window, a.max_q_len, a.max_blocks);
  a.whole = pages <= kWholePages ? 1 : 0;
  const int grid = grid_ctas(nt, a.device, a.B, a.Hkv, a.G, a.max_q_len, pages, a.whole != 0);
  if ((int64_t)a.B * a.Hkv * (((int64_t)a.G * a.max_q_len + 8 * nt - 1) / (8 * nt)) * std::max(pages, 1) > INT32_MAX / 2)
    throw std::runtime_error("b200.paged_attention_int8: more pages in the batch than 2^30");
  if (!a.whole) a.ws_pre = reinterpret_cast<int32_t*>(a.ws + (int64_t)grid * 4 * 2 * 8 * nt * (a.D + 2));
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
  return a.whole ? 1 : 2;
}

}  // namespace b200
