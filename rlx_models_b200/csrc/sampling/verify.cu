// Verification of drafted tokens (speculative sampling, Leviathan et al. 2023,
// Chen et al. 2023). With p_i = softmax(logits_i / T) the target's distribution
// at draft position i, q_i the drafter's and u_i given uniform numbers:
//
//   accept d_i while u_i q_i(d_i) < p_i(d_i);
//   at the first rejection draw from w = max(p_i - q_i, 0), if all are accepted
//   from w = p of the row behind the last draft: the token is the first whose
//   running sum of w exceeds u_last * sum(w);
//   T <= 0: accept while d_i is the (lowest) argmax, then take the argmax.
//
// Decisions are whole numbers, so what decides them is held in 64 bits: with
// 1.5e5 tokens the borders of the running sum lie 1e-5 apart and closer, and sums
// of 32-bit exponentials would move one draw in a thousand across a border.
// exp_nonpos below costs about a dozen double-precision operations a logit, which
// run under the loads of the logits (at 64 x 3.5 rows of 151936: 34 M logits,
// 136 MB or 21 us of HBM, 23 us of double-precision arithmetic).
//
// Two launches. stats_kernel: one CTA per (row, 8192 logits) leaves the chunk's
// maximum, sum of exponentials and argmax; rows are independent, so a single
// request's rows fill the GPU too. decide_kernel: a cluster of 8 CTAs per
// sequence joins the chunks, accepts, and draws: every CTA sums its slice of w in
// tiles of 512 tokens, the slice sums meet through distributed shared memory, and
// the CTA whose slice holds the border walks its tiles.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>

#include "../common/b200.cuh"
#include "../common/launch.h"
#include "../common/pdl_launch.h"

namespace b200 {
namespace verify {

namespace cg = cooperative_groups;

constexpr int kStatThreads = 256;
constexpr int kPerThread = 32;
constexpr int kChunk = kStatThreads * kPerThread;  // 8192
constexpr int kCluster = 8;
constexpr int kThreads = 256;
constexpr int kTile = 512;  // tokens per warp step: 16 per lane

// 2^(j / 64), filled once per CTA.
__device__ __forceinline__ void fill_table(double* tab) {
  for (int j = threadIdx.x; j < 64; j += blockDim.x) tab[j] = exp2((double)j * (1.0 / 64.0));
}

// e^x for x <= 0 given y = x * 64 / ln 2: y = 64 n + j + r with |r| <= 1/2, so
// e^x = 2^n 2^(j / 64) e^z, z = r ln 2 / 64, |z| < 0.00542: Taylor to z^5 leaves
// z^6 / 720 < 4e-17. Results below the normal range are 0.
__device__ __forceinline__ double exp_nonpos(double y, const double* tab) {
  const double magic = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are rint(y)
  if (!(y > -64.0 * 1000.0)) return 0.0;
  const double k = y + magic;
  const int i = __double2loint(k);
  const double z = (y - (k - magic)) * (0.693147180559945309417 / 64.0);
  double e = fma(z, 1.0 / 120.0, 1.0 / 24.0);
  e = fma(e, z, 1.0 / 6.0);
  e = fma(e, z, 0.5);
  e = fma(e, z, 1.0);
  e = fma(e, z, 1.0);
  const double r = tab[i & 63] * e;
  return __hiloint2double(__double2hiint(r) + ((i >> 6) << 20), __double2loint(r));
}

// NaN logits are never chosen, +inf counts as the largest finite number.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

__device__ __forceinline__ double warp_sum(double v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// last b with cu_rows[b] <= row
__device__ __forceinline__ int seq_of(const int32_t* cu, int B, int row) {
  int lo = 0, hi = B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kStatThreads) stats_kernel(VerifyArgs a) {
  __shared__ double tab[64];
  __shared__ float s_max[kStatThreads / 32];
  __shared__ int s_arg[kStatThreads / 32];
  __shared__ double s_sum[kStatThreads / 32];
  fill_table(tab);
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const float T = a.temperature[seq_of(a.cu_rows, a.B, row)];
  const float* x = a.logits + (int64_t)row * a.ld;
  const int lo = chunk * kChunk, hi = min(lo + kChunk, a.V);
  float v[kPerThread];
  if ((reinterpret_cast<uintptr_t>(x) & 15) == 0 && hi - lo == kChunk) {
#pragma unroll
    for (int i = 0; i < kPerThread / 4; ++i) {
      const float4 w = *reinterpret_cast<const float4*>(x + lo + (i * kStatThreads + tid) * 4);
      v[4 * i] = w.x;
      v[4 * i + 1] = w.y;
      v[4 * i + 2] = w.z;
      v[4 * i + 3] = w.w;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int at = lo + ((i >> 2) * kStatThreads + tid) * 4 + (i & 3);
      v[i] = at < hi ? x[at] : -INFINITY;
    }
  }
  float best = -INFINITY;
  int arg = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    v[i] = clean(v[i]);
    if (v[i] > best) {
      best = v[i];
      arg = lo + ((i >> 2) * kStatThreads + tid) * 4 + (i & 3);
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
    const int oa = __shfl_xor_sync(0xffffffffu, arg, o);
    if (ob > best || (ob == best && oa < arg)) {
      best = ob;
      arg = oa;
    }
  }
  if ((tid & 31) == 0) {
    s_max[tid >> 5] = best;
    s_arg[tid >> 5] = arg;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kStatThreads / 32; ++w) {
    const float ob = s_max[w];
    const int oa = s_arg[w];
    if (ob > best || (ob == best && oa < arg)) {
      best = ob;
      arg = oa;
    }
  }
  double sum = 0.0;
  if (T > 0.f && best != -INFINITY) {
    const double f = 64.0 * 1.44269504088896340736 / (double)T;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) sum += exp_nonpos(((double)v[i] - (double)best) * f, tab);
  }
  sum = warp_sum(sum);
  if ((tid & 31) == 0) s_sum[tid >> 5] = sum;
  __syncthreads();
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < kStatThreads / 32; ++w) t += s_sum[w];
    const int64_t at = (int64_t)row * a.chunks + chunk;
    a.part_max[at] = best;
    a.part_sum[at] = t;
    a.part_arg[at] = arg;
  }
}

struct RowStat {
  float max;
  double sum;
  int arg;
};

// One warp: the chunks of a row joined (every lane gets the result).
__device__ __forceinline__ RowStat row_stat(const VerifyArgs& a, int64_t row, double f, const double* tab) {
  const int lane = threadIdx.x & 31;
  float best = -INFINITY;
  int arg = 0x7fffffff;
  for (int c = lane; c < a.chunks; c += 32) {
    const float m = a.part_max[row * a.chunks + c];
    if (m > best) {
      best = m;
      arg = a.part_arg[row * a.chunks + c];
    }
  }
  for (int o = 16; o > 0; o >>= 1) {
    const float ob = __shfl_xor_sync(0xffffffffu, best, o);
    const int oa = __shfl_xor_sync(0xffffffffu, arg, o);
    if (ob > best || (ob == best && oa < arg)) {
      best = ob;
      arg = oa;
    }
  }
  double sum = 0.0;
  if (best != -INFINITY)
    for (int c = lane; c < a.chunks; c += 32)
      sum += a.part_sum[row * a.chunks + c] *
             exp_nonpos(((double)a.part_max[row * a.chunks + c] - (double)best) * f, tab);
  return {best, warp_sum(sum), arg};
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads) decide_kernel(VerifyArgs a) {
  extern __shared__ double tiles[];  // sums of this CTA's tiles
  __shared__ double tab[64];
  __shared__ double s_slice;         // sum of w over this CTA's slice
  __shared__ RowStat s_row;
  __shared__ double s_p;
  __shared__ int s_count, s_tok, s_last;
  cg::cluster_group cluster = cg::this_cluster();
  fill_table(tab);
  pdl_wait();
  pdl_trigger();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / kCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = min(max((int64_t)a.cu_rows[b], (int64_t)0), a.R);
  const int64_t r1 = min(max((int64_t)a.cu_rows[b + 1], r0), a.R);
  const int n = (int)min(r1 - r0 - 1, (int64_t)a.max_drafts);  // drafts; < 0: the sequence has no rows
  int32_t* out = a.tokens + (int64_t)b * (a.max_drafts + 1);
  const float T = a.temperature[b];
  const double f = T > 0.f ? 64.0 * 1.44269504088896340736 / (double)T : 0.0;
  const int64_t d0 = r0 - b;
  __syncthreads();

  // acceptance: one warp per drafted row, then the first refusal counts
  if (tid == 0) s_count = max(n, 0);
  __syncthreads();
  for (int i = warp; i < n; i += kThreads / 32) {
    const int64_t di = d0 + i;
    const int tok = di >= 0 && di < a.ND ? a.drafts[di] : -1;
    const RowStat st = row_stat(a, r0 + i, f, tab);
    bool ok = false;
    if (tok >= 0 && tok < a.V) {
      if (!(T > 0.f)) {
        ok = tok == st.arg;
      } else if (st.max != -INFINITY) {
        const float x = clean(a.logits[(r0 + i) * a.ld + tok]);
        const double p = exp_nonpos(((double)x - (double)st.max) * f, tab) / st.sum;
        const float q = a.probs != nullptr ? a.probs[di * a.ldp + tok] : 1.f;
        ok = (double)a.uniforms[r0 + i] * (double)(q > 0.f ? q : 0.f) < p;
      }
    }
    if (lane == 0 && !ok) atomicMin(&s_count, i);
  }
  __syncthreads();
  const int count = s_count;
  const int64_t row = r0 + count;
  if (warp == 0 && n >= 0) {
    const RowStat st = row_stat(a, row, f, tab);
    if (lane == 0) s_row = st;
  }
  __syncthreads();
  if (rank == 0) {
    if (tid == 0) a.accepted[b] = count;
    for (int i = tid; i <= a.max_drafts; i += kThreads) {
      if (i < count) out[i] = a.drafts[d0 + i];  // accepted: its index was in range
      else if (i > count || n < 0) out[i] = -1;
    }
  }
  if (n < 0) return;  // the whole cluster alike
  const RowStat st = s_row;
  if (!(T > 0.f) || st.max == -INFINITY) {  // argmax (0 for a row without a finite logit, as ops.argmax)
    if (rank == 0 && tid == 0) out[count] = st.max == -INFINITY ? 0 : st.arg;
    return;
  }

  // w over this CTA's slice, tile by tile
  const float* x = a.logits + row * a.ld;
  const int64_t di = d0 + count;
  const bool rejected = count < n && di >= 0 && di < a.ND;  // (a draft outside its list: drawn from p)
  const float* q = rejected && a.probs != nullptr ? a.probs + di * a.ldp : nullptr;
  const int gone = rejected && a.probs == nullptr ? a.drafts[di] : -1;  // a certain draft: q = 1 there
  const double inv = 1.0 / st.sum, mx = (double)st.max;
  auto weight = [&](int i, bool plain) -> double {
    double w = exp_nonpos(((double)clean(x[i]) - mx) * f, tab) * inv;
    if (!plain) {
      if (q != nullptr) {
        const float qi = q[i];
        w = fmax(w - (double)(qi > 0.f ? qi : 0.f), 0.0);
      }
      if (i == gone) w = 0.0;
    }
    return w;
  };
  const int all_tiles = (a.V + kTile - 1) / kTile;
  const int per = (all_tiles + kCluster - 1) / kCluster;
  const int tile0 = min(rank * per, all_tiles), tile1 = min(tile0 + per, all_tiles);
  bool plain = !rejected;
  double total = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int t = tile0 + warp; t < tile1; t += kThreads / 32) {
      double sum = 0.0;
#pragma unroll 4
      for (int i = 0; i < kTile / 32; ++i) {
        const int at = t * kTile + i * 32 + lane;
        if (at < a.V) sum += weight(at, plain);
      }
      sum = warp_sum(sum);
      if (lane == 0) tiles[t - tile0] = sum;
    }
    __syncthreads();
    if (tid == 0) {
      double s = 0.0;
      for (int t = 0; t < tile1 - tile0; ++t) s += tiles[t];
      s_slice = s;
    }
    cluster.sync();
    total = 0.0;
    for (int c = 0; c < kCluster; ++c) total += *cluster.map_shared_rank(&s_slice, c);
    if (total > 0.0 || plain) break;
    plain = true;  // p == q up to rounding, yet refused: draw from p
    cluster.sync();
  }
  const double target = (double)a.uniforms[r1 - 1] * total;
  // the slice that the border lies in; behind every border (rounding): the last slice with weight
  double before = 0.0;
  int owner = -1, fallback = 0;
  double owner_before = 0.0;
  for (int c = 0; c < kCluster; ++c) {
    const double s = *cluster.map_shared_rank(&s_slice, c);
    if (s > 0.0) fallback = c;
    if (owner < 0 && before + s > target) {
      owner = c;
      owner_before = before;
    }
    before += s;
  }
  const bool end = owner < 0;  // take the last token with weight of the fallback slice
  if (end) owner = fallback;
  if (rank == owner) {
    if (tid == 0) {
      double s = owner_before;
      int pick = -1, last = 0;
      for (int t = 0; t < tile1 - tile0; ++t) {
        if (tiles[t] > 0.0) last = t;
        if (!end && s + tiles[t] > target) {
          pick = t;
          break;
        }
        s += tiles[t];
      }
      s_tok = pick >= 0 ? pick : last;
      s_p = s;
      s_last = pick < 0 ? 1 : 0;
    }
    __syncthreads();
    if (warp == 0) {
      const int t = tile0 + s_tok;
      double s = s_p;
      int chosen = -1, last = 0;
      for (int i = 0; i < kTile / 32; ++i) {
        const int at = t * kTile + i * 32 + lane;
        const double w = at < a.V ? weight(at, plain) : 0.0;
        double inc = w;
        for (int o = 1; o < 32; o <<= 1) {
          const double v = __shfl_up_sync(0xffffffffu, inc, o);
          if (lane >= o) inc += v;
        }
        const unsigned some = __ballot_sync(0xffffffffu, w > 0.0);
        if (some != 0) last = t * kTile + i * 32 + 31 - __clz(some);
        const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && s + inc > target);
        if (hit != 0 && s_last == 0) {
          chosen = t * kTile + i * 32 + __ffs(hit) - 1;
          break;
        }
        s += __shfl_sync(0xffffffffu, inc, 31);
      }
      if (lane == 0) out[count] = chosen >= 0 ? chosen : last;
    }
  }
  cluster.sync();  // no CTA leaves while another reads its shared memory
}

}  // namespace verify

int verify_chunks(int V) { return (V + verify::kChunk - 1) / verify::kChunk; }

void verify_drafts_launch(const VerifyArgs& a, cudaStream_t st) {
  using namespace verify;
  if (a.B == 0) return;
  if (a.R > 0) launch_pdl(stats_kernel, dim3((unsigned)a.chunks, (unsigned)a.R), dim3(kStatThreads), 0, st, a);
  const int all_tiles = (a.V + kTile - 1) / kTile;
  const size_t smem = (size_t)((all_tiles + kCluster - 1) / kCluster) * sizeof(double);
  launch_pdl(decide_kernel, dim3((unsigned)a.B * kCluster), dim3(kThreads), smem, st, a);
}

}  // namespace b200
