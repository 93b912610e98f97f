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
// 1.5e5 tokens the borders of the drawn row's running sum lie 1e-5 apart and closer,
// and sums of 32-bit exponentials would move one draw in a thousand across a border;
// an acceptance needs them where u q lies next to p. Which rows are drawn or close is
// known after the statistics only, so all rows have them in 64 bits.
// An exponential (Exp64) takes 8 double-precision operations, so 34 M logits (64
// requests of 3.5 rows of 151936) are 15 us of the double-precision pipes under
// the 21 us that their 136 MB take from HBM.
//
// Two launches. stats_kernel: one CTA per (row, 8192 logits) leaves the chunk's
// maximum, sum of exponentials and argmax; rows are independent, so a single
// request's rows fill the GPU too. decide_kernel: a cluster of 8 CTAs per
// sequence joins the chunks, accepts, and draws: every CTA sums its slice of w in
// tiles of 512 tokens, the slice sums meet through distributed shared memory, and
// the CTA whose slice holds the border walks its tiles.
//
// On a B200 a request with 4 drafts takes 15.8 us (the latency of the two launches
// and a cluster's three meetings; 1024 threads a CTA instead of 512: 16.5), 64
// requests with up to 4 drafts 69 us: about 45 for the statistics, bound by
// instruction issue (27 a logit, 8 of them in 64 bits; chunks of 4096 logits with
// more CTAs an SM are slower), the rest for the draw from 64 rows of p and q.
#include <cooperative_groups.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cstdint>
#include <type_traits>

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
constexpr int kLaneTile = 16;
constexpr int kTile = 32 * kLaneTile;  // tokens per warp step
constexpr int kRows = 32;              // rows whose statistics a CTA keeps
constexpr float kMaxTemperature = 1e30f;

constexpr int kTable = 512;

// 2^(j / 512) by the Taylor series of e^(j ln 2 / 512), at compile time.
struct Exp2Table {
  double v[kTable];
  constexpr Exp2Table() : v{} {
    for (int j = 0; j < kTable; ++j) {
      const double x = j * (0.693147180559945309417 / kTable);
      double sum = 1.0;
      for (int k = 24; k > 0; --k) sum = 1.0 + sum * x / k;
      v[j] = sum;
    }
  }
};
__device__ constexpr Exp2Table kExp2Table{};

__device__ __forceinline__ void fill_table(double* tab) {
  for (int j = threadIdx.x; j < kTable; j += blockDim.x) tab[j] = kExp2Table.v[j];
}

// e^((x - max) / T) for x <= max in 64 bits: y = (x - max) 512 / (T ln 2) = 512 n + j + r with |r| <= 1/2, so the value
// is 2^n 2^(j / 512) e^z, z = r ln 2 / 512, |z| < 0.00068; Taylor to z^3 leaves z^4 / 24 < 9e-15 of it. Terms below
// e^-700 are 0 (`keep`), and so are those of -inf and NaN.
//
// y is one fma of x, f and c = -f max rounded, so all values of one maximum are off by the same factor, which `fix`
// takes out: the error of c, d = f max + c, is exact as an fma, and fix = e^(-d ln 2 / 512). A temperature below
// |max| 2^-34 acts like that one: other fp32 values lie 2^-24 |max| and more below max, 2^10 temperatures, where terms
// are 0 already. It bounds d by 2^-10, the terms of fix past the square by 4e-19.
struct Exp64 {
  double f, c;  // y = f x + c
  double fix;   // a kept term is fix times what `parts` gives
  float max, cut;
  const double* tab;
  __device__ __forceinline__ Exp64(float mx, float T, const double* table) : max(mx), tab(table) {
    const float t = fmaxf(T, fabsf(mx) * 0x1p-34f);
    f = kTable * 1.44269504088896340736 / (double)t;
    c = -f * (double)mx;
    const double z = fma(f, (double)mx, c) * (0.693147180559945309417 / kTable);
    fix = 1.0 - z + 0.5 * z * z;
    cut = -700.f * t;
  }
  __device__ __forceinline__ bool keep(float x) const { return x - max > cut; }
  // scale * e^z without the range check
  __device__ __forceinline__ void parts(float x, double& scale, double& e) const {
    constexpr double ln = 0.693147180559945309417 / kTable, magic = 6755399441055744.0;  // 1.5 * 2^52
    const double y = fma((double)x, f, c);
    const double k = y + magic;  // the sum's low bits are rint(y)
    const int i = __double2loint(k);
    const double r = y - (k - magic);
    e = fma(r, ln * ln * ln / 6.0, ln * ln / 2.0);
    e = fma(e, r, ln);
    e = fma(e, r, 1.0);
    const double t = tab[i & (kTable - 1)];
    scale = __hiloint2double(__double2hiint(t) + ((i >> 9) << 20), __double2loint(t));
  }
  __device__ __forceinline__ void add(float x, double& sum) const {  // of a term that is kept
    double scale, e;
    parts(x, scale, e);
    sum = fma(scale, e, sum);
  }
  __device__ __forceinline__ double operator()(float x) const {
    double scale, e;
    parts(x, scale, e);
    return keep(x) ? scale * e * fix : 0.0;
  }
};

__device__ __forceinline__ bool sampled(float T) { return T > 0.f; }
__device__ __forceinline__ float bounded(float T) { return T > kMaxTemperature ? kMaxTemperature : T; }  // (keeps NaN)

// NaN logits are never chosen, +inf counts as the largest finite number.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

__device__ __forceinline__ double warp_sum(double v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

__global__ void __launch_bounds__(kStatThreads, 4) stats_kernel(VerifyArgs a) {
  __shared__ double tab[kTable];
  __shared__ float s_max[kStatThreads / 32];
  __shared__ int s_arg[kStatThreads / 32];
  __shared__ double s_sum[kStatThreads / 32];
  __shared__ float s_t;
  fill_table(tab);
  pdl_wait();
  pdl_trigger();
  const int row = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x;
  const float* x = a.logits + (int64_t)row * a.ld;
  const int lo = chunk * kChunk, hi = min(lo + kChunk, a.V);
  if (tid == 0) s_t = 0.f;  // (a row of no sequence)
  __syncthreads();
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
  for (int b = tid; b < a.B; b += kStatThreads)  // the row's sequence: one round of loads, beside those of the logits
    if (a.cu_rows[b] <= row && row < a.cu_rows[b + 1]) s_t = a.temperature[b];
  float best = -INFINITY;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) best = fmaxf(best, v[i]);  // (NaN loses)
  if (best == INFINITY) {  // +inf counts as the largest finite number
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) v[i] = clean(v[i]);
    best = FLT_MAX;
  }
  __syncthreads();
  const float T = bounded(s_t);
  int arg = 0x7fffffff;
  if (!sampled(T)) {
#pragma unroll
    for (int i = kPerThread - 1; i >= 0; --i)
      if (v[i] == best && best != -INFINITY) arg = lo + ((i >> 2) * kStatThreads + tid) * 4 + (i & 3);
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
  if (sampled(T) && best != -INFINITY) {
    const Exp64 ex(best, T, tab);
    double part[2] = {0.0, 0.0};
    const float low = __fadd_ru(best, ex.cut);  // (not below the cut: the exponent of 2^n stays in range)
    if (low < best) {  // terms below it enter as e^-350 or less, which no sum of 1 and more sees (NaN loses)
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) ex.add(fmaxf(v[i], low), part[i & 1]);
      sum = (part[0] + part[1]) * ex.fix;
    } else {  // so cold that only the maximum counts
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) sum += v[i] == best ? 1.0 : 0.0;
    }
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
__device__ __forceinline__ RowStat row_stat(const VerifyArgs& a, int64_t row, float T, const double* tab) {
  const int lane = threadIdx.x & 31;
  const float* pm = a.part_max + row * a.chunks;
  float best = -INFINITY;
  int arg = 0x7fffffff;
  for (int c = lane; c < a.chunks; c += 32) {
    const float m = pm[c];
    const int i = a.part_arg[row * a.chunks + c];
    if (m > best) {
      best = m;
      arg = i;
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
  if (sampled(T) && best != -INFINITY) {
    const Exp64 ex(best, T, tab);
    for (int c = lane; c < a.chunks; c += 32) sum += a.part_sum[row * a.chunks + c] * ex(pm[c]);
  }
  return {best, warp_sum(sum), arg};
}

template <int kThreads, int kBlocks>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads, kBlocks) decide_kernel(VerifyArgs a) {
  constexpr int kWarps = kThreads / 32;
  extern __shared__ double tiles[];  // sums of this CTA's tiles
  __shared__ double tab[kTable];
  __shared__ double s_slice;         // sum of w over this CTA's slice
  __shared__ RowStat s_row[kRows];
  __shared__ double s_before;
  __shared__ int s_count, s_tile, s_end;
  cg::cluster_group cluster = cg::this_cluster();
  if (threadIdx.x == 0) s_count = 0x7fffffff;
  fill_table(tab);
  pdl_wait();
  pdl_trigger();
  const int rank = (int)cluster.block_rank(), b = blockIdx.x / kCluster;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = min(max((int64_t)a.cu_rows[b], (int64_t)0), a.R);
  const int64_t r1 = min(max((int64_t)a.cu_rows[b + 1], r0), a.R);
  const int n = (int)min(r1 - r0 - 1, (int64_t)a.max_drafts);  // drafts; < 0: the sequence has no rows
  int32_t* out = a.tokens + (int64_t)b * (a.max_drafts + 1);
  const float T = bounded(a.temperature[b]);
  const int64_t d0 = r0 - b;
  __syncthreads();

  // acceptance: one warp per row; the first refusal counts
  for (int i = warp; i <= n; i += kWarps) {
    const int64_t di = d0 + i;
    const int tok = i < n && di >= 0 && di < a.ND ? a.drafts[di] : -1;
    const bool token = tok >= 0 && tok < a.V;
    const float x = token ? clean(a.logits[(r0 + i) * a.ld + tok]) : 0.f;
    const float q = token && a.probs != nullptr ? a.probs[di * a.ldp + tok] : 1.f;
    const RowStat st = row_stat(a, r0 + i, T, tab);
    if (lane == 0 && i < kRows) s_row[i] = st;
    bool ok = false;
    if (token) {
      if (!sampled(T)) {
        ok = tok == st.arg;
      } else if (st.max != -INFINITY) {
        const double p = Exp64(st.max, T, tab)(x) / st.sum;
        ok = (double)a.uniforms[r0 + i] * (double)(q > 0.f ? q : 0.f) < p;
      }
    }
    if (lane == 0 && i < n && !ok) atomicMin(&s_count, i);
  }
  __syncthreads();
  const int count = min(s_count, max(n, 0));
  const int64_t row = r0 + count;
  if (n >= 0 && count >= kRows) {
    if (warp == 0) {
      const RowStat st = row_stat(a, row, T, tab);
      if (lane == 0) s_row[0] = st;
    }
    __syncthreads();
  }
  if (rank == 0) {
    if (tid == 0) a.accepted[b] = count;
    for (int i = tid; i <= a.max_drafts; i += kThreads) {
      if (i < count) out[i] = a.drafts[d0 + i];  // accepted: its index was in range
      else if (i > count || n < 0) out[i] = -1;
    }
  }
  if (n < 0) return;  // the whole cluster alike
  const RowStat st = s_row[count < kRows ? count : 0];
  if (!sampled(T) || st.max == -INFINITY) {  // argmax (0 for a row without a finite logit, as ops.argmax)
    if (rank == 0 && tid == 0) out[count] = st.max == -INFINITY ? 0 : st.arg;
    return;
  }

  // w over this CTA's slice, tile by tile; the loads of a tile are on their way together
  const float* x = a.logits + row * a.ld;
  const int64_t di = d0 + count;
  const bool rejected = count < n && di >= 0 && di < a.ND;  // (a draft outside its list: drawn from p)
  const float* q = rejected && a.probs != nullptr ? a.probs + di * a.ldp : nullptr;
  const int gone = rejected && a.probs == nullptr ? a.drafts[di] : INT32_MIN;  // a certain draft: q = 1 there
  const Exp64 ex(st.max, T, tab);
  const double inv = ex.fix / st.sum;
  bool plain = !rejected;
  // use(i, w) of the 16 tokens at0 + i * step of a lane. A tile inside the row needs no bounds, and a row whose largest
  // logit is an ordinary number no care for +inf (NaN and -inf fail `keep`).
  auto tile_of = [&](int at0, auto step, auto careful, auto&& use) {
    constexpr bool kCareful = decltype(careful)::value;
    constexpr int kStep = decltype(step)::value;
    const bool sub = !plain && q != nullptr;
    float xv[kLaneTile], qv[kLaneTile];
#pragma unroll
    for (int i = 0; i < kLaneTile; ++i) xv[i] = !kCareful || at0 + i * kStep < a.V ? x[at0 + i * kStep] : -INFINITY;
    if (sub) {
#pragma unroll
      for (int i = 0; i < kLaneTile; ++i) qv[i] = !kCareful || at0 + i * kStep < a.V ? q[at0 + i * kStep] : 0.f;
    } else {
#pragma unroll
      for (int i = 0; i < kLaneTile; ++i) qv[i] = 0.f;
    }
    const int skip = plain || gone < 0 ? -1 : gone - at0;
#pragma unroll
    for (int i = 0; i < kLaneTile; ++i) {
      const float xi = kCareful ? clean(xv[i]) : xv[i];
      double scale, e;
      ex.parts(xi, scale, e);
      const double v = fma(scale * e, inv, -(double)fmaxf(qv[i], 0.f));  // (NaN counts as 0)
      use(i, ex.keep(xi) && v > 0.0 && skip != i * kStep ? v : 0.0);
    }
  };
  using Spread = std::integral_constant<int, 32>;  // tokens of a lane 32 apart: coalesced loads
  using InRow = std::integral_constant<int, 1>;    // one behind the other: a lane's running sum is in order
  auto tile_weights = [&](int t, auto step, auto&& use) {
    const int at0 = t * kTile + (decltype(step)::value == 32 ? lane : lane * kLaneTile);
    if ((t + 1) * kTile <= a.V && st.max < FLT_MAX) tile_of(at0, step, std::false_type{}, use);
    else tile_of(at0, step, std::true_type{}, use);
  };
  const int all_tiles = (a.V + kTile - 1) / kTile;
  const int per = (all_tiles + kCluster - 1) / kCluster;
  const int tile0 = min(rank * per, all_tiles), mine = min(tile0 + per, all_tiles) - tile0;
  const int seg = (mine + 31) / 32;  // tiles per lane, in order, where one warp adds them up
  double total = 0.0, slice = 0.0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int t = warp; t < mine; t += kWarps) {
      double part[2] = {0.0, 0.0};
      tile_weights(tile0 + t, Spread{}, [&](int i, double w) { part[i & 1] += w; });
      const double sum = warp_sum(part[0] + part[1]);
      if (lane == 0) tiles[t] = sum;
    }
    __syncthreads();
    if (warp == 0) {
      double s = 0.0;
      for (int t = lane * seg; t < min(lane * seg + seg, mine); ++t) s += tiles[t];
      s = warp_sum(s);
      if (lane == 0) s_slice = s;
    }
    cluster.sync();
    slice = lane < kCluster ? *cluster.map_shared_rank(&s_slice, lane) : 0.0;  // lane c: the sum of slice c
    total = 0.0;
    for (int c = 0; c < kCluster; ++c) total += __shfl_sync(0xffffffffu, slice, c);
    if (total > 0.0 || plain) break;
    plain = true;  // p == q up to rounding, yet refused: draw from p
    cluster.sync();
  }
  const double target = (double)a.uniforms[r1 - 1] * total;
  // the slice that the border lies in; behind every border (rounding): the last slice with weight
  double before = 0.0, owner_before = 0.0;
  int owner = -1, fallback = 0;
  for (int c = 0; c < kCluster; ++c) {
    const double s = __shfl_sync(0xffffffffu, slice, c);
    if (s > 0.0) fallback = c;
    if (owner < 0 && before + s > target) {
      owner = c;
      owner_before = before;
    }
    before += s;
  }
  const bool end = owner < 0;  // take the last token with weight of the fallback slice
  if (rank == (end ? fallback : owner) && warp == 0) {
    // the tile: a running sum over the lanes' tiles, then over the tiles of the lane that holds the border
    double s = 0.0;
    int last = -1;
    for (int t = lane * seg; t < min(lane * seg + seg, mine); ++t) {
      s += tiles[t];
      if (tiles[t] > 0.0) last = t;
    }
    double inc = s;
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned hit = end ? 0u : __ballot_sync(0xffffffffu, last >= 0 && owner_before + inc > target);
    for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    if (lane == (hit != 0 ? __ffs(hit) - 1 : 0)) {
      s_tile = last;
      s_end = 1;
      s_before = 0.0;
      if (hit != 0) {
        double run = owner_before + inc - s;
        int pick = -1;
        for (int t = lane * seg; t < min(lane * seg + seg, mine); ++t) {
          if (tiles[t] > 0.0) pick = t;  // (rounding: the last one with weight holds it)
          if (run + tiles[t] > target) break;
          if (t + 1 < min(lane * seg + seg, mine)) run += tiles[t];
        }
        s_tile = pick;
        s_end = 0;
        s_before = run;
      }
    }
    __syncwarp();
    const int t = tile0 + max(s_tile, 0);
    double w[kLaneTile], own = 0.0;
    int last_i = -1;
    tile_weights(t, InRow{}, [&](int i, double v) {
      w[i] = v;
      own += v;
      if (v > 0.0) last_i = i;
    });
    double run = own;
    for (int o = 1; o < 32; o <<= 1) {
      const double v = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += v;
    }
    // the lane that holds the border; behind every border (rounding): the last lane with weight, at its end
    const unsigned some = __ballot_sync(0xffffffffu, last_i >= 0);
    const unsigned over = s_end != 0 ? 0u : __ballot_sync(0xffffffffu, last_i >= 0 && s_before + run > target);
    const int from = over != 0 ? __ffs(over) - 1 : (some != 0 ? 31 - __clz(some) : 0);
    if (lane == from) {
      double sum = s_before + run - own;
      int pick = max(last_i, 0);
      if (over != 0) {
        bool found = false;
#pragma unroll
        for (int i = 0; i < kLaneTile; ++i) {
          sum += w[i];
          if (!found && w[i] > 0.0 && sum > target) {
            pick = i;
            found = true;
          }
        }
      }
      out[count] = t * kTile + lane * kLaneTile + pick;
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
  // few sequences: more warps on each, the time is the latency of a cluster; many: 4 CTAs an SM hide it from one another
  if (a.B <= 16)
    launch_pdl(decide_kernel<512, 2>, dim3((unsigned)a.B * kCluster), dim3(512), smem, st, a);
  else
    launch_pdl(decide_kernel<256, 4>, dim3((unsigned)a.B * kCluster), dim3(256), smem, st, a);
}

}  // namespace b200
