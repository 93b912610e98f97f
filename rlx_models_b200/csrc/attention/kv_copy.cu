// Copies of whole KV blocks, dst[l, d_i] = src[l, s_i] for every layer l, pair i
// and tensor of a cache (K, V and, for 8-bit pages, their scales), in one launch:
// the partly filled block of a forked request, a prompt's blocks gathered out of
// the pool for a file or put back into it.
//
// Each byte is read once and written once, so HBM bounds it. A CTA copies 8 KB of
// one block, four 16-byte loads per thread in flight before the first store; the
// few bytes of a block's scales go with the first piece of its codes.
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <stdexcept>

#include "../common/b200.cuh"
#include "../common/launch.h"
#include "../common/pdl_launch.h"

namespace b200 {
namespace kvcopy {

constexpr int kThreads = 128;
constexpr int kVec = 4;
constexpr int64_t kPiece = (int64_t)kThreads * kVec * 16;

__device__ __forceinline__ bool aligned16(const void* a, const void* b, int64_t bytes) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | (uintptr_t)bytes) & 15) == 0;
}

__global__ void __launch_bounds__(kThreads) copy_kernel(KvCopyArgs a) {
  pdl_wait();
  pdl_trigger();
  const int64_t pair = blockIdx.x;
  const int layer = blockIdx.y, tid = threadIdx.x;
  const int64_t s = a.src_ids[pair], d = a.dst_ids[pair];
  if (s < 0 || d < 0) return;
  if (s >= a.src_blocks || d >= a.dst_blocks) {
    if (tid == 0) report_error(a.status, kErrBounds, (int)(s >= a.src_blocks ? s : d));
    return;
  }
  int piece = blockIdx.z;
  const bool first = piece == 0;
#pragma unroll 1
  for (int p = 0; p < a.parts; ++p) {
    const KvCopyArgs::Part& t = a.part[p];
    const uint8_t* src = t.src + layer * t.src_layer + s * t.bytes;
    uint8_t* dst = t.dst + layer * t.dst_layer + d * t.bytes;
    if (src == dst) {
      piece -= t.pieces;
      continue;
    }
    if (t.pieces == 0) {
      if (first)
        for (int64_t i = tid; i < t.bytes; i += kThreads) dst[i] = src[i];
      continue;
    }
    if (piece >= 0 && piece < t.pieces) {
      const int64_t lo = piece * kPiece, hi = min(lo + kPiece, t.bytes);
      if (aligned16(src, dst, t.bytes)) {
        uint4 v[kVec];
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int64_t o = lo + ((int64_t)i * kThreads + tid) * 16;
          if (o < hi) v[i] = __ldcs(reinterpret_cast<const uint4*>(src + o));
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
          const int64_t o = lo + ((int64_t)i * kThreads + tid) * 16;
          if (o < hi) __stcs(reinterpret_cast<uint4*>(dst + o), v[i]);
        }
      } else {
        for (int64_t i = lo + tid; i < hi; i += kThreads) dst[i] = src[i];
      }
    }
    piece -= t.pieces;
  }
}

}  // namespace kvcopy

void kv_copy_blocks_launch(const KvCopyArgs& args, cudaStream_t st) {
  using namespace kvcopy;
  KvCopyArgs a = args;
  if (a.n == 0 || a.layers == 0 || a.parts == 0) return;
  int pieces = 0;
  for (int p = 0; p < a.parts; ++p) {
    // the first part has its own pieces, for the small ones to ride on (an empty one: a launch of one piece)
    a.part[p].pieces = p > 0 && a.part[p].bytes < 1024 ? 0 : (int)((a.part[p].bytes + kPiece - 1) / kPiece);
    pieces += a.part[p].pieces;
  }
  if (pieces > 65535 || a.layers > 65535) throw std::runtime_error("b200.kv_copy_blocks: block or layer count too large");
  launch_pdl(copy_kernel, dim3((unsigned)a.n, (unsigned)a.layers, (unsigned)std::max(pieces, 1)), dim3(kThreads), 0, st, a);
}

}  // namespace b200
