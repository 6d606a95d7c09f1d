// bsattn_fork.hip -- the device side of a fork: a sequence that starts as
// another's first tokens, sharing the pages of its full blocks.
//
// One launch writes each new sequence's block-table row, length and capacity,
// its summaries (they lie by sequence, not by page), and its own copy of the
// last, partial block's page.  Bound by the bytes of those: at 32k tokens of
// 8 kv heads 1 MB of summaries and at most one page of 256 KB, both read and
// written, where a copy of the tokens would move 128 MB.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bsattn_device.h"

namespace bsattn {

// 16-byte pieces per thread and round (8 branches of 8191 bf16 tokens 4.7 us, 16
// of 16001 int8 5.5; with 8 pieces, a quarter of the workgroups, 5.2 and 6.0)
constexpr int kForkPieces = 2;

// grid (shares of the pieces, pairs)
__global__ __launch_bounds__(256) void k_fork(Geometry geo, ForkBatch fb) {
  const int i = blockIdx.y;
  const int src = fb.src[i], dst = fb.dst[i], tokens = fb.tokens[i];
  const int full = tokens / geo.tb, tail = fb.tail_to[i];
  const int first = blockIdx.x * 256 + threadIdx.x, step = gridDim.x * 256;
  const int32_t* from = block_table(geo, src);
  int32_t* to = geo.meta + geo.bt_off + (size_t)dst * geo.mbps;
  for (int b = first; b < full; b += step) to[b] = from[b];
  if (first == 0) {
    if (tail >= 0) to[full] = tail;
    geo.meta[dst] = tokens;
    geo.meta[geo.cap_off + dst] = (full + (tail >= 0 ? 1 : 0)) * geo.tb;
  }
  // pieces: the summaries of the full blocks, head by head, then the page
  const int per_head = full * (kHeadDim / 8);
  const int summaries = per_head * geo.hkv;
  const int pieces = summaries + (tail >= 0 ? (int)(geo.slab_bytes * geo.hkv / 16) : 0);
  const u32x4* page_from = (const u32x4*)(geo.pool + (size_t)max(fb.tail_from[i], 0) * geo.hkv * geo.slab_bytes);
  u32x4* page_to = (u32x4*)(geo.pool + (size_t)max(tail, 0) * geo.hkv * geo.slab_bytes);
  auto place = [&](int p, const u32x4*& a, u32x4*& b) __attribute__((always_inline)) {
    if (p < summaries) {
      const int h = p / per_head, at = p - h * per_head;
      a = (const u32x4*)summary_row(geo, src, h, 0) + at;
      b = (u32x4*)summary_row(geo, dst, h, 0) + at;
    } else {
      a = page_from + (p - summaries);
      b = page_to + (p - summaries);
    }
  };
  for (int p0 = first; p0 < pieces; p0 += kForkPieces * step) {
    const u32x4* a[kForkPieces];
    u32x4* b[kForkPieces];
    u32x4 x[kForkPieces];
#pragma unroll
    for (int j = 0; j < kForkPieces; ++j) {
      place(min(p0 + j * step, pieces - 1), a[j], b[j]);
      x[j] = *a[j];
    }
#pragma unroll
    for (int j = 0; j < kForkPieces; ++j)
      if (p0 + j * step < pieces) *b[j] = x[j];
  }
}

hipError_t launch_fork(const Geometry& g, const ForkBatch& fb, hipStream_t s, Timing* prof) {
  int64_t most = 1;
  for (int i = 0; i < fb.n; ++i)
    most = std::max(most, (int64_t)(fb.tokens[i] / g.tb) * (kHeadDim / 8) * g.hkv +
                              (fb.tail_to[i] >= 0 ? g.slab_bytes * g.hkv / 16 : 0));
  const int shares = (int)std::min<int64_t>((most + 256 * kForkPieces - 1) / (256 * kForkPieces), 256);
  launch(k_fork, dim3(shares, fb.n), dim3(256), 0, s, prof, kProfFork, g, fb);
  return hipGetLastError();
}

}  // namespace bsattn
