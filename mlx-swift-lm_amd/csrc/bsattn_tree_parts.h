// bsattn_tree_parts.h -- which units of a request's tokens a workgroup of a tree
// attention takes, in which order, and where its partials lie: integer code of
// the kernels (bsattn_tree.hip) that the host's tests run as well.
#pragma once

#include <stdint.h>

#include "bsattn_internal.h"

namespace bsattn {

#define BSATTN_BOTH __host__ __device__ __attribute__((always_inline)) inline

BSATTN_BOTH int least(int a, int b) { return a < b ? a : b; }
BSATTN_BOTH int greatest(int a, int b) { return a > b ? a : b; }

// What a request brings to a launch, and the units of its part
struct TreeRange {
  int T, N, P, lo, u0, units, cu;
  int lg;  // log2 of the heads of a group
};
// T: its tokens with the step's, taken: those of the step
BSATTN_BOTH TreeRange tree_range(const TreeBatch& tb, int i, int T, int taken, int group) {
  TreeRange r;
  r.T = T;
  r.N = least(least(taken, tb.max_tokens), r.T);
  r.P = r.T - r.N;
  r.lg = __builtin_ctz((unsigned)group);
  r.lo = tb.window > 0 ? greatest(0, r.P - tb.window + 1) : 0;  // the first token that a root sees
  r.u0 = r.lo >> 5;
  r.units = r.N > 0 ? ((r.T - 1) >> 5) - r.u0 + 1 : 0;
  // (more tokens than the launch was cut for, as when a graph replays after
  // further reservations: as many parts, of more units each)
  r.cu = tb.cu;
  if (r.units > tb.units[i]) {
    const int most = greatest(1, tb.part0[i + 1] - tb.part0[i]);
    r.cu = greatest(r.cu, ((r.units + most - 1) / most + 3) & ~3);
  }
  return r;
}
// parts of the request that are written
BSATTN_BOTH int tree_parts(const TreeRange& r) { return (r.units + r.cu - 1) / r.cu; }
// whether a request's only part writes the outputs
BSATTN_BOTH bool tree_direct(const TreeBatch& tb, int i) { return tb.part0[i + 1] - tb.part0[i] <= 1; }
// block of hq rows of a node's partials
BSATTN_BOTH int tree_row(const TreeBatch& tb, int i, int part, int node) { return tb.row0[i] + part * tb.max_tokens + node; }
// parts of the launch: padded so that the groups of a (part, head) lie a multiple
// of 8 workgroups apart, on one XCD, whose L2 then holds the K and V they share
BSATTN_BOTH int tree_grid(const TreeBatch& tb) { return tb.groups > 1 ? (tb.part0[tb.n] + 7) & ~7 : tb.part0[tb.n]; }

// The units of a part: those that every column sees whole (from fa on, `full` of
// them), then the others, in front of them and behind (at most 7 in all)
struct TreePart {
  int ua, fa, full, places;
  BSATTN_BOTH TreePart(const TreeBatch& tb, const TreeRange& r, int part) {
    ua = r.u0 + part * r.cu;
    const int ub = least(ua + r.cu, r.u0 + r.units);
    const int whole0 = tb.window > 0 ? (greatest(0, r.P + r.N - tb.window) + 31) >> 5 : 0, whole1 = r.P >> 5;
    fa = least(greatest(ua, whole0), ub);
    full = greatest(least(ub, whole1) - fa, 0);
    places = ub - ua;
  }
  // (places past the part's: its last one)
  BSATTN_BOTH int unit(int at) const {
    const int p = least(at, places - 1), k = ua + p - full;
    return p < full ? fa + p : k < fa ? k : k + full;
  }
};

}  // namespace bsattn
