// bsattn_step.hip -- the two ends of a verification step: the map from the
// requests' token counts to rows and page slots, and the accepted paths' way
// back into place.  Both move a few KB to a few hundred and are bound by the
// launch and the chains of dependent loads in it.
#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bsattn_append.h"
#include "bsattn_device.h"

namespace bsattn {

constexpr int kMapRows = 1024;  // rows of a map's workgroup

// ---------------------------------------------------------------------------
// The map.  Every workgroup first finds where the requests (n <= 64, a lane
// each) start and whether they fit, a wave looking at every fourth cache's
// lengths and capacities.  Then
//  - workgroup (x, c) writes the slots of rows [x kMapRows, ..) in cache c; a
//    row's request is the last that starts at or before it (a search in LDS);
//    those of cache 0 also write the rows' requests and, for chains, their
//    positions and ancestors;
//  - with parents, further workgroups of cache 0 take a tree per wave, a node
//    per lane: ancestors by doubling, six rounds of lane permutations (a walk
//    towards the root would be a chain of up to 64 loads).
// grid (workgroups of rows, then of trees; caches)
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void k_step_map(StepMap sm, int row_groups) {
  __shared__ int s_start[kMaxBatch], s_len[kMaxBatch], s_taken[kMaxBatch];
  __shared__ uint64_t s_fits[4];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), cache = blockIdx.y, n = sm.n;
  const int i = min(lane, n - 1);
  const int count = lane < n ? max(sm.counts[i], 0) : 0, seq = sm.ids[i];
  bool fits = lane < n && count <= sm.max_tokens;
  for (int c = wave; c < sm.caches; c += 32) {
    // (eight caches' words on their way at once: 36 caches 8.7 us one by one)
    int len[8], cap[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const StepCache& sc = sm.cache[min(c + 4 * j, sm.caches - 1)];
      len[j] = sc.meta[seq];
      cap[j] = sc.meta[sc.cap_off + seq];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) fits &= (int64_t)len[j] + count <= cap[j];
  }
  const uint64_t all = __ballot(fits);
  if (lane == 0) s_fits[wave] = all;
  const int own = sm.cache[cache].meta[seq];
  int64_t upto = count;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t below = __shfl_up(upto, d, 64);
    if (lane >= d) upto += below;
  }
  __syncthreads();
  if (wave == 0) {
    const bool take = ((s_fits[0] & s_fits[1] & s_fits[2] & s_fits[3]) >> lane & 1) && upto <= sm.rows;
    const int start = (int)min(upto - count, (int64_t)sm.rows), taken = take ? count : 0;
    s_start[lane] = lane < n ? start : INT32_MAX;
    s_taken[lane] = taken;
    s_len[lane] = own;
    if (blockIdx.x == 0 && lane < n) {
      sm.ends[(size_t)cache * n + lane] = own + taken;
      if (cache == 0) {
        sm.starts[lane] = start;
        sm.taken[lane] = taken;
        if (lane == n - 1) sm.starts[n] = (int)min(upto, (int64_t)sm.rows);
      }
    }
  }
  __syncthreads();
  if ((int)blockIdx.x >= row_groups) {
    const int r = 4 * (blockIdx.x - row_groups) + wave;
    if (cache != 0 || r >= n) return;
    const int start = s_start[r], taken = s_taken[r];
    const int up = lane < taken ? sm.parents[start + lane] : -1;
    int lost = up < -1 || up >= lane;
    int at = lost || up < 0 ? lane : up;
    uint64_t anc = 1ull << lane;
#pragma unroll
    for (int k = 0; k < 6; ++k) {  // each round twice as far towards the root
      anc |= __shfl(anc, at, 64);
      lost |= __shfl(lost, at, 64);
      at = __shfl(at, at, 64);
    }
    if (lane >= taken) return;
    if (lost) anc = 0;
    sm.ancestors[start + lane] = anc;
    sm.positions[start + lane] = s_len[r] + (lost ? 0 : __popcll(anc) - 1);
    return;
  }
  const StepCache& sc = sm.cache[cache];
  const int row1 = min((int)(blockIdx.x + 1) * kMapRows, sm.rows);
  for (int row = blockIdx.x * kMapRows + threadIdx.x; row < row1; row += 256) {
    int r = 0;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1)
      if (s_start[r + d] <= row) r += d;
    const int node = row - s_start[r];
    const bool there = node >= 0 && node < s_taken[r];
    const int p = s_len[r] + node;
    int slot = -1;
    if (there) slot = sc.meta[sc.bt_off + (size_t)sm.ids[r] * sc.mbps + p / sc.tb] * sc.tb + p % sc.tb;
    sm.slots[(size_t)cache * sm.rows + row] = slot;
    if (cache != 0) continue;
    sm.requests[row] = there ? r : -1;
    if (there && sm.parents) continue;  // (the tree's wave knows)
    sm.positions[row] = there ? p : 0;
    if (sm.ancestors) sm.ancestors[row] = !there ? 0 : node >= 63 ? ~0ull : (2ull << node) - 1;
  }
}

hipError_t launch_step_map(const StepMap& sm, hipStream_t s, Timing* prof) {
  static_assert(sizeof(StepMap) <= 4000, "a launch's arguments stay under 4 KiB");
  const int row_groups = (sm.rows + kMapRows - 1) / kMapRows;
  const int trees = sm.parents ? (sm.n + 3) / 4 : 0;
  launch(k_step_map, dim3(row_groups + trees, sm.caches), dim3(256), 0, s, prof, kProfMap, sm, row_groups);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------
// Kept paths.  A workgroup moves one (request, kv head)'s kept tokens: the lists
// ascend, so a token moves towards the front, perhaps to where another one still
// lies; everything is read into registers before the first store.  K goes by
// the 16 pieces of a token (8 dims each), V by the pieces of 8 tokens of a dim
// that the tiles are made of, each rebuilt from the codes or elements that move
// into it.  Then 64 or 128 threads fold the summaries of the blocks that are
// full now, in the appends' order, from the tiles.  Slots and lengths come from
// the step's arrays: the metadata is only written.  grid (Hkv, n)
// ---------------------------------------------------------------------------
// bytes of a token's 8 dims, and of 8 tokens' one dim
template <int KB>
struct Piece {
  typedef uint2 T;
};
template <>
struct Piece<0> {
  typedef u32x4 T;
};
template <>
struct Piece<4> {
  typedef uint32_t T;
};

// dims 2c, 2c + 1 of a full block's summary: the sums and roundings of fold_block,
// two dims a thread (a kept path that fills a block: 10.2 us with eight, 8.2 so)
template <int DT, int TB>
__device__ __forceinline__ uint32_t fold_pair(const uint32_t* blk, int c) {
  float a = 0.f, b = 0.f;
#pragma unroll 16
  for (int t = 0; t < TB; ++t) {
    const uint32_t w = blk[64 * t + c];
    const float x = DT == 0 ? lo_f(w) : __uint_as_float(w << 16), y = DT == 0 ? hi_f(w) : __uint_as_float(w & 0xFFFF0000u);
    a = t == 0 ? x : __fadd_rn(a, x);
    b = t == 0 ? y : __fadd_rn(b, y);
  }
  return pack2<DT>(__fmul_rn(a, 1.0f / TB), __fmul_rn(b, 1.0f / TB));
}

template <int DT, int KB, int TB>
__global__ __launch_bounds__(256) void k_keep(Geometry geo, StepRows sr, const int32_t* __restrict__ kept, int width,
                                              const int32_t* __restrict__ n_kept) {
  using T = typename Piece<KB>::T;
  __shared__ int s_from[kMaxNodes], s_slot[kMaxNodes];  // kept nodes; slots of the step's tokens
  __shared__ u32x4 s_blk[KB == 0 ? 64 : TB * KB / 16][16];  // a block's keys, or their code tile
  __shared__ u32x4 s_sb[KB ? TB : 1];
  const int h = blockIdx.x, i = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  // (everything that does not depend on another load is asked for at once)
  const int taken = min(sr.taken[i], kMaxNodes), start = sr.starts[i], seq = sr.ids[i], P = sr.ends[i] - taken;
  const int list = kept[(size_t)i * width + min(lane, width - 1)], many = n_kept[i];
  asm volatile("" ::"v"(list), "s"(many), "s"(start), "s"(P));
  if (taken <= 0) return;
  // the list, up to the first entry that does not ascend or is no node
  const int want = min(min(max(many, 0), width), taken);
  const int from = lane < want ? list : -1;
  const int before = __shfl_up(from, 1, 64);
  const uint64_t bad = __ballot(lane >= want || from < 0 || from >= taken || (lane > 0 && from <= before));
  const int m = bad ? __ffsll((unsigned long long)bad) - 1 : 64;
  if (tid < 64) {
    int slot = lane < taken ? sr.slots[start + lane] : -1;
    if ((int64_t)slot >= sr.pages * TB) slot = -1;
    s_slot[lane] = slot;
    s_from[lane] = lane < m ? from : -1;
  }
  if (h == 0 && tid == 0) geo.meta[seq] = P + m;
  __syncthreads();
  if (m == 0 || __ballot(lane < taken && s_slot[lane] < 0) != 0) return;
  auto slab = [&](int slot) { return geo.pool + ((size_t)(slot / TB) * geo.hkv + h) * geo.slab_bytes; };
  int sh;
  // where the key's dims 8c .. and the value's dim d of 8 tokens lie
  auto k_at = [&](int slot, int c) {
    uint8_t* s = slab(slot) + geo.k_off;
    if constexpr (KB == 0) return (T*)((uint16_t*)s + k_elem(slot % TB, 8 * c));
    else return (T*)(s + kq_byte(KB, slot % TB, 8 * c, &sh));
  };
  auto v_at = [&](int slot, int d) {
    uint8_t* s = slab(slot) + geo.v_off;
    if constexpr (KB == 0) return (T*)((uint16_t*)s + v_elem(TB, slot % TB & ~7, d));
    else return (T*)(s + vq_byte(KB, TB, slot % TB & ~7, d, &sh));
  };
  constexpr int NK = 4, NV = 5;  // pieces of K (64 tokens) and of V (9 groups of tokens) per thread
  T kp[NK], vp[NV];
#pragma unroll
  for (int x = 0; x < NK; ++x) {
    const int j = (tid >> 4) + 16 * x;
    if (j < m) kp[x] = *k_at(s_slot[s_from[j]], tid & 15);
  }
  u32x4 entry = u32x4{0u, 0u, 0u, 0u};
  if constexpr (KB != 0)
    if (tid < m) {
      const int slot = s_slot[s_from[tid]];
      entry = ((const u32x4*)(slab(slot) + geo.sb_off))[sb_entry(TB, slot % TB)];
    }
  const int g0 = P >> 3, g1 = (P + m - 1) >> 3;  // groups of 8 positions that change
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int grp = g0 + 2 * x + (tid >> 7), d = tid & 127;
    if (grp > g1) continue;
    T piece = *v_at(s_slot[max(8 * grp, P) - P], d);
    uint32_t part[8];  // (all eight are on their way before the first is needed)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int slot = s_slot[s_from[min(max(8 * grp + e - P, 0), m - 1)]];
      if constexpr (KB == 0) {
        part[e] = *((const uint16_t*)(slab(slot) + geo.v_off) + v_elem(TB, slot % TB, d));
      } else {
        const uint8_t* at = slab(slot) + geo.v_off + vq_byte(KB, TB, slot % TB, d, &sh);
        part[e] = ((uint32_t)*at >> sh) & ((1u << KB) - 1);
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = 8 * grp + e - P;
      const bool in = j >= 0 && j < m;
      auto with = [&](uint32_t word, int at, uint32_t mask) { return in ? (word & ~(mask << at)) | (part[e] << at) : word; };
      if constexpr (KB == 0) piece[e >> 1] = with(piece[e >> 1], 16 * (e & 1), 0xFFFFu);
      else if constexpr (KB == 4) piece = with(piece, 4 * q_nib(e), 0xFu);
      else if (e < 4) piece.x = with(piece.x, 8 * e, 0xFFu);
      else piece.y = with(piece.y, 8 * (e - 4), 0xFFu);
    }
    vp[x] = piece;
  }
  __builtin_amdgcn_s_waitcnt(0);  // every piece is in its register before any is overwritten
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NK; ++x) {
    const int j = (tid >> 4) + 16 * x;
    if (j < m) *k_at(s_slot[j], tid & 15) = kp[x];
  }
  if constexpr (KB != 0)
    if (tid < m) {
      const int slot = s_slot[tid];
      ((u32x4*)(slab(slot) + geo.sb_off))[sb_entry(TB, slot % TB)] = entry;
    }
#pragma unroll
  for (int x = 0; x < NV; ++x) {
    const int grp = g0 + 2 * x + (tid >> 7), d = tid & 127;
    if (grp <= g1) *v_at(s_slot[max(8 * grp, P) - P], d) = vp[x];
  }
  // summaries of the blocks that are full now, from the tiles
  for (int blk = P / TB; (blk + 1) * TB <= P + m; ++blk) {
    __threadfence_block();
    __syncthreads();
    const uint8_t* s = slab(s_slot[max(blk * TB, P) - P]);
    if constexpr (KB == 0) {
      for (int x = tid; x < TB * 16; x += 256)
        s_blk[x >> 4][x & 15] = *(const u32x4*)((const uint16_t*)(s + geo.k_off) + k_elem(x >> 4, 8 * (x & 15)));
    } else {
      for (int x = tid; x < TB * KB; x += 256) ((u32x4*)s_blk)[x] = ((const u32x4*)(s + geo.k_off))[x];
      if (tid < TB) s_sb[tid] = ((const u32x4*)(s + geo.sb_off))[tid];
    }
    __syncthreads();
    if constexpr (KB == 0) {
      if (tid < 64) ((uint32_t*)summary_row(geo, seq, h, blk))[tid] = fold_pair<DT, TB>((const uint32_t*)s_blk, tid);
    } else {
      if (tid < kHeadDim)
        summary_row(geo, seq, h, blk)[tid] = fold_block_q<KB ? KB : 4>((const uint8_t*)s_blk, (const uint16_t*)s_sb, TB, tid);
    }
  }
}

hipError_t launch_keep(const Geometry& g, const StepRows& sr, const int32_t* kept, int width, const int32_t* n_kept,
                       hipStream_t s, Timing* prof) {
  const dim3 grid(g.hkv, sr.n), blk(256);
  auto go = [&](auto kernel) { launch(kernel, grid, blk, 0, s, prof, kProfKeep, g, sr, kept, width, n_kept); };
  if (g.kv_bits == 4) g.tb == 64 ? go(k_keep<0, 4, 64>) : go(k_keep<0, 4, 32>);
  else if (g.kv_bits == 8) g.tb == 64 ? go(k_keep<0, 8, 64>) : go(k_keep<0, 8, 32>);
  else if (g.dtype == 0) g.tb == 64 ? go(k_keep<0, 0, 64>) : go(k_keep<0, 0, 32>);
  else g.tb == 64 ? go(k_keep<1, 0, 64>) : go(k_keep<1, 0, 32>);
  return hipGetLastError();
}

}  // namespace bsattn
