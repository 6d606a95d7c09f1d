// bsattn_rotate.hip -- rotary positions of queries and keys, alone or behind
// the per-head RMS norms that some models put there, in one pass over them.
//
// For a head x[0, 128) of the token at position p, with R rotated dims in
// pairs (a, b) = (x[2i], x[2i + 1]) (interleaved) or (x[i], x[i + R / 2])
// (halves), i < R / 2:
//   y = x * rsqrt(mean(x^2) + eps) * (offset + w)          (norm only)
//   phi = p * theta_i;  a' = m (a cos phi - b sin phi),  b' = m (a sin phi + b cos phi)
// Everything is fp32 and rounded once, to the output.  The angle is reduced
// in 64 bits: at position 2^20 an fp32 angle of theta_0 = 1 is off by 2^-4.
//
// Bound by memory: each head is read and written once (512 B), against about
// 65 VALU operations of a 16-lane row.  A workgroup takes up to 16 tokens of
// one sequence and a share of a tensor's heads.  A row of lanes stays with one
// token, so that what its dims are multiplied by (cosine and sine, with the
// weights of the norm in them) is in registers for every head, and asks for four
// heads ahead of the angles' arithmetic and of the four in hand.  8 x 2048 bf16
// tokens of 32 heads, 64 of 128 dims interleaved (268 MB): 48.6 us, 5.5 TB/s (a
// copy of 1 GiB reaches 4.8); with the cosines read from LDS for every head,
// rows that go through both tensors' heads and 160 operations a head 58 us,
// without heads under way 99.  8191 tokens normed and rotated, 64 + 4 heads, 96
// dims in halves (285 MB): 53 us (73 and 161); 8 x 512 of 32 + 8 heads (84 MB):
// 16.4 us (20).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bsattn_device.h"

namespace bsattn {

constexpr int kRotTok = 16;   // tokens per workgroup at the most
constexpr int kRotRound = 4;  // heads that a row has under way

// x of the lane 8 places on in its 16-lane row
__device__ __forceinline__ float row_half(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xF, 0xF, false));
}
__device__ __forceinline__ float row_sum(float x) {
  x += __uint_as_float(dpp_u32<kDppQuadXor1>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u32<kDppQuadXor2>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u32<kDppRowRor4>(__float_as_uint(x)));
  x += __uint_as_float(dpp_u32<kDppRowRor8>(__float_as_uint(x)));
  return x;
}

// How a dim meets the other of its pair: 8 lanes on (halves of all 128 dims),
// a whole number of lanes on (halves of R dims, 16 | R), in the same lane
// (interleaved), or anywhere.
enum RotateMode { kRotFull = 0, kRotLanes = 1, kRotInter = 2, kRotAny = 3 };

// What a lane's eight dims 8 c + e are multiplied by: y = a x + b (the other of
// the pair), with the norm's weights in both.  A dim that is not turned meets
// itself and takes half of each, which gives it back whole, infinities too.
struct Turn {
  float a[8], b[8];
  int other[8];  // the other dim (kRotAny)
};
template <bool NORM, int MODE>
__device__ __forceinline__ Turn turn_of(const RotateBatch& rb, const float* w, int c, const float* cs,
                                        const float* sn) {
  const int half = rb.dims >> 1;
  Turn t;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = 8 * c + e;
    const bool turned = d < rb.dims;
    const bool low = MODE == kRotInter ? e % 2 == 0 : d < half;
    const int i = MODE == kRotInter ? d >> 1 : low ? d : d - half;
    const int other = !turned ? d : MODE == kRotInter ? d ^ 1 : low ? d + half : d - half;
    t.a[e] = turned ? cs[turned ? i : 0] : 0.5f;
    t.b[e] = turned ? (low ? -sn[turned ? i : 0] : sn[turned ? i : 0]) : 0.5f;
    if constexpr (NORM) {
      t.a[e] *= w[d];
      t.b[e] *= w[other];
    }
    t.other[e] = other;
  }
  return t;
}

// One row's share of a head: 8 dims of x in fp32, normed and rotated.  partner:
// the lane of the others, times 4 (kRotLanes); xs: the row's LDS slot (kRotAny).
template <int DT, bool NORM, int MODE>
__device__ __forceinline__ u32x4 rotate_row(const RotateBatch& rb, u32x4 raw, const Turn& t, int c, int partner,
                                            float* xs) {
  float x[8], y[8];
  unpack8<DT>(raw, x);
  if constexpr (NORM) {
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(x[e], x[e], sq);
    const float r = rsqrtf(row_sum(sq) * (1.0f / kHeadDim) + rb.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= r;
  }
  if constexpr (MODE == kRotAny) {
    // through LDS, one slot a row (only its own lanes use it, in order)
#pragma unroll
    for (int e = 0; e < 8; ++e) xs[8 * c + e] = x[e];
    wave_lds_order();
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float other;
    if constexpr (MODE == kRotFull) other = row_half(x[e]);
    else if constexpr (MODE == kRotLanes) other = __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(x[e])));
    else if constexpr (MODE == kRotInter) other = x[e ^ 1];
    else other = xs[t.other[e]];
    y[e] = __builtin_fmaf(x[e], t.a[e], other * t.b[e]);
  }
  if constexpr (MODE == kRotInter) {
    // (the other in the lane is not the dim itself)
    if (rb.dims < kHeadDim) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * c + e >= rb.dims) y[e] = x[e] * (2.0f * t.a[e]);
    }
  }
  if constexpr (MODE == kRotAny) wave_lds_order();
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = cvt_pk<DT>(y[2 * e], y[2 * e + 1]);
  return o;
}

// grid (token tiles of 1 << tsh, shares of the heads of one tensor, then of the
// other's, sequences); 16 rows of 16 lanes, lane c of a row holds dims
// 8c .. 8c + 7 of one (head, token).  A row stays with one token, whose
// cosines, sines and weights its lanes keep, and goes through the share's heads,
// kRotRound of them under way.  ONCE: the inputs are more than the caches keep.
template <int DT, bool NORM, int MODE, bool ONCE>
__global__ __launch_bounds__(256) void k_rotate(const int32_t* __restrict__ lens, RotateBatch rb) {
  __shared__ __align__(16) float s_cs[kRotTok][kHeadDim / 2], s_sn[kRotTok][kHeadDim / 2];
  __shared__ float s_x[MODE == kRotAny ? 16 : 1][MODE == kRotAny ? kHeadDim + 4 : 1];
  __shared__ float s_w[NORM ? kHeadDim : 1];
  const int bi = blockIdx.z, t0 = blockIdx.x << rb.tsh;
  const int ntok = min(1 << rb.tsh, rb.L - t0);
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
  const int which = (int)blockIdx.y >= rb.shares0, share = (int)blockIdx.y - (which ? rb.shares0 : 0);
  const int heads = rb.heads[which], h0 = share * rb.share, nh = min(rb.share, heads - h0);
  // this row's token, first head and number of heads (places that do not exist
  // read some place that does)
  const int hstep = 16 >> rb.tsh;
  const int t = min(row & ((1 << rb.tsh) - 1), ntok - 1), hr = min(row >> rb.tsh, nh - 1);
  const bool exists = (row & ((1 << rb.tsh) - 1)) == t && (row >> rb.tsh) == hr;
  const int mine = exists ? (nh - hr + hstep - 1) / hstep : 0, rounds = (nh + hstep - 1) / hstep;
  const int64_t step = hstep * rb.sh[which], ostep = (int64_t)hstep * rb.L * kHeadDim;
  const uint16_t* from = rb.x[which] + (int64_t)(rb.b0 + bi) * rb.sb[which] + (int64_t)(h0 + hr) * rb.sh[which] +
                         (int64_t)(t0 + t) * rb.sl[which] + 8 * c;
  uint16_t* to = rb.out[which] + (((int64_t)(rb.b0 + bi) * heads + h0 + hr) * rb.L + t0 + t) * kHeadDim + 8 * c;
  int left = max(mine, 1);  // heads from `from` on
  u32x4 raw[kRotRound];
  auto load = [&](int j) __attribute__((always_inline)) {
    if constexpr (ONCE) raw[j] = __builtin_nontemporal_load((const u32x4*)from);
    else raw[j] = *(const u32x4*)from;
    from += left > 1 ? step : 0;
    --left;
  };
#pragma unroll
  for (int j = 0; j < kRotRound; ++j) load(j);
  if constexpr (NORM) {
    if (threadIdx.x < kHeadDim) s_w[threadIdx.x] = to_f32<DT>(rb.w[which][threadIdx.x]) + rb.woff;
  }
  // the angles of this tile's tokens
  const int half = rb.dims >> 1;
  const int first = rb.pos ? 0 : lens[rb.ids[bi]];
  for (int at = threadIdx.x >> rb.hsh; at < ntok; at += 256 >> rb.hsh) {
    const int i = threadIdx.x & ((1 << rb.hsh) - 1);
    if (i < half) {
      const int p = rb.pos ? rb.pos[(size_t)(rb.b0 + bi) * rb.L + t0 + at] : first + t0 + at;
      const double turns = (double)p * (rb.theta[i] * 0.15915494309189533577);
      const float x = (float)(2.0 * (turns - __builtin_rint(turns)));  // half turns, in [-1, 1]
      float sn, cn;
      sincospif(x, &sn, &cn);
      s_cs[at][i] = cn * rb.m;
      s_sn[at][i] = sn * rb.m;
    }
  }
  __syncthreads();
  const Turn turn = turn_of<NORM, MODE>(rb, s_w, c, s_cs[t], s_sn[t]);
  const int partner = ((threadIdx.x & 48) + (turn.other[0] >> 3)) << 2;
  for (int i0 = 0; i0 < rounds; i0 += kRotRound) {
#pragma unroll
    for (int j = 0; j < kRotRound; ++j) {
      const u32x4 o = rotate_row<DT, NORM, MODE>(rb, raw[j], turn, c, partner, s_x[MODE == kRotAny ? row : 0]);
      load(j);
      if (i0 + j < mine) *(u32x4*)to = o;
      to += ostep;
    }
  }
}

template <int DT, bool NORM, bool ONCE>
static void rotate_dispatch(const int32_t* lens, const RotateBatch& rb, dim3 grid, hipStream_t s, Timing* prof) {
  const dim3 blk(256);
  const int kd = kProfRotate;
  if (rb.interleaved) launch(k_rotate<DT, NORM, kRotInter, ONCE>, grid, blk, 0, s, prof, kd, lens, rb);
  else if (rb.dims == kHeadDim) launch(k_rotate<DT, NORM, kRotFull, ONCE>, grid, blk, 0, s, prof, kd, lens, rb);
  else if (rb.dims % 16 == 0) launch(k_rotate<DT, NORM, kRotLanes, ONCE>, grid, blk, 0, s, prof, kd, lens, rb);
  else launch(k_rotate<DT, NORM, kRotAny, ONCE>, grid, blk, 0, s, prof, kd, lens, rb);
}

// Inputs of this many bytes and more are loaded past the caches: written by the
// kernel before, 42 MB take 17.9 us kept and 21.9 past them, 84 MB 36 both, 126
// MB 57.9 and 54.6, 336 MB 131 and 117.
constexpr int64_t kRotOnce = 96 << 20;

template <int DT, bool NORM>
static void rotate_dispatch(const int32_t* lens, const RotateBatch& rb, dim3 grid, bool once, hipStream_t s,
                            Timing* prof) {
  if (once) rotate_dispatch<DT, NORM, true>(lens, rb, grid, s, prof);
  else rotate_dispatch<DT, NORM, false>(lens, rb, grid, s, prof);
}

hipError_t launch_rotate(const Geometry& g, RotateBatch rb, int n, hipStream_t s, Timing* prof) {
  const int heads = rb.heads[0] + rb.heads[1];
  rb.tsh = 0;
  while ((1 << rb.tsh) < std::min(rb.L, kRotTok)) ++rb.tsh;
  rb.hsh = 0;
  while ((2 << rb.hsh) < rb.dims) ++rb.hsh;
  const int64_t tiles = ((int64_t)rb.L + (1 << rb.tsh) - 1) >> rb.tsh;
  // shares of the heads: about 2048 workgroups where there is work for them, of
  // one round of every row and more (2 x 134, 2 x 143 and 2 x 42 MB: 48.6, 53.1
  // and 16.4 us; with 1024 49.4, 51.6 and 17.1, with 4096 47.6, 55.4 and 20.4)
  const int64_t want = 2048;
  const int64_t most = std::max<int64_t>(1, ((int64_t)heads << rb.tsh) / 64);
  const int shares = (int)std::min<int64_t>(most, std::max<int64_t>(1, want / (tiles * n)));
  rb.share = (heads + shares - 1) / shares;
  // (whole rounds of every row)
  const int whole = std::max(1, (16 * kRotRound) >> rb.tsh);
  rb.share = (rb.share + whole - 1) / whole * whole;
  rb.shares0 = (rb.heads[0] + rb.share - 1) / rb.share;
  const dim3 grid((unsigned)tiles, rb.shares0 + (rb.heads[1] + rb.share - 1) / rb.share, n);
  const bool norm = rb.w[0] != nullptr, once = (int64_t)n * heads * rb.L * kHeadDim * 2 >= kRotOnce;
  if (g.dtype == 0) norm ? rotate_dispatch<0, true>(g.meta, rb, grid, once, s, prof) : rotate_dispatch<0, false>(g.meta, rb, grid, once, s, prof);
  else norm ? rotate_dispatch<1, true>(g.meta, rb, grid, once, s, prof) : rotate_dispatch<1, false>(g.meta, rb, grid, once, s, prof);
  return hipGetLastError();
}

}  // namespace bsattn
