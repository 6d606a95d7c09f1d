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
// 130 VALU operations of a 16-lane row.  A workgroup takes up to 16 tokens of
// one sequence and a share of the heads, so that a token's cosines and sines
// (in LDS) serve every head of the share; each row asks for four heads ahead of
// the angles' arithmetic and of the four in hand.  8 x 2048 bf16 tokens of 32
// heads, 64 of 128 dims interleaved (268 MB): 58 us, 4.6 TB/s (a copy of 1 GiB
// reaches 4.8); one head at a time 99 us, the cosines read as pairs 64.  8191
// tokens normed and rotated, 64 + 4 heads, 96 dims in halves (285 MB): 73 us
// (161; 92 with the halves' exchange through LDS, whose banks it met 8 times
// over, instead of a lane permutation).
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

__device__ __forceinline__ void read8(const float* p, float* x) {
  const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = a[e];
    x[4 + e] = b[e];
  }
}

// One row's share of a head: 8 dims of x in fp32, normed and rotated.  cs, sn:
// the token's cosines and sines; xs: the row's LDS slot (kRotAny).
template <int DT, bool NORM, int MODE>
__device__ __forceinline__ u32x4 rotate_row(const RotateBatch& rb, u32x4 raw, const float* w, int c, const float* cs,
                                            const float* sn, float* xs) {
  const int half = rb.dims >> 1;
  float x[8], y[8];
  unpack8<DT>(raw, x);
  if constexpr (NORM) {
    float sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(x[e], x[e], sq);
    const float r = rsqrtf(row_sum(sq) * (1.0f / kHeadDim) + rb.eps);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w[e];
  }
  if constexpr (MODE == kRotFull || MODE == kRotLanes) {
    const int lanes = MODE == kRotFull ? 8 : half >> 3;
    const bool low = c < lanes, turned = MODE == kRotFull || c < 2 * lanes;
    const int at = 8 * (MODE == kRotFull ? c & 7 : low ? c : turned ? c - lanes : 0);
    const int partner = ((threadIdx.x & 48) + (low ? c + lanes : turned ? c - lanes : c)) << 2;
    float co[8], si[8];
    read8(cs + at, co);
    read8(sn + at, si);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float other;
      if constexpr (MODE == kRotFull) other = row_half(x[e]);
      else other = __int_as_float(__builtin_amdgcn_ds_bpermute(partner, __float_as_int(x[e])));
      y[e] = __builtin_fmaf(x[e], co[e], (low ? -other : other) * si[e]);
      if (!turned) y[e] = x[e];
    }
  } else if constexpr (MODE == kRotInter) {
    const f32x4 co = *(const f32x4*)(cs + 4 * c), si = *(const f32x4*)(sn + 4 * c);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool turned = 4 * c + j < half;
      const float a = x[2 * j], b = x[2 * j + 1];
      y[2 * j] = turned ? __builtin_fmaf(a, co[j], -b * si[j]) : a;
      y[2 * j + 1] = turned ? __builtin_fmaf(b, co[j], a * si[j]) : b;
    }
  } else {
    // through LDS, one slot a row (only its own lanes use it, in order)
#pragma unroll
    for (int e = 0; e < 8; ++e) xs[8 * c + e] = x[e];
    wave_lds_order();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * c + e;
      y[e] = x[e];
      if (d < rb.dims) {
        const bool low = d < half;
        const int i = low ? d : d - half;
        const float other = xs[low ? d + half : i];
        y[e] = __builtin_fmaf(x[e], cs[i], (low ? -other : other) * sn[i]);
      }
    }
    wave_lds_order();
  }
  u32x4 o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = cvt_pk<DT>(y[2 * e], y[2 * e + 1]);
  return o;
}

// grid (token tiles of 1 << tsh, shares of the heads, sequences); 16 rows of
// 16 lanes, lane c of a row holds dims 8c .. 8c + 7 of one (head, token); a row
// has kRotRound of them under way.
template <int DT, bool NORM, int MODE>
__global__ __launch_bounds__(256) void k_rotate(const int32_t* __restrict__ lens, RotateBatch rb) {
  __shared__ __align__(16) float s_cs[kRotTok][kHeadDim / 2], s_sn[kRotTok][kHeadDim / 2];
  __shared__ float s_x[MODE == kRotAny ? 16 : 1][MODE == kRotAny ? kHeadDim + 4 : 1];
  const int bi = blockIdx.z, t0 = blockIdx.x << rb.tsh;
  const int ntok = min(1 << rb.tsh, rb.L - t0);
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
  const int heads = rb.heads[0] + rb.heads[1];
  const int h0 = blockIdx.y * rb.share, h1 = min(h0 + rb.share, heads);
  const int half = rb.dims >> 1;
  const int items = (h1 - h0) << rb.tsh;
  auto place = [&](int it, int& which, int& hx, int& t) __attribute__((always_inline)) {
    t = it & ((1 << rb.tsh) - 1);
    const int head = h0 + (it >> rb.tsh);
    which = head >= rb.heads[0];
    hx = which ? head - rb.heads[0] : head;
    return it < items && t < ntok;
  };
  u32x4 raw[kRotRound];
  auto load = [&](int it0) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < kRotRound; ++j) {
      int which, hx, t;
      if (place(it0 + 16 * j, which, hx, t))
        raw[j] = *(const u32x4*)(rb.x[which] + (int64_t)(rb.b0 + bi) * rb.sb[which] + (int64_t)hx * rb.sh[which] +
                                 (int64_t)(t0 + t) * rb.sl[which] + 8 * c);
    }
  };
  load(row);
  float w[2][8];
  if constexpr (NORM) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      unpack8<DT>(*(const u32x4*)(rb.w[i] + 8 * c), w[i]);
#pragma unroll
      for (int e = 0; e < 8; ++e) w[i][e] += rb.woff;
    }
  }
  // the angles of this tile's tokens
  const int first = rb.pos ? 0 : lens[rb.ids[bi]];
  for (int t = threadIdx.x >> rb.hsh; t < ntok; t += 256 >> rb.hsh) {
    const int i = threadIdx.x & ((1 << rb.hsh) - 1);
    if (i < half) {
      const int p = rb.pos ? rb.pos[(size_t)(rb.b0 + bi) * rb.L + t0 + t] : first + t0 + t;
      const double turns = (double)p * (rb.theta[i] * 0.15915494309189533577);
      const float x = (float)(2.0 * (turns - __builtin_rint(turns)));  // half turns, in [-1, 1]
      float sn, cn;
      sincospif(x, &sn, &cn);
      s_cs[t][i] = cn * rb.m;
      s_sn[t][i] = sn * rb.m;
    }
  }
  __syncthreads();
  for (int it0 = row; it0 < items; it0 += 16 * kRotRound) {
    // (a row's 16 lanes go together; rows of a wave may differ)
#pragma unroll
    for (int j = 0; j < kRotRound; ++j) {
      int which, hx, t;
      if (place(it0 + 16 * j, which, hx, t)) {
        float wj[8];
        if constexpr (NORM) {
#pragma unroll
          for (int e = 0; e < 8; ++e) wj[e] = which ? w[1][e] : w[0][e];
        }
        const u32x4 o = rotate_row<DT, NORM, MODE>(rb, raw[j], wj, c, s_cs[t], s_sn[t], s_x[MODE == kRotAny ? row : 0]);
        *(u32x4*)(rb.out[which] + (((size_t)(rb.b0 + bi) * rb.heads[which] + hx) * rb.L + t0 + t) * kHeadDim + 8 * c) = o;
      }
    }
    load(it0 + 16 * kRotRound);
  }
}

template <int DT, bool NORM>
static void rotate_dispatch(const int32_t* lens, const RotateBatch& rb, dim3 grid, hipStream_t s, Timing* prof) {
  const dim3 blk(256);
  const int kd = kProfRotate;
  if (rb.interleaved) launch(k_rotate<DT, NORM, kRotInter>, grid, blk, 0, s, prof, kd, lens, rb);
  else if (rb.dims == kHeadDim) launch(k_rotate<DT, NORM, kRotFull>, grid, blk, 0, s, prof, kd, lens, rb);
  else if (rb.dims % 16 == 0) launch(k_rotate<DT, NORM, kRotLanes>, grid, blk, 0, s, prof, kd, lens, rb);
  else launch(k_rotate<DT, NORM, kRotAny>, grid, blk, 0, s, prof, kd, lens, rb);
}

hipError_t launch_rotate(const Geometry& g, RotateBatch rb, int n, hipStream_t s, Timing* prof) {
  const int heads = rb.heads[0] + rb.heads[1];
  rb.tsh = 0;
  while ((1 << rb.tsh) < std::min(rb.L, kRotTok)) ++rb.tsh;
  rb.hsh = 0;
  while ((2 << rb.hsh) < rb.dims) ++rb.hsh;
  const int64_t tiles = ((int64_t)rb.L + (1 << rb.tsh) - 1) >> rb.tsh;
  // shares of the heads: about 4096 workgroups where there is work for them
  // (2 x 134 MB: 67 us with 2048, 58 with 4096 and 6144), of one round of
  // every row and more
  const int64_t want = 4096;
  const int64_t most = std::max<int64_t>(1, ((int64_t)heads << rb.tsh) / 64);
  const int shares = (int)std::min<int64_t>(most, std::max<int64_t>(1, want / (tiles * n)));
  rb.share = (heads + shares - 1) / shares;
  // (whole rounds of every row)
  const int whole = std::max(1, (16 * kRotRound) >> rb.tsh);
  rb.share = (rb.share + whole - 1) / whole * whole;
  const dim3 grid((unsigned)tiles, (heads + rb.share - 1) / rb.share, n);
  const bool norm = rb.w[0] != nullptr;
  if (g.dtype == 0) norm ? rotate_dispatch<0, true>(g.meta, rb, grid, s, prof) : rotate_dispatch<0, false>(g.meta, rb, grid, s, prof);
  else norm ? rotate_dispatch<1, true>(g.meta, rb, grid, s, prof) : rotate_dispatch<1, false>(g.meta, rb, grid, s, prof);
  return hipGetLastError();
}

}  // namespace bsattn
