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
// 100 VALU operations of a 16-lane row.  A workgroup takes kTok tokens of one
// sequence and a share of the heads, so that the token's cosines and sines
// (one per thread and round, in LDS) serve every head of the share.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bsattn_device.h"

namespace bsattn {

constexpr int kRotTok = 16;  // tokens per workgroup

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

// FULL: the halves layout over all 128 dims, whose pairs lie 8 lanes apart.
// grid (token tiles, shares of the heads, sequences); 16 rows of 16 lanes,
// lane c of a row holds dims 8c .. 8c + 7 of one (head, token).
template <int DT, bool NORM, bool FULL>
__global__ __launch_bounds__(256) void k_rotate(const int32_t* __restrict__ lens, RotateBatch rb) {
  __shared__ f32x2 s_cs[kRotTok][kHeadDim / 2];
  __shared__ float s_x[FULL ? 1 : 16][FULL ? 1 : kHeadDim + 4];
  const int bi = blockIdx.z, t0 = blockIdx.x * kRotTok;
  const int ntok = min(kRotTok, rb.L - t0);
  const int row = threadIdx.x >> 4, c = threadIdx.x & 15;
  const int heads = rb.heads[0] + rb.heads[1];
  const int h0 = blockIdx.y * rb.share, h1 = min(h0 + rb.share, heads);
  const int half = rb.dims >> 1;
  // the angles of this tile's tokens
  const int first = rb.pos ? 0 : lens[rb.ids[bi]];
  for (int e = threadIdx.x; e < ntok * half; e += 256) {
    const int t = e / half, i = e - t * half;
    const int p = rb.pos ? rb.pos[(size_t)(rb.b0 + bi) * rb.L + t0 + t] : first + t0 + t;
    const double turns = (double)p * (rb.theta[i] * 0.15915494309189533577);
    const float x = (float)(2.0 * (turns - __builtin_rint(turns)));  // half turns, in [-1, 1]
    s_cs[t][i] = f32x2{cospif(x) * rb.m, sinpif(x) * rb.m};
  }
  __syncthreads();
  const int items = (h1 - h0) * ntok;
  for (int it = row; it < items; it += 16) {
    // (a row's 16 lanes enter together; rows of a wave may differ in their trip counts)
    const int hh = it / ntok, t = it - hh * ntok;
    const int head = h0 + hh;
    const int which = head >= rb.heads[0];
    const int hx = which ? head - rb.heads[0] : head;
    const uint16_t* src = rb.x[which] + (int64_t)(rb.b0 + bi) * rb.sb[which] + (int64_t)hx * rb.sh[which] +
                          (int64_t)(t0 + t) * rb.sl[which] + 8 * c;
    float x[8];
    unpack8<DT>(*(const u32x4*)src, x);
    if constexpr (NORM) {
      float w[8], sq = 0.f;
      unpack8<DT>(*(const u32x4*)(rb.w[which] + 8 * c), w);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = __builtin_fmaf(x[e], x[e], sq);
      const float r = rsqrtf(row_sum(sq) * (1.0f / kHeadDim) + rb.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * r * (rb.woff + w[e]);
    }
    float y[8];
    if constexpr (FULL) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float other = row_half(x[e]);
        const f32x2 cs = s_cs[t][8 * (c & 7) + e];
        y[e] = __builtin_fmaf(x[e], cs[0], (c < 8 ? -other : other) * cs[1]);
      }
    } else if (rb.interleaved) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const int i = 4 * c + (e >> 1);
        const f32x2 cs = i < half ? s_cs[t][i] : f32x2{1.f, 0.f};
        y[e] = __builtin_fmaf(x[e], cs[0], -x[e + 1] * cs[1]);
        y[e + 1] = __builtin_fmaf(x[e + 1], cs[0], x[e] * cs[1]);
      }
    } else {
      // pairs of any distance: through LDS, one slot a row (only its own
      // lanes use it, in order)
#pragma unroll
      for (int e = 0; e < 8; ++e) s_x[row][8 * c + e] = x[e];
      wave_lds_order();
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = 8 * c + e;
        if (d < rb.dims) {
          const bool low = d < half;
          const float other = s_x[row][low ? d + half : d - half];
          const f32x2 cs = s_cs[t][low ? d : d - half];
          y[e] = __builtin_fmaf(x[e], cs[0], (low ? -other : other) * cs[1]);
        } else {
          y[e] = x[e];
        }
      }
      wave_lds_order();
    }
    u32x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = pack2<DT>(y[2 * e], y[2 * e + 1]);
    *(u32x4*)(rb.out[which] + (((size_t)(rb.b0 + bi) * rb.heads[which] + hx) * rb.L + t0 + t) * kHeadDim + 8 * c) = o;
  }
}

template <int DT, bool NORM>
static void rotate_dispatch(const int32_t* lens, const RotateBatch& rb, dim3 grid, hipStream_t s, Timing* prof) {
  if (rb.dims == kHeadDim && !rb.interleaved)
    launch(k_rotate<DT, NORM, true>, grid, dim3(256), 0, s, prof, kProfRotate, lens, rb);
  else
    launch(k_rotate<DT, NORM, false>, grid, dim3(256), 0, s, prof, kProfRotate, lens, rb);
}

hipError_t launch_rotate(const Geometry& g, RotateBatch rb, int n, hipStream_t s, Timing* prof) {
  const int tiles = (rb.L + kRotTok - 1) / kRotTok, heads = rb.heads[0] + rb.heads[1];
  rb.share = heads;
  const dim3 grid(tiles, (heads + rb.share - 1) / rb.share, n);
  const bool norm = rb.w[0] != nullptr;
  if (g.dtype == 0) norm ? rotate_dispatch<0, true>(g.meta, rb, grid, s, prof) : rotate_dispatch<0, false>(g.meta, rb, grid, s, prof);
  else norm ? rotate_dispatch<1, true>(g.meta, rb, grid, s, prof) : rotate_dispatch<1, false>(g.meta, rb, grid, s, prof);
  return hipGetLastError();
}

}  // namespace bsattn
