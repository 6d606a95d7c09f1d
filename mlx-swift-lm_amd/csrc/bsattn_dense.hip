// bsattn_dense.hip -- attention of one new token per sequence over every
// token of its paged cache (or the last `window` ones):
//   o = sum_t p_t v_t / (sum_t p_t + exp(sink - m)),  p_t = exp(scale q.k_t - m)
// for 16-bit and affine caches.
//
// Bound by the bytes of K and V: each is read once, by one workgroup.  The
// tokens of a (sequence, kv head) are cut into parts of `cu` units of 32
// tokens, one workgroup of four waves each, wave w taking units w, w + 4, ...
// of the part; the parts are joined by k_dense_join.  A wave works in
// registers alone, one unit at a time with MFMA 16x16x32:
//   S^T[token][head] = K[token][:] . Q^T      (A = K rows, B = Q^T)
//   O^T[dim][head]  += V^T[dim][token] . P^T  (A = V^T,    B = P^T)
// In both products a lane (column n, group g) holds head n's share of tokens
// 8g .. 8g + 7, so P goes from one to the other without a shuffle, and the
// running maximum and sum of a head live in its own lanes.
//
// The 16 columns hold a group of G heads 16 / G times.  Where there are two
// copies or more, columns 0-7 multiply V by P rounded to 16 bits and columns
// 8-15 by what that rounding left, so P enters with 16 (bf16) or 22 (fp16)
// bits at no further cost; groups of 16 heads take a second product for it.
//
// The softmax's reference is only raised when a score passes it by more than
// 2^kSlack: the sums are the same for any reference, and a raise costs moves
// across the lanes and a pass over O.
#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "bsattn_append.h"
#include "bsattn_codes.h"
#include "bsattn_device.h"

namespace bsattn {

constexpr float kSlack = 6.0f;
constexpr float kTop = 14.0f;
constexpr float kLog2e = 1.4426950408889634f;

// x of the lane 8 columns on
__device__ __forceinline__ float column8(float x) {
  return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xF, 0xF, false));
}

template <int DT>
__device__ __forceinline__ float lo16(uint32_t w) { return to_f32<DT>((uint16_t)(w & 0xFFFFu)); }
template <int DT>
__device__ __forceinline__ float hi16(uint32_t w) { return to_f32<DT>((uint16_t)(w >> 16)); }

// B operand of x[0, 8) (tokens 8g .. 8g + 7 of this lane's head): hi rounded
// to 16 bits, lo what the rounding left.  Narrow groups: the one that this
// lane's column takes (rest: 1 in columns 8-15, else 0), in hi.
template <int DT, bool WIDE>
__device__ __forceinline__ void split_operand(const float* x, float rest, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t h = cvt_pk<DT>(x[2 * j], x[2 * j + 1]);
    if constexpr (WIDE) {
      hi[j] = h;
      lo[j] = cvt_pk<DT>(x[2 * j] - lo16<DT>(h), x[2 * j + 1] - hi16<DT>(h));
    } else {
      hi[j] = cvt_pk<DT>(__builtin_fmaf(-rest, lo16<DT>(h), x[2 * j]), __builtin_fmaf(-rest, hi16<DT>(h), x[2 * j + 1]));
    }
  }
}

// The range of a sequence that the call sees: tokens [lo, len), units of 32
// from u0 on.
struct DenseRange {
  int len, lo, u0, units;
};
__device__ __forceinline__ DenseRange dense_range(const Geometry& geo, const DenseBatch& db, int seq) {
  DenseRange r;
  r.len = uniform(geo.meta[seq]);
  r.lo = db.window > 0 ? max(0, r.len - db.window) : 0;
  r.u0 = r.lo >> 5;
  r.units = r.len > 0 ? ((r.len - 1) >> 5) - r.u0 + 1 : 0;
  return r;
}

// KIND: 0 fp16, 1 bf16, 4 / 8 affine codes (fp16 queries).
// grid (parts of all entries, Hkv)
template <int KIND, bool WIDE>
__global__ __launch_bounds__(256) void k_dense(Geometry geo, DenseBatch db, const uint16_t* __restrict__ q,
                                               uint16_t* __restrict__ out, float* __restrict__ partials) {
  constexpr int DT = KIND == 1 ? 1 : 0;
  constexpr bool Q = KIND >= 4;
  constexpr int KB = Q ? KIND : 4;
  constexpr int NK = Q ? 2 * QCode<KB>::KF : 8;   // K fragments of a unit
  constexpr int NV = Q ? 8 / QCode<KB>::DPF : 8;  // V fragments of a unit
  constexpr int HC = WIDE ? 16 : 8;               // heads that the workgroup can hold
  // P's range: fp16 weights are lifted to at most 2^14, so that small ones keep
  // their bits (bf16 has fp32's range).  In a quantized cache a weight also
  // meets its token's scale: where one of 2 or more turns up, the weights are
  // at most 1 from there on (65504 times that still fits).
  float lift = DT == 0 ? kTop - kSlack : 0.0f;
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __align__(16) float s_o[4][HC][kHeadDim + 4];
  const int h = blockIdx.y;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  // the entry whose parts hold this workgroup's
  const int bi = __popcll(__ballot(lane < db.n && db.part0[lane] <= (int)blockIdx.x)) - 1;
  const int part = (int)blockIdx.x - uniform(db.part0[bi]);
  const int seq = uniform(db.ids[bi]);
  const int G = geo.group;
  const DenseRange r = dense_range(geo, db, seq);
  const int parts = (r.units + db.cu - 1) / db.cu;
  if (part >= max(parts, 1)) return;
  const int ua = r.u0 + part * db.cu, ub = min(ua + db.cu, r.u0 + r.units);
  u32x4 qf[4];
  {
    const uint16_t* src = q + ((size_t)bi * geo.hq + h * G + (n & (G - 1))) * kHeadDim + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[s] = *(const u32x4*)(src + 32 * s);
  }
  const int sh = geo.tb == 64 ? 1 : 0;
  const int32_t* bt = block_table(geo, seq);
  int pbase = ua >> sh;  // the block whose page lane 0 holds
  int pages = bt[min(pbase + lane, geo.mbps - 1)];
  const float rest = n >= 8 ? 1.0f : 0.0f;

  u32x4 kf[NK], vf[NV];
  u32x4 sb[Q ? 8 : 1];
  auto slab_of = [&](int u) __attribute__((always_inline)) -> const uint8_t* {
    int b = (u >> sh) - pbase;
    if (b >= 64) {
      pbase += b;
      pages = bt[min(pbase + lane, geo.mbps - 1)];
      b = 0;
    }
    const int page = __builtin_amdgcn_readlane(pages, b);
    return geo.pool + ((size_t)page * geo.hkv + h) * geo.slab_bytes;
  };
  auto load_k = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const int sub = u & sh;
    const u32x4* p = (const u32x4*)(slab + geo.k_off) + sub * (NK * 64) + lane;
#pragma unroll
    for (int i = 0; i < NK; ++i) kf[i] = __builtin_nontemporal_load(p + i * 64);
  };
  auto load_v = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const int sub = u & sh;
    const u32x4* p = (const u32x4*)(slab + geo.v_off) + sub * 64 + lane;
#pragma unroll
    for (int i = 0; i < NV; ++i) vf[i] = __builtin_nontemporal_load(p + (i << sh) * 64);
  };
  auto load_sb = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const int sub = u & sh;
    const u32x4* p = (const u32x4*)(slab + geo.sb_off) + g * (geo.tb >> 2) + 8 * sub;
#pragma unroll
    for (int e = 0; e < 8; ++e) sb[Q ? e : 0] = p[e];
  };

  f32x4 o[8], ob0 = f32x4{0.f, 0.f, 0.f, 0.f}, ob1 = ob0;
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, base = 0.0f, l = 0.0f;

  // the queries' share of the code offsets (see bsattn_quant.hip): qk is the
  // QK operand, qs / qb its sum and q's over each 64 dims
  u32x4 qk[4];
  float q0 = 0.f, q1 = 0.f, q0c = 0.f, q1c = 0.f;
  uint32_t code_base = 0;
  if constexpr (Q) {
    code_base = f16_pair_1024();
    const u32x4 ones = u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
    const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      qk[s] = qf[s];
      if constexpr (KB == 4) {
        qk[s][1] = f16x2_unit16(qf[s][1]);
        qk[s][3] = f16x2_unit16(qf[s][3]);
      }
    }
    q0 = mfma_f16(ones, qf[1], mfma_f16(ones, qf[0], zero))[0];
    q1 = mfma_f16(ones, qf[3], mfma_f16(ones, qf[2], zero))[0];
    q0c = kDecOff * mfma_f16(ones, qk[1], mfma_f16(ones, qk[0], zero))[0];
    q1c = kDecOff * mfma_f16(ones, qk[3], mfma_f16(ones, qk[2], zero))[0];
  }

  int u = ua + wave;
  if (u < ub) {
    const uint8_t* slab = slab_of(u);
    load_k(slab, u);
    if constexpr (Q) load_sb(slab, u);
    load_v(slab, u);
  }
  while (u < ub) {
    const int next = u + 4;
    const bool more = next < ub;
    const uint8_t* slab = more ? slab_of(next) : nullptr;
    __builtin_amdgcn_sched_barrier(0);
    // scores of tokens 32 u + 8 g + e, in the log2 domain
    float pv[8];
    if constexpr (!Q) {
      f32x4 acc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; ++s) acc[t] = mfma16x16x32<DT>(kf[4 * t + s], qf[s], acc[t]);
      }
      if (more) load_k(slab, next);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = acc[e >> 2][e & 3] * db.sl2;
    } else {
      f32x4 r0[2], r1[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4* kt = kf + t * QCode<KB>::KF;
        r0[t] = f32x4{-q0c, -q0c, -q0c, -q0c};
        r1[t] = f32x4{-q1c, -q1c, -q1c, -q1c};
        r0[t] = mfma_f16(k_operand<KB>(kt, 0, code_base), qk[0], r0[t]);
        r0[t] = mfma_f16(k_operand<KB>(kt, 1, code_base), qk[1], r0[t]);
        r1[t] = mfma_f16(k_operand<KB>(kt, 2, code_base), qk[2], r1[t]);
        r1[t] = mfma_f16(k_operand<KB>(kt, 3, code_base), qk[3], r1[t]);
      }
      if (more) load_k(slab, next);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float sc = lo_f(sb[e][0]) * r0[e >> 2][e & 3];
        sc = __builtin_fmaf(hi_f(sb[e][0]), r1[e >> 2][e & 3], sc);
        sc = __builtin_fmaf(lo_f(sb[e][1]), q0, sc);
        sc = __builtin_fmaf(hi_f(sb[e][1]), q1, sc);
        pv[e] = sc * db.sl2;
      }
    }
    // tokens that the query does not see: no score, and nothing of what lies
    // there (old pages hold anything) reaches the products
    const bool edge = 32 * u < r.lo || 32 * u + 32 > r.len;
    if (edge) {
      const int t0 = 32 * u + 8 * g;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (t0 + e < r.lo || t0 + e >= r.len) {
          pv[e] = -INFINITY;
          if constexpr (Q) sb[e] = u32x4{0u, 0u, 0u, 0u};
        }
    }
    if constexpr (Q) {
      uint32_t any = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) any |= sb[e][2];
      if (lift > 0.0f && __any((any & 0x40004000u) != 0)) {  // exponents of 2 and more
        const float f = __builtin_amdgcn_exp2f(-kTop);
        lift -= kTop;
        base += kTop;
        l *= f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] *= f;
        ob0 *= f;
        ob1 *= f;
      }
    }
    float mx = pv[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, pv[e]);
    if (__any(mx > m + kSlack)) {
      const float top = fmaxf(m, max_over_groups(mx));
      const float f = top == m ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      m = top;
      base = (top == -INFINITY ? 0.0f : top) - lift;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[dt] *= f;
      if constexpr (Q) {
        ob0 *= f;
        ob1 *= f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pv[e] = __builtin_amdgcn_exp2f(pv[e] - base);
      l += pv[e];
    }
    u32x4 hi, lo;
    split_operand<DT, WIDE>(pv, rest, hi, lo);
    if constexpr (!Q) {
      if (edge) {
        const int t0 = 32 * u + 8 * g;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int ta = t0 + 2 * j, tb = ta + 1;
          const uint32_t keep = (ta >= r.lo && ta < r.len ? 0x0000FFFFu : 0u) | (tb >= r.lo && tb < r.len ? 0xFFFF0000u : 0u);
#pragma unroll
          for (int dt = 0; dt < 8; ++dt) vf[dt][j] &= keep;
        }
      }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        o[dt] = mfma16x16x32<DT>(vf[dt], hi, o[dt]);
        if constexpr (WIDE) o[dt] = mfma16x16x32<DT>(vf[dt], lo, o[dt]);
      }
    } else {
      // sum_t p v_bias per dim group (every row of ob the same), and
      // P_g = p * v_scale_g against the codes; the codes' offset of 1024 is
      // taken off with the same P_g, unit by unit
      u32x4 vb0, vb1;
      float p0[8], p1[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t a = sb[2 * j][3], b = sb[2 * j + 1][3];
        vb0[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        vb1[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = KB == 4 && (e & 2) ? pv[e] * kUnit16 : pv[e];  // int4's unit-16 elements
        p0[e] = x * lo_f(sb[e][2]);
        p1[e] = x * hi_f(sb[e][2]);
      }
      if (more) load_sb(slab, next);
      ob0 = mfma_f16(vb0, hi, ob0);
      ob1 = mfma_f16(vb1, hi, ob1);
      if constexpr (WIDE) {
        ob0 = mfma_f16(vb0, lo, ob0);
        ob1 = mfma_f16(vb1, lo, ob1);
      }
      const u32x4 off = u32x4{0xE400E400u, 0xE400E400u, 0xE400E400u, 0xE400E400u};  // -1024
      u32x4 h0, l0, h1, l1;
      split_operand<0, WIDE>(p0, rest, h0, l0);
      split_operand<0, WIDE>(p1, rest, h1, l1);
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) {
        const u32x4 a = v_operand<KB, 1>(vf, dt, 0, code_base);
        const u32x4& ph = dt < 4 ? h0 : h1;
        o[dt] = mfma_f16(off, ph, o[dt]);
        o[dt] = mfma_f16(a, ph, o[dt]);
        if constexpr (WIDE) {
          const u32x4& pl = dt < 4 ? l0 : l1;
          o[dt] = mfma_f16(off, pl, o[dt]);
          o[dt] = mfma_f16(a, pl, o[dt]);
        }
      }
    }
    if (more) load_v(slab, next);
    __builtin_amdgcn_sched_barrier(0);
    u = next;
  }

  // the waves' shares, then the part's
  l = sum_over_groups(l);
  if (n < G) {
    if (g == 0) {
      s_m[wave][n] = m == -INFINITY ? m : base;
      s_l[wave][n] = l;
    }
  }
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) {
    f32x4 x = o[dt];
    if constexpr (Q) x += dt < 4 ? ob0 : ob1;
    if constexpr (!WIDE) {
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] += column8(x[i]);
    }
    if (n < G) *(f32x4*)&s_o[wave][n][16 * dt + 4 * g] = x;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < G * kHeadDim; e += 256) {
    const int head = e >> 7, d = e & 127;
    float M = s_m[0][head];
#pragma unroll
    for (int w = 1; w < 4; ++w) M = fmaxf(M, s_m[w][head]);
    float L = 0.f, a = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float mw = s_m[w][head];
      const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - M);
      L += f * s_l[w][head];
      a += f * s_o[w][head][d];
    }
    const int hq = h * G + head;
    if (parts <= 1) {
      if (db.sinks && r.len > 0) {
        const float sk = db.sinks[hq] * kLog2e, top = fmaxf(M, sk);
        const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
        L = L * f + (sk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sk - top));
        a *= f;
      }
      out[((size_t)bi * geo.hq + hq) * kHeadDim + d] = from_f32<DT>(L == 0.f ? 0.f : a / L);
    } else {
      float* pp = partials + ((size_t)blockIdx.x * geo.hq + hq) * (kHeadDim + 2);
      pp[d] = a;
      if (d == 0) {
        pp[kHeadDim] = M;
        pp[kHeadDim + 1] = L;
      }
    }
  }
}

// The parts of one (entry, query head) joined; grid (Hq, n)
template <int DT>
__global__ __launch_bounds__(128) void k_dense_join(Geometry geo, DenseBatch db, const float* __restrict__ partials,
                                                    uint16_t* __restrict__ out) {
  const int hq = blockIdx.x, bi = blockIdx.y, d = threadIdx.x;
  const DenseRange r = dense_range(geo, db, db.ids[bi]);
  const int parts = (r.units + db.cu - 1) / db.cu;
  if (parts <= 1) return;
  const float* pp = partials + ((size_t)db.part0[bi] * geo.hq + hq) * (kHeadDim + 2);
  const size_t step = (size_t)geo.hq * (kHeadDim + 2);
  const float sk = db.sinks ? db.sinks[hq] * kLog2e : -INFINITY;
  float M = sk, L = 0.f, a = 0.f;
  for (int p = 0; p < parts; ++p) M = fmaxf(M, pp[p * step + kHeadDim]);
  for (int p = 0; p < parts; ++p) {
    const float mp = pp[p * step + kHeadDim];
    const float f = mp == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mp - M);
    L += f * pp[p * step + kHeadDim + 1];
    a += f * pp[p * step + d];
  }
  if (sk != -INFINITY) L += __builtin_amdgcn_exp2f(sk - M);
  out[((size_t)bi * geo.hq + hq) * kHeadDim + d] = from_f32<DT>(L == 0.f ? 0.f : a / L);
}

// The parts of a launch: units per part (db.cu) and each entry's first part,
// from the most units that it can see.  Returns the number of parts.
int dense_plan(const Geometry& g, const int32_t* units, DenseBatch& db) {
  int64_t all = 0;
  int most = 1;
  for (int i = 0; i < db.n; ++i) {
    all += units[i];
    most = std::max(most, units[i]);
  }
  const int64_t want = 4 * (int64_t)std::max(g.cus, 1);
  db.cu = (int)std::min<int64_t>(most, std::max<int64_t>(4, (all * g.hkv + want - 1) / want));
  while (true) {
    db.cu = (db.cu + 3) & ~3;
    int64_t parts = 0;
    for (int i = 0; i < db.n; ++i) {
      db.part0[i] = (int32_t)parts;
      parts += std::max(1, (units[i] + db.cu - 1) / db.cu);
    }
    if (parts == db.n || parts * g.hq <= kPrefillRows) return (int)parts;
    db.cu *= 2;
  }
}

template <int KIND>
static void dense_dispatch(const Geometry& g, const DenseBatch& db, dim3 grid, const uint16_t* q, uint16_t* out,
                           float* partials, hipStream_t s, Timing* prof) {
  if (g.group > 8) launch(k_dense<KIND, true>, grid, dim3(256), 0, s, prof, kProfDense, g, db, q, out, partials);
  else launch(k_dense<KIND, false>, grid, dim3(256), 0, s, prof, kProfDense, g, db, q, out, partials);
}

template <int DT>
static hipError_t join_dispatch(const Geometry& g, const DenseBatch& db, const float* ws, uint16_t* out,
                                hipEvent_t done, hipStream_t s, Timing* prof) {
  const dim3 grid(g.hq, db.n), blk(128);
  if (done && !prof)  // (the event is the dispatch's own: no packet of its own behind it)
    hipExtLaunchKernelGGL(k_dense_join<DT>, grid, blk, 0u, s, nullptr, done, 0u, g, db, ws, out);
  else
    launch(k_dense_join<DT>, grid, blk, 0, s, prof, kProfCombine, g, db, ws, out);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && done && prof) e = hipEventRecord(done, s);
  return e;
}

hipError_t launch_dense(const Geometry& g, const DenseBatch& db, int parts, const void* q, void* out, float* ws,
                        hipEvent_t done, hipStream_t s, Timing* prof) {
  const dim3 grid(parts, g.hkv);
  const uint16_t* qq = (const uint16_t*)q;
  uint16_t* oo = (uint16_t*)out;
  if (g.kv_bits == 4) dense_dispatch<4>(g, db, grid, qq, oo, ws, s, prof);
  else if (g.kv_bits == 8) dense_dispatch<8>(g, db, grid, qq, oo, ws, s, prof);
  else if (g.dtype == 0) dense_dispatch<0>(g, db, grid, qq, oo, ws, s, prof);
  else dense_dispatch<1>(g, db, grid, qq, oo, ws, s, prof);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || parts == db.n) return e;
  return g.dtype == 0 ? join_dispatch<0>(g, db, ws, oo, done, s, prof) : join_dispatch<1>(g, db, ws, oo, done, s, prof);
}

}  // namespace bsattn
