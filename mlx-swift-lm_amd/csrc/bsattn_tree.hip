// bsattn_tree.hip -- attention of a tree of drafted tokens over the paged cache:
// node j of a request, N nodes behind P tokens, sees the tokens t < P (or those
// at the last `window` positions up to its own) and its ancestors P + a,
//   o = sum_t p_t v_t / (sum_t p_t + exp(sink - m)),  p_t = exp(scale q.k_t - m)
// for 16-bit and affine caches.
//
// A workgroup takes a part of one (request, kv head)'s tokens, in units of 32,
// for a group of the columns, each a (node, query head) pair:
//   S^T[token][col] = K[token][:] . Q^T      (A = K rows, B = Q^T)
//   O^T[dim][col]  += V^T[dim][token] . P^T  (A = V^T,    B = P^T)
// with MFMA 16x16x32.  A lane (column n, group g) holds column n's share of tokens
// 8g .. 8g + 7 in both, so P goes from one to the other without a shuffle.  P
// enters as two 16-bit parts, for 16 (bf16) or 22 (fp16) bits, whatever the columns
// (bf16 values as fp16 where that holds their size, and P as one fp16 number, took
// half of those products, 361 for 414 us with 256 columns over 8 x 32k tokens; but
// weights had 11 bits, and a value of 2^-20 with all the weight, beside an unattended
// one of 1, was off by several of bf16's half steps).  Affine codes enter
// as 1024 + c (K, fp16) and c (V, bf16), exactly; scales and biases act on scores
// and weights.
//
// What bounds it: 64 columns and fewer the reads; above, the order within a wave:
// a unit's scores, its softmax and its products follow each other, and the two
// waves of a SIMD hide only a part of that.  A wave's unit of 32 tokens by 32
// columns is 52 products (of 16 cycles) beside 92 VALU instructions (256 columns,
// bf16; 105 with 64), 48 beside 296 for int8 and 307 for int4, exponentials (16)
// and the codes' conversion included (counted over whole launches).  The matrix
// cores are busy for 50% of the SIMDs' time with 256 bf16 columns and 28% with
// affine caches; waves wait for 30 to 34% of theirs.  Passes: 64 columns over 8 x
// 32k bf16 tokens 200 us (1074 MB: 5.4 TB/s, a plain streaming read 154 us), 256 414
// (664 TFLOP/s; 51% of a large product's rate), 100 over 4 x 131k int4 502, 96 over
// 4 x 262k int8 477.
#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "bsattn_append.h"
#include "bsattn_codes.h"
#include "bsattn_device.h"
#include "bsattn_tree_parts.h"

namespace bsattn {

constexpr float kTreeLog2e = 1.4426950408889634f;
// The softmax's reference is raised when a score passes it by more than 2^kSlack
constexpr float kTreeSlack = 6.0f;
constexpr float kTreeTop = 14.0f;

__device__ __forceinline__ TreeRange tree_range(const Geometry& geo, const TreeBatch& tb, int i) {
  return tree_range(tb, i, geo.meta[tb.ids[i]], tb.taken[i], geo.group);
}

// slabs of the units that a wave takes, the block table read through the scalar cache
struct TreePages {
  const int32_t* bt;
  int h, sh;  // sh: log2 of the units per block
  __device__ __forceinline__ TreePages(const Geometry& geo, int seq, int h_) : h(h_) {
    sh = geo.tb == 64 ? 1 : 0;
    bt = block_table(geo, seq);
  }
  __device__ __forceinline__ int page(int unit) const {
    return *((const __attribute__((address_space(4))) int32_t*)(uintptr_t)(bt + (unit >> sh)));
  }
  __device__ __forceinline__ const uint8_t* slab(const Geometry& geo, int page) const {
    return geo.pool + ((size_t)page * geo.hkv + h) * geo.slab_bytes;
  }
};

// weights x[0, 8) as an operand's two parts: hi rounded to 16 bits, lo what the
// rounding left.  one: bf16 -1 in the low half, and in the high half (from
// minus_one: as constants of the product they come out wrong with this compiler)
struct MinusOne {
  uint32_t lo, hi;
};
__device__ __forceinline__ MinusOne minus_one() {
  return MinusOne{(uint32_t)__builtin_amdgcn_mov_dpp(0x0000BF80, 0xE4, 0xF, 0xF, false),
                  (uint32_t)__builtin_amdgcn_mov_dpp((int)0xBF800000u, 0xE4, 0xF, 0xF, false)};
}
template <int DT>
__device__ __forceinline__ void tree_split(const float* x, const MinusOne& one, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = cvt_pk<DT>(x[2 * j], x[2 * j + 1]);
    hi[j] = w;
    if constexpr (DT == 1) {
      // (a product with -1 and 0 gives the difference in one instruction, exactly)
      auto less = [&](uint32_t c, float v) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), __builtin_bit_cast(bf16x2, c), v, false);
      };
      lo[j] = cvt_pk<1>(less(one.lo, x[2 * j]), less(one.hi, x[2 * j + 1]));
    } else {
      lo[j] = cvt_pk<0>(x[2 * j] - lo_f(w), x[2 * j + 1] - hi_f(w));
    }
  }
}

// eight codes as bf16 (exact): an int4 word (element e in nibble q_nib(e)), or two
// int8 words
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
  return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
}
__device__ __forceinline__ u32x4 nib_to_bf16(uint32_t w) {
  const uint32_t a = w & 0x0F0F0F0Fu, b = (w >> 4) & 0x0F0F0F0Fu;
  auto el = [&](int e) {
    const int nb = q_nib(e);
    return (float)(((nb & 1 ? b : a) >> (8 * (nb >> 1))) & 0xFFu);
  };
  return u32x4{bf16_pair(el(0), el(1)), bf16_pair(el(2), el(3)), bf16_pair(el(4), el(5)), bf16_pair(el(6), el(7))};
}
__device__ __forceinline__ u32x4 byte_to_bf16(uint32_t lo, uint32_t hi) {
  auto el = [&](int e) { return (float)(((e < 4 ? lo : hi) >> (8 * (e & 3))) & 0xFFu); };
  return u32x4{bf16_pair(el(0), el(1)), bf16_pair(el(2), el(3)), bf16_pair(el(4), el(5)), bf16_pair(el(6), el(7))};
}
// a workgroup barrier that orders LDS only: the global loads of later units stay
// in flight across it
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// which of the tokens t0 .. t0 + 7 a node sees: bit e of the cached ones (from
// `from` on) and of the tree's, which begin at token P
__device__ __forceinline__ uint32_t seen_tokens(const uint64_t* s_seen, const int* s_from, int node, int P, int t0) {
  const uint64_t seen = s_seen[node];
  auto below = [](int x) { return (1u << min(max(x, 0), 8)) - 1; };
  const int a = P - t0;
  const uint32_t cached = seen ? below(a) & ~below(s_from[node] - t0) : 0u;
  const uint32_t tree = a > 0 ? (a < 8 ? (uint32_t)(seen << a) : 0u) : a > -64 ? (uint32_t)(seen >> -a) : 0u;
  return (cached | tree) & 0xFFu;
}

// What a workgroup takes of the launch: grid (tree_grid's parts, kv heads, column
// groups)
struct TreePlace {
  int i, h, group, part;  // i: -1 where there is nothing
};
__device__ __forceinline__ TreePlace tree_place(const TreeBatch& tb) {
  TreePlace p;
  const int lane = threadIdx.x & 63, at = blockIdx.x;
  p.h = blockIdx.y;
  p.group = blockIdx.z;
  int last = 0;
  if (tb.n > 1) last = uniform(__popcll(__ballot(lane < tb.n && tb.part0[min(lane, tb.n - 1)] <= at)) - 1);
  p.i = at < tb.part0[tb.n] ? last : -1;
  p.part = at - tb.part0[max(p.i, 0)];
  return p;
}

// Each node's ancestors, those in its window, and the first cached token it
// sees, by the first 64 threads
__device__ __forceinline__ void tree_nodes(const TreeBatch& tb, const TreeRange& r, int start, uint64_t* s_seen, int* s_from) {
  const int j = threadIdx.x;
  if (j >= kMaxNodes) return;
  uint64_t seen = j < r.N ? tb.ancestors[start + j] : 0;
  const int depth = __popcll(seen) - 1;
  s_from[j] = tb.window > 0 ? r.P + depth - tb.window + 1 : 0;
  if (tb.window > 0)
    for (int k = depth + 1; k > tb.window; --k) seen &= seen - 1;  // (the furthest come first)
  s_seen[j] = seen;
}

// What was noted: a value that is infinite or no number is so in the output of
// every column that sees its token, whatever its weight
template <int DT, int KB, int CT>
__device__ __forceinline__ void tree_odd(const Geometry& geo, const TreeRange& r, int seq, int h, const uint2* noted,
                                         const uint64_t* s_seen, const int* s_from, int col0, int cols, f32x4 (&o)[CT][8]) {
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, sh = geo.tb == 64 ? 1 : 0;
  if (!__any(noted[lane & 7].y != 0)) return;
#pragma unroll 1
  for (int x = 0; x < 8; ++x) {
    const int unit = uniform((int)noted[x].x);
#pragma unroll 1
    for (uint32_t odd = (uint32_t)uniform((int)noted[x].y); odd; odd &= odd - 1) {
      const int t = __ffs(odd) - 1, tok = 32 * (unit & sh) + t;
      const int32_t page = block_table(geo, seq)[unit >> sh];
      const uint8_t* own = geo.pool + ((size_t)page * geo.hkv + h) * geo.slab_bytes;
      float v[32];
#pragma unroll
      for (int y = 0; y < 32; ++y) {
        const int d = 16 * (y >> 2) + 4 * g + (y & 3);
        if constexpr (KB == 0) {
          v[y] = to_f32<DT>(((const uint16_t*)(own + geo.v_off))[v_elem(geo.tb, tok, d)]);
        } else {
          int bit;
          const uint2 f = *(const uint2*)(own + geo.sb_off + 16 * sb_entry(geo.tb, tok) + 8);
          const float code = (float)(own[geo.v_off + vq_byte(KB, geo.tb, tok, d, &bit)] >> bit & ((1 << KB) - 1));
          v[y] = y < 16 ? __builtin_fmaf(lo_f(f.x), code, lo_f(f.y)) : __builtin_fmaf(hi_f(f.x), code, hi_f(f.y));
        }
        if (__builtin_isfinite(v[y])) v[y] = 0.f;
      }
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        const int node = min(col0 + 16 * ct + n, cols - 1) >> r.lg;
        const bool ok = seen_tokens(s_seen, s_from, node, r.P, 32 * unit + t) & 1;
#pragma unroll
        for (int y = 0; y < 32; ++y) o[ct][y >> 2][y & 3] += ok ? v[y] : 0.f;
      }
    }
  }
}

// Columns first .. first + count - 1 out of W shares (references s_m, sums s_l,
// o), four dims a thread: the outputs, or the part's partials
template <int DT, int W, int C, int THREADS>
__device__ __forceinline__ void tree_write(const Geometry& geo, const TreeBatch& tb, const TreeRange& r, int i, int h, int part,
                                           int start, int first, int count, bool direct, const float (&s_m)[W][C],
                                           const float (&s_l)[W][C], const float (*s_o)[C][kHeadDim + 4],
                                           const uint64_t* s_seen, uint16_t* __restrict__ out, float* __restrict__ partials) {
  const int d = 4 * (threadIdx.x & 31);
#pragma unroll 4
  for (int c0 = 0; c0 < C; c0 += THREADS / 32) {
    const int c = c0 + (threadIdx.x >> 5);
    if (C % (THREADS / 32) != 0 && c >= C) break;
    const int col = min(first + c, first + count - 1), node = col >> r.lg, hq = (h << r.lg) + col - (node << r.lg);
    float M = s_m[0][c];
#pragma unroll
    for (int v = 1; v < W; ++v) M = fmaxf(M, s_m[v][c]);
    float L = 0.f;
    f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < W; ++v) {
      const float mv = s_m[v][c];
      const float f = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - M);
      L += f * s_l[v][c];
      const f32x4 x = *(const f32x4*)&s_o[v][c][d];
      if (mv != -INFINITY) a += f * x;
    }
    if (c >= count) continue;
    if (s_seen[node] == 0) {  // absent: nothing is seen
      M = -INFINITY;
      L = 0.f;
      a = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    if (direct) {
      if (tb.sinks && M != -INFINITY) {
        const float sk = tb.sinks[hq] * kTreeLog2e, top = fmaxf(M, sk), f = __builtin_amdgcn_exp2f(M - top);
        L = L * f + (sk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sk - top));
        a *= f;
      }
      a = L == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : a / L;
      *(uint2*)(out + ((int64_t)(start + node) * geo.hq + hq) * kHeadDim + d) =
          make_uint2(pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3]));
    } else {
      float* pp = partials + ((int64_t)tree_row(tb, i, part, node) * geo.hq + hq) * kPartial;
      // (partials are 130 floats apart)
      *(float2*)(pp + d) = make_float2(a[0], a[1]);
      *(float2*)(pp + d + 2) = make_float2(a[2], a[3]);
      if (d == 0) *(float2*)(pp + kHeadDim) = make_float2(M, L);
    }
  }
}

template <int KB>
struct Raw {  // a lane's part of a 16-bit operand fragment, as stored
  typedef uint2 T;
};
template <>
struct Raw<0> {
  typedef u32x4 T;
};
template <>
struct Raw<4> {
  typedef uint32_t T;
};

// ---------------------------------------------------------------------------
// CW waves hold up to CT column tiles each and take the same units; TW such teams
// take different ones, UB each per step.  A unit passes through LDS, as 16-bit
// operands: each wave of the team brings its share of the fragments, loaded a
// step before.  So K and V are read, and affine codes converted, once for all of
// the columns (each wave on its own with its own loads: 64 columns 208, 256 485 us
// over 8 x 32k bf16 tokens; 100 columns over 4 x 131k int4 800).  A team of one
// wave (CW 1) needs no barrier, and one place for its unit.
// grid: see tree_place
// ---------------------------------------------------------------------------
template <int DT, int KB, int CT, int CW>
__global__ __launch_bounds__(CW == 1 ? 256 : 512, 2) void k_tree(Geometry geo, TreeBatch tb, const uint16_t* __restrict__ q,
                                                                uint16_t* __restrict__ out, float* __restrict__ partials) {
  static_assert(KB == 0 || DT == 0, "affine caches: fp16");
  constexpr int W = CW == 1 ? 4 : 8, TW = W / CW, SLOTS = CW == 1 ? 1 : 2;
  // units of a team, and of the workgroup, in a step.  16-bit caches: four, however
  // many teams there are (256 columns over 8 x 32k bf16 tokens, 1 and 4: 418 and 403
  // us); affine ones one per team, since their units' pieces and entries then stay in
  // fewer registers (132 columns over 8 x 16k int8 tokens, 1 and 4: 280 and 328 us for
  // the step; 1 and 2, 96 over 4 x 262k int8 487 and 518, 100 over 4 x 131k int4 503
  // and 508)
  constexpr int UB = KB == 0 && CW > 2 ? CW / 2 : 1, STEP = TW * UB;
  constexpr int F = 8 / CW;  // K, and V, operand fragments of a unit that a wave brings: cw + CW x
  static_assert(4 % STEP == 0, "parts are cut in fours");
  // P's type.  Weights times scales need bf16's range, and codes are exact in it
  constexpr int PT = KB ? 1 : DT;
  // fp16 weights are lifted to at most 2^14, so that small ones keep their bits
  constexpr float kLift = PT == 0 ? kTreeTop - kTreeSlack : 0.0f;
  constexpr int COLS = 16 * CT * CW;
  using R = typename Raw<KB>::T;
  // units ([slot][unit of a step][8 K, 8 V fragments][lane]), and in the end the
  // teams' sums
  constexpr int RING = SLOTS * STEP * 16 * 64, SUMS = TW * COLS * (kHeadDim + 4) / 4;
  __shared__ u32x4 s_mem[RING > SUMS ? RING : SUMS];
  // (affine) the tokens' scales and biases: K's in 32 bits, times the scores' scale
  __shared__ f32x4 s_kent[KB ? SLOTS * STEP : 1][KB ? 32 : 1];
  __shared__ uint2 s_vent[KB ? SLOTS * STEP : 1][KB ? 32 : 1];
  __shared__ uint64_t s_seen[kMaxNodes];
  __shared__ int s_from[kMaxNodes];
  __shared__ uint2 s_odd[TW][8];  // units with values that are infinite or no numbers, and their tokens
  __shared__ float s_m[TW][COLS], s_l[TW][COLS];

  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4, cw = wave % CW, tw = wave / CW;
  const TreePlace at = tree_place(tb);
  if (at.i < 0) return;
  const int i = at.i, h = at.h, part = at.part;
  const TreeRange r = tree_range(geo, tb, i);
  const int first = at.group * COLS, cols = r.N << r.lg;
  if (first >= cols || part * r.cu >= r.units) return;
  const bool direct = tree_direct(tb, i);
  const int start = uniform(tb.starts[i]), seq = tb.ids[i];
  const TreePart pt(tb, r, part);
  // the wave's column tiles, spread evenly over the team; waves w and w + 4 share a
  // SIMD, so that the teams' fuller waves lie on different ones.  (Two a wave as far
  // as they go, 96 columns over 4 x 262k int8 tokens 546, spread 486 us; 132 over
  // 8 x 16k ones 336 and 290 for the step.)
  const int tiles = min((cols - first + 15) >> 4, CT * CW), turn = wave >= 4 && CW < 8 ? CW - 1 - cw : cw;
  const int own = CW == 1 ? CT : tiles / CW + (turn < tiles % CW ? 1 : 0);
  const int tile0 = CW == 1 ? 0 : tiles / CW * turn + min(turn, tiles % CW), col0 = first + 16 * tile0;
  const int steps = (pt.places + STEP - 1) / STEP;  // the team's units of step s: places STEP s + TW u + tw

  // --- units from memory, and their pages a step ahead
  TreePages pages(geo, seq, h);
  int unit_next[UB], page_next[UB];
  auto ask = [&](int step) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      unit_next[u] = pt.unit(STEP * step + TW * u + tw);
      page_next[u] = pages.page(unit_next[u]);
    }
  };
  R rk[UB][F], rv[UB][F];
  [[maybe_unused]] u32x4 re[UB];
  const uint32_t lane16 = (uint32_t)lane * 16;
  const uint32_t ent_at = 16u * (uint32_t)(((lane >> 3) & 3) * (geo.tb >> 2) + (lane & 7));
  auto load = [&](int next) __attribute__((always_inline)) {  // the units asked for; then asks for step `next`
    const uint8_t* slab[UB];
    int sub[UB];
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      slab[u] = pages.slab(geo, page_next[u]);
      sub[u] = unit_next[u] & pages.sh;
    }
    ask(next);
    // (a lane's offset, kept in 32 bits up to here: the loads add it to a uniform address)
    uint32_t at = lane16;
    asm volatile("" : "+v"(at));
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const uint8_t *ks = slab[u] + geo.k_off, *vs = slab[u] + geo.v_off;
#pragma unroll
      for (int x = 0; x < F; ++x) {
        const int f = cw + CW * x;
        if constexpr (KB == 0) {
          rk[u][x] = *(const R*)(ks + (8 * sub[u] + f) * 1024 + at);
          rv[u][x] = *(const R*)(vs + ((f << pages.sh) + sub[u]) * 1024 + at);
        } else if constexpr (KB == 4) {
          rk[u][x] = *(const R*)(ks + (2 * sub[u] + (f >> 2)) * 1024 + 4 * (f & 3) + at);
          rv[u][x] = *(const R*)(vs + (((f >> 2) << pages.sh) + sub[u]) * 1024 + 4 * (f & 3) + at);
        } else {
          rk[u][x] = *(const R*)(ks + (4 * sub[u] + (f >> 1)) * 1024 + 8 * (f & 1) + at);
          rv[u][x] = *(const R*)(vs + (((f >> 1) << pages.sh) + sub[u]) * 1024 + 8 * (f & 1) + at);
        }
      }
      if constexpr (KB != 0) re[u] = *(const u32x4*)(slab[u] + geo.sb_off + sub[u] * 128 + ent_at);
    }
  };
  ask(0);
  load(1);

  if (threadIdx.x < 8 * TW) s_odd[threadIdx.x >> 3][threadIdx.x & 7] = make_uint2(0u, 0u);
  tree_nodes(tb, r, start, s_seen, s_from);
  // scores are products times |scale|, of queries with its sign: the largest is
  // found on the products.  (-inf, of what is not seen, times it is -inf)
  const float sc = fmaxf(fabsf(tb.sl2), 1e-30f);
  const uint32_t qflip = tb.sl2 < 0.f ? 0x80008000u : 0u;
  u32x4 qf[CT][4];
  [[maybe_unused]] float q0[CT], q1[CT], q0c[CT], q1c[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int col = min(col0 + 16 * ct + n, cols - 1), node = col >> r.lg;
    const uint16_t* src = q + (int64_t)(start + node) * tb.qr + (int64_t)((h << r.lg) + col - (node << r.lg)) * tb.qh + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[ct][s] = *(const u32x4*)(src + 32 * s) ^ qflip;
    if constexpr (KB != 0) {
      // the queries' sums over each 64 dims: of q, and of the QK operand (int4:
      // with its unit-16 elements scaled) times 1024
      const u32x4 ones = u32x4{0x3C003C00u, 0x3C003C00u, 0x3C003C00u, 0x3C003C00u};
      const f32x4 zero = f32x4{0.f, 0.f, 0.f, 0.f};
      q0[ct] = mfma_f16(ones, qf[ct][1], mfma_f16(ones, qf[ct][0], zero))[0];
      q1[ct] = mfma_f16(ones, qf[ct][3], mfma_f16(ones, qf[ct][2], zero))[0];
      if constexpr (KB == 4)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          qf[ct][s][1] = f16x2_unit16(qf[ct][s][1]);
          qf[ct][s][3] = f16x2_unit16(qf[ct][s][3]);
        }
      q0c[ct] = mfma_f16(ones, qf[ct][1], mfma_f16(ones, qf[ct][0], zero))[0] * -kDecOff;
      q1c[ct] = mfma_f16(ones, qf[ct][3], mfma_f16(ones, qf[ct][2], zero))[0] * -kDecOff;
    }
  }
  [[maybe_unused]] const uint32_t code_base = KB ? f16_pair_1024() : 0u;

  // --- and into LDS, as 16-bit operands
  auto stage = [&](int step, int slot) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < UB; ++u) {
      const int place = STEP * step + TW * u + tw, at = slot * STEP + TW * u + tw;
      u32x4* to = s_mem + at * 16 * 64 + lane;
#pragma unroll
      for (int x = 0; x < F; ++x) {
        const int f = cw + CW * x;
        if constexpr (KB == 0) {
          to[f * 64] = rk[u][x];
          to[(8 + f) * 64] = rv[u][x];
        } else if constexpr (KB == 4) {
          to[f * 64] = nib_to_f16_dec(rk[u][x], code_base);
          to[(8 + f) * 64] = nib_to_bf16(rv[u][x]);
        } else {
          to[f * 64] = byte_to_f16(rk[u][x].x, rk[u][x].y);
          to[(8 + f) * 64] = byte_to_bf16(rv[u][x].x, rv[u][x].y);
        }
      }
      if (place >= pt.full) {
        // Some columns do not see all of the unit.  Values of tokens that none sees
        // (old pages hold anything) are taken as zeros; so are infinities and NaN,
        // which a weight of zero does not take out of a product: they are noted, and
        // reach the columns that see them at the end.  Of affine caches these are
        // tokens with such scales or biases, for their 64 dims.
        const int unit = pt.unit(place);
        uint32_t odd = 0;
        if constexpr (KB == 0) {
          const int t0 = 32 * unit + 8 * g;
          constexpr uint32_t INF = DT == 0 ? 0x7C00u : 0x7F80u;
          u32x4 any = u32x4{0u, 0u, 0u, 0u};
#pragma unroll 1
          for (int f = 8 + cw; f < 16; f += CW) {
            u32x4 v = to[f * 64];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int a = t0 + 2 * j;
              const uint32_t w = v[j] & ((a >= r.lo && a < r.T ? 0x0000FFFFu : 0u) | (a + 1 >= r.lo && a + 1 < r.T ? 0xFFFF0000u : 0u));
              const uint32_t bad = ((w & INF) == INF ? 0xFFFFu : 0u) | ((w >> 16 & INF) == INF ? 0xFFFF0000u : 0u);
              any[j] |= bad;
              v[j] = w & ~bad;
            }
            to[f * 64] = v;
          }
          if (__any((any[0] | any[1] | any[2] | any[3]) != 0))
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const uint64_t who = __ballot((any[e >> 1] >> (16 * (e & 1)) & 1) != 0);
#pragma unroll
              for (int gg = 0; gg < 4; ++gg)
                if (who >> (16 * gg) & 0xFFFF) odd |= 1u << (8 * gg + e);
            }
        } else {
          auto inf = [](uint32_t w) {
            return ((w & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((w >> 16 & 0x7C00u) == 0x7C00u ? 0xFFFF0000u : 0u);
          };
          const uint32_t bad = inf(re[u][2]) | inf(re[u][3]);
          odd = (uint32_t)__ballot(bad != 0 && lane < 32);
          re[u][2] &= ~bad;
          re[u][3] &= ~bad;
        }
        if (odd && lane == 0 && place < pt.places) {
          uint2* note = &s_odd[tw][place - pt.full];
          note->x = unit;
          atomicOr(&note->y, odd);
        }
      }
      if constexpr (KB != 0)
        if (cw == 0) {
          s_kent[at][lane & 31] = sc * f32x4{lo_f(re[u][0]), hi_f(re[u][0]), lo_f(re[u][1]), hi_f(re[u][1])};
          s_vent[at][lane & 31] = make_uint2(re[u][2], re[u][3]);
        }
    }
  };
  auto sync = [&]() __attribute__((always_inline)) {
    if constexpr (CW == 1) wave_lds_order();
    else lds_barrier();
  };

  f32x4 o[CT][8];
  float m[CT], base[CT], limit[CT];  // limit: the product (affine caches: exponent) past which the reference is raised
  // the weights' sums, as they enter the products: of 16-bit caches by a product
  // with ones (rows alike)
  f32x4 l[CT];
  [[maybe_unused]] float ob0[CT], ob1[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[ct][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    m[ct] = limit[ct] = -INFINITY;
    base[ct] = 0.f;
    l[ct] = f32x4{0.f, 0.f, 0.f, 0.f};
    if constexpr (KB != 0) ob0[ct] = ob1[ct] = 0.f;
  }
  const MinusOne one = minus_one();
  [[maybe_unused]] const uint32_t unit_pair = PT == 0 ? 0x3C003C00u : 0x3F803F80u;
  [[maybe_unused]] const u32x4 ones = u32x4{unit_pair, unit_pair, unit_pair, unit_pair};

  auto compute = [&](auto count, int place, int at) __attribute__((always_inline)) {  // at: the unit in the ring
    constexpr int C = decltype(count)::value;  // the wave's column tiles
    const u32x4* in = s_mem + at * 16 * 64 + lane;
    [[maybe_unused]] const f32x4* kent = s_kent[KB ? at : 0] + 8 * g;
    [[maybe_unused]] const uint2* vent = s_vent[KB ? at : 0] + 8 * g;
    // S^T: entry e is token 8 g + e of the unit.  Affine caches: the codes' products
    // of each 64 dims, then with the token's scales and biases, which makes the
    // exponents: times the scale, and less the reference
    float sv[C][8];
    f32x4 acc[C][KB ? 4 : 2];
#pragma unroll
    for (int ct = 0; ct < C; ++ct)
#pragma unroll
      for (int x = 0; x < (KB ? 4 : 2); ++x) {
        float c = 0.f;
        if constexpr (KB != 0) c = x < 2 ? q0c[ct] : q1c[ct];
        acc[ct][x] = f32x4{c, c, c, c};
      }
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const u32x4 a = in[(4 * t + s) * 64];
        const int x = (KB ? 2 * (s >> 1) : 0) + t;
#pragma unroll
        for (int ct = 0; ct < C; ++ct) acc[ct][x] = mfma16x16x32<DT>(a, qf[ct][s], acc[ct][x]);
      }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      f32x4 k = f32x4{0.f, 0.f, 0.f, 0.f};
      if constexpr (KB != 0) k = kent[e];
#pragma unroll
      for (int ct = 0; ct < C; ++ct) {
        if constexpr (KB == 0) {
          sv[ct][e] = acc[ct][e >> 2][e & 3];
        } else {
          float x = __builtin_fmaf(k[3], q1[ct], -base[ct]);
          x = __builtin_fmaf(k[2], q0[ct], x);
          x = __builtin_fmaf(k[1], acc[ct][2 + (e >> 2)][e & 3], x);
          sv[ct][e] = __builtin_fmaf(k[0], acc[ct][e >> 2][e & 3], x);
        }
      }
    }
    if (place >= pt.full) {
#pragma unroll
      for (int ct = 0; ct < C; ++ct) {
        const uint32_t mask =
            seen_tokens(s_seen, s_from, min(col0 + 16 * ct + n, cols - 1) >> r.lg, r.P, 32 * pt.unit(place) + 8 * g);
#pragma unroll
        for (int e = 0; e < 8; ++e) sv[ct][e] = mask >> e & 1 ? sv[ct][e] : -INFINITY;
      }
    }
    // the largest scores, and one branch for all columns' references
    float mx[C];
    bool raise = false;
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
      mx[ct] = sv[ct][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) mx[ct] = fmaxf(mx[ct], sv[ct][e]);
      raise = raise || mx[ct] > limit[ct];
    }
    if (__any(raise)) {
#pragma unroll
      for (int ct = 0; ct < C; ++ct) {
        const float most = max_over_groups(mx[ct]), was = base[ct];
        const float top = fmaxf(m[ct], KB ? was + most : most * sc);
        const bool same = top == m[ct];
        const float f = same ? 1.0f : __builtin_amdgcn_exp2f(m[ct] - top);
        m[ct] = top;
        base[ct] = (top == -INFINITY ? 0.0f : top) - kLift;
        limit[ct] = KB ? (top == -INFINITY ? top : kTreeSlack) : (top + kTreeSlack) / sc;
        if constexpr (KB != 0) {
          const float less = same ? 0.0f : was - base[ct];
#pragma unroll
          for (int e = 0; e < 8; ++e) sv[ct][e] += less;
        }
        l[ct] *= f;
        if constexpr (KB != 0) {
          ob0[ct] *= f;
          ob1[ct] *= f;
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[ct][dt] *= f;
      }
    }
    // the weights, as operands' two parts; affine caches: times the value scales,
    // o_d = sum_t (p_t vs_j) c_td + sum_t p_t vb_j for group j of 64 dims
    u32x4 hi[C][KB ? 2 : 1], lo[C][KB ? 2 : 1];
    [[maybe_unused]] float w0[C][KB ? 8 : 1], w1[C][KB ? 8 : 1];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      uint2 sb = make_uint2(0u, 0u);
      if constexpr (KB != 0) sb = vent[e];
#pragma unroll
      for (int ct = 0; ct < C; ++ct) {
        const float p = __builtin_amdgcn_exp2f(KB ? sv[ct][e] : __builtin_fmaf(sv[ct][e], sc, -base[ct]));
        if constexpr (KB == 0) {
          sv[ct][e] = p;
        } else {
          l[ct][0] += p;
          // (a multiplication with a 16-bit operand is an addition of 0 as well)
          w0[ct][e] = __builtin_fmaf(p, lo_f(sb.x), 0.0f);
          w1[ct][e] = __builtin_fmaf(p, hi_f(sb.x), 0.0f);
          ob0[ct] = __builtin_fmaf(p, lo_f(sb.y), ob0[ct]);
          ob1[ct] = __builtin_fmaf(p, hi_f(sb.y), ob1[ct]);
        }
      }
    }
#pragma unroll
    for (int ct = 0; ct < C; ++ct) {
      if constexpr (KB == 0) {
        tree_split<PT>(sv[ct], one, hi[ct][0], lo[ct][0]);
        l[ct] = mfma16x16x32<PT>(ones, hi[ct][0], l[ct]);
        l[ct] = mfma16x16x32<PT>(ones, lo[ct][0], l[ct]);
      } else {
        tree_split<1>(w0[ct], one, hi[ct][0], lo[ct][0]);
        tree_split<1>(w1[ct], one, hi[ct][1], lo[ct][1]);
      }
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const u32x4 v = in[(8 + dt) * 64];
      constexpr int HALF = KB ? 4 : 8;
#pragma unroll
      for (int ct = 0; ct < C; ++ct) o[ct][dt] = mfma16x16x32<PT>(v, hi[ct][dt / HALF], o[ct][dt]);
#pragma unroll
      for (int ct = 0; ct < C; ++ct) o[ct][dt] = mfma16x16x32<PT>(v, lo[ct][dt / HALF], o[ct][dt]);
    }
  };

  __syncthreads();
  auto run = [&](auto count) __attribute__((always_inline)) {
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      const int slot = SLOTS == 1 ? 0 : s & 1;
      stage(s, slot);
      load(s + 2);
      sync();
      if constexpr (decltype(count)::value > 0)
#pragma unroll 1
        for (int u = 0; u < UB; ++u) {
          const int place = STEP * s + TW * u + tw;
          if (place < pt.places) compute(count, place, slot * STEP + TW * u + tw);
        }
      if constexpr (SLOTS == 1) sync();
    }
  };
  // (a wave's barriers are those of its own loop: all waves reach as many)
  if (CW == 1 || own == CT) run(std::integral_constant<int, CT>{});
  else if (CT > 1 && own == 1) run(std::integral_constant<int, 1>{});
  else run(std::integral_constant<int, 0>{});
  __syncthreads();
  tree_odd<DT, KB, CT>(geo, r, seq, h, s_odd[tw], s_seen, s_from, col0, cols, o);

  // the teams' shares joined
  float (*s_o)[COLS][kHeadDim + 4] = (float (*)[COLS][kHeadDim + 4])s_mem;
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    if (ct >= own) break;
    const int c = 16 * (tile0 + ct) + n;
    const float lc = KB ? sum_over_groups(l[ct][0]) : l[ct][0];
    if (g == 0) {
      s_m[tw][c] = m[ct] == -INFINITY ? m[ct] : base[ct];
      s_l[tw][c] = lc;
    }
    float b0 = 0.f, b1 = 0.f;
    if constexpr (KB != 0) {
      b0 = sum_over_groups(ob0[ct]);
      b1 = sum_over_groups(ob1[ct]);
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      f32x4 x = o[ct][dt];
      if constexpr (KB != 0) x += dt < 4 ? b0 : b1;
      *(f32x4*)&s_o[tw][c][16 * dt + 4 * g] = x;
    }
  }
  __syncthreads();
  tree_write<DT, TW, COLS, 64 * W>(geo, tb, r, i, h, part, start, first, min(cols - first, COLS), direct, s_m, s_l, s_o, s_seen,
                                   out, partials);
}

// The parts of each (node, query head) joined: 32 lanes with four dims each take
// the parts four at a time; ROWS of them share a (node, head) where there are many
// parts.  grid (Hq, nodes of all requests, 8 / ROWS a workgroup)
template <int DT, int ROWS>
__global__ __launch_bounds__(256) void k_tree_join(Geometry geo, TreeBatch tb, const float* __restrict__ ws,
                                                   uint16_t* __restrict__ out) {
  __shared__ __align__(16) float s_o[8][kHeadDim];
  __shared__ float s_ml[8][2];
  const int slot = threadIdx.x >> 5, c = threadIdx.x & 31, y = slot % ROWS;
  const int hq = blockIdx.x, which = blockIdx.y * (8 / ROWS) + slot / ROWS;
  const int i = min(which / tb.max_tokens, tb.n - 1), node = which - i * tb.max_tokens;
  const TreeRange r = tree_range(geo, tb, ROWS == 8 ? uniform(i) : i);
  // (requests of one part: the launch before wrote the output, and they have no
  // partials.  The loads go by the parts of the launch and do not wait for the lengths)
  const int cut = tb.part0[i + 1] - tb.part0[i], most = which < tb.n * tb.max_tokens && cut > 1 ? cut : 0;
  const bool there = most > 0 && node < r.N;
  float M = -INFINITY, L = 0.f;
  f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
  const int parts = there ? tree_parts(r) : 0;
  for (int p0 = y; p0 < most; p0 += 4 * ROWS) {
    f32x4 x[4];
    float m[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int p = min(p0 + j * ROWS, most - 1);
      const float2* part = (const float2*)(ws + ((int64_t)tree_row(tb, i, p, node) * geo.hq + hq) * kPartial);
      const float2 xa = part[2 * c], xb = part[2 * c + 1], ml = part[kHeadDim / 2];
      x[j] = f32x4{xa.x, xa.y, xb.x, xb.y};
      // (without a token that is seen: no reference, and a sum of 0, or NaN)
      m[j] = p0 + j * ROWS < parts ? ml.x : -INFINITY;
      l[j] = p0 + j * ROWS < parts ? ml.y : 0.f;
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = fmaxf(top, m[j]);
    const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
    L *= f;
    a *= f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float w = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[j] - top);
      L += w * l[j];
      if (m[j] != -INFINITY) a += w * x[j];
    }
    M = top;
  }
  if constexpr (ROWS > 1) {
    *(f32x4*)&s_o[slot][4 * c] = a;
    if (c == 0) {
      s_ml[slot][0] = M;
      s_ml[slot][1] = L;
    }
    __syncthreads();
    if (y != 0) return;
    float top = M;
#pragma unroll
    for (int x = 1; x < ROWS; ++x) top = fmaxf(top, s_ml[slot + x][0]);
    const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
    L *= f;
    a *= f;
#pragma unroll
    for (int x = 1; x < ROWS; ++x) {
      const float mx = s_ml[slot + x][0], w = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mx - top);
      L += w * s_ml[slot + x][1];
      if (mx != -INFINITY) a += w * *(const f32x4*)&s_o[slot + x][4 * c];
    }
    M = top;
  }
  if (!there) return;
  if (tb.sinks && M != -INFINITY) {
    const float sk = tb.sinks[hq] * kTreeLog2e, top = fmaxf(M, sk), f = __builtin_amdgcn_exp2f(M - top);
    L = L * f + (sk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sk - top));
    a *= f;
  }
  a = L == 0.f ? f32x4{0.f, 0.f, 0.f, 0.f} : a / L;
  *(uint2*)(out + ((int64_t)(tb.starts[i] + node) * geo.hq + hq) * kHeadDim + 4 * c) =
      make_uint2(pack2<DT>(a[0], a[1]), pack2<DT>(a[2], a[3]));
}

template <int DT, int KB>
static void tree_dispatch(const Geometry& g, const TreeBatch& tb, const uint16_t* q, uint16_t* out, float* ws,
                          hipStream_t s, Timing* prof) {
  const dim3 grid(tree_grid(tb), g.hkv, tb.groups);
  auto go = [&](auto kernel, int threads) { launch(kernel, grid, dim3(threads), 0, s, prof, kProfTree, g, tb, q, out, ws); };
  if (tb.tiles == 1) go(k_tree<DT, KB, 1, 1>, 256);
  else if (tb.tiles == 2) go(k_tree<DT, KB, 2, 1>, 256);
  else if (tb.tiles == 4) tb.narrow ? go(k_tree<DT, KB, 1, 4>, 512) : go(k_tree<DT, KB, 2, 2>, 512);
  else if (tb.tiles == 8) tb.narrow ? go(k_tree<DT, KB, 1, 8>, 512) : go(k_tree<DT, KB, 2, 4>, 512);
  else go(k_tree<DT, KB, 2, 8>, 512);
}

static_assert(sizeof(Geometry) + sizeof(TreeBatch) <= 4000, "a launch's arguments stay under 4 KiB");
hipError_t launch_tree(const Geometry& g, const TreeBatch& tb, const void* q, void* out, float* ws, hipEvent_t done,
                       hipStream_t s, Timing* prof) {
  const uint16_t* qq = (const uint16_t*)q;
  uint16_t* oo = (uint16_t*)out;
  if (g.kv_bits == 4) tree_dispatch<0, 4>(g, tb, qq, oo, ws, s, prof);
  else if (g.kv_bits == 8) tree_dispatch<0, 8>(g, tb, qq, oo, ws, s, prof);
  else if (g.dtype == 0) tree_dispatch<0, 0>(g, tb, qq, oo, ws, s, prof);
  else tree_dispatch<1, 0>(g, tb, qq, oo, ws, s, prof);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !ws) return e;
  int most = 1;
  for (int i = 0; i < tb.n; ++i) most = std::max(most, tb.part0[i + 1] - tb.part0[i]);
  const bool many = most > 8;
  const int nodes = tb.n * tb.max_tokens;
  const dim3 grid(g.hq, many ? nodes : (nodes + 7) / 8), blk(256);
  const float* cws = ws;
  auto join = [&](auto kernel) {
    if (done && !prof)  // (the event is the dispatch's own: no packet of its own behind it)
      hipExtLaunchKernelGGL(kernel, grid, blk, 0u, s, nullptr, done, 0u, g, tb, cws, oo);
    else
      launch(kernel, grid, blk, 0, s, prof, kProfCombine, g, tb, cws, oo);
  };
  if (g.dtype == 0) many ? join(k_tree_join<0, 8>) : join(k_tree_join<0, 1>);
  else many ? join(k_tree_join<1, 8>) : join(k_tree_join<1, 1>);
  e = hipGetLastError();
  if (e == hipSuccess && done && prof) e = hipEventRecord(done, s);
  return e;
}

}  // namespace bsattn
