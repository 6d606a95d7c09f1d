// bsattn_dense.hip -- attention of one new token per sequence over every
// token of its paged cache (or the last `window` ones):
//   o = sum_t p_t v_t / (sum_t p_t + exp(sink - m)),  p_t = exp(scale q.k_t - m)
// for 16-bit and affine caches.
//
// Bound by the bytes of K and V: each is read once, by one workgroup.  8
// sequences of 32k bf16 tokens, 8 kv heads (1.07 GB): 163 us with the join, 6.6
// TB/s, where a streaming read of as much takes 154; 4 of 131k int4 tokens (604
// MB) 99 us, 90 with nothing but the loads; 4 of 262k int8 tokens in 16-head
// groups (1.14 GB) 179 us, loads alone 170.
// The tokens of a (sequence, kv head) are cut into parts of `cu` units of 32
// tokens, one workgroup of four waves each, wave w taking every fourth unit of
// the part; the parts are joined by k_dense_join.  A wave works in registers
// alone, one unit at a time with MFMA 16x16x32, and asks for the next unit's K
// as soon as this one's is used, its V likewise.  Nothing may stand in front of
// those loads' waits: a block-table entry read as a vector, loads behind a
// branch, or scales that have to move between registers made every unit wait
// for all of them (131k int4 tokens: 99 us, 112 before):
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
//
// Blocks that several sequences of a call share (forks) are read once for as
// many of them as the columns hold (16 / G queries), as a job of their own
// whose partials join those of each sequence's rest.
#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "bsattn_append.h"
#include "bsattn_codes.h"
#include "bsattn_device.h"

namespace bsattn {

constexpr float kSlack = 6.0f;
constexpr float kTop = 14.0f;
constexpr float kLog2e = 1.4426950408889634f;

// What the 16 columns hold: a group of up to 8 heads of one entry; a group of
// 16, or the queries of a shared job's members; the latter where another job of
// the launch reads the same blocks.
enum Columns { kNarrow, kWide, kAgain };

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
template <int DT, Columns C>
__device__ __forceinline__ void split_operand(const float* x, float rest, u32x4& hi, u32x4& lo) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t h = cvt_pk<DT>(x[2 * j], x[2 * j + 1]);
    if constexpr (C != kNarrow) {
      hi[j] = h;
      lo[j] = cvt_pk<DT>(x[2 * j] - lo16<DT>(h), x[2 * j + 1] - hi16<DT>(h));
    } else {
      hi[j] = cvt_pk<DT>(__builtin_fmaf(-rest, lo16<DT>(h), x[2 * j]), __builtin_fmaf(-rest, hi16<DT>(h), x[2 * j + 1]));
    }
  }
}

// The same from weights that are shared out (quantized caches): x holds the
// lane's tokens, all eight, or (narrow) four of them (odd: the last four).  hi, lo
// as split_operand's.
template <Columns C, int NT>
__device__ __forceinline__ void weight_operand(const float (&x)[NT], bool odd, u32x4& hi, u32x4& lo) {
  uint32_t h[NT / 2], r[NT / 2];
#pragma unroll
  for (int j = 0; j < NT / 2; ++j) {
    h[j] = cvt_pk<0>(x[2 * j], x[2 * j + 1]);
    r[j] = cvt_pk<0>(x[2 * j] - lo16<0>(h[j]), x[2 * j + 1] - hi16<0>(h[j]));
  }
  if constexpr (C != kNarrow) {
    hi = u32x4{h[0], h[1], h[2], h[3]};
    lo = u32x4{r[0], r[1], r[2], r[3]};
  } else {
    uint32_t got[2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      got[j] = __float_as_uint(column8(__uint_as_float(odd ? h[j] : r[j])));
    hi = u32x4{odd ? got[0] : h[0], odd ? got[1] : h[1], odd ? r[0] : got[0], odd ? r[1] : got[1]};
  }
}

// The tokens of an entry's own job: [lo, len), units of 32 from u0 on.
struct DenseRange {
  int len, lo, u0, units;
};
__device__ __forceinline__ DenseRange dense_range(const Geometry& geo, const DenseBatch& db, const DenseJob& job) {
  DenseRange r;
  r.len = uniform(geo.meta[job.seq]);
  r.lo = db.window > 0 ? max(0, r.len - db.window) : 32 * job.from;
  r.u0 = r.lo >> 5;
  r.units = r.len > r.lo ? ((r.len - 1) >> 5) - r.u0 + 1 : 0;
  return r;
}

// One workgroup's part: units of a job, in the order in which its waves take
// them (wave w the places w, w + 4, ...): `full` units from fa on, whose tokens
// are all seen, then up to two at the ends of the range that are not.
struct DensePart {
  int h;                        // the kv head
  int entry, first, count, rows;  // members order[first] .. (entry: the first); their partials' first block (-1: the output itself)
  int seq, fa, full, places, head;  // head: the first of the two units (or the only one)
  DenseRange r;
  __device__ __forceinline__ int unit(int place) const {
    return place < full ? fa + place : place == full ? head : r.u0 + r.units - 1;
  }
};
__device__ __forceinline__ DensePart dense_part(const Geometry& geo, const DenseBatch& db, float* partials) {
  DensePart w;
  const int lane = threadIdx.x & 63;
  const int at = db.heads_first ? blockIdx.y : blockIdx.x;
  w.h = db.heads_first ? blockIdx.x : blockIdx.y;
  // the job whose parts hold this workgroup's
  static_assert(kMaxDenseJobs <= 128, "two jobs a lane");
  auto holds = [&](int j) { return j < db.jobs && db.job[j].part0 <= at; };
  int j = 0;
  if (db.jobs > 1) j = uniform(__popcll(__ballot(holds(lane))) + __popcll(__ballot(holds(lane + 64))) - 1);
  const DenseJob job = db.job[j];
  w.entry = job.entry;
  w.first = job.first;
  w.count = job.count;
  w.seq = job.seq;
  const int part = at - job.part0;
  const bool alone = w.count == 1;
  if (alone) w.r = dense_range(geo, db, job);
  else w.r = DenseRange{32 * job.units, 0, 0, job.units};
  // (more tokens than the launch was cut for, as when a graph replays after
  // further reservations: as many parts, of more units each)
  int cu = db.cu;
  if (alone && w.r.units > job.units) {
    const int most = max(1, (job.units + cu - 1) / cu);
    cu = max(cu, ((w.r.units + most - 1) / most + 3) & ~3);
  }
  const int parts = (w.r.units + cu - 1) / cu;
  const bool direct = alone && parts <= 1 && job.of < 0;
  w.rows = direct ? -1 : job.row0 + part * w.count;
  if (alone && part == 0 && w.h == 0 && partials && threadIdx.x == 0)
    ((DenseJoin*)partials)[w.entry] =
        DenseJoin{job.shared0, job.step, job.shared, job.row0 - job.shared, job.shared + parts};
  const int end = w.r.u0 + w.r.units;
  const int ua = w.r.u0 + part * cu, ub = min(ua + cu, end);
  const bool first = ua == w.r.u0 && 32 * ua < w.r.lo;
  const bool last = ub == end && 32 * ub > w.r.len && !(first && ub == ua + 1);
  w.places = max(ub - ua, 0);
  w.fa = ua + first;
  w.full = w.places - first - last;
  w.head = first ? ua : ub - 1;
  // (an entry of no tokens has one part, whose output is zeros)
  if (w.places == 0) w.full = direct && part == 0 ? 0 : -1;
  return w;
}

// Slabs of the units that a wave takes: the block table is read through the
// scalar cache one unit ahead (a vector load here would put its wait in front
// of the fragments on their way).
struct DensePages {
  const int32_t* bt;
  int h, sh, unit, page;  // sh: log2 of the units per block; the unit asked for last, and its page
  __device__ __forceinline__ DensePages(const Geometry& geo, const DensePart& w, int place) {
    h = w.h;
    sh = geo.tb == 64 ? 1 : 0;
    bt = block_table(geo, w.seq);
    ask(w, place);
  }
  // (places past the part's ask for its last one; a sequence without tokens for
  // its first table entry, which names some page of the pool at all times)
  __device__ __forceinline__ void ask(const DensePart& w, int place) {
    unit = w.places > 0 ? w.unit(min(place, w.places - 1)) : 0;
    page = *((const __attribute__((address_space(4))) int32_t*)(uintptr_t)(bt + (unit >> sh)));
  }
  __device__ __forceinline__ const uint8_t* slab(const Geometry& geo) const {
    return geo.pool + ((size_t)page * geo.hkv + h) * geo.slab_bytes;
  }
};

// 16 bytes at a uniform address plus a lane's offset: read once, unless another
// shared job reads them, too (8 branches of 8191 bf16 tokens, two jobs: 14.1 us
// as if read once, 12.2 so; four prompts of 16001 int8 tokens, one job each,
// with fork and append 53 us read once and 61 so, out of different caches in
// turn)
template <Columns C>
__device__ __forceinline__ u32x4 stream16(const uint8_t* base, uint32_t at) {
  if constexpr (C == kAgain) return *(const u32x4*)(base + at);
  return __builtin_nontemporal_load((const u32x4*)(base + at));
}
// a lane's offset, kept in 32 bits up to here (the load then adds it to the
// uniform address itself)
__device__ __forceinline__ uint32_t offset32(uint32_t at) {
  asm volatile("" : "+v"(at));
  return at;
}

// The four waves' shares of a part joined: this wave's o (lane (column n, group
// g), dims 16 dt + 4 g ..), sums l over its own tokens, and their reference
// (-inf: no token); written as the output (one part) or as partials (o,
// reference, l).  Column c holds head c % G of member c / G.
template <int DT, Columns C>
__device__ __forceinline__ void dense_finish(const Geometry& geo, const DenseBatch& db, const DensePart& w,
                                             const f32x4 (&o)[8], float ref, float l, uint16_t* __restrict__ out,
                                             float* __restrict__ partials) {
  __shared__ float s_m[4][16], s_l[4][16];
  __shared__ __align__(16) float s_o[4][C == kNarrow ? 8 : 16][kHeadDim + 4];
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4, G = geo.group, h = w.h;
  const int cols = G * w.count;
  l = sum_over_groups(l);
  if (n < cols) {
    if (g == 0) {
      s_m[wave][n] = ref;
      s_l[wave][n] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) *(f32x4*)&s_o[wave][n][16 * dt + 4 * g] = o[dt];
  }
  __syncthreads();
  for (int e = threadIdx.x; e < cols * kHeadDim; e += 256) {
    const int col = e >> 7, d = e & 127;
    float M = s_m[0][col];
#pragma unroll
    for (int v = 1; v < 4; ++v) M = fmaxf(M, s_m[v][col]);
    float L = 0.f, a = 0.f;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float mv = s_m[v][col];
      const float f = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - M);
      L += f * s_l[v][col];
      a += f * s_o[v][col][d];
    }
    const int member = C != kNarrow ? col / G : 0, hq = h * G + col - member * G;
    if (w.rows < 0) {
      if (db.sinks && w.r.len > 0) {
        const float sk = db.sinks[hq] * kLog2e, top = fmaxf(M, sk);
        const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
        L = L * f + (sk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sk - top));
        a *= f;
      }
      out[((size_t)w.entry * geo.hq + hq) * kHeadDim + d] = from_f32<DT>(L == 0.f ? 0.f : a / L);
    } else {
      float* pp = partials + kJoinRows * kPartial + ((size_t)(w.rows + member) * geo.hq + hq) * kPartial;
      pp[d] = a;
      if (d == 0) {
        pp[kHeadDim] = M;
        pp[kHeadDim + 1] = L;
      }
    }
  }
}

// q's row for this lane's column (columns past the members' repeat the first's)
template <Columns C>
__device__ __forceinline__ const uint16_t* dense_query(const Geometry& geo, const DenseBatch& db, const DensePart& w,
                                                       const uint16_t* __restrict__ q) {
  const int n = threadIdx.x & 15, G = geo.group;
  int bi = w.entry;
  if constexpr (C != kNarrow) {
    const int member = n / G;
    if (member > 0 && member < w.count) bi = db.order[w.first + member];
  }
  return q + ((size_t)bi * geo.hq + w.h * G + (n & (G - 1))) * kHeadDim;
}

// 16-bit caches.  grid (parts of all entries, Hkv), or the other way round
template <int DT, Columns C>
__global__ __launch_bounds__(256, 2) void k_dense(Geometry geo, DenseBatch db, const uint16_t* __restrict__ q,
                                               uint16_t* __restrict__ out, float* __restrict__ partials) {
  // P's range: fp16 weights are lifted to at most 2^14, so that small ones keep
  // their bits (bf16 has fp32's range)
  constexpr float kLift = DT == 0 ? kTop - kSlack : 0.0f;
  const DensePart w = dense_part(geo, db, partials);
  if (w.full < 0) return;  // nothing here: past the sequence's end
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  int place = wave;  // of the unit that a step takes
  DensePages pages(geo, w, place);
  u32x4 qf[4];
  {
    const uint16_t* src = dense_query<C>(geo, db, w, q) + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[s] = *(const u32x4*)(src + 32 * s);
  }
  const float rest = n >= 8 ? 1.0f : 0.0f;
  const uint32_t at = (uint32_t)lane * 16;
  u32x4 kf[8], vf[8];
  auto load_k = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const uint8_t* p = slab + geo.k_off + (u & pages.sh) * 8192;
    const uint32_t x = offset32(at);
#pragma unroll
    for (int i = 0; i < 8; ++i) kf[i] = stream16<C>(p + i * 1024, x);
  };
  auto load_v = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const uint8_t* p = slab + geo.v_off + (u & pages.sh) * 1024;
    const uint32_t x = offset32(at);
#pragma unroll
    for (int i = 0; i < 8; ++i) vf[i] = stream16<C>(p + (i << pages.sh) * 1024, x);
  };
  f32x4 o[8];
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, base = 0.0f, l = 0.0f;
  // EDGE: some of the unit's tokens are not seen.  MORE: the wave has another
  // unit, which is asked for (without a branch: behind one the compiler must
  // wait as if nothing had been)
  auto step = [&](auto edge, auto m_) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge)::value, MORE = decltype(m_)::value;
    const int next = pages.unit;
    const uint8_t* slab = pages.slab(geo);
    if constexpr (MORE) pages.ask(w, place + 8);
    __builtin_amdgcn_sched_barrier(0);
    // scores of tokens 32 u + 8 g + e, in the log2 domain; the next unit's K
    // is asked for as soon as this one's is used, its V likewise
    float pv[8];
    f32x4 acc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) acc[t] = mfma16x16x32<DT>(kf[4 * t + s], qf[s], acc[t]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_k(slab, next);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 8; ++e) pv[e] = acc[e >> 2][e & 3] * db.sl2;
    // tokens that the query does not see: no score, and nothing of what lies
    // there (old pages hold anything) reaches the products
    if constexpr (EDGE) {
      const int t0 = 32 * w.unit(place) + 8 * g;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const bool a = t0 + 2 * j >= w.r.lo && t0 + 2 * j < w.r.len;
        const bool b = t0 + 2 * j + 1 >= w.r.lo && t0 + 2 * j + 1 < w.r.len;
        if (!a) pv[2 * j] = -INFINITY;
        if (!b) pv[2 * j + 1] = -INFINITY;
        const uint32_t keep = (a ? 0x0000FFFFu : 0u) | (b ? 0xFFFF0000u : 0u);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) vf[dt][j] &= keep;
      }
    }
    float mx = pv[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) mx = fmaxf(mx, pv[e]);
    if (__any(mx > m + kSlack)) {
      const float top = fmaxf(m, max_over_groups(mx));
      const float f = top == m ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      m = top;
      base = (top == -INFINITY ? 0.0f : top) - kLift;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[dt] *= f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      pv[e] = __builtin_amdgcn_exp2f(pv[e] - base);
      l += pv[e];
    }
    u32x4 hi, lo;
    split_operand<DT, C>(pv, rest, hi, lo);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      o[dt] = mfma16x16x32<DT>(vf[dt], hi, o[dt]);
      if constexpr (C != kNarrow) o[dt] = mfma16x16x32<DT>(vf[dt], lo, o[dt]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_v(slab, next);
    __builtin_amdgcn_sched_barrier(0);
  };
  {
    // (a wave without a unit asks for the part's last one, too: behind a branch
    // the loop would wait for everything under way)
    const int u = pages.unit;
    const uint8_t* slab = pages.slab(geo);
    pages.ask(w, place + 4);
    load_k(slab, u);
    load_v(slab, u);
  }
  // (a wave's units are all full ones, but for its last)
  for (; place + 4 < w.places; place += 4) step(std::false_type(), std::true_type());
  if (place < w.full) step(std::false_type(), std::false_type());
  else if (place < w.places) step(std::true_type(), std::false_type());
  if constexpr (C == kNarrow) {
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[dt][i] += column8(o[dt][i]);
  }
  dense_finish<DT, C>(geo, db, w, o, m == -INFINITY ? m : base, l, out, partials);
}

// Affine caches of KB bits, dequantised inside the products (the codes as fp16
// operands: bsattn_codes.h).  Per group j of 64 dims and token t,
//   s_t = sum_j ks_j (sum_d q_d c_d) + kb_j Q_j,   Q_j = sum_d q_d
//   o_d = sum_t (p_t vs_j) c_td + sum_t p_t vb_j
// with the codes' offset of 1024 taken off after the first product (K: 1024 sum
// q') and by a product of the same operand with -1024 (V).  The VALU work for each code and score bounds the kernel, so
// the two copies of a narrow group's heads share the scores: columns 0-7 take
// the unit's even QK tile (tokens 8g .. 8g + 3 of lane group g), columns 8-15
// the odd one (8g + 4 .. 8g + 7), and exchange what PV needs of the other: the
// rounded weights go to columns 0-7, what the rounding left to 8-15.  sum p vb
// stays fp32 and per lane until the end.
// grid as k_dense's
template <int KB, Columns C>
__global__ __launch_bounds__(256, 2) void k_dense_q(Geometry geo, DenseBatch db, const uint16_t* __restrict__ q,
                                                 uint16_t* __restrict__ out, float* __restrict__ partials) {
  constexpr int NK = 2 * QCode<KB>::KF, NV = 8 / QCode<KB>::DPF;  // K and V fragments of a unit
  constexpr int NT = C == kNarrow ? 4 : 8;                              // tokens of a unit whose scores a lane holds
  const DensePart w = dense_part(geo, db, partials);
  if (w.full < 0) return;  // nothing here: past the sequence's end
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n = lane & 15, g = lane >> 4;
  const bool odd = C == kNarrow && n >= 8;
  const int tok0 = 8 * g + (odd ? 4 : 0);
  int place = wave;  // of the unit that a step takes
  DensePages pages(geo, w, place);
  u32x4 qf[4];
  {
    const uint16_t* src = dense_query<C>(geo, db, w, q) + 8 * g;
#pragma unroll
    for (int s = 0; s < 4; ++s) qf[s] = *(const u32x4*)(src + 32 * s);
  }
  const uint32_t code_base = f16_pair_1024();
  const uint32_t at = (uint32_t)lane * 16;
  // scales and biases: a lane loads one token's (token lane & 31 of the unit, in
  // the slab's order), and reads the NT of its scores through LDS
  __shared__ u32x4 s_sb[4][32];
  const uint32_t sb_at = 16u * (uint32_t)(((lane >> 3) & 3) * (geo.tb >> 2) + (lane & 7));
  u32x4 kf[NK], vf[NV], sbx;
  auto load_k = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const uint8_t* p = slab + geo.k_off + (u & pages.sh) * (NK * 1024);
    const uint32_t x = offset32(at);
#pragma unroll
    for (int i = 0; i < NK; ++i) kf[i] = stream16<C>(p + i * 1024, x);
  };
  auto load_v = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    const uint8_t* p = slab + geo.v_off + (u & pages.sh) * 1024;
    const uint32_t x = offset32(at);
#pragma unroll
    for (int i = 0; i < NV; ++i) vf[i] = stream16<C>(p + (i << pages.sh) * 1024, x);
  };
  auto load_sb = [&](const uint8_t* slab, int u) __attribute__((always_inline)) {
    sbx = stream16<C>(slab + geo.sb_off + (u & pages.sh) * 128, offset32(sb_at));
  };

  // the queries' sums over each 64 dims: of q, and of the QK operand (int4:
  // with its unit-16 elements scaled) times 1024
  u32x4 qk[4];
  float q0, q1, q0c, q1c;
  {
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
    q0c = mfma_f16(ones, qk[1], mfma_f16(ones, qk[0], zero))[0] * kDecOff;
    q1c = mfma_f16(ones, qk[3], mfma_f16(ones, qk[2], zero))[0] * kDecOff;
    q0 = mfma_f16(ones, qf[1], mfma_f16(ones, qf[0], zero))[0];
    q1 = mfma_f16(ones, qf[3], mfma_f16(ones, qf[2], zero))[0];
  }

  f32x4 o[8];
#pragma unroll
  for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  // P's range: lifted to at most 2^14 as for fp16 caches.  A weight also meets
  // its token's scale; in units where a product would pass 2^15 the scales of
  // that half of the dims are lowered by as much, and its sums with them, so
  // that the other tokens' weights keep their bits (all weights at most 1 from
  // the first scale of 2 on, whatever its own weight, put them among fp16's
  // subnormals: outputs were off by 8 half steps of fp16 at their root mean
  // square where one token in 32 had such a scale and e^-12 of the largest
  // weight).  Done with the raise
  // of the reference, behind one branch: 4 x 131k int4 tokens 99.6 us (99.0
  // before); with scales of 10 everywhere 117 (115), on one token in 32 108 (103).
  constexpr float kLift = kTop - kSlack;
  float m = -INFINITY, base = 0.0f, limit = -INFINITY, l = 0.0f, ob0 = 0.0f, ob1 = 0.0f;
  uint32_t lower = 0x3C003C00u;  // what the scales of dims 0-63 and 64-127 are multiplied by (fp16)
  // 1 / x of a power of two
  auto inverse = [](float x) { return __uint_as_float(0x7F000000u - __float_as_uint(x)); };

  // EDGE: some of the unit's tokens are not seen.  MORE: the wave has another
  // unit, which is asked for (without a branch: behind one the compiler must
  // wait as if nothing had been)
  auto step = [&](auto edge, auto m_) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge)::value, MORE = decltype(m_)::value;
    const int next = pages.unit;
    const uint8_t* slab = pages.slab(geo);
    if constexpr (MORE) pages.ask(w, place + 8);
    __builtin_amdgcn_sched_barrier(0);
    f32x4 r0[2], r1[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const u32x4* kt = kf + t * QCode<KB>::KF;
      r0[t] = mfma_f16(k_operand<KB>(kt, 0, code_base), qk[0], f32x4{0.f, 0.f, 0.f, 0.f});
      r1[t] = mfma_f16(k_operand<KB>(kt, 2, code_base), qk[2], f32x4{0.f, 0.f, 0.f, 0.f});
      r0[t] = mfma_f16(k_operand<KB>(kt, 1, code_base), qk[1], r0[t]);
      r1[t] = mfma_f16(k_operand<KB>(kt, 3, code_base), qk[3], r1[t]);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_k(slab, next);
    __builtin_amdgcn_sched_barrier(0);
    s_sb[wave][lane & 31] = sbx;
    wave_lds_order();
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_sb(slab, next);
    __builtin_amdgcn_sched_barrier(0);
    u32x4 sb[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) sb[i] = s_sb[wave][8 * g + (odd ? 4 : 0) + i];
    // scores over the reference, in the log2 domain
    float pv[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float a = (C != kNarrow ? r0[i >> 2][i & 3] : odd ? r0[1][i] : r0[0][i]) - q0c;
      const float b = (C != kNarrow ? r1[i >> 2][i & 3] : odd ? r1[1][i] : r1[0][i]) - q1c;
      float x = lo_f(sb[i][0]) * a;
      x = __builtin_fmaf(hi_f(sb[i][0]), b, x);
      x = __builtin_fmaf(lo_f(sb[i][1]), q0, x);
      x = __builtin_fmaf(hi_f(sb[i][1]), q1, x);
      pv[i] = __builtin_fmaf(x, db.sl2, -base);
    }
    // tokens that the query does not see: no score, and nothing of what lies
    // there (old pages hold anything) reaches the products
    if constexpr (EDGE) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int t = 32 * w.unit(place) + tok0 + i;
        if (t < w.r.lo || t >= w.r.len) {
          pv[i] = -INFINITY;
          sb[i][2] = sb[i][3] = 0u;
        }
      }
    }
    float mx = pv[0];
    uint32_t scales = sb[0][2];
#pragma unroll
    for (int i = 1; i < NT; ++i) {
      mx = fmaxf(mx, pv[i]);
      scales |= sb[i][2];
    }
    // (weights are at most 2^14: only a scale of 2 or more can pass 2^15; then
    // the largest weight and scale say whether one does)
    bool move = mx > limit || lower != 0x3C003C00u;
    if (__any((scales & 0x40004000u) != 0)) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) most = fmaxf(most, fmaxf(fabsf(lo_f(sb[i][2])), fabsf(hi_f(sb[i][2]))));
      move = move || most * __builtin_amdgcn_exp2f(mx) >= 32768.0f;
    }
    if (__any(move)) {
      if constexpr (C == kNarrow) mx = fmaxf(mx, column8(mx));
      const float top = fmaxf(m, base + max_over_groups(mx)), was = base;
      const float f = top == m ? 1.0f : __builtin_amdgcn_exp2f(m - top);
      base = (top == -INFINITY ? 0.0f : top) - kLift;
      limit = top == -INFINITY ? top : kTop;
      m = top;
      l *= f;
      ob0 *= f;
      ob1 *= f;
      float w0 = 0.f, w1 = 0.f;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        pv[i] += was - base;
        float p = pv[i];
        asm volatile("" : "+v"(p));  // (not taken out of here to be shared with the weights below)
        p = __builtin_amdgcn_exp2f(p);
        w0 = fmaxf(w0, fabsf(lo_f(sb[i][2])) * p);
        w1 = fmaxf(w1, fabsf(hi_f(sb[i][2])) * p);
      }
      if constexpr (C == kNarrow) {
        w0 = fmaxf(w0, column8(w0));
        w1 = fmaxf(w1, column8(w1));
      }
      // 2^(14 - e) for products of 2^e and more, e >= 15 (at most 2^14 * 65504)
      auto factor = [](float x) {
        return x < 32768.0f ? 1.0f : __uint_as_float((268u - min(__float_as_uint(x) >> 23, 157u)) << 23);
      };
      w0 = factor(max_over_groups(w0));
      w1 = factor(max_over_groups(w1));
      const float f0 = f * w0 * inverse(lo_f(lower)), f1 = f * w1 * inverse(hi_f(lower));
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) o[dt] *= dt < 4 ? f0 : f1;
      lower = cvt_pk<0>(w0, w1);
#pragma unroll
      for (int i = 0; i < NT; ++i) sb[i][2] = f16x2_mul(sb[i][2], lower);
    }
    float p0[NT], p1[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const float p = __builtin_amdgcn_exp2f(pv[i]);
      l += p;
      ob0 = __builtin_fmaf(lo_f(sb[i][3]), p, ob0);
      ob1 = __builtin_fmaf(hi_f(sb[i][3]), p, ob1);
      const float x = KB == 4 && (i & 2) ? p * kUnit16 : p;  // int4's unit-16 elements
      p0[i] = lo_f(sb[i][2]) * x;
      p1[i] = hi_f(sb[i][2]) * x;
    }
    const u32x4 off = u32x4{0xE400E400u, 0xE400E400u, 0xE400E400u, 0xE400E400u};  // -1024
    u32x4 h0, l0, h1, l1;
    weight_operand<C>(p0, odd, h0, l0);
    weight_operand<C>(p1, odd, h1, l1);
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) {
      const u32x4 a = v_operand<KB, 1>(vf, dt, 0, code_base);
      const u32x4& ph = dt < 4 ? h0 : h1;
      o[dt] = mfma_f16(off, ph, o[dt]);
      o[dt] = mfma_f16(a, ph, o[dt]);
      if constexpr (C != kNarrow) {
        const u32x4& pl = dt < 4 ? l0 : l1;
        o[dt] = mfma_f16(off, pl, o[dt]);
        o[dt] = mfma_f16(a, pl, o[dt]);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (MORE) load_v(slab, next);
    __builtin_amdgcn_sched_barrier(0);
  };
  {
    // (a wave without a unit asks for the part's last one, too: behind a branch
    // the loop would wait for everything under way)
    const int u = pages.unit;
    const uint8_t* slab = pages.slab(geo);
    pages.ask(w, place + 4);
    load_k(slab, u);
    load_sb(slab, u);
    load_v(slab, u);
  }
  // (a wave's units are all full ones, but for its last)
  for (; place + 4 < w.places; place += 4) step(std::false_type(), std::true_type());
  if (place < w.full) step(std::false_type(), std::false_type());
  else if (place < w.places) step(std::true_type(), std::false_type());
  ob0 = sum_over_groups(ob0);
  ob1 = sum_over_groups(ob1);
  if constexpr (C == kNarrow) {
    ob0 += column8(ob0);
    ob1 += column8(ob1);
    l += column8(l);
  }
  const float f0 = inverse(lo_f(lower)), f1 = inverse(hi_f(lower));
#pragma unroll
  for (int dt = 0; dt < 8; ++dt)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (C == kNarrow) o[dt][i] += column8(o[dt][i]);
      o[dt][i] = __builtin_fmaf(o[dt][i], dt < 4 ? f0 : f1, dt < 4 ? ob0 : ob1);
    }
  dense_finish<0, C>(geo, db, w, o, m == -INFINITY ? m : base, l, out, partials);
}

// The parts of one (entry, query head) joined, those of its shared job first:
// rows of 32 lanes with four dims each take the parts in turn, four of them
// asked for at once, and are summed in order at the end.  (Joined by the
// workgroup that arrives last, with device-scope partials, one sequence of 4k
// tokens takes 11.5 us, against 5.1 and 3.3 for the two launches.)  grid (Hq, n)
constexpr int kRows = 8, kRound = 4;
template <int DT>
__global__ __launch_bounds__(32 * kRows) void k_dense_join(const float* __restrict__ ws,
                                                           const float* __restrict__ sinks,
                                                           uint16_t* __restrict__ out) {
  __shared__ __align__(16) float s_o[kRows][kHeadDim];
  __shared__ float s_ml[kRows][2];
  const int hq = blockIdx.x, hqs = gridDim.x, bi = blockIdx.y;
  const int row = threadIdx.x >> 5, c = threadIdx.x & 31;
  const DenseJoin at = ((const DenseJoin*)ws)[bi];
  const float* partials = ws + kJoinRows * kPartial;
  if (at.parts <= 1 && at.shared == 0) return;  // (the launch before wrote the output)
  float M = -INFINITY, L = 0.f;
  f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int p0 = row; p0 < at.parts; p0 += kRows * kRound) {
    f32x4 x[kRound];
    float m[kRound], l[kRound];
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      const int p = min(p0 + j * kRows, at.parts - 1);
      const int block = p < at.shared ? at.shared0 + p * at.step : at.own0 + p;
      const float2* part = (const float2*)(partials + ((size_t)block * hqs + hq) * kPartial);
      const float2 xa = part[2 * c], xb = part[2 * c + 1], ml = part[kHeadDim / 2];
      x[j] = f32x4{xa.x, xa.y, xb.x, xb.y};
      m[j] = p0 + j * kRows < at.parts ? ml.x : -INFINITY;
      l[j] = ml.y;
    }
    float top = M;
#pragma unroll
    for (int j = 0; j < kRound; ++j) top = fmaxf(top, m[j]);
    const float f = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - top);
    L *= f;
    a *= f;
#pragma unroll
    for (int j = 0; j < kRound; ++j) {
      const float g = m[j] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[j] - top);
      L += g * l[j];
      if (m[j] != -INFINITY) a += g * x[j];
    }
    M = top;
  }
  *(f32x4*)&s_o[row][4 * c] = a;
  if (c == 0) {
    s_ml[row][0] = M;
    s_ml[row][1] = L;
  }
  __syncthreads();
  if (threadIdx.x >= kHeadDim) return;
  const int d = threadIdx.x;
  const float sk = sinks ? sinks[hq] * kLog2e : -INFINITY;
  float top = sk;
#pragma unroll
  for (int i = 0; i < kRows; ++i) top = fmaxf(top, s_ml[i][0]);
  float Ls = sk == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sk - top), as = 0.f;
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const float mi = s_ml[i][0];
    const float f = mi == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mi - top);
    Ls += f * s_ml[i][1];
    if (mi != -INFINITY) as += f * s_o[i][d];
  }
  out[((size_t)bi * hqs + hq) * kHeadDim + d] = from_f32<DT>(Ls == 0.f ? 0.f : as / Ls);
}

template <Columns C>
static void dense_dispatch(const Geometry& g, const DenseBatch& db, dim3 grid, const uint16_t* q, uint16_t* out,
                           float* ws, hipStream_t s, Timing* prof) {
  const dim3 blk(256);
  const int kd = kProfDense;
  if (g.kv_bits == 4) launch(k_dense_q<4, C>, grid, blk, 0, s, prof, kd, g, db, q, out, ws);
  else if (g.kv_bits == 8) launch(k_dense_q<8, C>, grid, blk, 0, s, prof, kd, g, db, q, out, ws);
  else if (g.dtype == 0) launch(k_dense<0, C>, grid, blk, 0, s, prof, kd, g, db, q, out, ws);
  else launch(k_dense<1, C>, grid, blk, 0, s, prof, kd, g, db, q, out, ws);
}

template <int DT>
static hipError_t join_dispatch(const Geometry& g, const DenseBatch& db, const float* ws, uint16_t* out,
                                hipEvent_t done, hipStream_t s, Timing* prof) {
  const dim3 grid(g.hq, db.n), blk(32 * kRows);
  if (done && !prof)  // (the event is the dispatch's own: no packet of its own behind it)
    hipExtLaunchKernelGGL(k_dense_join<DT>, grid, blk, 0u, s, nullptr, done, 0u, ws, db.sinks, out);
  else
    launch(k_dense_join<DT>, grid, blk, 0, s, prof, kProfCombine, ws, db.sinks, out);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && done && prof) e = hipEventRecord(done, s);
  return e;
}

static_assert(sizeof(Geometry) + sizeof(DenseBatch) <= 4000, "a launch's arguments stay under 4 KiB");
hipError_t launch_dense(const Geometry& g, const DenseBatch& db, int parts, const void* q, void* out, float* ws,
                        hipEvent_t done, hipStream_t s, Timing* prof) {
  const dim3 grid = db.heads_first ? dim3(g.hkv, parts) : dim3(parts, g.hkv);
  const uint16_t* qq = (const uint16_t*)q;
  uint16_t* oo = (uint16_t*)out;
  const bool wide = g.group > 8 || db.job[0].count > 1;  // (shared jobs come first)
  if (db.again) dense_dispatch<kAgain>(g, db, grid, qq, oo, ws, s, prof);
  else if (wide) dense_dispatch<kWide>(g, db, grid, qq, oo, ws, s, prof);
  else dense_dispatch<kNarrow>(g, db, grid, qq, oo, ws, s, prof);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !ws) return e;
  return g.dtype == 0 ? join_dispatch<0>(g, db, ws, oo, done, s, prof) : join_dispatch<1>(g, db, ws, oo, done, s, prof);
}

}  // namespace bsattn
