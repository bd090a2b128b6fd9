// Losses on logits: token log-probabilities (forward and backward), the clipped policy loss with a KL term and the paired
// preference loss, each with its gradient in the logits. Loops like the reference's train on them (mote/train/dpo.py:217,
// kto.py:151, rlvr.py:308: clip and AdamW after such a loss).
//
// Per row (one position) with logits z, temperature T, x = z / T and target y:
//   logp = x_y - lse(x),  dlogp/dz_j = ([j == y] - exp(x_j - lse)) / T
// The target's column is kept out of the sum: with m the largest of the OTHER logits, ref(m) = m / T to a whole power of two
// (see Ex), s = sum_{j != y} exp(x_j - ref(m)) and a = x_y - ref(m),
//   a >= 0: logp = -log1p(s e^-a)          1 - p_y = X / (1 + X), X = s e^-a
//   a <  0: logp = a - log1p(s - 1 + e^a)  1 - p_y = s / (s + e^a)
// so that neither logp nor 1 - p_y cancels where the model is sure of its target (p_y -> 1). The exponentials and their sums
// are fp32, a position's logp is kept in 64 bits, and the sums over positions are in 64 bits.
//
// By their bytes all kernels are memory-bound (2 or 4 read per logit, as many written for a gradient); the exponential is next:
// one ex2 per logit at 16 per clock and SM takes 0.73 of the time in which the copy bandwidth reads a bf16 logit. Only the stream
// and the gradient of long rows come near either.
#pragma once

#include <cfloat>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <type_traits>

#include "mt_types.h"
#include "ptx.cuh"

namespace moteopt {
namespace loss {

constexpr float kNegInf = -INFINITY;
constexpr double kLog2e = 1.4426950408889634074;
// ex2.approx's mean relative error below -1 is -5.05e-8, the same for every binade (measured over 4e6 arguments each). A
// sequence would add up thousands of them.
constexpr float kEx2Bias = 5.05e-8f;
constexpr double kLn2 = 0.69314718055994530942;

// logits [seqs][tokens][vocab], the last axis contiguous, and the targets [seqs][tokens]
struct Rows {
  const char* z;
  const int64_t* y;
  int64_t z_seq, z_tok;   // strides in elements
  int64_t y_seq, y_tok;
  uint32_t n;             // rows: seqs * tokens, below 2^27
  uint32_t tokens;
  uint32_t vocab;
  const int32_t* cu;      // packed: n_seqs + 1 row offsets, or null. Rows outside [cu[0], cu[n_seqs]) do not count
  int n_seqs;
  float c_hi, c_lo;       // log2(e) / T as two floats, c_lo > 0 (see Ex)
  double t, inv_t;        // T and 1 / T
};

struct Per {              // fp32 values per position, broadcast where a stride is 0
  const float* p;
  int64_t seq, tok;
  __device__ float at(uint32_t s, uint32_t t) const { return p[s * seq + t * tok]; }
};

struct Policy {
  Per adv, old_lp, ref_lp, weight;   // ref_lp.p, weight.p may be null
  double clip_lo, clip_hi, kl;       // 1 - low, 1 + high, the KL term's coefficient
  double inv_div;                    // 1 / divisor where it is a host number
  const float* div;                  // or the divisor on the device
};

__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
// Two fp32 values in one register pair, and a multiply-add of both at once
using F2 = uint64_t;
__device__ __forceinline__ F2 pack2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(F2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 fma2(F2 x, F2 y, F2 z) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
  return r;
}

// The exponentials of a row about a logit m, with c = c_hi + c_lo = log2(e) / T: 2^(z c - b) 2^16 is exp(z / T - ref(m)), where
// ref(m) is m / T rounded to a whole power of two, base(m) = rint(m c). Sums about different m then differ by powers of two,
// exactly. c_hi has 12 bits, so that what the first multiply-add leaves to the second is not lost under half a unit of its
// result (with one float for c, or a full one for c_hi, its rounding leans every exponent of a row the same way: 5e-8 of a sum,
// and the sums of thousands of positions keep it). b is base + 16: ex2 is asked for values below -1 only, where its relative
// error has the mean of -5.05e-8 that row_stat takes out. So exponents are rounded between 16 and 32, twice, by 2^-20 at most: an
// exponential is off by up to 1.3e-6, mostly by 2e-7. c_lo > 0 keeps -inf a -inf.
//
// Where |m c| >= 2^18 (a far m: a mask of -1e9, say), ref(m) is m / T itself and m is taken from z first: the difference is
// exact where its exponential is not 0, and b is kAbove alone. A product with m there would leave half a unit of m c, which is
// 128 from 2^32 on. Loops over a row branch once (two<true>): the subtraction in all rows would be one of five instructions.
constexpr float kAbove = 16.f, kFix = 65536.f;   // 2^kAbove
struct Base {
  float b;     // rint(m c)
  bool near;
  __device__ Base(float m, const Rows& R) {
    const float p = fmaf(m, R.c_hi, m * R.c_lo);
    b = rintf(p);
    near = fabsf(p) < 0x1p18f;   // not of infinities and NaN
  }
};
__device__ __forceinline__ double ref_of(float m, const Rows& R) {
  const Base b(m, R);
  return b.near ? b.b * kLn2 : m * R.inv_t;
}
struct Ex {
  F2 hi, lo, nb;
  float sub;   // a far m, else 0
  __device__ Ex(float m, const Rows& R, float up = 0.f) {   // up: a power of two that the values carry (policy_row)
    if (m == kNegInf) m = 0.f;
    const Base base(m, R);
    sub = base.near ? 0.f : m;
    const float b = (base.near ? base.b : 0.f) + kAbove - up;
    hi = pack2(R.c_hi, R.c_hi);
    lo = pack2(R.c_lo, R.c_lo);
    nb = pack2(-b, -b);
  }
  __device__ __forceinline__ bool far() const { return sub != 0.f; }
  template <bool kFar>
  __device__ __forceinline__ void two(F2 z, float& e0, float& e1) const {
    float t0, t1;
    if (kFar) z = fma2(z, pack2(1.f, 1.f), pack2(-sub, -sub));
    unpack2(fma2(z, lo, fma2(z, hi, nb)), t0, t1);
    e0 = ex2(t0);
    e1 = ex2(t1);
  }
  template <bool kFar>
  __device__ __forceinline__ float sum(F2 z) const {
    float e0, e1;
    two<kFar>(z, e0, e1);
    return e0 + e1;
  }
  __device__ __forceinline__ float one(float z) const {   // of any row
    float e0, e1;
    z -= sub;
    two<false>(pack2(z, z), e0, e1);
    return e0;
  }
};
// exp(ref(m) - ref(to)), the factor of a partial sum that moves from m to a larger logit
__device__ __forceinline__ float rescale(float m, float to, const Rows& R) {
  if (m == kNegInf) return 0.f;
  const Base a(m, R), b(to, R);
  if (a.near && b.near) return __int_as_float((static_cast<int>(fmaxf(a.b - b.b, -126.f)) + 127) << 23);
  return expf(static_cast<float>(ref_of(m, R) - ref_of(to, R)));
}

__device__ __forceinline__ float lo_bf16(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float hi_bf16(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t to_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
constexpr uint32_t kNegInf2 = 0xff80ff80u;   // two bf16 -inf

// A 32-bit word of logits: two bf16 or one fp32
template <typename T>
struct Word;
template <>
struct Word<__nv_bfloat16> {
  static constexpr int kPer = 2;
  static constexpr uint32_t kEmpty = kNegInf2;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return max_bf16x2(a, b); }
  static __device__ __forceinline__ float top(uint32_t w) { return fmaxf(lo_bf16(w), hi_bf16(w)); }
  static __device__ __forceinline__ uint32_t drop(uint32_t w, uint32_t at) {   // -inf in place of element `at`
    return at ? (w & 0xffffu) | 0xff800000u : (w & 0xffff0000u) | 0xff80u;
  }
};
template <>
struct Word<float> {
  static constexpr int kPer = 1;
  static constexpr uint32_t kEmpty = 0xff800000u;
  static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }
  static __device__ __forceinline__ float top(uint32_t w) { return __uint_as_float(w); }
  static __device__ __forceinline__ uint32_t drop(uint32_t, uint32_t) { return 0xff800000u; }
};

__device__ __forceinline__ float load_one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ float warp_max(float v) {   // NaN is left out: the exponentials carry it
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Programmatic dependent launch: `pdl_wait` returns when the launch before this one has ended and its writes are visible
// (at once where the launch has no such attribute), `pdl_go` lets the next launch's blocks be placed early.
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_go() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// A line's 16 bytes as pairs of fp32: 4 of bf16, 2 of fp32. A line's exponentials are added up before they join a lane's sum:
// bf16 logits take few values, so the roundings of a long chain of sums lean (20000 of them: 2e-8 of the sum).
template <typename T>
struct Pairs;
template <>
struct Pairs<__nv_bfloat16> {
  static constexpr int kN = 4;
  F2 p[4];
  __device__ __forceinline__ explicit Pairs(const uint4& v)
      : p{pack2(lo_bf16(v.x), hi_bf16(v.x)), pack2(lo_bf16(v.y), hi_bf16(v.y)), pack2(lo_bf16(v.z), hi_bf16(v.z)),
          pack2(lo_bf16(v.w), hi_bf16(v.w))} {}
  template <bool kFar>
  __device__ __forceinline__ float sum(const Ex& ex) const {
    return (ex.sum<kFar>(p[0]) + ex.sum<kFar>(p[1])) + (ex.sum<kFar>(p[2]) + ex.sum<kFar>(p[3]));
  }
  template <bool kFar>
  __device__ __forceinline__ uint4 scaled(const Ex& ex, float f) const {   // f exp, rounded once
    float a[8];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      ex.two<kFar>(p[u], a[2 * u], a[2 * u + 1]);
      a[2 * u] *= f;
      a[2 * u + 1] *= f;
    }
    return make_uint4(to_bf16x2(a[0], a[1]), to_bf16x2(a[2], a[3]), to_bf16x2(a[4], a[5]), to_bf16x2(a[6], a[7]));
  }
};
template <>
struct Pairs<float> {
  static constexpr int kN = 2;
  F2 p[2];
  __device__ __forceinline__ explicit Pairs(const uint4& v)
      : p{pack2(bits(v.x), bits(v.y)), pack2(bits(v.z), bits(v.w))} {}
  static __device__ __forceinline__ float bits(uint32_t w) { return __uint_as_float(w); }
  template <bool kFar>
  __device__ __forceinline__ float sum(const Ex& ex) const {
    return ex.sum<kFar>(p[0]) + ex.sum<kFar>(p[1]);
  }
  template <bool kFar>
  __device__ __forceinline__ uint4 scaled(const Ex& ex, float f) const {
    float a[4];
    ex.two<kFar>(p[0], a[0], a[1]);
    ex.two<kFar>(p[1], a[2], a[3]);
    return make_uint4(__float_as_uint(a[0] * f), __float_as_uint(a[1] * f), __float_as_uint(a[2] * f), __float_as_uint(a[3] * f));
  }
};

// (largest logit m, sum of exp(x - ref(m))) of a part of a row. Written to other blocks' shared memory as one value of 8 bytes
// (store_remote).
struct alignas(8) Part {
  float m, s;
};
__device__ __forceinline__ Part warp_join(Part p, const Rows& R) {
  const float M = warp_max(p.m);
  return Part{M, warp_sum(p.s == 0.f ? 0.f : p.s * rescale(p.m, M, R))};
}

// What a row's sums give (see the top of this file). The differences and the results are in 64 bits; exp, the logarithm and
// the quotient between them are fp32 functions, which keep 6e-8 of values of at most 1 in size: log(1 + X) is k log 2 +
// log(f) + c with 1 + X = 2^k f, 3/4 <= f < 3/2, and c what the fp32 sum 1 + X lost. In 64 bits throughout, these functions
// took a lane 1500 cycles and as many instructions as the row itself.
struct RowStat {
  double logp, lse;
  float f;      // exp(ref(m) - lse): p_j = exp(x_j - ref(m)) f
  float rest;   // 1 - p_y
};
__device__ __forceinline__ RowStat row_stat(float zy, float m, float s, const Rows& R) {
  const double x = zy * R.inv_t, ref = ref_of(m, R), a = x - ref;
  const bool up = a >= 0.0;
  const float q = expf(static_cast<float>(up ? -a : a));
  const float X = up ? (s == 0.f ? 0.f : s * q) : (s - 1.f) + q;
  const float u = 1.f + X, inv = 1.f / u;
  const int k = (__float_as_int(u) - 0x3f400000) >> 23;
  const float f = __int_as_float(__float_as_int(u) - (k << 23));
  const float bias = kEx2Bias * s * (up ? q : 1.f) * inv;   // ex2's, in the others' share of the whole sum
  double l = k * kLn2 + static_cast<double>(logf(f) + (X - (u - 1.f)) * inv + bias);
  if (X != X) l = static_cast<double>(X);
  RowStat r;
  r.logp = up ? -l : a - l;
  r.lse = (up ? x : ref) + l;
  r.f = (up ? q : 1.f) * inv;
  r.rest = (up ? X : s) * inv;
  if (zy == INFINITY) r.logp = r.lse = static_cast<double>(r.f = r.rest = NAN);   // inf - inf
  return r;
}

// The policy loss of one row, unscaled by the weight and the divisor. The ratio is an fp32 exponential of a 64-bit
// difference, and taken in 64 bits where it lies within 1e-5 of a border, at which the gradient jumps, and beyond e^80, where
// fp32 ends: an advantage or a weight may bring what it gives back into range. A ratio of a finite difference stays finite, so
// that an advantage of 0 makes it 0. k(d) = e^d - d - 1 is its series below 1 in size (the difference would cancel):
// 2 / (n + 2)! falls below 2^-24 at n = 9.
constexpr double kFarLog = 80.0;
struct RowLoss {
  double loss, kl, slope;   // slope: dloss/dlogp
  bool clipped;
};
__device__ __forceinline__ RowLoss policy_row_loss(double logp, const Policy& P, float old_lp, float ref_lp, bool has_ref,
                                                   float adv) {
  const double A = adv, d_old = logp - static_cast<double>(old_lp);
  double r = expf(static_cast<float>(d_old));
  if (d_old > kFarLog || fabs(r - P.clip_hi) < 1e-5 * P.clip_hi || fabs(r - P.clip_lo) < 1e-5 * P.clip_lo) {
    r = exp(d_old);
    if (d_old < INFINITY) r = fmin(r, DBL_MAX);
  }
  const double held_r = fmin(fmax(r, P.clip_lo), P.clip_hi);
  const double free = r * A, held = (r != r ? r : held_r) * A;
  RowLoss L;
  L.clipped = held < free;
  L.loss = L.clipped ? -held : -free;
  L.slope = L.clipped ? 0.0 : -free;
  L.kl = 0.0;
  if (has_ref) {
    const double far = static_cast<double>(ref_lp) - logp;
    double e;
    if (far > kFarLog) {   // the 1 is below 64 bits
      e = exp(far);
      L.kl = e - far;
    } else {
      const float d = static_cast<float>(far), m1 = expm1f(d);
      float k = m1 - d;
      if (fabsf(d) < 1.f) {
        k = 1.f / 11.f;
#pragma unroll
        for (int n = 10; n >= 3; --n) k = fmaf(k, d, 1.f) * (1.f / n);
        k = fmaf(k, d, 1.f) * (0.5f * d * d);
      }
      L.kl = k;
      e = m1;
    }
    if (P.kl != 0.0) {
      L.loss += P.kl * L.kl;
      L.slope -= P.kl * e;
    }
  }
  return L;
}

// The policy loss of a row: its sums' terms, and its gradient's factors: 2^up f exp(x_j - ref(m)), gy at the target. A slope
// beyond 2^96 stays in 64 bits to the factors, and what is left above 2^64 goes into the exponents (Ex): products with small
// probabilities are finite then, and those with a probability of 0 (one below 2^-126 counts as 0) are 0.
struct PolicyRow {
  double part[4];
  float f, gy, up;
};
__device__ __forceinline__ PolicyRow policy_row(const Policy& P, const RowStat& st, float wt, float adv, float old_lp,
                                                float ref_lp, double inv_t) {
  const RowLoss L = policy_row_loss(st.logp, P, old_lp, ref_lp, P.ref_lp.p != nullptr, adv);
  const double w = wt, inv = P.div ? 1.0 / static_cast<double>(*P.div) : P.inv_div, slope = w * L.slope * inv * inv_t;
  const float g = static_cast<float>(slope);
  PolicyRow r = {{w * L.loss * inv, w, w * L.kl * inv, L.clipped ? w : 0.0}, -g * st.f, g * st.rest, 0.f};
  if (fabsf(g) >= 0x1p96f) {   // not of NaN
    const double h = fmin(fmax(slope, -0x1p1020), 0x1p1020);
    double f = -h * st.f;
    while (fabs(f) >= 0x1p64) {
      f *= 0x1p-64;
      r.up += 64.f;
    }
    r.f = static_cast<float>(f);
    r.gy = static_cast<float>(h * st.rest);
  }
  return r;
}

__device__ __forceinline__ bool in_packed(const Rows& R, uint32_t row) {
  if (R.cu == nullptr) return true;
  return static_cast<int64_t>(row) >= R.cu[0] && static_cast<int64_t>(row) < R.cu[R.n_seqs];
}

// ---------------------------------------------------------------------------------------------------------------------
// A row in vectors of 16 bytes: `head` elements up to the first aligned one, then `vecs` vectors, then `tail` elements
template <typename T>
struct Split {
  static constexpr uint32_t kPer = 16 / sizeof(T);
  uint32_t head, vecs, tail;
  __device__ Split(const T* p, uint32_t vocab) {
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uint64_t>(p) & 15) / sizeof(T);
    head = min(off ? kPer - off : 0u, vocab);
    vecs = (vocab - head) / kPer;
    tail = vocab - head - vecs * kPer;
  }
  // element of the edge thread `i` < head + tail
  __device__ uint32_t edge(uint32_t i) const { return i < head ? i : vecs * kPer + i; }
};
__device__ __forceinline__ uint4 load_vec(const void* p) {
  uint4 v;
  asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
template <typename T>
__device__ __forceinline__ void drop_target(uint4& v, uint32_t at) {   // element `at` of the vector
  const uint32_t w = at / Word<T>::kPer, h = at % Word<T>::kPer;
  if (w == 0) v.x = Word<T>::drop(v.x, h);
  if (w == 1) v.y = Word<T>::drop(v.y, h);
  if (w == 2) v.z = Word<T>::drop(v.z, h);
  if (w == 3) v.w = Word<T>::drop(v.w, h);
}
template <typename T>
__device__ __forceinline__ uint32_t vec_max(uint32_t top, const uint4& v) {
  using W = Word<T>;
  return W::max(W::max(W::max(top, v.x), W::max(v.y, v.z)), v.w);
}

// kBehind[i]: the bytes of a line behind its first 2 i, as masks of its words
__constant__ const uint4 kBehind[9] = {
    {0xffffffffu, 0xffffffffu, 0xffffffffu, 0xffffffffu}, {0xffff0000u, 0xffffffffu, 0xffffffffu, 0xffffffffu},
    {0u, 0xffffffffu, 0xffffffffu, 0xffffffffu},          {0u, 0xffff0000u, 0xffffffffu, 0xffffffffu},
    {0u, 0u, 0xffffffffu, 0xffffffffu},                   {0u, 0u, 0xffff0000u, 0xffffffffu},
    {0u, 0u, 0u, 0xffffffffu},                            {0u, 0u, 0u, 0xffff0000u},
    {0u, 0u, 0u, 0u}};
template <typename T>
__device__ __forceinline__ uint4 behind(uint32_t elems) {
  return kBehind[elems * (sizeof(T) / 2)];
}
__device__ __forceinline__ void put_in(uint4& v, const uint4& m, uint32_t other) {   // `other` where the mask is 0
  v.x = (v.x & m.x) | (other & ~m.x);
  v.y = (v.y & m.y) | (other & ~m.y);
  v.z = (v.z & m.z) | (other & ~m.z);
  v.w = (v.w & m.w) | (other & ~m.w);
}
__device__ __forceinline__ void put_out(uint4& v, const uint4& m, uint32_t other) {   // where it is 1
  put_in(v, make_uint4(~m.x, ~m.y, ~m.z, ~m.w), other);
}

// `n` elements of a line from `from` stay, the others become -inf
template <typename T>
__device__ __forceinline__ void keep(uint4& v, uint32_t from, uint32_t n) {
#pragma unroll
  for (uint32_t i = 0; i < 16 / sizeof(T); ++i)
    if (i < from || i >= from + n) drop_target<T>(v, i);
}
// 16 bytes from byte `by` (1 to 15) of two lines (uniform over a row)
__device__ __forceinline__ uint4 shift_lines(const uint4& a, const uint4& b, uint32_t by) {
  uint32_t w[5];
  switch (by >> 2) {
    case 0: w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x; break;
    case 1: w[0] = a.y, w[1] = a.z, w[2] = a.w, w[3] = b.x, w[4] = b.y; break;
    case 2: w[0] = a.z, w[1] = a.w, w[2] = b.x, w[3] = b.y, w[4] = b.z; break;
    default: w[0] = a.w, w[1] = b.x, w[2] = b.y, w[3] = b.z, w[4] = b.w; break;
  }
  const uint32_t sh = (by & 3u) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], sh), __funnelshift_r(w[1], w[2], sh), __funnelshift_r(w[2], w[3], sh),
                    __funnelshift_r(w[3], w[4], sh));
}
// 16 bytes of shared memory from any element
__device__ __forceinline__ uint4 load_shifted(const unsigned char* p, uint32_t off) {
  const uint4* const l = reinterpret_cast<const uint4*>(p + (off & ~15u));
  const uint32_t by = off & 15u;
  return by ? shift_lines(l[0], l[1], by) : l[0];
}

// A thread's running maximum and sum. The maximum moves only when a logit is more than kSlack units of log2 above it, so the
// sum is rescaled hardly ever.
constexpr float kSlack = kAbove - 1.f;
struct Running {
  float m, s0, s1, limit;
  Ex ex;
  __device__ explicit Running(const Rows& R) : m(kNegInf), s0(0.f), s1(0.f), limit(kSlack), ex(kNegInf, R) {}
  template <typename T, int kN>
  __device__ __forceinline__ void add(const uint4 (&v)[kN], const Rows& R) {
    using W = Word<T>;
    uint32_t t = W::kEmpty;
#pragma unroll
    for (int k = 0; k < kN; ++k) t = vec_max<T>(t, v[k]);
    const float top = W::top(t), above = (top - m) * R.c_hi;
    if (!(above <= limit)) {   // hardly ever, or always about a far m, whose limit is a NaN (above itself may be -inf)
      if (above > kSlack) {
        const float by = rescale(m, top, R);
        s0 *= by;
        s1 *= by;
        m = top;
        ex = Ex(top, R);
        limit = ex.far() ? NAN : kSlack;
      }
      if (ex.far()) {
#pragma unroll
        for (int k = 0; k < kN; ++k) (k & 1 ? s1 : s0) += Pairs<T>(v[k]).template sum<true>(ex);
        return;
      }
    }
#pragma unroll
    for (int k = 0; k < kN; ++k) (k & 1 ? s1 : s0) += Pairs<T>(v[k]).template sum<false>(ex);
  }
  __device__ __forceinline__ Part part() const { return Part{m, (s0 + s1) * kFix}; }
};

// Gradient lines [i, n) by kStride of an output row from lines of shared memory `off` bytes from `src`: f exp(x - ref(m))
template <typename T, uint32_t kStride, int kUnroll>
__device__ __forceinline__ void gradient_lines(uint4* __restrict__ out, const unsigned char* src, uint32_t off, uint32_t i,
                                               uint32_t n, const Ex& ex, float f) {
  if ((off & 15u) == 0 && !ex.far()) {   // the two rows are aligned alike
    const uint4* const in = reinterpret_cast<const uint4*>(src + static_cast<int32_t>(off));
    for (; i + (kUnroll - 1) * kStride < n; i += kUnroll * kStride) {
      uint4 v[kUnroll];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) v[k] = in[i + k * kStride];
#pragma unroll
      for (int k = 0; k < kUnroll; ++k) out[i + k * kStride] = Pairs<T>(v[k]).template scaled<false>(ex, f);
    }
#pragma unroll 1
    for (; i < n; i += kStride) out[i] = Pairs<T>(in[i]).template scaled<false>(ex, f);
  } else if (!ex.far()) {
#pragma unroll 1
    for (; i < n; i += kStride) out[i] = Pairs<T>(load_shifted(src, i * 16 + off)).template scaled<false>(ex, f);
  } else {
#pragma unroll 1
    for (; i < n; i += kStride) out[i] = Pairs<T>(load_shifted(src, i * 16 + off)).template scaled<true>(ex, f);
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_arrive_relaxed() { asm volatile("barrier.cluster.arrive.relaxed.aligned;"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_remote(void* local, uint32_t rank, float a, float b) {   // 8 bytes in rank's copy
  uint32_t dst;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(a), "f"(b) : "memory");
}

constexpr int kMaxCluster = 16;

// The four sums of one cluster's blocks' terms, in a fixed order: the threads with `has` hold their block's term k
__device__ __forceinline__ void cluster_sums(double part, bool has, int k, float* out) {
  __shared__ double sh_block[kMaxCluster][4];
  const uint32_t rank = cluster_rank();
  uint32_t blocks;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  cluster_wait();   // every block runs (arrived at its start)
  if (has) {
    uint32_t dst;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(&sh_block[rank][k])), "r"(0));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(dst), "d"(part) : "memory");
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (rank == 0 && threadIdx.x < 4) {
    double t = 0.0;
    for (uint32_t b = 0; b < blocks; ++b) t += sh_block[b][threadIdx.x];
    out[threadIdx.x] = static_cast<float>(t);
  }
}

// The sums of a row from its threads' parts, given to every thread. One block, or a cluster of `cl` blocks whose warps 0
// write their block's part into every block's shared memory.
template <int kThreads>
__device__ __forceinline__ Part row_join(Part p, int cl, uint32_t rank, const Rows& R, Part* sh_warp, Part* sh_block) {
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  p = warp_join(p, R);
  if (lane == 0) sh_warp[warp] = p;
  __syncthreads();
  Part b = lane < kWarps ? sh_warp[lane] : Part{kNegInf, 0.f};
  b = warp_join(b, R);
  if (cl > 1) {
    cluster_wait();   // every block of the cluster runs (arrived at its start)
    if (warp == 0) {   // the only writes to be seen by other blocks
      if (lane < cl) store_remote(sh_block + rank, lane, b.m, b.s);
      __syncwarp();
      cluster_arrive();
    } else {
      cluster_arrive_relaxed();
    }
    cluster_wait();
    b = lane < cl ? sh_block[lane] : Part{kNegInf, 0.f};
    b = warp_join(b, R);
  }
  return b;
}

// ---------------------------------------------------------------------------------------------------------------------
// The gradient from kept row values: d_j = g ([j == y] - exp(x_j - lse)) / T with one coefficient g per row. Rows with g = 0
// are written as zeros.
struct Kept {
  Per logp, lse, coef;       // per position ...
  const double* logp64;      // ... or by row: the preference loss's own [n] arrays. An fp32 lse of 8 to 16 would be off by
  const double* lse64;       // up to 4.8e-7, and every probability of the gradient with it
  const float* coef_row;
  const double* pair_loss;   // preference: the first block adds up the pairs' losses
  int pairs;
  float* loss;
};
// A factor near fp32's end, whose product with kFix would overflow: its power of two goes into the exponents (Ex)
__device__ __forceinline__ void lift(float& f, float& up) {
  if (fabsf(f) >= 0x1p96f) {
    f *= 0x1p-64f;
    up += 64.f;
  }
}
// exp(x_j - lse) = exp(x_j - ref(m)) exp(ref(m) - lse) with m = lse T
struct KeptRow {
  float m, f, gy, up;   // d_j = 2^up exp(x_j - ref(m)) f, gy at the target
};
__device__ __forceinline__ float kept_coef(const Kept& K, uint32_t row, uint32_t seq, uint32_t tok) {
  return K.coef_row ? K.coef_row[row] : K.coef.at(seq, tok);
}
__device__ __forceinline__ KeptRow kept_row(const Kept& K, const Rows& R, uint32_t row, uint32_t seq, uint32_t tok, float coef) {
  const double lse = K.lse64 ? K.lse64[row] : K.lse.at(seq, tok);
  const float lp = K.logp64 ? static_cast<float>(K.logp64[row]) : K.logp.at(seq, tok);
  const float g = static_cast<float>(coef * R.inv_t);
  KeptRow r;
  r.m = static_cast<float>(lse * R.t);
  const Base b(r.m, R);
  if (b.near) {
    r.f = -g * expf(static_cast<float>(b.b * kLn2 - lse));
    r.up = 0.f;
  } else {   // a far lse may be a large number away from m / T: in the exponents, where nothing overflows before the result does
    r.f = -g;
    r.up = static_cast<float>((r.m * R.inv_t - lse) * kLog2e);
  }
  lift(r.f, r.up);
  r.gy = -expm1f(lp) * g;
  return r;
}
__device__ __forceinline__ void sum_pairs(const Kept& K) {   // one warp, in a fixed order
  const int lane = threadIdx.x & 31;
  double v = 0.0;
  for (int i = lane; i < K.pairs; i += 32) v += __ldcg(K.pair_loss + i);
  v = warp_sum(v);
  if (lane == 0) *K.loss = static_cast<float>(v);
}

// ---------------------------------------------------------------------------------------------------------------------
// The preference loss of a pair (chosen sequence i, rejected sequence i + pairs), one block each: the sums of the two
// sequences' log-probabilities in 64 bits, u = beta ((s_i - ref_i) - (s_j - ref_j)), and each sequence's coefficient written
// to its rows.
struct PairArgs {
  Rows R;
  int pairs;
  const float* ref;      // [2 pairs], or null
  double beta, eps, inv_div;
  const float* div;
  int average;
  const double* logp64;
  float* coef;           // [n], or null (no gradient)
  double* pair_loss;
  float* rewards;        // [2 pairs]
  float* seq_logp;       // [2 pairs]
};
template <int kThreads, bool kShort>
__device__ __forceinline__ void pair_loss(const PairArgs& A, uint32_t pair) {   // all threads of a block
  // kShort: few positions, whose time is that of fetching the code: loops that are not unrolled (4 x 64 x 271 bf16, preference
  // loss: 8.0 against 8.4 us; with 1024 and more positions a sequence they take 1 to 2 us longer). The mean's count has a loop of
  // its own: in one loop with the sums it costs those without a mean as much (20 x 1678 x 256: 18.5 against 16.0 us).
  const Rows& R = A.R;
  __shared__ double sh_s[2][kThreads / 32];
  __shared__ int sh_n[2][kThreads / 32];
  __shared__ float sh_c[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int64_t b[2], e[2];
  double sum[2] = {0.0, 0.0};
  int cnt[2] = {0, 0};
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t q = pair + static_cast<int64_t>(k) * A.pairs, n = R.n;
    if (R.cu) {   // held to the rows there are, between the first offset and the last (in_packed)
      const int64_t lo = max(static_cast<int64_t>(R.cu[0]), static_cast<int64_t>(0));
      const int64_t hi = min(static_cast<int64_t>(R.cu[R.n_seqs]), n);
      b[k] = min(max(static_cast<int64_t>(R.cu[q]), lo), max(lo, hi));
      e[k] = min(max(static_cast<int64_t>(R.cu[q + 1]), b[k]), max(b[k], hi));
    } else {
      b[k] = q * R.tokens;
      e[k] = b[k] + R.tokens;
    }
    if (A.average) {
      for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kThreads) {
        const uint32_t row = static_cast<uint32_t>(i), seq = row / R.tokens, tok = row - seq * R.tokens;
        MO_CHECK(row < R.n);
        if (R.y[seq * R.y_seq + tok * R.y_tok] >= 0) {
          sum[k] += __ldcg(A.logp64 + i);
          ++cnt[k];
        }
      }
    } else if (kShort) {   // logp64 is 0 where a position does not count
#pragma unroll 1
      for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kThreads) sum[k] += __ldcg(A.logp64 + i);
    } else {
      for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kThreads) sum[k] += __ldcg(A.logp64 + i);
    }
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    sum[k] = warp_sum(sum[k]);
    cnt[k] = __reduce_add_sync(0xffffffffu, cnt[k]);
    if (lane == 0) {
      sh_s[k][warp] = sum[k];
      sh_n[k][warp] = cnt[k];
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double s[2], n[2], rw[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      double t = 0.0;
      int c = 0;
      for (int w = 0; w < kThreads / 32; ++w) {
        t += sh_s[k][w];
        c += sh_n[k][w];
      }
      n[k] = A.average ? static_cast<double>(max(c, 1)) : 1.0;
      s[k] = t / n[k];
      const int q = pair + k * A.pairs;
      rw[k] = A.beta * (s[k] - (A.ref ? static_cast<double>(A.ref[q]) : 0.0));
      A.rewards[q] = static_cast<float>(rw[k]);
      A.seq_logp[q] = static_cast<float>(s[k]);
    }
    const double u = rw[0] - rw[1], inv = A.div ? 1.0 / static_cast<double>(*A.div) : A.inv_div;
    // -log sigmoid(u) = max(-u, 0) + log1p(e^-|u|); sigmoid(-u) = e^-|u| / (1 + e^-|u|) or 1 / (1 + e^-|u|)
    const double t = exp(-fabs(u)), l = log1p(t);
    const double up = (u > 0.0 ? 0.0 : -u) + l, down = (u < 0.0 ? 0.0 : u) + l;
    const double q = 1.0 / (1.0 + t), sn = (u >= 0.0 ? t : 1.0) * q, sp = (u >= 0.0 ? 1.0 : t) * q;
    // a term without weight is left out: with a target of probability 0 on one side, the other term is infinite
    A.pair_loss[pair] = ((A.eps < 1.0 ? (1.0 - A.eps) * up : 0.0) + (A.eps > 0.0 ? A.eps * down : 0.0)) * inv;
    const double du = A.beta * (A.eps * sp - (1.0 - A.eps) * sn) * inv;
    sh_c[0] = static_cast<float>(du / n[0]);
    sh_c[1] = static_cast<float>(-du / n[1]);
  }
  __syncthreads();
  if (A.coef == nullptr) return;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float c = sh_c[k];
    if (kShort) {
#pragma unroll 1
      for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kThreads) A.coef[i] = c;
    } else {
      for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kThreads) A.coef[i] = c;
    }
  }
  __syncthreads();   // sh_c is the next pair's
}
constexpr int kPairThreads = 256;
__global__ void __launch_bounds__(kPairThreads) pair_kernel(const __grid_constant__ PairArgs A) {
  pdl_wait();
  pdl_go();
  pair_loss<kPairThreads, false>(A, blockIdx.x);
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows a warp can hold: a warp takes a tile of `per_warp` rows. Their 16-byte lines come into shared memory by cp.async (a
// line may hold up to 15 bytes beside the row: the same aligned line, so nothing beyond the allocation), which lifts every
// alignment and stride question and keeps all of a tile in flight at once. kG lanes work on a row in lines of 16 bytes,
// 32 / kG rows at a time: the quarter of a warp that shared memory serves at once reads 128 bytes in a row whatever the rows'
// pitch, and the maximum and the sum take 3 shuffles for four rows. kL, where it is not 0: no lane has more lines of a row, and
// the loops over them are unrolled (64 x 1024 x 271 bf16, forward: 14.3 us without, 12.2 with).
//
// One warp of the block then forms the values of all its rows, a lane each (64 x 1024 x 271 bf16, policy loss: 22.6 us; with
// each warp for its own rows, on 8 of its lanes, 24.6. The gradient from kept values needs no sums: a barrier for its rows' few
// values costs more, 13.8 against 13.4 us, than it saves). Then, for the gradient, the exponentials again from shared memory,
// by the lines of the output.
//
// Many warps, each with one tile, and not few with the next tile already on its way: a warp waits on its own arithmetic more
// than on memory (with two buffers for half the warps, 16 x 1024 x 4096: policy loss 78 against 57 us).
constexpr int kTileWarps = 4;
constexpr int kTileRows = 8;           // most rows of a tile: 64 x 1024 x 271 bf16, forward, at 4, 8 and 16 rows, loops not
                                       // unrolled: 16.2, 14.5 and 18.2 us (fewer rows: more of a warp's instructions are not
                                       // its rows'; more: too few warps an SM), policy loss 31.7, 27.5 and 31.2 us
constexpr int kTileBytes = 9216;       // most bytes of a tile: 6 blocks of 4 warps in an SM's shared memory
enum Mode { kForward, kPolicyLoss, kGradient, kPreference };   // kPreference: of one cluster

struct TileArgs {
  Rows R;
  int per_warp;
  uint32_t pitch;                      // bytes of a row's lines in shared memory, and 16 to read over
  float* logp;                         // [n], or null
  float* lse;                          // [n], or null
  double* logp64;                      // [n] with lse64 (outside a cluster) and coef [n] (preference), or null
  double* lse64;
  float* coef;
  Policy P;
  void* grad;                          // [n][vocab], or null
  double* partials;                    // [blocks][4] (policy)
  float* sums;                         // or, of one cluster, the sums themselves
  Kept K;                              // (gradient)
  PairArgs pair;                       // (preference)
};

template <int kG>
__device__ __forceinline__ float group_max(float v) {
  if (kG == 32) return warp_max(v);
#pragma unroll
  for (int o = kG / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int kG>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = kG / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Between the rows' log-probabilities and their gradients: the pairs, dealt out to the cluster's blocks. What a block writes
// to global memory in front of a barrier of the cluster is seen by the others behind it.
template <int kThreads>
__device__ __forceinline__ void cluster_pairs(const PairArgs& A, const Kept& K) {
  uint32_t blocks;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  for (uint32_t p = cluster_rank(); p < static_cast<uint32_t>(A.pairs); p += blocks) pair_loss<kThreads, true>(A, p);
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (cluster_rank() == 0 && threadIdx.x < 32) sum_pairs(K);
}

template <typename T, int kG, int kL, Mode kMode>
__device__ __forceinline__ void tile_rows(const TileArgs& A, unsigned char* sm, int chosen, double& sum) {
  using W = Word<T>;
  constexpr uint32_t kPer = 16 / sizeof(T);
  constexpr int kAtOnce = 32 / kG;
  // a row's (m, s, target logit, counts), then (m, f, gy, up; -inf where its gradient is 0)
  __shared__ float4 sh_row[kTileWarps * kTileRows];
  const Rows& R = A.R;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, group = lane / kG;
  const uint32_t gl = lane % kG;
  const uint32_t all = blockIdx.x * kTileWarps * static_cast<uint32_t>(A.per_warp);   // the block's first row
  const int block_rows = all < R.n ? static_cast<int>(min(static_cast<uint32_t>(kTileWarps * A.per_warp), R.n - all)) : 0;
  const uint32_t first = all + warp * static_cast<uint32_t>(A.per_warp);
  const int rows = max(0, min(A.per_warp, block_rows - warp * A.per_warp));
  unsigned char* const base = sm + static_cast<size_t>(warp) * A.per_warp * A.pitch;
  float4* const own = sh_row + warp * A.per_warp;

  // lane r: its row
  uint32_t y = 0;
  int64_t y64 = -1;
  uint64_t addr = 0;
  bool live = false;
  if (lane < rows) {
    const uint32_t row = first + lane, seq = row / R.tokens, tok = row - seq * R.tokens;
    y64 = in_packed(R, row) ? R.y[seq * R.y_seq + tok * R.y_tok] : -1;
    addr = reinterpret_cast<uint64_t>(R.z) + (seq * R.z_seq + tok * R.z_tok) * sizeof(T);
    live = y64 >= 0;
    if (kMode == kPolicyLoss && A.P.weight.p) live = live && A.P.weight.at(seq, tok) != 0.f;
  }
  const bool has_y = live && y64 < static_cast<int64_t>(R.vocab);
  if (has_y) y = static_cast<uint32_t>(y64);
  const uint32_t skew = static_cast<uint32_t>(addr & 15) / sizeof(T);   // elements in front of the row in its first line
  const uint32_t lines = (skew + R.vocab + kPer - 1) / kPer;
  const uint32_t have = live ? lines : 0;
  // the lots' lines: a lane asks for those that it will sum
#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += kAtOnce) {
    const int r = r0 + group;
    const uint64_t a = (__shfl_sync(0xffffffffu, addr, r & 31) & ~15ull) + gl * 16;
    const uint32_t nl = __shfl_sync(0xffffffffu, have, r & 31);
    MO_CHECK(nl == 0 || (nl + 1) * 16 <= A.pitch);
    MO_CHECK(kL == 0 || nl <= kL * kG);
    const uint32_t dst = smem_u32(base + static_cast<size_t>(r) * A.pitch) + gl * 16;
    if (kL > 0) {
#pragma unroll
      for (int k = 0; k < kL; ++k)
        if (gl + k * kG < nl)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + k * kG * 16), "l"(a + k * kG * 16) : "memory");
    } else {
#pragma unroll 4
      for (uint32_t l = 0; gl + l < nl; l += kG)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + l * 16), "l"(a + l * 16) : "memory");
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");

  // the chosen warp's lane r: the inputs of the block's row r
  const bool values = warp == chosen && lane < block_rows;
  float wt = 1.f, adv = 0.f, old_lp = 0.f, ref_lp = 0.f;
  if (kMode == kPolicyLoss && values) {
    const uint32_t row = all + lane, seq = row / R.tokens, tok = row - seq * R.tokens;
    if (A.P.weight.p) wt = A.P.weight.at(seq, tok);
    adv = A.P.adv.at(seq, tok);
    old_lp = A.P.old_lp.at(seq, tok);
    if (A.P.ref_lp.p) ref_lp = A.P.ref_lp.at(seq, tok);
  }
  if (kMode == kGradient) {
    pdl_wait();   // the logits and targets are inputs; the rows' coefficients may come from the launch before
    if (A.K.pair_loss && blockIdx.x == 0 && warp == 0) sum_pairs(A.K);
    if (lane < rows) {
      float4 v = make_float4(0.f, 0.f, 0.f, kNegInf);
      const uint32_t row = first + lane, seq = row / R.tokens, tok = row - seq * R.tokens;
      const float coef = live ? kept_coef(A.K, row, seq, tok) : 0.f;
      if (coef != 0.f) {
        const KeptRow k = kept_row(A.K, R, row, seq, tok, coef);
        v = make_float4(k.m, k.f, k.gy, k.up);
      }
      own[lane] = v;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  if (kMode != kGradient) {
    // lane r: takes the target out of its row, and what lies beside the row in its first and last line
    uint4* const mine = reinterpret_cast<uint4*>(base + static_cast<size_t>(lane) * A.pitch);
    float zy = NAN;
    if (live) {
      if (has_y) {
        T* const at = reinterpret_cast<T*>(mine) + skew + y;
        zy = load_one(at);
        *at = static_cast<T>(kNegInf);
      }
      const uint32_t tail = skew + R.vocab - (lines - 1) * kPer;
      if (skew != 0) put_in(mine[0], behind<T>(skew), W::kEmpty);
      if (tail != kPer) put_out(mine[lines - 1], behind<T>(tail), W::kEmpty);
    }
    if (lane < rows) own[lane] = make_float4(kNegInf, 0.f, zy, live ? 1.f : 0.f);
    __syncwarp();
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += kAtOnce) {
      const int r = r0 + group;
      uint32_t nl = __shfl_sync(0xffffffffu, have, r & 31);
      if (r >= rows) nl = 0;
      const uint4* const row = reinterpret_cast<const uint4*>(base + static_cast<size_t>(r) * A.pitch) + gl;
      uint32_t top = W::kEmpty;
      float s0 = 0.f, s1 = 0.f, m;
      if (kL > 0) {
        uint4 v[kL > 0 ? kL : 1];
#pragma unroll
        for (int k = 0; k < kL; ++k) {
          v[k] = make_uint4(W::kEmpty, W::kEmpty, W::kEmpty, W::kEmpty);
          if (gl + k * kG < nl) v[k] = row[k * kG];
        }
#pragma unroll
        for (int k = 0; k < kL; ++k) top = vec_max<T>(top, v[k]);
        m = group_max<kG>(W::top(top));
        const Ex ex(m, R);
        if (ex.far()) {
#pragma unroll
          for (int k = 0; k < kL; ++k) (k & 1 ? s1 : s0) += Pairs<T>(v[k]).template sum<true>(ex);
        } else {
#pragma unroll
          for (int k = 0; k < kL; ++k) (k & 1 ? s1 : s0) += Pairs<T>(v[k]).template sum<false>(ex);
        }
      } else {
#pragma unroll 4
        for (uint32_t l = 0; gl + l < nl; l += kG) top = vec_max<T>(top, row[l]);
        m = group_max<kG>(W::top(top));
        const Ex ex(m, R);
        if (ex.far()) {
#pragma unroll 1
          for (uint32_t l = 0; gl + l < nl; l += kG) s0 += Pairs<T>(row[l]).template sum<true>(ex);
        } else {
#pragma unroll 4
          for (uint32_t l = 0; gl + l < nl; l += kG) s0 += Pairs<T>(row[l]).template sum<false>(ex);
        }
      }
      const float s = group_sum<kG>(s0 + s1) * kFix;
      if (gl == 0 && r < rows) *reinterpret_cast<float2*>(own + r) = make_float2(m, s);
    }
    __syncthreads();
    if (warp == chosen) {
      const float4 v = values ? sh_row[lane] : make_float4(0.f, 0.f, 0.f, 0.f);
      const bool counts = v.w != 0.f;
      RowStat st = {0.0, 0.0, 0.f, 0.f};
      double part[4] = {0.0, 0.0, 0.0, 0.0};
      float up = 0.f;
      if (counts) {
        st = row_stat(v.z, v.x, v.y, R);
        if (kMode == kPolicyLoss) {
          const PolicyRow p = policy_row(A.P, st, wt, adv, old_lp, ref_lp, R.inv_t);
#pragma unroll
          for (int k = 0; k < 4; ++k) part[k] = p.part[k];
          st.f = p.f;
          st.rest = p.gy;
          up = p.up;
        }
      }
      if (values) {
        const uint32_t row = all + lane;
        if (A.logp) A.logp[row] = static_cast<float>(st.logp);
        if (A.lse) A.lse[row] = static_cast<float>(st.lse);
        if (A.logp64) {
          A.logp64[row] = st.logp;
          if (A.lse64) A.lse64[row] = st.lse;
          A.coef[row] = 0.f;
        }
        if (kMode != kForward) sh_row[lane] = make_float4(v.x, st.f, st.rest, counts ? up : kNegInf);
      }
      if (kMode == kPolicyLoss) {   // lane k < 4: the block's sum k
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const double t = warp_sum(part[k]);
          if (lane == k) sum = t;
        }
        if (A.sums == nullptr && lane < 4) A.partials[static_cast<size_t>(blockIdx.x) * 4 + lane] = sum;
      }
    }
    if (kMode == kForward) return;
    if (kMode == kPreference) {
      cluster_pairs<kTileWarps * 32>(A.pair, A.K);
      if (lane < rows) {
        const float coef = __ldcg(A.coef + first + lane), g = static_cast<float>(coef * R.inv_t);
        const float4 v = own[lane];
        float f = -g * v.y, up = v.w;
        lift(f, up);
        own[lane] = make_float4(v.x, f, g * v.z, coef != 0.f ? up : kNegInf);
      }
      __syncwarp();
    }
    if (A.grad == nullptr) return;
  }
  if (kMode == kPolicyLoss) __syncthreads();

#pragma unroll 1
  for (int r0 = 0; r0 < rows; r0 += kAtOnce) {
    const int r = r0 + group;
    const uint32_t sk = __shfl_sync(0xffffffffu, skew, r & 31);
    if (r >= rows) continue;
    const float4 v = own[r];
    T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(first + r) * R.vocab;
    const Split<T> so(out, R.vocab);
    uint4* const ov = reinterpret_cast<uint4*>(out + so.head);
    const unsigned char* const row = base + static_cast<size_t>(r) * A.pitch;
    if (v.w == kNegInf) {
      for (uint32_t l = gl; l < so.vecs; l += kG) ov[l] = make_uint4(0, 0, 0, 0);
      for (uint32_t i = gl; i < so.head + so.tail; i += kG) store_one(out + so.edge(i), 0.f);
      continue;
    }
    const Ex ex(v.x, R, v.w);
    const float k1 = v.y * kFix;
    const uint32_t off = (sk + so.head) * static_cast<uint32_t>(sizeof(T));
    if (kL > 0 && (off & 15u) == 0 && !ex.far()) {
      const uint4* const in = reinterpret_cast<const uint4*>(row + off) + gl;
#pragma unroll
      for (int k = 0; k < kL; ++k)
        if (gl + k * kG < so.vecs) ov[gl + k * kG] = Pairs<T>(in[k * kG]).template scaled<false>(ex, k1);
    } else {
      gradient_lines<T, kG, 2>(ov, row, off, gl, so.vecs, ex, k1);
    }
    for (uint32_t i = gl; i < so.head + so.tail; i += kG) {
      const uint32_t j = so.edge(i);
      store_one(out + j, ex.one(load_one(reinterpret_cast<const T*>(row) + sk + j)) * k1);
    }
  }
  __syncwarp();   // the targets' elements, written above
  if (has_y) {
    const float4 v = own[lane];
    if (v.w != kNegInf) store_one(static_cast<T*>(A.grad) + static_cast<size_t>(first + lane) * R.vocab + y, v.z);
  }
}

template <typename T, int kG, int kL, Mode kMode>
__global__ void __launch_bounds__(kTileWarps * 32, kMode == kPreference ? 4 : 8) tile_kernel(const __grid_constant__ TileArgs A) {
  extern __shared__ __align__(16) unsigned char sm[];
  const bool one_cluster = kMode == kPolicyLoss && A.sums != nullptr;
  if (kMode != kGradient && kMode != kPreference) pdl_go();
  if (one_cluster) cluster_arrive_relaxed();
  // the block's rows' values are formed by one warp, another one in the next block: a warp's number is its scheduler's
  const int chosen = blockIdx.x % kTileWarps;
  double sum = 0.0;
  tile_rows<T, kG, kL, kMode>(A, sm, chosen, sum);
  if (one_cluster) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    cluster_sums(sum, static_cast<int>(threadIdx.x >> 5) == chosen && lane < 4, lane, A.sums);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long rows, forward only: a stream of pieces of `lines` lines, a warp each, in batches of kBatch lines a lane. A warp has its
// own ring of kStages batches in shared memory, filled by cp.async two batches ahead, over the end of a piece into its next
// one, and each lane reads what it asked for itself. join_kernel puts a row's parts together.
struct StreamArgs {
  Rows R;
  uint32_t pieces;      // of a row
  uint32_t n;           // pieces in all
  uint32_t lines;       // of a piece: a multiple of a batch's
  Part* parts;          // [n]
};
constexpr int kStreamThreads = 128, kStreamBlocks = 7, kBatch = 4, kStages = 3;
constexpr int kAhead = 8;   // pieces that may be known and not done: kStages batches of different ones and the next, rounded up
constexpr size_t kStreamSmem = static_cast<size_t>(kStreamThreads) * kStages * kBatch * 16;

template <typename T>
__global__ void __launch_bounds__(kStreamThreads, kStreamBlocks) stream_kernel(const __grid_constant__ StreamArgs A) {
  extern __shared__ __align__(16) unsigned char sm[];
  __shared__ uint4 sh_known[kStreamThreads / 32][kAhead];
  using W = Word<T>;
  constexpr uint32_t kPer = 16 / sizeof(T), kLines = 32 * kBatch, kElems = kLines * kPer;
  const Rows& R = A.R;
  const uint32_t lane = threadIdx.x & 31, step = gridDim.x * (kStreamThreads / 32);
  uint32_t piece = blockIdx.x * (kStreamThreads / 32) + (threadIdx.x >> 5);
  pdl_go();
  if (piece >= A.n) return;
  // this lane's place in its warp's ring, and the warp's pieces
  uint4* const ring = reinterpret_cast<uint4*>(sm) + (threadIdx.x >> 5) * (kStages * kLines) + lane;
  uint4* const known = sh_known[threadIdx.x >> 5];

  // The asking side. A piece: its lines (0: nothing to read), the elements in front of the row in its first line, the row's
  // end and the target, in elements from the first line's begin. A piece without lines still takes a (void) batch, so that
  // both sides count the same.
  uint32_t ask_piece = piece, asked = 0, ask_lines = 0, ask_count = 0, ask_stage = 0;
  uint64_t ask_at = 0;
  const auto look = [&] {
    uint4 b = make_uint4(0, 0, 0, 0xffffffffu);
    if (ask_piece < A.n) {
      const uint32_t row = ask_piece / A.pieces, from = (ask_piece - row * A.pieces) * A.lines;
      const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
      const int64_t y = in_packed(R, row) ? R.y[seq * R.y_seq + tok * R.y_tok] : -1;
      const uint64_t a = reinterpret_cast<uint64_t>(R.z) + (seq * R.z_seq + tok * R.z_tok) * sizeof(T);
      const uint32_t skew = static_cast<uint32_t>(a & 15) / sizeof(T), lines = (skew + R.vocab + kPer - 1) / kPer;
      if (y >= 0 && from < lines) {
        b.x = min(A.lines, lines - from);
        b.y = from == 0 ? skew : 0;
        b.z = skew + R.vocab - from * kPer;
        if (y < static_cast<int64_t>(R.vocab)) b.w = skew + static_cast<uint32_t>(y) - from * kPer;   // wraps in front
        ask_at = (a & ~15ull) + (static_cast<uint64_t>(from) + lane) * 16;
      }
    }
    ask_lines = b.x;
    if (lane == 0) known[ask_count % kAhead] = b;
    ++ask_count;
    __syncwarp();
  };
  const auto request = [&] {
    const uint32_t dst = smem_u32(ring) + ask_stage * (kLines * 16);
    if (asked + kLines <= ask_lines) {
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 512 * k), "l"(ask_at + 512 * k) : "memory");
    } else {
#pragma unroll
      for (uint32_t k = 0; k < kBatch; ++k)
        if (asked + lane + 32 * k < ask_lines)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + 512 * k), "l"(ask_at + 512 * k) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    ask_stage = ask_stage == kStages - 1 ? 0 : ask_stage + 1;
    asked += kLines;
    ask_at += kLines * 16;
    if (asked >= ask_lines) {
      ask_piece += step;
      asked = 0;
      look();
    }
  };
  look();
#pragma unroll 1
  for (int k = 0; k < kStages - 1; ++k) request();

  uint32_t count = 0, stage = 0;
  for (; piece < A.n; piece += step, ++count) {
    const uint4 b = known[count % kAhead];
    Running run(R);
    for (uint32_t done = 0;;) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      const uint4* const at = ring + stage * kLines;
      stage = stage == kStages - 1 ? 0 : stage + 1;
      uint4 v[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) v[k] = at[32 * k];
      request();   // into the batch that was read before this one
      const uint32_t e0 = done * kPer, there = b.w - e0;
      if ((b.x < done + kLines) | (b.z - e0 < kElems) | (e0 < b.y)) {   // an edge of the row, or the piece's end
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) {
          const uint32_t line = done + lane + 32 * k, e = line * kPer;
          const uint32_t from = line == 0 ? b.y : 0;
          keep<T>(v[k], from, line < b.x ? min(kPer, b.z - e) - from : 0);
        }
      }
      if (there < kElems) {   // the target
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k)
          if (there / kPer == lane + 32 * k) drop_target<T>(v[k], there % kPer);
      }
      run.add<T>(v, R);
      done += kLines;
      if (done >= b.x) break;
    }
    const Part p = warp_join(run.part(), R);
    if (lane == 0) A.parts[piece] = p;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Rows from their pieces' parts, a warp each
struct JoinArgs {
  Rows R;
  uint32_t pieces;
  const Part* parts;
  float* logp;
  float* lse;
  double* logp64;
  double* lse64;
  float* coef;
};
constexpr int kJoinThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ JoinArgs A) {
  const Rows& R = A.R;
  const int lane = threadIdx.x & 31;
  const uint32_t row = blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5);
  pdl_go();
  if (row >= R.n) return;
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const int64_t y = in_packed(R, row) ? R.y[seq * R.y_seq + tok * R.y_tok] : -1;
  float zy = NAN;
  if (y >= 0 && y < static_cast<int64_t>(R.vocab))
    zy = load_one(reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok) + y);
  pdl_wait();
  RowStat st = {0.0, 0.0, 0.f, 0.f};
  if (y >= 0) {
    Part p = {kNegInf, 0.f};
    for (uint32_t i = lane; i < A.pieces; i += 32) {
      const Part q = A.parts[static_cast<size_t>(row) * A.pieces + i];
      const float M = fmaxf(p.m, q.m);
      p.s = (p.s == 0.f ? 0.f : p.s * rescale(p.m, M, R)) + (q.s == 0.f ? 0.f : q.s * rescale(q.m, M, R));
      p.m = M;
    }
    p = warp_join(p, R);
    st = row_stat(zy, p.m, p.s, R);
  }
  if (lane == 0) {
    if (A.logp) A.logp[row] = static_cast<float>(st.logp);
    if (A.lse) A.lse[row] = static_cast<float>(st.lse);
    if (A.logp64) {
      A.logp64[row] = st.logp;
      A.lse64[row] = st.lse;
      A.coef[row] = 0.f;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long rows, the policy loss: a row per block, or per cluster of blocks that take a slice each. A slice's 16-byte lines come
// into shared memory at once by cp.async, so a block has all its bytes in flight and several blocks of an SM are at different
// stages: each row is read once, however often the kernel goes over it. Every thread masks, maximises and sums the lines that
// it loaded itself; the blocks' parts meet in distributed shared memory; one thread forms the row's values, and all go over
// the slice again for the gradient, by the lines of the output.
//
// Nothing is full (4 x 1024 x 32768 bf16: 109 us, 0.75 of the copy bandwidth's rate; special-function units 0.63, issue slots
// 0.53, DRAM 0.55): a block loads, exchanges, forms its values and stores in turn, and three of them share an SM. Blocks that
// stay, and ask for the next row's lines while they store this one's gradient, took 115 us.
// Exponentials again instead of kept ones: 32 fp32 exponentials a thread in registers left two blocks of 512 threads an SM,
// whose chain of load, cluster exchange and row values then stands between them (8192 rows of 131072: 1497 us).
struct SliceArgs {
  Rows R;
  int cl;               // blocks per row
  float* logp;          // [n]
  Policy P;
  void* grad;           // [n][vocab], or null
  double* partials;     // [n][4]
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads, kThreads == 128 ? 6 : 3) slice_kernel(const __grid_constant__ SliceArgs A) {
  extern __shared__ __align__(16) unsigned char sm[];
  using W = Word<T>;
  constexpr uint32_t kPer = 16 / sizeof(T);
  __shared__ Part sh_warp[kThreads / 32], sh_block[kMaxCluster];
  __shared__ float sh_g[3];
  __shared__ float sh_in[4];   // the row's target logit, advantage, old and reference log-probability
  const Rows& R = A.R;
  const uint32_t rank = A.cl > 1 ? cluster_rank() : 0;
  const uint32_t row = blockIdx.x / A.cl;
  MO_CHECK(row < R.n && rank < static_cast<uint32_t>(A.cl));
  pdl_go();
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const T* const z = reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok);
  T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(row) * R.vocab;
  // the slice [e0, e1) is cut at the output's lines where there is a gradient, at the input's otherwise
  const Split<T> so(A.grad ? out : z, R.vocab);
  const uint32_t share = (so.vecs + A.cl - 1) / A.cl;
  const uint32_t v0 = min(rank * share, so.vecs), v1 = min(v0 + share, so.vecs);
  const bool last = rank == static_cast<uint32_t>(A.cl) - 1;
  const uint32_t e0 = rank == 0 ? 0 : so.head + v0 * kPer, e1 = last ? R.vocab : so.head + v1 * kPer;
  // this thread's element beside the output's lines, if any
  uint32_t je = 0xffffffffu;
  if (rank == 0 && threadIdx.x < so.head) je = threadIdx.x;
  if (last && threadIdx.x >= 32 && threadIdx.x < 32 + so.tail) je = so.head + so.vecs * kPer + threadIdx.x - 32;

  int64_t y64 = R.y[seq * R.y_seq + tok * R.y_tok];
  if (A.P.weight.p && A.P.weight.at(seq, tok) == 0.f) y64 = -1;
  if (y64 < 0) {   // the whole cluster
    if (rank == 0 && threadIdx.x == 0) A.logp[row] = 0.f;
    if (rank == 0 && threadIdx.x < 4) A.partials[static_cast<size_t>(row) * 4 + threadIdx.x] = 0.0;
    if (A.grad) {
      if (je != 0xffffffffu) store_one(out + je, 0.f);
      for (uint32_t i = v0 + threadIdx.x; i < v1; i += kThreads)
        reinterpret_cast<uint4*>(out + so.head)[i] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  if (A.cl > 1) cluster_arrive_relaxed();

  const uint64_t a0 = reinterpret_cast<uint64_t>(z + e0);
  const uint32_t skew = static_cast<uint32_t>(a0 & 15) / sizeof(T);             // elements in front of e0 in line 0
  const uint32_t lines = e1 > e0 ? (skew + (e1 - e0) + kPer - 1) / kPer : 0;
  MO_CHECK(lines <= share + 3);
  const uint32_t dst = smem_u32(sm);
  for (uint32_t i = threadIdx.x; i < lines; i += kThreads)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * 16), "l"((a0 & ~15ull) + i * 16ull) : "memory");
  asm volatile("cp.async.commit_group;" ::: "memory");
  const bool has_y = y64 < static_cast<int64_t>(R.vocab);
  const uint32_t y = has_y ? static_cast<uint32_t>(y64) : 0xffffffffu;
  if (threadIdx.x < 4) {   // read by thread 0 behind row_join's barrier
    float x = NAN;
    if (threadIdx.x == 0) {
      if (has_y) x = load_one(z + y);
    } else {
      const Per& per = threadIdx.x == 1 ? A.P.adv : threadIdx.x == 2 ? A.P.old_lp : A.P.ref_lp;
      if (per.p) x = per.at(seq, tok);
    }
    sh_in[threadIdx.x] = x;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");

  // a thread's own lines: what lies beside the slice in the first and the last one, and the target, become -inf
  uint4* const line = reinterpret_cast<uint4*>(sm);
  const uint32_t len = e1 - e0, ty = y - e0 < len ? skew + (y - e0) : 0xffffffffu;
  if (threadIdx.x == 0 && skew != 0 && lines > 0) put_in(line[0], behind<T>(skew), W::kEmpty);
  if (lines > 0 && threadIdx.x == (lines - 1) % kThreads)
    put_out(line[lines - 1], behind<T>(skew + len - (lines - 1) * kPer), W::kEmpty);
  if (ty != 0xffffffffu && threadIdx.x == ty / kPer % kThreads) drop_target<T>(line[ty / kPer], ty % kPer);
  Running run(R);
  uint32_t at = threadIdx.x;
  for (; at + 3 * kThreads < lines; at += 4 * kThreads) {
    const uint4 v[4] = {line[at], line[at + kThreads], line[at + 2 * kThreads], line[at + 3 * kThreads]};
    run.add<T>(v, R);
  }
#pragma unroll 1
  for (; at < lines; at += kThreads) {
    const uint4 v[1] = {line[at]};
    run.add<T>(v, R);
  }
  const Part p = row_join<kThreads>(run.part(), A.cl, rank, R, sh_warp, sh_block);
  if (threadIdx.x == 0) {
    const RowStat st = row_stat(sh_in[0], p.m, p.s, R);
    const float wt = A.P.weight.p ? A.P.weight.at(seq, tok) : 1.f;
    const PolicyRow v = policy_row(A.P, st, wt, sh_in[1], sh_in[2], sh_in[3], R.inv_t);
    sh_g[0] = v.f;
    sh_g[1] = v.gy;
    sh_g[2] = v.up;
    if (rank == 0) {
      A.logp[row] = static_cast<float>(st.logp);
      double* const o = A.partials + static_cast<size_t>(row) * 4;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = v.part[k];
    }
  }
  if (A.grad == nullptr) return;
  __syncthreads();
  const Ex ex(p.m, R, sh_g[2]);
  const float f = sh_g[0] * kFix, gy = sh_g[1];
  if (je != 0xffffffffu) {
    const T* const x = reinterpret_cast<const T*>(sm) + skew + (je - e0);
    store_one(out + je, je == y ? gy : ex.one(load_one(x)) * f);
  }
  // output line i of the row is at byte i * 16 + (skew + head - e0) * size of the slice (the sum may wrap, not the address)
  gradient_lines<T, kThreads, 4>(reinterpret_cast<uint4*>(out + so.head) + v0, sm,
                                 v0 * 16 + (skew + so.head - e0) * static_cast<uint32_t>(sizeof(T)), threadIdx.x, v1 - v0, ex,
                                 f);
  const uint32_t yl = (y - so.head) / kPer;   // the target's line, if it lies in one of this slice's
  if (y - so.head < so.vecs * kPer && yl >= v0 && yl < v1 && threadIdx.x == (yl - v0) % kThreads) store_one(out + y, gy);
}

// ---------------------------------------------------------------------------------------------------------------------
// Long rows, the gradient from kept row values: elementwise, so a row is cut into pieces of kGradVecs lines a thread.
struct GradArgs {
  Rows R;
  Kept K;
  void* grad;
  uint32_t pieces;        // blocks per row
};
// 4096 rows of 131072 bf16 at 256 x 4 lines a block 356 us, 128 x 4 344, 128 x 8 341, 512 x 2 437
constexpr int kGradThreads = 128, kGradVecs = 8;

template <typename T>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const __grid_constant__ GradArgs A) {
  const Rows& R = A.R;
  constexpr uint32_t kPer = 16 / sizeof(T);
  // from the last row to the first: what the forward pass read last is still in L2
  const uint32_t row = R.n - 1 - blockIdx.x / A.pieces, piece = blockIdx.x % A.pieces;
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const T* const z = reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok);
  T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(row) * R.vocab;
  const Split<T> so(out, R.vocab);
  MO_CHECK(row < R.n);
  const int64_t y64 = R.y[seq * R.y_seq + tok * R.y_tok];
  const uint32_t begin = piece * (kGradThreads * kGradVecs) + threadIdx.x;
  // an output line's elements: one line of the input, or two and a shift where the two rows are aligned differently
  const uint64_t a = reinterpret_cast<uint64_t>(z + so.head);
  const uint32_t by = static_cast<uint32_t>(a & 15);
  const uint4* const zv = reinterpret_cast<const uint4*>(a & ~15ull);
  uint4 v[kGradVecs], w[kGradVecs];
  if (y64 >= 0) {   // inputs: read before the launch in front of this one has ended
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k) {
      const uint32_t at = begin + k * kGradThreads;
      if (at < so.vecs) v[k] = load_vec(zv + at);
    }
    if (by) {
#pragma unroll
      for (int k = 0; k < kGradVecs; ++k) {
        const uint32_t at = begin + k * kGradThreads;
        if (at < so.vecs) w[k] = load_vec(zv + at + 1);
      }
    }
  }
  pdl_wait();
  if (A.K.pair_loss && blockIdx.x == 0 && threadIdx.x < 32) sum_pairs(A.K);
  const float coef = y64 >= 0 ? kept_coef(A.K, row, seq, tok) : 0.f;
  const bool edge = piece == 0 && threadIdx.x < so.head + so.tail;
  const uint32_t je = so.edge(threadIdx.x);
  uint4* const ov = reinterpret_cast<uint4*>(out + so.head);
  if (coef == 0.f) {
    if (edge) store_one(out + je, 0.f);
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k) {
      const uint32_t at = begin + k * kGradThreads;
      if (at < so.vecs) ov[at] = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const KeptRow r = kept_row(A.K, R, row, seq, tok, coef);
  const Ex ex(r.m, R, r.up);
  const float f = r.f * kFix;
  const uint32_t y = y64 < static_cast<int64_t>(R.vocab) ? static_cast<uint32_t>(y64) : 0xffffffffu;
  if (edge) store_one(out + je, je == y ? r.gy : ex.one(load_one(z + je)) * f);
  const auto write = [&](auto far) {
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k) {
      const uint32_t at = begin + k * kGradThreads;
      if (at >= so.vecs) break;
      const uint4 d = Pairs<T>(by ? shift_lines(v[k], w[k], by) : v[k]).template scaled<decltype(far)::value>(ex, f);
      // the preference loss has read the logits before: a gradient that leaves L2 first leaves them there (4 x 1024 x 32768
      // bf16: 137 against 147 us)
      if (A.K.pair_loss) __stcs(ov + at, d);
      else ov[at] = d;
      const uint32_t e = so.head + at * kPer;
      if (y - e < kPer) store_one(out + y, r.gy);
    }
  };
  if (ex.far()) write(std::true_type());
  else write(std::false_type());
}

// ---------------------------------------------------------------------------------------------------------------------
// Sums of `n` rows of four partials, in a fixed order: block b adds up its contiguous share. With one block the result goes
// to out32, else a block's to out64[b].
struct SumArgs {
  const double* partials;
  uint32_t n;
  double* out64;
  float* out32;
};
constexpr int kSumThreads = 512;
__global__ void __launch_bounds__(kSumThreads) sum_kernel(const __grid_constant__ SumArgs A) {
  __shared__ double sh[kSumThreads / 32][4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t share = (A.n + gridDim.x - 1) / gridDim.x;
  const uint32_t begin = min(A.n, blockIdx.x * share), end = min(A.n, begin + share);
  pdl_wait();
  pdl_go();
  double v[4] = {0.0, 0.0, 0.0, 0.0};
  for (uint32_t i = begin + threadIdx.x; i < end; i += kSumThreads) {
    const double2 a = reinterpret_cast<const double2*>(A.partials)[2 * static_cast<size_t>(i)];
    const double2 b = reinterpret_cast<const double2*>(A.partials)[2 * static_cast<size_t>(i) + 1];
    v[0] += a.x;
    v[1] += a.y;
    v[2] += b.x;
    v[3] += b.y;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    v[k] = warp_sum(v[k]);
    if (lane == 0) sh[warp][k] = v[k];
  }
  __syncthreads();
  if (threadIdx.x < 4) {
    double t = 0.0;
    for (int w = 0; w < kSumThreads / 32; ++w) t += sh[w][threadIdx.x];
    if (gridDim.x == 1) A.out32[threadIdx.x] = static_cast<float>(t);
    else A.out64[static_cast<size_t>(blockIdx.x) * 4 + threadIdx.x] = t;
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The pairs' losses added up where no gradient pass does it
__global__ void __launch_bounds__(32) pair_sum_kernel(const __grid_constant__ Kept K) {
  pdl_wait();
  sum_pairs(K);
}

}  // namespace loss
}  // namespace moteopt
