// Losses on logits: token log-probabilities (forward and backward), the clipped policy loss with a KL term and the paired
// preference loss, each with its gradient in the logits. The steps that train on them are the reference's post-training
// loops (mote/train/dpo.py:217, kto.py:151, rlvr.py:308: clip and AdamW after such a loss).
//
// Per row (one position) with logits z, temperature T, x = z / T and target y:
//   logp = x_y - lse(x),  dlogp/dz_j = ([j == y] - exp(x_j - lse)) / T
// The target's column is kept out of the sum: with m the largest of the OTHER logits, s = sum_{j != y} exp(x_j - m/T) and
// a = x_y - m/T,
//   a >= 0: logp = -log1p(s e^-a)          1 - p_y = X / (1 + X), X = s e^-a
//   a <  0: logp = a - log1p(s - 1 + e^a)  1 - p_y = s / (s + e^a)
// so that neither logp nor 1 - p_y cancels where the model is sure of its target (p_y -> 1). These few values of a row are
// formed in 64 bits; the exponentials and the sums inside a thread are fp32.
//
// All kernels are memory-bound in principle (2 or 4 bytes read per logit, as many written for a gradient); the exponential
// is next: one ex2 per logit at 16 per clock and SM is 0.73 of the copy bandwidth's rate for bf16 logits read once.
#pragma once

#include <cooperative_groups.h>
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "mt_types.h"
#include "ptx.cuh"

namespace moteopt {
namespace loss {

constexpr float kNegInf = -INFINITY;
constexpr double kLog2e = 1.4426950408889634074;
// ex2.approx's mean relative error below -1 is -5.05e-8, the same for every binade (measured over 4e6 arguments each). It
// is a bias, so it would add up over the thousands of positions of a sequence; a row's sum, but for the 1 of its largest
// element, is multiplied by the inverse.
constexpr double kEx2Bias = 1.0 + 5.05e-8;

// logits [seqs][tokens][vocab], the last axis contiguous, and the targets [seqs][tokens]
struct Rows {
  const char* z;
  const int64_t* y;
  int64_t z_seq, z_tok;   // strides in elements
  int64_t y_seq, y_tok;
  uint32_t n;             // rows: seqs * tokens, below 2^31
  uint32_t tokens;
  uint32_t vocab;
  const int32_t* cu;      // packed: n_seqs + 1 row offsets, or null. Rows outside [cu[0], cu[n_seqs]) do not count
  int n_seqs;
  float c_hi, c_lo;       // log2(e) / T as two floats, c_lo > 0 (see ex2_of)
  double inv_t;
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

// 2^((z - m) c) for z <= m, c = c_hi + c_lo. One rounding of the whole product: log2(e) rounded to one float is a relative
// error of 1.3e-8 in every exponent, which the same sums would carry. c_lo > 0 keeps -inf a -inf.
__device__ __forceinline__ float ex2(float t) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(t));
  return r;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

struct Ex {               // the constants of one row's exponentials, two at a time
  uint64_t neg_m, hi, lo;
  __device__ Ex(float m, float c_hi, float c_lo) : neg_m(pack2(-m, -m)), hi(pack2(c_hi, c_hi)), lo(pack2(c_lo, c_lo)) {}
  __device__ __forceinline__ void two(float z0, float z1, float& e0, float& e1) const {
    const uint64_t d = add2(pack2(z0, z1), neg_m);
    float t0, t1;
    unpack2(fma2(d, hi, mul2(d, lo)), t0, t1);
    e0 = ex2(t0);
    e1 = ex2(t1);
  }
};
__device__ __forceinline__ float ex_one(float z, float m, float c_hi, float c_lo) {
  const float d = z - m;
  return ex2(fmaf(d, c_hi, d * c_lo));
}
// exp((m - to) / T), the factor of a partial sum that moves to another maximum: once a thread, by expf
__device__ __forceinline__ float rescale(float m, float to, float inv_t) { return m == kNegInf ? 0.f : expf((m - to) * inv_t); }

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

// (largest logit, sum) of a part of a row
struct Part {
  float m, s;
};
__device__ __forceinline__ Part warp_join(Part p, float inv_t) {
  const float M = warp_max(p.m);
  return Part{M, warp_sum(p.s == 0.f ? 0.f : p.s * rescale(p.m, M, inv_t))};
}

// What a row's sums give (see the top of this file)
struct RowStat {
  double logp, lse;
  float f;      // exp(m / T - lse): p_j = exp((z_j - m) / T) f
  float rest;   // 1 - p_y
};
__device__ __forceinline__ RowStat row_stat(float zy, float m, float s32, double inv_t) {
  const double s = s32 >= 1.f ? 1.0 + (static_cast<double>(s32) - 1.0) * kEx2Bias : static_cast<double>(s32);
  const double a = (static_cast<double>(zy) - static_cast<double>(m)) * inv_t;
  const bool up = a >= 0.0;
  const double q = exp(up ? -a : a);
  const double X = up ? (s == 0.0 ? 0.0 : s * q) : (s - 1.0) + q;
  const double l = log1p(X), inv = 1.0 / (1.0 + X);
  RowStat r;
  r.logp = up ? -l : a - l;
  r.lse = static_cast<double>(up ? zy : m) * inv_t + l;
  r.f = static_cast<float>((up ? q : 1.0) * inv);
  r.rest = static_cast<float>((up ? X : s) * inv);
  if (zy == INFINITY) r.logp = r.lse = static_cast<double>(r.f = r.rest = NAN);   // inf - inf
  return r;
}

// The policy loss of one row, unscaled by the weight and the divisor
struct RowLoss {
  double loss, kl, slope;   // slope: dloss/dlogp
  bool clipped;
};
__device__ __forceinline__ RowLoss policy_row_loss(double logp, const Policy& P, float old_lp, float ref_lp, bool has_ref,
                                                   float adv) {
  const double A = adv, r = exp(logp - static_cast<double>(old_lp));
  const double held_r = fmin(fmax(r, P.clip_lo), P.clip_hi);
  const double free = r * A, held = (r != r ? r : held_r) * A;
  RowLoss L;
  L.clipped = held < free;
  L.loss = L.clipped ? -held : -free;
  L.slope = L.clipped ? 0.0 : -free;
  L.kl = 0.0;
  if (has_ref) {
    const double d = static_cast<double>(ref_lp) - logp, e = expm1(d);
    L.kl = e - d;
    if (P.kl != 0.0) {
      L.loss += P.kl * L.kl;
      L.slope -= P.kl * e;
    }
  }
  return L;
}

__device__ __forceinline__ bool in_packed(const Rows& R, uint32_t row) {
  if (R.cu == nullptr) return true;
  return static_cast<int64_t>(row) >= R.cu[0] && static_cast<int64_t>(row) < R.cu[R.n_seqs];
}

// ---------------------------------------------------------------------------------------------------------------------
// Short rows: a warp takes `per_warp` rows. Their 16-byte lines come into shared memory by cp.async (a line may hold up to
// 15 bytes beside the row: the same aligned line, so nothing beyond the allocation), which lifts every alignment and stride
// question and keeps all of a warp's rows in flight at once. Then per row the maximum and the sum over the warp's lanes; then
// one lane per row for the row's values in 64 bits (they would cost a warp more than the whole row if every lane formed them
// for one row); then, for the gradient, the exponentials again from shared memory.
constexpr int kTileWarps = 4;
constexpr int kTileRows = 16;          // most rows of a warp
constexpr int kTileBytes = 9216;       // most bytes of a warp's rows: 6 blocks of 4 warps in an SM's shared memory

struct TileArgs {
  Rows R;
  int per_warp;
  uint32_t pitch;                      // bytes of a row's lines in shared memory
  float* logp;                         // [n], or null
  float* lse;                          // [n], or null
  double* logp64;                      // [n] with coef [n] (preference), or null
  float* coef;
  Policy P;
  void* grad;                          // [n][vocab], or null
  double* partials;                    // [warps][4] (policy)
};

template <typename T, bool kPolicy>
__global__ void __launch_bounds__(kTileWarps * 32) tile_kernel(const __grid_constant__ TileArgs A) {
  extern __shared__ __align__(16) unsigned char sm[];
  using W = Word<T>;
  const Rows& R = A.R;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t tile = blockIdx.x * kTileWarps + warp;
  const uint32_t first = tile * static_cast<uint32_t>(A.per_warp);
  pdl_go();
  if (first >= R.n) return;
  const int rows = static_cast<int>(min(static_cast<uint32_t>(A.per_warp), R.n - first));
  unsigned char* const base = sm + static_cast<size_t>(warp) * A.per_warp * A.pitch;

  // lane r: its row
  uint32_t seq = 0, tok = 0, y = 0;
  int64_t y64 = -1;
  uint64_t addr = 0;
  float wt = 1.f;
  if (lane < rows) {
    const uint32_t row = first + lane;
    seq = row / R.tokens;
    tok = row - seq * R.tokens;
    y64 = in_packed(R, row) ? R.y[seq * R.y_seq + tok * R.y_tok] : -1;
    addr = reinterpret_cast<uint64_t>(R.z) + (seq * R.z_seq + tok * R.z_tok) * sizeof(T);
    if (kPolicy && A.P.weight.p) wt = A.P.weight.at(seq, tok);
  }
  const bool live = y64 >= 0 && wt != 0.f;
  const bool has_y = live && y64 < static_cast<int64_t>(R.vocab);
  if (has_y) y = static_cast<uint32_t>(y64);
  const unsigned live_rows = __ballot_sync(0xffffffffu, live);
  for (int r = 0; r < rows; ++r) {
    if (!(live_rows >> r & 1)) continue;
    const uint64_t a = __shfl_sync(0xffffffffu, addr, r);
    const uint32_t lines = (static_cast<uint32_t>(a & 15) + R.vocab * static_cast<uint32_t>(sizeof(T)) + 15) / 16;
    MO_CHECK(lines * 16 <= A.pitch);
    const uint32_t dst = smem_u32(base + static_cast<size_t>(r) * A.pitch);
    for (uint32_t v = lane; v < lines; v += 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + v * 16), "l"((a & ~15ull) + v * 16) : "memory");
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
  float adv = 0.f, old_lp = 0.f, ref_lp = 0.f;
  if (kPolicy && live) {
    adv = A.P.adv.at(seq, tok);
    old_lp = A.P.old_lp.at(seq, tok);
    if (A.P.ref_lp.p) ref_lp = A.P.ref_lp.at(seq, tok);
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncwarp();

  // lane r: takes the target out of its row, and what lies beside the row in its first and last word
  const uint32_t skew = static_cast<uint32_t>(addr & 15) / sizeof(T);   // elements in front of the row
  const uint32_t w_begin = skew / W::kPer, w_end = (skew + R.vocab + W::kPer - 1) / W::kPer;
  uint32_t* const mine = reinterpret_cast<uint32_t*>(base + static_cast<size_t>(lane) * A.pitch);
  float zy = NAN;
  if (live) {
    if (W::kPer == 2) {
      if (skew & 1) mine[w_begin] = W::drop(mine[w_begin], 0);
      if ((skew + R.vocab) & 1) mine[w_end - 1] = W::drop(mine[w_end - 1], 1);
    }
    if (has_y) {
      const uint32_t e = skew + y, w = e / W::kPer;
      zy = W::kPer == 2 ? ((e & 1) ? hi_bf16(mine[w]) : lo_bf16(mine[w])) : __uint_as_float(mine[w]);
      mine[w] = W::drop(mine[w], e % W::kPer);
    }
  }
  __syncwarp();

  float m_mine = kNegInf, s_mine = 0.f;
  for (int r = 0; r < rows; ++r) {
    if (!(live_rows >> r & 1)) continue;
    const uint32_t b = __shfl_sync(0xffffffffu, w_begin, r), e = __shfl_sync(0xffffffffu, w_end, r);
    const uint32_t* row = reinterpret_cast<const uint32_t*>(base + static_cast<size_t>(r) * A.pitch);
    uint32_t top = W::kEmpty;
#pragma unroll 4
    for (uint32_t w = b + lane; w < e; w += 32) top = W::max(top, row[w]);
    const float m = warp_max(W::top(top));
    const float mm = m == kNegInf ? 0.f : m;
    const Ex ex(mm, R.c_hi, R.c_lo);
    float s = 0.f, s2 = 0.f;
#pragma unroll 4
    for (uint32_t w = b + lane; w < e; w += 32) {
      const uint32_t v = row[w];
      if (W::kPer == 2) {
        float e0, e1;
        ex.two(lo_bf16(v), hi_bf16(v), e0, e1);
        s += e0;
        s2 += e1;
      } else {
        s += ex_one(__uint_as_float(v), mm, R.c_hi, R.c_lo);
      }
    }
    s = warp_sum(s + s2);
    if (lane == r) {
      m_mine = m;
      s_mine = s;
    }
  }

  // lane r: the row's values
  RowStat st = {0.0, 0.0, 0.f, 0.f};
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  float g = 0.f;
  if (live) {
    st = row_stat(zy, m_mine, s_mine, R.inv_t);
    if (kPolicy) {
      const RowLoss L = policy_row_loss(st.logp, A.P, old_lp, ref_lp, A.P.ref_lp.p != nullptr, adv);
      const double w = wt, inv = A.P.div ? 1.0 / static_cast<double>(*A.P.div) : A.P.inv_div;
      part[0] = w * L.loss * inv;
      part[1] = w;
      part[2] = w * L.kl * inv;
      part[3] = L.clipped ? w : 0.0;
      g = static_cast<float>(w * L.slope * inv * R.inv_t);
    }
  }
  if (lane < rows) {
    const uint32_t row = first + lane;
    if (A.logp) A.logp[row] = static_cast<float>(st.logp);
    if (A.lse) A.lse[row] = static_cast<float>(st.lse);
    if (A.logp64) {
      A.logp64[row] = st.logp;
      A.coef[row] = 0.f;
    }
  }
  if (!kPolicy) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double v = warp_sum(part[k]);
    if (lane == k) A.partials[static_cast<size_t>(tile) * 4 + k] = v;
  }
  if (A.grad == nullptr) return;

  const float gf = -g * st.f;
  for (int r = 0; r < rows; ++r) {
    T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(first + r) * R.vocab;
    const bool on = live_rows >> r & 1;
    const uint32_t b = __shfl_sync(0xffffffffu, w_begin, r), e = __shfl_sync(0xffffffffu, w_end, r);
    const uint32_t sk = __shfl_sync(0xffffffffu, skew, r);
    const float k = __shfl_sync(0xffffffffu, gf, r);
    const float m = __shfl_sync(0xffffffffu, m_mine, r);
    const uint32_t* row = reinterpret_cast<const uint32_t*>(base + static_cast<size_t>(r) * A.pitch);
    if (!on) {
      for (uint32_t j = lane; j < R.vocab; j += 32) store_one(out + j, 0.f);
      continue;
    }
    const float mm = m == kNegInf ? 0.f : m;
    if (W::kPer == 2) {
      const Ex ex(mm, R.c_hi, R.c_lo);
      // the output's pairs fall on 4 bytes where its row's alignment has the parity of the input's
      const bool wide = ((reinterpret_cast<uint64_t>(out) >> 1) & 1) == (sk & 1);
      T* const o = out - static_cast<int>(sk);
#pragma unroll 4
      for (uint32_t w = b + lane; w < e; w += 32) {
        float e0, e1;
        const uint32_t v = row[w];
        ex.two(lo_bf16(v), hi_bf16(v), e0, e1);
        const uint32_t d = to_bf16x2(e0 * k, e1 * k);
        const bool in0 = 2 * w >= sk, in1 = 2 * w + 1 < sk + R.vocab;
        if (wide && in0 && in1) {
          *reinterpret_cast<uint32_t*>(o + 2 * w) = d;
        } else {
          if (in0) *reinterpret_cast<uint16_t*>(o + 2 * w) = static_cast<uint16_t>(d);
          if (in1) *reinterpret_cast<uint16_t*>(o + 2 * w + 1) = static_cast<uint16_t>(d >> 16);
        }
      }
    } else {
#pragma unroll 4
      for (uint32_t w = b + lane; w < e; w += 32)
        store_one(out + (w - b), ex_one(__uint_as_float(row[w]), mm, R.c_hi, R.c_lo) * k);
    }
  }
  __syncwarp();   // the targets' elements, written as 0 above
  if (has_y) store_one(static_cast<T*>(A.grad) + static_cast<size_t>(first + lane) * R.vocab + y, g * st.rest);
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

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void store_remote(void* local, uint32_t rank, float a, float b) {   // 8 bytes in rank's copy
  uint32_t dst;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(dst), "f"(a), "f"(b) : "memory");
}

constexpr int kMaxCluster = 16;

// The sums of a row from its threads' parts, given to every thread. One block, or a cluster of `cl` blocks whose warps 0
// write their block's part into every block's shared memory.
template <int kThreads>
__device__ __forceinline__ Part row_join(Part p, int cl, uint32_t rank, float inv_t, Part* sh_warp, Part* sh_block) {
  constexpr int kWarps = kThreads / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  p = warp_join(p, inv_t);
  if (lane == 0) sh_warp[warp] = p;
  __syncthreads();
  Part b = lane < kWarps ? sh_warp[lane] : Part{kNegInf, 0.f};
  b = warp_join(b, inv_t);
  if (cl > 1) {
    cluster_wait();   // every block of the cluster runs (arrived at its start)
    if (warp == 0 && lane < cl) store_remote(sh_block + rank, lane, b.m, b.s);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    b = lane < cl ? sh_block[lane] : Part{kNegInf, 0.f};
    b = warp_join(b, inv_t);
  }
  return b;
}

// ---------------------------------------------------------------------------------------------------------------------
// Long rows, forward only: a row per block (or per cluster of blocks where there are few rows), read once in vectors with a
// running maximum and sum per thread.
struct RowArgs {
  Rows R;
  int cl;               // blocks per row
  float* logp;
  float* lse;
  double* logp64;
  float* coef;
};
constexpr int kRowThreads = 256;

template <typename T>
__global__ void __launch_bounds__(kRowThreads) row_kernel(const __grid_constant__ RowArgs A) {
  constexpr int kUnroll = 4;
  using W = Word<T>;
  __shared__ Part sh_warp[kRowThreads / 32], sh_block[kMaxCluster];
  const Rows& R = A.R;
  const uint32_t rank = A.cl > 1 ? cluster_rank() : 0;
  const uint32_t row = blockIdx.x / A.cl;
  MO_CHECK(row < R.n && rank < static_cast<uint32_t>(A.cl));
  pdl_go();
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const int64_t y64 = in_packed(R, row) ? R.y[seq * R.y_seq + tok * R.y_tok] : -1;
  if (y64 < 0) {   // the whole cluster
    if (rank == 0 && threadIdx.x == 0) {
      if (A.logp) A.logp[row] = 0.f;
      if (A.lse) A.lse[row] = 0.f;
      if (A.logp64) {
        A.logp64[row] = 0.0;
        A.coef[row] = 0.f;
      }
    }
    return;
  }
  if (A.cl > 1) cluster_arrive();
  const T* const z = reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok);
  const bool has_y = y64 < static_cast<int64_t>(R.vocab);
  const uint32_t y = has_y ? static_cast<uint32_t>(y64) : 0xffffffffu;
  const Split<T> sp(z, R.vocab);
  const float zy = has_y ? load_one(z + y) : NAN;
  const float inv_t = static_cast<float>(R.inv_t);
  const uint32_t yv = has_y && y >= sp.head ? (y - sp.head) / sp.kPer : 0xffffffffu, ye = (y - sp.head) % sp.kPer;
  const uint32_t share = (sp.vecs + A.cl - 1) / A.cl, begin = rank * share, end = min(begin + share, sp.vecs);
  const uint4* const zv = reinterpret_cast<const uint4*>(z + sp.head);
  Part p = {kNegInf, 0.f};
  if (rank == 0 && threadIdx.x < sp.head + sp.tail) {
    const uint32_t j = sp.edge(threadIdx.x);
    if (j != y) {
      p.m = load_one(z + j);
      p.s = p.m == kNegInf ? 0.f : ex_one(p.m, p.m, R.c_hi, R.c_lo);   // 1, or NaN
    }
  }
  for (uint32_t i = begin + threadIdx.x; i < end; i += kRowThreads * kUnroll) {
    uint4 v[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const uint32_t at = i + k * kRowThreads;
      v[k] = make_uint4(W::kEmpty, W::kEmpty, W::kEmpty, W::kEmpty);
      if (at < end) v[k] = load_vec(zv + at);
    }
    uint32_t top = W::kEmpty;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      if (i + k * kRowThreads == yv) drop_target<T>(v[k], ye);
      top = vec_max<T>(top, v[k]);
    }
    const float t = W::top(top);
    if (t > p.m) {
      p.s *= rescale(p.m, t, inv_t);
      p.m = t;
    }
    const float mm = p.m == kNegInf ? 0.f : p.m;
    const Ex ex(mm, R.c_hi, R.c_lo);
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
      const uint32_t q[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
      float e0, e1;
      if (W::kPer == 2) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          ex.two(lo_bf16(q[u]), hi_bf16(q[u]), e0, e1);
          s0 += e0;
          s1 += e1;
        }
      } else {
#pragma unroll
        for (int u = 0; u < 4; u += 2) {
          ex.two(__uint_as_float(q[u]), __uint_as_float(q[u + 1]), e0, e1);
          s0 += e0;
          s1 += e1;
        }
      }
    }
    p.s += s0 + s1;
  }
  p = row_join<kRowThreads>(p, A.cl, rank, inv_t, sh_warp, sh_block);
  if (rank == 0 && threadIdx.x == 0) {
    const RowStat st = row_stat(zy, p.m, p.s, R.inv_t);
    if (A.logp) A.logp[row] = static_cast<float>(st.logp);
    if (A.lse) A.lse[row] = static_cast<float>(st.lse);
    if (A.logp64) {
      A.logp64[row] = st.logp;
      A.coef[row] = 0.f;
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Long rows, the policy loss and its gradient in one pass: a row's exponentials stay in the registers of one block, or of a
// cluster of blocks (32 a thread), relative to each thread's own maximum; when the row's sum is known each thread scales
// them by one factor. Each logit is read once, exponentiated once, and its gradient written once.
struct HeldArgs {
  Rows R;
  int cl;
  float* logp;
  Policy P;
  void* grad;
  double* partials;     // [n][4]
};

template <typename T, int kThreads>
__global__ void __launch_bounds__(kThreads) held_kernel(const __grid_constant__ HeldArgs A) {
  using W = Word<T>;
  constexpr int kPer = 16 / sizeof(T), kVecs = 32 / kPer;
  __shared__ Part sh_warp[kThreads / 32], sh_block[kMaxCluster];
  __shared__ float sh_g[2];
  __shared__ float sh_in[4];   // the row's target logit, advantage, old and reference log-probability
  const Rows& R = A.R;
  const uint32_t rank = A.cl > 1 ? cluster_rank() : 0;
  const uint32_t row = blockIdx.x / A.cl;
  MO_CHECK(row < R.n && rank < static_cast<uint32_t>(A.cl));
  pdl_go();
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const int64_t y64 = R.y[seq * R.y_seq + tok * R.y_tok];
  const T* const z = reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok);
  T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(row) * R.vocab;
  const Split<T> sp(z, R.vocab);
  const Split<T> so(out, R.vocab);
  const uint32_t share = (sp.vecs + A.cl - 1) / A.cl, begin = rank * share, end = min(begin + share, sp.vecs);
  MO_CHECK(share <= static_cast<uint32_t>(kThreads * kVecs));
  const bool wide = so.head == sp.head;   // both rows start at the same place of a 16-byte line
  const bool edge = rank == 0 && threadIdx.x < sp.head + sp.tail;
  const uint32_t je = sp.edge(threadIdx.x);
  if (y64 < 0 || (A.P.weight.p && A.P.weight.at(seq, tok) == 0.f)) {   // the whole cluster
    if (rank == 0 && threadIdx.x < 4) {
      A.partials[static_cast<size_t>(row) * 4 + threadIdx.x] = 0.0;
      if (threadIdx.x == 0) A.logp[row] = 0.f;
    }
    if (A.grad) {
      if (wide) {
        if (edge) store_one(out + je, 0.f);
        for (uint32_t i = begin + threadIdx.x; i < end; i += kThreads)
          reinterpret_cast<uint4*>(out + sp.head)[i] = make_uint4(0, 0, 0, 0);
      } else {
        for (uint32_t j = rank * kThreads + threadIdx.x; j < R.vocab; j += kThreads * A.cl) store_one(out + j, 0.f);
      }
    }
    return;
  }
  if (A.cl > 1) cluster_arrive();
  const bool has_y = y64 < static_cast<int64_t>(R.vocab);
  const uint32_t y = has_y ? static_cast<uint32_t>(y64) : 0xffffffffu;
  const uint32_t yv = has_y && y >= sp.head ? (y - sp.head) / kPer : 0xffffffffu, ye = (y - sp.head) % kPer;
  const uint4* const zv = reinterpret_cast<const uint4*>(z + sp.head);
  uint4 v[kVecs];
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const uint32_t at = begin + threadIdx.x + k * kThreads;
    v[k] = make_uint4(W::kEmpty, W::kEmpty, W::kEmpty, W::kEmpty);
    if (at < end) v[k] = load_vec(zv + at);
  }
  float xe = kNegInf;
  if (edge && je != y) xe = load_one(z + je);
  if (threadIdx.x < 4) {   // read by thread 0 behind row_join's barrier
    const Per& per = threadIdx.x == 1 ? A.P.adv : threadIdx.x == 2 ? A.P.old_lp : A.P.ref_lp;
    float x = NAN;
    if (threadIdx.x == 0) {
      if (has_y) x = load_one(z + y);
    } else if (per.p) {
      x = per.at(seq, tok);
    }
    sh_in[threadIdx.x] = x;
  }
  uint32_t top = W::kEmpty;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    if (begin + threadIdx.x + k * kThreads == yv) drop_target<T>(v[k], ye);
    top = vec_max<T>(top, v[k]);
  }
  const float m = fmaxf(W::top(top), xe), mm = m == kNegInf ? 0.f : m;
  const Ex ex(mm, R.c_hi, R.c_lo);
  float e[32], s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const uint32_t q[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
    if (W::kPer == 2) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        ex.two(lo_bf16(q[u]), hi_bf16(q[u]), e[k * 8 + 2 * u], e[k * 8 + 2 * u + 1]);
        s0 += e[k * 8 + 2 * u];
        s1 += e[k * 8 + 2 * u + 1];
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; u += 2) {
        ex.two(__uint_as_float(q[u]), __uint_as_float(q[u + 1]), e[k * 4 + u], e[k * 4 + u + 1]);
        s0 += e[k * 4 + u];
        s1 += e[k * 4 + u + 1];
      }
    }
  }
  const float ee = ex_one(xe, mm, R.c_hi, R.c_lo);
  const float inv_t = static_cast<float>(R.inv_t);
  const Part p = row_join<kThreads>(Part{m, s0 + s1 + ee}, A.cl, rank, inv_t, sh_warp, sh_block);
  if (threadIdx.x == 0) {
    const RowStat st = row_stat(sh_in[0], p.m, p.s, R.inv_t);
    const RowLoss L = policy_row_loss(st.logp, A.P, sh_in[2], sh_in[3], A.P.ref_lp.p != nullptr, sh_in[1]);
    const double w = A.P.weight.p ? A.P.weight.at(seq, tok) : 1.f;
    const double inv = A.P.div ? 1.0 / static_cast<double>(*A.P.div) : A.P.inv_div;
    const float g = static_cast<float>(w * L.slope * inv * R.inv_t);
    sh_g[0] = -g * st.f;
    sh_g[1] = g * st.rest;
    if (rank == 0) {
      A.logp[row] = static_cast<float>(st.logp);
      double* const o = A.partials + static_cast<size_t>(row) * 4;
      o[0] = w * L.loss * inv;
      o[1] = w;
      o[2] = w * L.kl * inv;
      o[3] = L.clipped ? w : 0.0;
    }
  }
  if (A.grad == nullptr) return;
  __syncthreads();
  const float f = sh_g[0] * rescale(m, p.m, inv_t), gy = sh_g[1];
  if (edge) store_one(out + je, je == y ? gy : ee * f);
#pragma unroll
  for (int k = 0; k < kVecs; ++k) {
    const uint32_t at = begin + threadIdx.x + k * kThreads;
    if (at >= end) continue;
    T* const o = out + sp.head + at * kPer;
    if (wide) {
      uint4 d;
      if (W::kPer == 2) {
        d.x = to_bf16x2(e[k * 8] * f, e[(k * 8 + 1) & 31] * f);
        d.y = to_bf16x2(e[(k * 8 + 2) & 31] * f, e[(k * 8 + 3) & 31] * f);
        d.z = to_bf16x2(e[(k * 8 + 4) & 31] * f, e[(k * 8 + 5) & 31] * f);
        d.w = to_bf16x2(e[(k * 8 + 6) & 31] * f, e[(k * 8 + 7) & 31] * f);
      } else {
        d = make_uint4(__float_as_uint(e[k * 4] * f), __float_as_uint(e[(k * 4 + 1) & 31] * f),
                       __float_as_uint(e[(k * 4 + 2) & 31] * f), __float_as_uint(e[(k * 4 + 3) & 31] * f));
      }
      *reinterpret_cast<uint4*>(o) = d;
    } else {
#pragma unroll
      for (int u = 0; u < kPer; ++u) store_one(o + u, e[k * kPer + u] * f);
    }
    if (at == yv) store_one(o + ye, gy);
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The gradient from kept row values: d_j = g ([j == y] - exp(x_j - lse)) / T with one coefficient g per row. Elementwise, so
// a row may be cut anywhere. Rows with g = 0 are written as zeros and not read.
struct GradArgs {
  Rows R;
  Per logp, lse, coef;    // per position ...
  const double* logp64;   // ... or by row: the preference loss's own [n] arrays
  const float* lse_row;
  const float* coef_row;
  void* grad;
  uint32_t pieces;        // blocks per row (grad_kernel)
  const double* pair_loss;   // preference: block 0 adds up the pairs' losses
  int pairs;
  float* loss;
};
struct GradRow {
  bool live;
  uint32_t y;
  float g, gy, l_hi, l_lo;   // g / T, the target's gradient, lse log2(e) as two floats
};
__device__ __forceinline__ GradRow grad_row(const GradArgs& A, uint32_t row, uint32_t seq, uint32_t tok) {
  const Rows& R = A.R;
  GradRow r;
  r.y = 0xffffffffu;
  const int64_t y64 = R.y[seq * R.y_seq + tok * R.y_tok];
  const float c = A.coef_row ? A.coef_row[row] : A.coef.at(seq, tok);
  r.live = y64 >= 0 && c != 0.f;
  if (!r.live) return r;
  const double lse = A.lse_row ? A.lse_row[row] : A.lse.at(seq, tok);
  const double lp = A.logp64 ? A.logp64[row] : static_cast<double>(A.logp.at(seq, tok));
  r.g = static_cast<float>(c * R.inv_t);
  r.gy = static_cast<float>(-expm1(lp) * c * R.inv_t);
  r.l_hi = static_cast<float>(lse * kLog2e);
  r.l_lo = static_cast<float>(lse * kLog2e - static_cast<double>(r.l_hi));
  if (y64 < static_cast<int64_t>(R.vocab)) r.y = static_cast<uint32_t>(y64);
  return r;
}
struct GradEx {   // -g 2^(z c - lse log2(e)): the large product and its small rest are rounded apart, then added
  uint64_t hi, lo, l_hi, l_lo, g;
  __device__ GradEx(const GradRow& r, const Rows& R)
      : hi(pack2(R.c_hi, R.c_hi)), lo(pack2(R.c_lo, R.c_lo)), l_hi(pack2(-r.l_hi, -r.l_hi)), l_lo(pack2(-r.l_lo, -r.l_lo)),
        g(pack2(-r.g, -r.g)) {}
  __device__ __forceinline__ void two(float z0, float z1, float& d0, float& d1) const {
    const uint64_t z = pack2(z0, z1);
    float t0, t1;
    unpack2(add2(fma2(z, hi, l_hi), fma2(z, lo, l_lo)), t0, t1);
    unpack2(mul2(pack2(ex2(t0), ex2(t1)), g), d0, d1);
  }
  __device__ __forceinline__ float one(float z) const {
    float d0, d1;
    two(z, z, d0, d1);
    return d0;
  }
};
constexpr int kGradThreads = 256, kGradVecs = 4;

__device__ __forceinline__ void sum_pairs(const GradArgs& A) {   // one warp, in a fixed order
  const int lane = threadIdx.x & 31;
  double v = 0.0;
  for (int i = lane; i < A.pairs; i += 32) v += A.pair_loss[i];
  v = warp_sum(v);
  if (lane == 0) *A.loss = static_cast<float>(v);
}

template <typename T>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const __grid_constant__ GradArgs A) {
  const Rows& R = A.R;
  constexpr int kPer = 16 / sizeof(T);
  const uint32_t row = blockIdx.x / A.pieces, piece = blockIdx.x - row * A.pieces;
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const T* const z = reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok);
  T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(row) * R.vocab;
  const Split<T> sp(z, R.vocab);
  const bool wide = Split<T>(out, R.vocab).head == sp.head;
  pdl_wait();
  if (A.pair_loss && blockIdx.x == 0 && threadIdx.x < 32) sum_pairs(A);
  MO_CHECK(row < R.n);
  const GradRow r = grad_row(A, row, seq, tok);
  const uint32_t begin = piece * (kGradThreads * kGradVecs) + threadIdx.x;
  const bool edge = piece == 0 && threadIdx.x < sp.head + sp.tail;
  const uint32_t je = sp.edge(threadIdx.x);
  if (!r.live) {
    if (edge) store_one(out + je, 0.f);
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k) {
      const uint32_t at = begin + k * kGradThreads;
      if (at >= sp.vecs) break;
      T* const o = out + sp.head + at * kPer;
      if (wide) {
        *reinterpret_cast<uint4*>(o) = make_uint4(0, 0, 0, 0);
      } else {
#pragma unroll
        for (int u = 0; u < kPer; ++u) store_one(o + u, 0.f);
      }
    }
    return;
  }
  const GradEx ex(r, R);
  const uint32_t yv = r.y != 0xffffffffu && r.y >= sp.head ? (r.y - sp.head) / kPer : 0xffffffffu, ye = (r.y - sp.head) % kPer;
  const uint4* const zv = reinterpret_cast<const uint4*>(z + sp.head);
  uint4 v[kGradVecs];
#pragma unroll
  for (int k = 0; k < kGradVecs; ++k) {
    const uint32_t at = begin + k * kGradThreads;
    if (at < sp.vecs) v[k] = load_vec(zv + at);
  }
  if (edge) store_one(out + je, je == r.y ? r.gy : ex.one(load_one(z + je)));
#pragma unroll
  for (int k = 0; k < kGradVecs; ++k) {
    const uint32_t at = begin + k * kGradThreads;
    if (at >= sp.vecs) break;
    const uint32_t q[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
    T* const o = out + sp.head + at * kPer;
    uint32_t d[4];
    if (sizeof(T) == 2) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float d0, d1;
        ex.two(lo_bf16(q[u]), hi_bf16(q[u]), d0, d1);
        d[u] = to_bf16x2(d0, d1);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; u += 2) {
        float d0, d1;
        ex.two(__uint_as_float(q[u]), __uint_as_float(q[u + 1]), d0, d1);
        d[u] = __float_as_uint(d0);
        d[u + 1] = __float_as_uint(d1);
      }
    }
    if (wide) {
      *reinterpret_cast<uint4*>(o) = make_uint4(d[0], d[1], d[2], d[3]);
    } else if (sizeof(T) == 2) {
#pragma unroll
      for (int u = 0; u < kPer; ++u) reinterpret_cast<uint16_t*>(o)[u] = static_cast<uint16_t>(d[u >> 1] >> (16 * (u & 1)));
    } else {
#pragma unroll
      for (int u = 0; u < kPer; ++u) reinterpret_cast<uint32_t*>(o)[u] = d[u & 3];
    }
    if (at == yv) store_one(o + ye, r.gy);
  }
}

// Short rows: a warp per row, in words of 4 bytes (16-byte vectors would leave most lanes of a row of a few hundred logits
// without one).
template <typename T>
__global__ void __launch_bounds__(kGradThreads) grad_short_kernel(const __grid_constant__ GradArgs A) {
  using W = Word<T>;
  const Rows& R = A.R;
  const int lane = threadIdx.x & 31;
  const uint32_t row = blockIdx.x * (kGradThreads / 32) + (threadIdx.x >> 5);
  pdl_wait();
  if (A.pair_loss && blockIdx.x == 0 && threadIdx.x < 32) sum_pairs(A);
  if (row >= R.n) return;
  const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
  const T* const z = reinterpret_cast<const T*>(R.z) + (seq * R.z_seq + tok * R.z_tok);
  T* const out = static_cast<T*>(A.grad) + static_cast<size_t>(row) * R.vocab;
  const GradRow r = grad_row(A, row, seq, tok);
  if (!r.live) {
    for (uint32_t j = lane; j < R.vocab; j += 32) store_one(out + j, 0.f);
    return;
  }
  const GradEx ex(r, R);
  // words of the input; an output whose row has the other parity is stored element by element
  const uint32_t sk = W::kPer == 2 ? (reinterpret_cast<uint64_t>(z) >> 1) & 1 : 0;
  const bool wide = W::kPer == 1 || ((reinterpret_cast<uint64_t>(out) >> 1) & 1) == sk;
  const uint32_t words = (sk + R.vocab + W::kPer - 1) / W::kPer;
  const T* const zw = z - sk;
  T* const ow = out - sk;
#pragma unroll 4
  for (uint32_t w = lane; w < words; w += 32) {
    if (W::kPer == 1) {
      store_one(out + w, w == r.y ? r.gy : ex.one(load_one(z + w)));
      continue;
    }
    const uint32_t j = 2 * w - sk;   // wraps where only the second element lies in the row
    const bool in0 = j < R.vocab, in1 = j + 1 < R.vocab;
    float z0 = 0.f, z1 = 0.f;
    if (in0 && in1) {
      const uint32_t v = *reinterpret_cast<const uint32_t*>(zw + 2 * w);
      z0 = lo_bf16(v);
      z1 = hi_bf16(v);
    } else if (in0) {
      z0 = load_one(zw + 2 * w);
    } else {
      z1 = load_one(zw + 2 * w + 1);
    }
    float d0, d1;
    ex.two(z0, z1, d0, d1);
    if (j == r.y) d0 = r.gy;
    if (j + 1 == r.y) d1 = r.gy;
    const uint32_t d = to_bf16x2(d0, d1);
    if (wide && in0 && in1) {
      *reinterpret_cast<uint32_t*>(ow + 2 * w) = d;
    } else {
      if (in0) *reinterpret_cast<uint16_t*>(ow + 2 * w) = static_cast<uint16_t>(d);
      if (in1) *reinterpret_cast<uint16_t*>(ow + 2 * w + 1) = static_cast<uint16_t>(d >> 16);
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Row values of the policy loss from kept log-probabilities (rows too long to be held): a thread per row.
struct PolicyRowsArgs {
  Rows R;
  Policy P;
  const double* logp64;
  float* logp;
  float* coef;
  double* partials;       // [blocks][4]
};
__global__ void __launch_bounds__(256) policy_rows_kernel(const __grid_constant__ PolicyRowsArgs A) {
  const Rows& R = A.R;
  __shared__ double sh[8][4];
  const uint32_t row = blockIdx.x * 256 + threadIdx.x;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_go();
  double part[4] = {0.0, 0.0, 0.0, 0.0};
  if (row < R.n) {
    const uint32_t seq = row / R.tokens, tok = row - seq * R.tokens;
    const float wt = A.P.weight.p ? A.P.weight.at(seq, tok) : 1.f;
    const bool live = R.y[seq * R.y_seq + tok * R.y_tok] >= 0 && wt != 0.f;
    float g = 0.f, lp = 0.f;
    if (live) {
      const double l = A.logp64[row];
      const RowLoss L = policy_row_loss(l, A.P, A.P.old_lp.at(seq, tok), A.P.ref_lp.p ? A.P.ref_lp.at(seq, tok) : 0.f,
                                        A.P.ref_lp.p != nullptr, A.P.adv.at(seq, tok));
      const double w = wt, inv = A.P.div ? 1.0 / static_cast<double>(*A.P.div) : A.P.inv_div;
      part[0] = w * L.loss * inv;
      part[1] = w;
      part[2] = w * L.kl * inv;
      part[3] = L.clipped ? w : 0.0;
      g = static_cast<float>(w * L.slope * inv);
      lp = static_cast<float>(l);
    }
    A.coef[row] = g;
    A.logp[row] = lp;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const double v = warp_sum(part[k]);
    if (lane == 0) sh[warp][k] = v;
  }
  __syncthreads();
  if (threadIdx.x < 4) {
    double v = 0.0;
    for (int w = 0; w < 8; ++w) v += sh[w][threadIdx.x];
    A.partials[static_cast<size_t>(blockIdx.x) * 4 + threadIdx.x] = v;
  }
}

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
constexpr int kPairThreads = 256;
__global__ void __launch_bounds__(kPairThreads) pair_kernel(const __grid_constant__ PairArgs A) {
  const Rows& R = A.R;
  __shared__ double sh_s[2][kPairThreads / 32];
  __shared__ int sh_n[2][kPairThreads / 32];
  __shared__ float sh_c[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  pdl_go();
  int64_t b[2], e[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t q = blockIdx.x + static_cast<int64_t>(k) * A.pairs, n = R.n;
    if (R.cu) {   // held to the rows there are
      b[k] = min(max(static_cast<int64_t>(R.cu[q]), static_cast<int64_t>(0)), n);
      e[k] = min(max(static_cast<int64_t>(R.cu[q + 1]), b[k]), n);
    } else {
      b[k] = q * R.tokens;
      e[k] = b[k] + R.tokens;
    }
    double s = 0.0;
    int cnt = 0;
    for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kPairThreads) {
      const uint32_t row = static_cast<uint32_t>(i), seq = row / R.tokens, tok = row - seq * R.tokens;
      MO_CHECK(row < R.n);
      if (R.y[seq * R.y_seq + tok * R.y_tok] >= 0) {
        s += A.logp64[i];
        ++cnt;
      }
    }
    s = warp_sum(s);
    cnt = __reduce_add_sync(0xffffffffu, cnt);
    if (lane == 0) {
      sh_s[k][warp] = s;
      sh_n[k][warp] = cnt;
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    double s[2], n[2], rw[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      double t = 0.0;
      int c = 0;
      for (int w = 0; w < kPairThreads / 32; ++w) {
        t += sh_s[k][w];
        c += sh_n[k][w];
      }
      n[k] = A.average ? static_cast<double>(max(c, 1)) : 1.0;
      s[k] = t / n[k];
      const int q = blockIdx.x + k * A.pairs;
      rw[k] = A.beta * (s[k] - (A.ref ? static_cast<double>(A.ref[q]) : 0.0));
      A.rewards[q] = static_cast<float>(rw[k]);
      A.seq_logp[q] = static_cast<float>(s[k]);
    }
    const double u = rw[0] - rw[1], inv = A.div ? 1.0 / static_cast<double>(*A.div) : A.inv_div;
    // -log sigmoid(u) = max(-u, 0) + log1p(e^-|u|); sigmoid(-u) = e^-|u| / (1 + e^-|u|) or 1 / (1 + e^-|u|)
    const double t = exp(-fabs(u)), l = log1p(t);
    const double up = (u > 0.0 ? 0.0 : -u) + l, down = (u < 0.0 ? 0.0 : u) + l;
    const double sn = (u >= 0.0 ? t : 1.0) / (1.0 + t), sp = (u >= 0.0 ? 1.0 : t) / (1.0 + t);
    A.pair_loss[blockIdx.x] = ((1.0 - A.eps) * up + A.eps * down) * inv;
    const double du = A.beta * (A.eps * sp - (1.0 - A.eps) * sn) * inv;
    sh_c[0] = static_cast<float>(du / n[0]);
    sh_c[1] = static_cast<float>(-du / n[1]);
  }
  if (A.coef == nullptr) return;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float c = sh_c[k];
    for (int64_t i = b[k] + threadIdx.x; i < e[k]; i += kPairThreads) A.coef[i] = c;
  }
}

// The pairs' losses added up where no gradient pass does it
__global__ void __launch_bounds__(32) pair_sum_kernel(const __grid_constant__ GradArgs A) {
  pdl_wait();
  sum_pairs(A);
}

}  // namespace loss
}  // namespace moteopt
