// token_kernels.cuh -- log-probabilities of tokens from a policy's logits, and
// the gradients that flow back into the logits.
//
// A row is one step's logits x[0..V).  With z = x / temperature,
//   lse = log sum_v exp z_v,  p_v = exp(z_v - lse),
//   logprob = z_tok - lse,    entropy H = lse - sum_v p_v z_v,
//   d logprob / d x_v = (1[v = tok] - p_v) / temperature,
//   d H / d x_v       = -p_v (log p_v + H) / temperature.
// Everything is computed in base 2: with c = log2(e) / temperature and an
// offset M (an element near the maximum, times c, rounded to a whole number, and 9),
//   d_v = x_v c - M,  S0 = sum 2^d_v,  S1 = sum 2^d_v d_v,  t = S1 / S0,
//   logprob = ln2 (d_tok - log2 S0),   H = ln2 (log2 S0 - t),
// one fused multiply-add and one ex2 an element, and the gradient for incoming
// (a, b) of (logprob, H) is
//   a 1[v = tok] / temperature - 2^d_v (A + B d_v),
//   A = (a - b ln2 t) / (S0 temperature),  B = b ln2 / (S0 temperature).
// The sums and the row's statistics are fp32 (each thread's partial sum covers
// at most V / threads elements); the logprob itself is formed in fp64 from
// them, so that it is rounded once.
#pragma once
#include <math.h>

#include "common.cuh"
#include "rlscan.h"

namespace rls {
namespace tok {

constexpr float kLn2 = 0.693147180559945309f;
// Where a row's maximum is so large that M = m c is rounded by whole units
// (logits at the type's lowest value in a whole row, infinities), x c - M is
// useless and S0 leaves [kLeast, kMost]; such rows, and rows with NaN, are
// summed again with d = (x - m) c, the far form.
constexpr float kFar = 1e15f;
constexpr float kLeast = 2e-4f, kMost = 1e12f;
// An offset stays until an element lies this far (in powers of two) above where
// it put its own: any offset near the maximum serves, and a warp whose lanes each kept
// their own maximum would move one of them at almost every step.  Offsets lie kLift above the
// element, so that every d is below 0: ex2.approx is off to one side there, to
// the other above 0 (see logprob_of).
constexpr float kSlack = 8.f, kLift = 9.f;
constexpr float kDeep = -16384.f;  // 2^kDeep is 0: keeps 2^d * d finite at d = -inf

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 lanes in one instruction.
struct F2 {
  unsigned long long u;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.u) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void split(F2 a, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(a.u));
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 ex2(F2 a) {
  float x, y;
  split(a, x, y);
  return f2(ex2(x), ex2(y));
}

// ---- mask ------------------------------------------------------------------
// One element a step, any of the types below; non-zero counts (NaN too).
struct Mask {
  const void* p;
  int kind;  // RLS_MASK_*
};

__device__ __forceinline__ bool mask_at(const Mask& m, int64_t i) {
  switch (m.kind) {
    case RLS_MASK_U8: return reinterpret_cast<const uint8_t*>(m.p)[i] != 0;
    case RLS_MASK_F32: return reinterpret_cast<const float*>(m.p)[i] != 0.f;
    case RLS_MASK_BF16: return bf16_bits_to_float(reinterpret_cast<const unsigned short*>(m.p)[i]) != 0.f;
    case RLS_MASK_I32: return reinterpret_cast<const int32_t*>(m.p)[i] != 0;
    case RLS_MASK_I64: return reinterpret_cast<const int64_t*>(m.p)[i] != 0;
    default: return true;
  }
}

// Bits 0 .. 3: steps i .. i + 3 (i a multiple of 4; none past the end M).
__device__ __forceinline__ unsigned mask_four(const Mask& m, int64_t i, int64_t M) {
  if (m.kind == RLS_MASK_NONE) return i + 4 <= M ? 15u : (1u << (M - i)) - 1u;
  if (m.kind == RLS_MASK_U8 && i + 4 <= M && ((uintptr_t)m.p & 3) == 0) {
    const unsigned w = *reinterpret_cast<const unsigned*>(reinterpret_cast<const uint8_t*>(m.p) + i);
    return ((w & 0xffu) != 0) | ((w & 0xff00u) != 0) << 1 | ((w & 0xff0000u) != 0) << 2 | ((w & 0xff000000u) != 0) << 3;
  }
  unsigned b = 0;
  for (int e = 0; e < 4; ++e)
    if (i + e < M && mask_at(m, i + e)) b |= 1u << e;
  return b;
}

// ---- rows ------------------------------------------------------------------
// row / seq by a multiplication, for rows below 2^31 (else by a division):
// q = (umulhi(n, mul) + n) >> shift, shift = ceil(log2 seq),
// mul = ceil(2^(32 + shift) / seq) - 2^32.
struct Divide {
  int64_t by;
  unsigned mul, shift;
  bool wide;
  __host__ static Divide of(int64_t by, int64_t most) {
    Divide d{by, 0, 0, most > 0x7fffffffLL || by > 0x7fffffffLL};
    if (d.wide) return d;
    while ((1LL << d.shift) < by) ++d.shift;
    const unsigned long long two = 1ull << (32 + d.shift);
    d.mul = (unsigned)((two + (unsigned long long)by - 1) / (unsigned long long)by - (1ull << 32));
    return d;
  }
  __device__ __forceinline__ int64_t operator()(int64_t n) const {
    if (wide) return n / by;
    const unsigned m = (unsigned)n;
    return (int64_t)((__umulhi(m, mul) + m) >> shift);
  }
};

template <class T>
struct Rows {
  const T* x;          // logits
  int64_t es, ss;      // strides of env and step in elements
  int64_t rows, seq;   // rows = envs * seq
  Divide env;          // a row's env
  int V;
  const int64_t* tokens;
  Mask mask;
  const int* order;    // null, or what rls_row_order made of the mask
  float c;             // log2(e) / temperature, rounded
  double c64, c_off;   // the same, not rounded; c64 / c - 1
  float inv_temp;
  bool flat;           // es == seq * ss

  __device__ __forceinline__ int64_t at(int64_t row) const {
    if (flat) return row * ss;
    const int64_t e = env(row);
    return e * es + (row - e * seq) * ss;
  }
};

template <class T>
struct GradRows {
  T* g;
  int64_t es, ss;
  bool flat;
  bool alike;  // every row lies within 16 bytes as its logits do
  __device__ __forceinline__ int64_t at(int64_t row, const Rows<T>& in) const {
    if (flat) return row * ss;
    const int64_t e = in.env(row);
    return e * es + (row - e * in.seq) * ss;
  }
};

// What a row's reduction leaves: m the maximum that d is taken from, S0, t,
// and whether d has the far form.  alone: one element holds all of S0 and S1 (all others
// are exactly 0), so the entropy is 0 and not the rounding of its parts.
struct RowStats {
  float m, s0, t;
  bool far, alone;
  // long rows, near form: the share of S0 and the mean of d of all but the token
  float others = -1.f, t_others = 0.f;
};

// A long row's record (RLS_ROW_STATS floats, two 16-byte words): m, S0, t and
// flags; and, written by the policy loss, the derivative a of the loss by the
// row's log-probability, the weighted term, the KL estimate and the drift.
constexpr int kFlagClipped = 1, kFlagFar = 2, kFlagKept = 4;
__device__ __forceinline__ float4 stats_word(const RowStats& r, int flags) {
  return make_float4(r.m, r.s0, r.t, __int_as_float(flags | (r.far ? kFlagFar : 0)));
}
__device__ __forceinline__ RowStats stats_of(const float4& q) {
  return RowStats{q.x, q.y, q.z, (__float_as_int(q.w) & kFlagFar) != 0, false, -1.f, 0.f};
}

// d of one element under the row's statistics.
struct Shift {
  float c, off;  // d = x c - off, or (x - off) c in the far form
  bool far;
  __device__ __forceinline__ float operator()(float x) const { return far ? (x - off) * c : fmaf(x, c, -off); }
};
// What d is taken from: m c to a whole number, and kLift.  Sums move to a larger offset by a
// power of two then, exactly (ex2.approx of a whole number is one).
__device__ __forceinline__ float offset_of(float m, float c) { return rintf(m * c) + kLift; }
__device__ __forceinline__ Shift shift_of(const RowStats& r, float c) {
  return Shift{c, r.far ? r.m : offset_of(r.m, c), r.far};
}

__device__ __forceinline__ double log2_of(float s0) {
  int e;
  const float f = frexpf(s0, &e);
  return (double)e + (double)log2f(f);
}

// fp64, so that what follows from it (the ratio of the policy loss) does not
// carry the rounding of the fp32 output.  Two errors that S0 has in common over
// all rows are taken out to first order, since sums of many log-probabilities
// (the preference loss's) would add them up: c was rounded, which moves log S0 by
// the mean of d times the relative error; and ex2.approx lies 5.0e-8 low on
// average for d below 0 (measured; 3.4e-8 high above), except at the far form's
// maximum, where d is 0.
//
// Where the sum of the others is known apart from the token's term, q =
// (others / token's) gives logprob = -log(1 + q) with the relative accuracy of
// q, however close to 0 it is (a sum that the token's term dominates would not).
__device__ __forceinline__ double logprob_of(float x_tok, const RowStats& r, float c, double c64, double c_off) {
  const Shift sh = shift_of(r, c);
  if (!r.far && r.others >= 0.f) {
    if (x_tok == -INFINITY) return -INFINITY;  // c_off times an infinite d would be NaN
    const double d = (double)x_tok * (double)c - (double)sh.off;
    const double l = log2_of(r.others) - d + c_off * ((double)r.t_others - d) + 7.2e-8;  // log2 q
    if (l > 0.0) return -(l * 0.693147180559945309417 + (double)log1pf(exp2f(-(float)l)));
    const float lf = (float)l, low = lf > -INFINITY ? (float)(l - (double)lf) : 0.f;
    float q = exp2f(lf);
    q = fmaf(q, low * kLn2, q);
    return q == 0.f ? 0.0 : -(double)log1pf(q);
  }
  if (ex2(sh(x_tok)) == r.s0) return 0.0;  // the others are below fp32's reach
  const double res = r.far ? 0.0 : (double)r.m * (double)c - (double)sh.off;  // d at the maximum
  const double low = r.far ? 7.2e-8 * (double)(1.f - __frcp_rn(r.s0)) : 7.2e-8;
  const double log_s0 = log2_of(r.s0) - res + c_off * ((double)r.t - res) + low;
  return (((double)x_tok - (double)r.m) * c64 - log_s0) * 0.693147180559945309417;
}
__device__ __forceinline__ float entropy_of(const RowStats& r) {
  if (r.alone) return 0.f;
  return (float)((log2_of(r.s0) - (double)r.t) * 0.693147180559945309417);
}

// The gradient's coefficients for incoming (a, b) of (logprob, entropy).
struct RowGrad {
  float A, B;  // -2^d (A + B d), and at the token token_grad() instead
};
__device__ __forceinline__ RowGrad row_grad(float a, float b, const RowStats& r, float inv_temp) {
  const float k = inv_temp / r.s0, bl = b * kLn2;
  return RowGrad{(a - bl * r.t) * k, bl * k};
}
// At the token, from 1 - p with a p that is 1 where the token is all there is.
__device__ __forceinline__ float token_grad(float x, const Shift& sh, float a, float b, float s0, float t,
                                            float inv_temp) {
  const float d = sh(x);
  const float p = ex2(d) / s0;
  return inv_temp * (a * (1.f - p) - b * kLn2 * p * (fmaxf(d, kDeep) - t));
}
template <bool ENT>
__device__ __forceinline__ float grad_at(float x, const Shift& sh, const RowGrad& g) {
  const float d = sh(x);
  const float e = ex2(d);
  if constexpr (ENT) return -e * fmaf(g.B, fmaxf(d, kDeep), g.A);
  else return -e * g.A;
}

// ---- 16-byte vectors ---------------------------------------------------------
template <class T>
struct Vec;
template <>
struct Vec<float> {
  static constexpr int N = 4;
  static constexpr unsigned kLowest = 0xff800000u;  // -inf
  __device__ __forceinline__ static void unpack(const uint4& u, float (&f)[4]) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  }
  __device__ __forceinline__ static uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
  // -inf becomes finite (and as good as -inf: 2^d is 0, and the products with d stay finite); NaN stays.
  __device__ __forceinline__ static uint4 bound(const uint4& u) {
    uint4 o;
    constexpr unsigned low = 0xdd800000u;  // -2^60, below -kFar
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(o.x) : "r"(u.x), "r"(low));
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(o.y) : "r"(u.y), "r"(low));
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(o.z) : "r"(u.z), "r"(low));
    asm("max.NaN.f32 %0, %1, %2;" : "=r"(o.w) : "r"(u.w), "r"(low));
    return o;
  }
  // The vector with -inf for element e.
  __device__ __forceinline__ static uint4 without(uint4 u, int e) {
    if (e == 0) u.x = 0xff800000u;
    if (e == 1) u.y = 0xff800000u;
    if (e == 2) u.z = 0xff800000u;
    if (e == 3) u.w = 0xff800000u;
    return u;
  }
  __device__ __forceinline__ static float top(const uint4& u) {
    return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
  }
  __device__ __forceinline__ static F2 pair(const uint4& u, int k) {
    return k == 0 ? f2(__uint_as_float(u.x), __uint_as_float(u.y)) : f2(__uint_as_float(u.z), __uint_as_float(u.w));
  }
  __device__ __forceinline__ static uint4 join(const F2 (&g)[2]) {
    float f[4];
    split(g[0], f[0], f[1]);
    split(g[1], f[2], f[3]);
    return pack(f);
  }
  __device__ __forceinline__ static F2 two(const float* p) {
    const float2 v = *reinterpret_cast<const float2*>(p);
    return f2(v.x, v.y);
  }
  __device__ __forceinline__ static float get(const float* p) { return *p; }
  __device__ __forceinline__ static float put(float v) { return v; }
};
template <>
struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static constexpr unsigned kLowest = 0xff80ff80u;
  __device__ __forceinline__ static void unpack(const uint4& u, float (&f)[8]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f[2 * k] = __uint_as_float(w[k] << 16);
      f[2 * k + 1] = __uint_as_float(w[k] & 0xffff0000u);
    }
  }
  // The gradient leaves in the logits' type: one rounding, to nearest even.
  __device__ __forceinline__ static uint4 pack(const float (&f)[8]) {
    unsigned w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * k], f[2 * k + 1]);
      w[k] = *reinterpret_cast<const unsigned*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ static unsigned max2(unsigned a, unsigned b) {
    unsigned o;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(o) : "r"(a), "r"(b));
    return o;
  }
  __device__ __forceinline__ static uint4 bound(const uint4& u) {
    uint4 o;
    constexpr unsigned low = 0xdd80dd80u;  // -2^60, below -kFar
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.x) : "r"(u.x), "r"(low));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.y) : "r"(u.y), "r"(low));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.z) : "r"(u.z), "r"(low));
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(o.w) : "r"(u.w), "r"(low));
    return o;
  }
  __device__ __forceinline__ static uint4 without(uint4 u, int e) {
    const unsigned keep = e & 1 ? 0x0000ffffu : 0xffff0000u, low = e & 1 ? 0xff800000u : 0x0000ff80u;
    if (e >> 1 == 0) u.x = (u.x & keep) | low;
    if (e >> 1 == 1) u.y = (u.y & keep) | low;
    if (e >> 1 == 2) u.z = (u.z & keep) | low;
    if (e >> 1 == 3) u.w = (u.w & keep) | low;
    return u;
  }
  __device__ __forceinline__ static float top(const uint4& u) {
    const unsigned m = max2(max2(u.x, u.y), max2(u.z, u.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  __device__ __forceinline__ static F2 pair(const uint4& u, int k) {
    const unsigned w = k == 0 ? u.x : k == 1 ? u.y : k == 2 ? u.z : u.w;
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ __forceinline__ static uint4 join(const F2 (&g)[4]) {
    float f[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) split(g[k], f[2 * k], f[2 * k + 1]);
    return pack(f);
  }
  __device__ __forceinline__ static F2 two(const __nv_bfloat16* p) {
    const unsigned w = *reinterpret_cast<const unsigned*>(p);
    return f2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  __device__ __forceinline__ static float get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
  __device__ __forceinline__ static __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// A row cut at 16-byte boundaries: `head` elements, `nvec` vectors, `tail`.
struct Cut {
  int head, nvec, tail;
};
template <class T>
__device__ __forceinline__ Cut cut_row(const T* p, int V) {
  constexpr int N = Vec<T>::N;
  int head = (int)((16u - (unsigned)((uintptr_t)p & 15)) & 15u) / (int)sizeof(T);
  if (head > V) head = V;
  const int nvec = (int)((unsigned)(V - head) / (unsigned)N);
  return Cut{head, nvec, V - head - nvec * N};
}

// ---- running statistics --------------------------------------------------------
// s0 = sum 2^d and s1 = sum 2^d d of the elements seen, with d taken from off, the
// offset of one of them, m, that no other exceeds by kSlack; without an entropy
// to compute, s1 takes each group's largest d for all of its elements, which serves for
// logprob_of's small correction.  m starts at -kFar, not -inf, so that no
// difference of two offsets is NaN; elements below it count as 0 (rows that have
// nothing above it take the far form).
template <bool ENT>
struct Run {
  float m = -kFar, off, s0 = 0.f, s1 = 0.f;
  __device__ __forceinline__ explicit Run(float c) : off(offset_of(-kFar, c)) {}
  // Moves to a larger element's offset.
  __device__ __forceinline__ void raise(float mx, float c) {
    const float to = offset_of(mx, c), by = off - to;
    const float k = ex2(by);
    s1 = fmaf(s0, fmaxf(by, kDeep), s1) * k;
    s0 *= k;
    m = mx;
    off = to;
  }
  template <int K>
  __device__ __forceinline__ void add(const float (&x)[K], float c) {
    float mx = x[0];
#pragma unroll
    for (int k = 1; k < K; ++k) mx = fmaxf(mx, x[k]);
    if (fmaf(mx, c, -off) > kSlack - kLift) raise(mx, c);
    float e[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float d = fmaf(x[k], c, -off);
      e[k] = ex2(d);
      if constexpr (ENT) s1 = fmaf(e[k], fmaxf(d, kDeep), s1);
    }
#pragma unroll
    for (int w = 1; w < K; w *= 2)
#pragma unroll
      for (int k = 0; k + w < K; k += 2 * w) e[k] += e[k + w];
    s0 += e[0];
    if constexpr (!ENT) s1 = fmaf(e[0], fmaxf(fmaf(mx, c, -off), kDeep), s1);
  }
  // M whole vectors at once; `at` places NT apart is where the token lies from the
  // first of them (anything else: not among them), `e` its element, left out.
  template <class T, int M, int NT>
  __device__ __forceinline__ void add_vectors(uint4 (&u)[M], float c, int at, int e) {
    constexpr int P = Vec<T>::N / 2;
    if constexpr (ENT) {
#pragma unroll
      for (int k = 0; k < M; ++k) u[k] = Vec<T>::bound(u[k]);
    }
    float mx = Vec<T>::top(u[0]);
#pragma unroll
    for (int k = 1; k < M; ++k) mx = fmaxf(mx, Vec<T>::top(u[k]));
    float dm = fmaf(mx, c, -off);
    if (dm > kSlack - kLift || (unsigned)at <= (unsigned)((M - 1) * NT)) {  // one branch for the two
#pragma unroll
      for (int k = 0; k < M; ++k)
        if (at == k * NT) u[k] = ENT ? Vec<T>::bound(Vec<T>::without(u[k], e)) : Vec<T>::without(u[k], e);
      mx = Vec<T>::top(u[0]);
#pragma unroll
      for (int k = 1; k < M; ++k) mx = fmaxf(mx, Vec<T>::top(u[k]));
      if (fmaf(mx, c, -off) > kSlack - kLift) raise(mx, c);
      dm = fmaf(mx, c, -off);
    }
    const F2 cc = f2(c, c), no = f2(-off, -off);
    F2 sum, by;
#pragma unroll
    for (int k = 0; k < M; ++k)
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const F2 d = fma2(Vec<T>::pair(u[k], q), cc, no);
        const F2 e = ex2(d);
        const bool first = k == 0 && q == 0;
        sum = first ? e : add2(sum, e);
        if constexpr (ENT) by = first ? mul2(e, d) : fma2(e, d, by);
      }
    float x, y;
    split(sum, x, y);
    x += y;
    s0 += x;
    if constexpr (ENT) {
      split(by, x, y);
      s1 += x + y;
    } else {
      s1 = fmaf(x, fmaxf(dm, kDeep), s1);
    }
  }
  __device__ __forceinline__ void join(float om, float ooff, float os0, float os1) {
    const bool up = om > m;
    const float to = up ? ooff : off;
    const float d0 = off - to, d1 = ooff - to;
    const float k0 = ex2(d0), k1 = ex2(d1);
    s1 = fmaf(s0, fmaxf(d0, kDeep), s1) * k0 + fmaf(os0, fmaxf(d1, kDeep), os1) * k1;
    s0 = s0 * k0 + os0 * k1;
    if (up) m = om;
    off = to;
  }
};

template <bool ENT>
__device__ __forceinline__ void warp_join(Run<ENT>& r, int width = 32) {
  for (int o = width / 2; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, r.m, o);
    const float oo = __shfl_xor_sync(0xffffffffu, r.off, o);
    const float a = __shfl_xor_sync(0xffffffffu, r.s0, o);
    const float b = __shfl_xor_sync(0xffffffffu, r.s1, o);
    r.join(om, oo, a, b);
  }
}

// ---- the policy loss -------------------------------------------------------------
struct Policy {
  const float* old_lp;
  const float* adv;
  bool adv_row;          // adv holds one value a row of the batch
  const float* ref;      // may be null
  float lo, hi, dual;    // ratio bounds
  // their logarithms as sums of two floats; -inf, +inf where there is none
  float2 log_lo, log_hi, log_dual;
  float kl_coef;
  int kl_kind;
  float ent_coef;
  // weight of a step's term: w; or norm[0], over norm[1 + env] for the mean by sequence
  int reduction;
  const float* norm;     // null: w alone
  float w;
};

__device__ __forceinline__ float policy_weight(const Policy& p, int64_t env) {
  if (!p.norm) return p.w;
  const float n0 = p.norm[0];
  return p.reduction == RLS_REDUCE_SEQUENCE ? n0 / p.norm[1 + env] : n0;
}

struct PolicyTerm {
  float loss, d;         // the step's term and its derivative by the logprob
  float kl;
  bool clipped;
};

// A difference of log-probabilities as the sum of two floats (low: what the first leaves).
struct Diff {
  float x, low;
};
__device__ __forceinline__ Diff diff(double a, float b) {
  const double d = a - (double)b;
  const float x = (float)d;
  return Diff{x, fabsf(x) < INFINITY ? (float)(d - (double)x) : 0.f};
}
// The same of two floats, exactly (Knuth's two-sum).
__device__ __forceinline__ Diff diff(float a, float b) {
  const float x = __fsub_rn(a, b), v = __fsub_rn(x, a);
  const float low = __fsub_rn(__fsub_rn(a, __fsub_rn(x, v)), __fadd_rn(b, v));
  return Diff{x, fabsf(x) < INFINITY ? low : 0.f};
}
__device__ __forceinline__ Diff minus(Diff d) { return Diff{-d.x, -d.low}; }
__device__ __forceinline__ bool above(Diff d, float2 bound) {
  return (d.x - bound.x) + (d.low - bound.y) > 0.f;  // d.x - bound.x is exact where it is small
}
__device__ __forceinline__ bool below(Diff d, float2 bound) {
  return (d.x - bound.x) + (d.low - bound.y) < 0.f;
}

// r - 1 - log r
__device__ __forceinline__ float drift_of(Diff lr) {
  return expm1f(lr.x) - lr.x;
}

// -min(r A, clip(r) A), at most -dual A where A < 0, plus the KL estimate:
// k1 = lp - ref, k2 = (lp - ref)^2 / 2, k3 = exp(ref - lp) - (ref - lp) - 1.
// Whether the clip holds is decided on log r with twice fp32's digits (exact for
// fp32 inputs), against the logarithms of the caller's bounds: the derivative jumps there,
// and exp's rounding would put steps near a bound on either side of it (in fp32
// exp(-0.22314358) may round to 0.8f; it is 0.79999998).  lr = lp - old, away = lp - ref.
__device__ __forceinline__ PolicyTerm policy_term(const Policy& p, Diff lr, float adv, Diff away) {
  PolicyTerm o;
  float gain = expf(lr.x);
  if (gain < INFINITY) gain = fmaf(gain, lr.low, gain);
  else if (adv == 0.f && lr.x < INFINITY) gain = 0.f;  // a ratio past fp32's range, times 0
  gain *= adv;
  const bool up = above(lr, p.log_hi), down = below(lr, p.log_lo), far = above(lr, p.log_dual);
  o.clipped = adv > 0.f ? up : adv < 0.f && (down || far);
  const float held = adv > 0.f ? p.hi : down ? p.lo : p.dual;
  o.loss = o.clipped ? -held * adv : -gain;
  o.d = o.clipped ? 0.f : -gain;
  o.kl = 0.f;
  if (p.ref) {
    const Diff x = minus(away);
    float dk;
    if (p.kl_kind == RLS_KL_K1) { o.kl = -x.x; dk = 1.f; }
    else if (p.kl_kind == RLS_KL_K2) { o.kl = 0.5f * x.x * x.x; dk = -x.x; }
    else {
      float e = expm1f(x.x);
      if (e < INFINITY) e = fmaf(e + 1.f, x.low, e);
      o.kl = e - x.x;
      dk = -e;
    }
    if (p.kl_coef != 0.f) {
      o.loss = fmaf(p.kl_coef, o.kl, o.loss);
      o.d = fmaf(p.kl_coef, dk, o.d);
    }
  }
  return o;
}

// ---- sums over steps ---------------------------------------------------------------
// loss, KL, drift, clipped, entropy, steps: fp64 per thread, then per CTA, then
// the CTAs' in their order, so that the result does not depend on timing.
constexpr int kSums = 6;
struct SumOut {
  double* partials;   // [CTAs][kSums]
  unsigned* ticket;   // CTAs done; the last one resets it
  float* loss;
  float* stats;       // may be null
};

// Adds the CTA's sums to the call's; every thread of every CTA calls it once.
// NT >= 32 kSums.
template <int NT>
__device__ __forceinline__ void finish_sums(double (&sum)[kSums], const SumOut& o) {
  static_assert(NT >= 32 * kSums, "a warp for each sum");
  __shared__ double part[NT / 32][kSums];
  __shared__ bool last;
#pragma unroll
  for (int k = 0; k < kSums; ++k)
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], d);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < kSums; ++k) part[warp][k] = sum[k];
  __syncthreads();
  if (threadIdx.x < kSums) {
    double s = 0;
    for (int w = 0; w < NT / 32; ++w) s += part[w][threadIdx.x];
    o.partials[(int64_t)blockIdx.x * kSums + threadIdx.x] = s;
    __threadfence();
  }
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(o.ticket, 1u) == gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  // warp k adds sum k: lanes in strides over the CTAs, then the lanes
  double s = 0;
  if (warp < kSums)
    for (int64_t b = lane; b < gridDim.x; b += 32) s += __ldcg(&o.partials[b * kSums + warp]);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
  if (warp < kSums && lane == 0) part[0][warp] = s;
  __syncthreads();
  if (threadIdx.x < kSums) {
    const double n = part[0][5], v = part[0][threadIdx.x];
    if (threadIdx.x == 0) *o.loss = (float)v;
    else if (o.stats) o.stats[threadIdx.x - 1] = (float)(threadIdx.x == 5 ? v : n > 0 ? v / n : 0.0);
  }
  if (threadIdx.x == 0) *o.ticket = 0u;
}

// ---- where a row's incoming gradients come from --------------------------------
// Given per step.
struct GivenGrad {
  static constexpr bool kPolicy = false;
  const float* g_lp;
  const float* g_ent;  // may be null
};

// Those of the policy loss, for an incoming gradient of `scale` of the loss
// itself, or *g where g is set.
struct PolicyGrad {
  static constexpr bool kPolicy = true;
  Policy p;
  float scale;
  const float* g;
  bool force;
  SumOut sums;
  unsigned* error;  // the workspace's error word
  unsigned tries;   // of a wait on the team
  // the gradient at hand was made for that very scale
  __device__ __forceinline__ bool skip() const { return g && !force && *g == scale; }
  __device__ __forceinline__ float up() const { return g ? *g : scale; }
};

enum Mode { kFwd, kBwd, kBoth };

// ---- any row: one CTA a row ------------------------------------------------------
// The simplest form: for rows beyond the slots of a full cluster, and gradients whose
// rows do not lie as their logits do.  The second pass reads the row from L2, as far
// as that holds the rows at work (8 x 1024 x 131072 bf16, ragged, loss and gradient: 783 us
// a call, against 590 from shared memory).
template <bool ENT, int NT>
__device__ __forceinline__ void block_join(Run<ENT>& r, float c) {
  __shared__ float4 part[NT / 32];
  warp_join<ENT>(r);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();  // the last row's parts are read
  if (lane == 0) part[warp] = make_float4(r.m, r.off, r.s0, r.s1);
  __syncthreads();
  constexpr int W = NT / 32;
  const float4 q = part[lane < W ? lane : 0];
  Run<ENT> z(c);
  z.m = q.x; z.off = q.y;
  z.s0 = lane < W ? q.z : 0.f;
  z.s1 = lane < W ? q.w : 0.f;
  warp_join<ENT>(z);
  // The lanes join in different orders, so their last bits may differ; every
  // thread goes on with lane 0's (the same in each warp): branches on it hold
  // barriers.
  r.m = __shfl_sync(0xffffffffu, z.m, 0);
  r.off = __shfl_sync(0xffffffffu, z.off, 0);
  r.s0 = __shfl_sync(0xffffffffu, z.s0, 0);
  r.s1 = __shfl_sync(0xffffffffu, z.s1, 0);
}

template <int NT>
__device__ __forceinline__ float block_max(float v) {
  __shared__ float part[NT / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < NT / 32; ++w) v = fmaxf(v, part[w]);
  return v;
}
template <int NT>
__device__ __forceinline__ float block_sum(float v) {
  __shared__ float part[NT / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = part[0];
  for (int w = 1; w < NT / 32; ++w) v += part[w];
  return v;
}

// The far form: two plain passes, the true maximum first.
template <class T, bool ENT, int NT>
__device__ __noinline__ RowStats far_stats(const T* x, int V, float c) {
  float m = -INFINITY;
  for (int64_t v = threadIdx.x; v < V; v += NT) m = fmaxf(m, Vec<T>::get(x + v));
  m = block_max<NT>(m);
  float s0 = 0.f, s1 = 0.f;
  for (int64_t v = threadIdx.x; v < V; v += NT) {
    const float d = (Vec<T>::get(x + v) - m) * c;
    const float e = ex2(d);
    s0 += e;
    s1 = fmaf(e, fmaxf(d, kDeep), s1);
  }
  s0 = block_sum<NT>(s0);
  s1 = block_sum<NT>(s1);
  return RowStats{m, s0, s1 / s0, true, s0 == 1.f && s1 == 0.f};
}

template <class T, bool ENT, int NT, int U>
__device__ __forceinline__ RowStats row_stats(const T* x, int V, float c) {
  constexpr int N = Vec<T>::N;
  const Cut cut = cut_row(x, V);
  Run<ENT> run(c);
  const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
  const unsigned low = Vec<T>::kLowest;
  for (int64_t v0 = threadIdx.x; v0 < cut.nvec; v0 += (int64_t)NT * U) {
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t v = v0 + (int64_t)k * NT;
      u[k] = v < cut.nvec ? __ldg(xv + v) : make_uint4(low, low, low, low);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float f[N];
      Vec<T>::unpack(u[k], f);
      run.add(f, c);
    }
  }
  const int ends = cut.head + cut.tail;
  if ((int)threadIdx.x < ends) {
    const int64_t i = (int)threadIdx.x < cut.head ? (int)threadIdx.x : V - ends + (int)threadIdx.x;
    const float f[1] = {Vec<T>::get(x + i)};
    run.add(f, c);
  }
  block_join<ENT, NT>(run, c);
  if (!(run.s0 >= kLeast && run.s0 <= kMost)) return far_stats<T, ENT, NT>(x, V, c);
  const float d = fmaf(run.m, c, -run.off), e = ex2(d);
  const bool alone = ENT && run.s0 == e && run.s1 == e * d;
  return RowStats{run.m, run.s0, alone ? d : run.s1 / run.s0, false, alone};
}

template <class T, int NT>
__device__ __forceinline__ void zero_row(T* g, int V) {
  const Cut cut = cut_row(g, V);
  uint4* gv = reinterpret_cast<uint4*>(g + cut.head);
  for (int64_t v = threadIdx.x; v < cut.nvec; v += NT) __stcs(gv + v, make_uint4(0, 0, 0, 0));
  const int ends = cut.head + cut.tail;
  if ((int)threadIdx.x < ends) g[(int)threadIdx.x < cut.head ? (int)threadIdx.x : V - ends + (int)threadIdx.x] = Vec<T>::put(0.f);
}

template <class T, bool ENT, int NT, int U>
__device__ __forceinline__ void grad_row(const T* x, T* g, int V, int64_t tok, const RowStats& r, float a, float b,
                                         float c, float inv_temp) {
  const Shift sh = shift_of(r, c);
  const RowGrad rg = row_grad(a, b, r, inv_temp);
  auto at_token = [&](float y) { return token_grad(y, sh, a, b, r.s0, r.t, inv_temp); };
  constexpr int N = Vec<T>::N;
  const Cut cut = cut_row(x, V);
  const bool same = (((uintptr_t)x ^ (uintptr_t)g) & 15) == 0;
  const uint4* xv = reinterpret_cast<const uint4*>(x + cut.head);
  for (int64_t v0 = threadIdx.x; v0 < cut.nvec; v0 += (int64_t)NT * U) {
    uint4 u[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t v = v0 + (int64_t)k * NT;
      if (v < cut.nvec) u[k] = __ldcs(xv + v);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t v = v0 + (int64_t)k * NT;
      if (v >= cut.nvec) break;
      float f[N];
      Vec<T>::unpack(u[k], f);
      const int64_t i0 = cut.head + v * N;
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = i0 + e == tok ? at_token(f[e]) : grad_at<ENT>(f[e], sh, rg);
      if (same) {
        __stcs(reinterpret_cast<uint4*>(g + i0), Vec<T>::pack(f));
      } else {
#pragma unroll
        for (int e = 0; e < N; ++e) g[i0 + e] = Vec<T>::put(f[e]);
      }
    }
  }
  const int ends = cut.head + cut.tail;
  if ((int)threadIdx.x < ends) {
    const int64_t i = (int)threadIdx.x < cut.head ? (int)threadIdx.x : V - ends + (int)threadIdx.x;
    const float f = Vec<T>::get(x + i);
    g[i] = Vec<T>::put(i == tok ? at_token(f) : grad_at<ENT>(f, sh, rg));
  }
}

// Outputs per row; entropy and stats may be null.
struct RowOut {
  float* logprob;
  float* entropy;
  float4* stats;  // long rows' records
};

template <class T, bool ENT, int MODE, class Src, int NT, int U>
__global__ void __launch_bounds__(NT) cta_rows_kernel(Rows<T> in, RowOut out, GradRows<T> gr, Src src) {
  if constexpr (Src::kPolicy && MODE == kBwd) {
    if (src.skip()) return;
  }
  for (int64_t row = blockIdx.x; row < in.rows; row += gridDim.x) {
    const T* x = in.x + in.at(row);
    T* g = MODE == kFwd || !gr.g ? nullptr : gr.g + gr.at(row, in);
    if (!mask_at(in.mask, row)) {
      if constexpr (MODE != kBwd) {
        if (threadIdx.x == 0) {
          out.logprob[row] = 0.f;
          if (out.entropy) out.entropy[row] = 0.f;
          if (out.stats) out.stats[2 * row] = out.stats[2 * row + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      if (g) zero_row<T, NT>(g, in.V);
      continue;
    }
    const int64_t tok = in.tokens[row];
    const bool ok = tok >= 0 && tok < in.V;
    RowStats r;
    float a = 0.f, b = 0.f;
    if constexpr (MODE != kBwd) {
      const float xt = ok ? Vec<T>::get(x + tok) : NAN;
      r = row_stats<T, ENT, NT, U>(x, in.V, in.c);
      const double lp = logprob_of(xt, r, in.c, in.c64, in.c_off);
      float ent = 0.f;
      if constexpr (ENT) ent = entropy_of(r);
      int flags = kFlagKept;
      if constexpr (Src::kPolicy) {
        const int64_t env = in.env(row);
        const Policy& p = src.p;
        const PolicyTerm o = policy_term(p, diff(lp, p.old_lp[row]), p.adv[p.adv_row ? env : row],
                                         diff(lp, p.ref ? p.ref[row] : 0.f));
        const float w = policy_weight(p, env);
        a = w * o.d;
        if constexpr (ENT) b = -w * p.ent_coef;
        if (o.clipped) flags |= kFlagClipped;
        if (threadIdx.x == 0) {
          const float term = ENT && p.ent_coef != 0.f ? o.loss - p.ent_coef * ent : o.loss;
          out.stats[2 * row + 1] = make_float4(a, w * term, o.kl, drift_of(diff(lp, p.old_lp[row])));
        }
      }
      if (threadIdx.x == 0) {
        out.logprob[row] = (float)lp;
        if (out.entropy) out.entropy[row] = ent;
        if (out.stats) out.stats[2 * row] = stats_word(r, flags);
      }
    } else {
      r = stats_of(out.stats[2 * row]);
      if constexpr (Src::kPolicy) {
        a = out.stats[2 * row + 1].x;
        if constexpr (ENT) b = -policy_weight(src.p, in.env(row)) * src.p.ent_coef;
      } else {
        a = src.g_lp ? src.g_lp[row] : 0.f;
        if constexpr (ENT) b = src.g_ent[row];
      }
    }
    if (g) {
      if constexpr (Src::kPolicy) { a *= src.up(); b *= src.up(); }
      if (!ok) a = NAN;
      if (a == 0.f && b == 0.f) zero_row<T, NT>(g, in.V);
      else grad_row<T, ENT, NT, U>(x, g, in.V, tok, r, a, b, in.c, in.inv_temp);
    }
  }
}

// ---- long rows ------------------------------------------------------------------
// A team of 1 to 8 CTAs (a cluster) of NT threads works on one row at a time; each
// CTA takes one stretch of the row's 16-byte vectors, each thread every NT-th vector
// of the stretch.  What a vector was read into (registers, or a slot of shared
// memory that no other thread reads) is refilled with a later one, of the next row at
// the end of a row, as soon as its last use is over: so loads are always in flight, across the
// row's one barrier (the join of the statistics) too.
__device__ __forceinline__ void copy16(uint4* to, const uint4* from) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(to);
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// The same for a number that unrolling makes constant, at most N.
template <int N>
__device__ __forceinline__ void copy_wait_upto(int n) {
  if constexpr (N == 0) copy_wait<0>();
  else if (n == N) copy_wait<N>();
  else copy_wait_upto<N - 1>(n);
}

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Stores to the same shared variable of another CTA of the cluster.
__device__ __forceinline__ void store_remote(float4* p, unsigned rank, float4 v) {
  unsigned at = (unsigned)__cvta_generic_to_shared(p), there;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

constexpr int kMostCtas = 8;  // of a cluster (the portable limit)

// Every warp's value to every warp of the row's CTAs: `mine` (one per warp) goes to all
// CTAs' tables, of which two take turns, so that one barrier a call suffices.
//
// Across CTAs there are two ways.  A cluster barrier with release and acquire
// waits for all of the thread's earlier stores, gradients on their way to memory among
// them (measured at 131072 bf16 logits: 462 us with it, 432 us without, for 4081 rows of
// loss and gradient); so where there are such stores the values travel as
// asynchronous stores that count down an mbarrier of the CTA they go to.
template <int NT, bool CL, bool ASYNC>
struct Table {
  static constexpr int kWarps = NT / 32;
  static constexpr int kMost = CL ? kWarps * kMostCtas : kWarps;
  float4 at[2][kMost];
  unsigned long long bar[CL && ASYNC ? 2 : 1];
};

__device__ __forceinline__ void bar_init(unsigned long long* bar) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((unsigned)__cvta_generic_to_shared(bar)) : "memory");
}
__device__ __forceinline__ void bar_expect(unsigned long long* bar, unsigned bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"((unsigned)__cvta_generic_to_shared(bar)),
               "r"(bytes) : "memory");
}
// Polled without ordering (an acquire at each try would invalidate L1 each time);
// bar_acquire orders what follows a wait that succeeded.
__device__ __forceinline__ bool bar_try(unsigned long long* bar, unsigned parity) {
  unsigned ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"((unsigned)__cvta_generic_to_shared(bar)), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ void bar_acquire(unsigned long long* bar, unsigned parity) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%0], %1;\n\t}"
      ::"r"((unsigned)__cvta_generic_to_shared(bar)), "r"(parity) : "memory");
}
__device__ __forceinline__ void store_async(float4* p, unsigned long long* bar, unsigned rank, float4 v) {
  const unsigned at = (unsigned)__cvta_generic_to_shared(p), b = (unsigned)__cvta_generic_to_shared(bar);
  unsigned there, its;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(its) : "r"(b), "r"(rank));
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(there),
               "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w), "r"(its) : "memory");
}

// What a thread keeps of its exchanges.
struct Turns {
  unsigned n = 0;
  unsigned* error;      // where a wait that ran out is noted
  unsigned tries;       // of a wait, each suspended for a while
  // A wait of this warp ran out (from the row's next barrier on: of the CTA).  Nothing is sent,
  // expected or awaited any more -- a barrier whose phase did not end takes no other
  // arrival -- and the rows' results are NaN.  The others of the team miss this one's
  // values and run out in their turn.
  bool broken = false;
};

template <int NT, bool CL, bool ASYNC>
__device__ __forceinline__ const float4* exchange(Table<NT, CL, ASYNC>& t, Turns& turn, float4 mine, unsigned rank,
                                                  unsigned size) {
  const unsigned which = turn.n & 1, parity = (turn.n >> 1) & 1;
  float4* tab = t.at[which];
  ++turn.n;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if constexpr (CL && ASYNC) {
    if (turn.broken) return tab;
    // Each warp of the team sends size x 16 bytes; this CTA's barrier gets 16 from each.
    // A barrier is used again two exchanges on: whoever sends then has had this CTA's
    // values of the exchange between, which its warps send after this wait.
    unsigned long long* bar = &t.bar[which];
    if (threadIdx.x == 0) bar_expect(bar, size * (NT / 32) * 16);
    if (lane < size) store_async(tab + rank * (NT / 32) + warp, bar, lane, mine);
    bool done = false;
    for (unsigned k = 0; k < turn.tries && !done; ++k) done = bar_try(bar, parity);
    if (done) bar_acquire(bar, parity);
    turn.broken = __any_sync(0xffffffffu, !done);
    if (turn.broken && lane == 0) atomicOr(turn.error, 8u);
  } else if constexpr (CL) {
    if (lane < size) store_remote(tab + rank * (NT / 32) + warp, lane, mine);
    cluster_barrier();
  } else {
    if (lane == 0) tab[warp] = mine;
    __syncthreads();
  }
  return tab;
}

// Joins (m, s0, s1) over groups of WIDTH lanes: to the common maximum first, then
// plain sums.
template <int WIDTH>
__device__ __forceinline__ void gather(float& m, float& s0, float& s1, float c) {
  float top = m;
  if constexpr (WIDTH == 32) {
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(top) : "f"(m));
  } else {
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  const float by = offset_of(m, c) - offset_of(top, c);
  const float k = ex2(by);
  s1 = fmaf(s0, fmaxf(by, kDeep), s1) * k;
  s0 *= k;
  m = top;
#pragma unroll
  for (int o = WIDTH / 2; o > 0; o >>= 1) {
    s0 += __shfl_xor_sync(0xffffffffu, s0, o);
    s1 += __shfl_xor_sync(0xffffffffu, s1, o);
  }
}

__device__ __forceinline__ float incoming_entropy(const PolicyGrad& s, float w, float) { return -w * s.p.ent_coef; }
__device__ __forceinline__ float incoming_entropy(const GivenGrad&, float, float b) { return b; }

// A row's statistics where the team's were not to be had.
__device__ __forceinline__ RowStats no_stats() { return RowStats{NAN, NAN, NAN, true, false, -1.f, 0.f}; }

// The rows of a team, in order, and what its CTA and threads have of each.
template <class T, bool ENT, int MODE, class Src, int NT, bool CL>
struct Walk {
  static constexpr int N = Vec<T>::N;
  const Rows<T>& in;
  const RowOut& out;
  const GradRows<T>& gr;
  const Src& src;
  const int tid = threadIdx.x;
  const unsigned rank = CL ? cluster_rank() : 0, size = CL ? cluster_size() : 1;
  const int log_size = !CL || size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3;  // sizes are powers of two
  const int64_t teams = gridDim.x >> log_size;
  int64_t next = blockIdx.x >> log_size;  // the team's next place in the order of the rows
  const int64_t kept = in.order ? in.order[0] : 0;
  unsigned window = 0;  // without an order: which of the next 32 rows are to be worked on; the others only get their zeros
  int left = 0;

  __device__ __forceinline__ Walk(const Rows<T>& i, const RowOut& o, const GradRows<T>& g, const Src& s)
      : in(i), out(o), gr(g), src(s) {}

  __device__ __forceinline__ bool wanted(int64_t row) const {
    if (row >= in.rows || !mask_at(in.mask, row)) return false;
    if constexpr (MODE == kBwd && Src::kPolicy) return ENT || out.stats[2 * row + 1].x != 0.f;
    if constexpr (MODE == kBwd && !Src::kPolicy) {
      bool some = src.g_lp && src.g_lp[row] != 0.f;
      if constexpr (ENT) some = some || src.g_ent[row] != 0.f;
      return some;
    }
    return true;
  }
  __device__ __forceinline__ void zeros(int64_t row) const {
    T* g = gr.g + gr.at(row, in);
    const Cut cut = cut_row(g, in.V);
    int v0;
    const int n = stretch(cut, v0);
    uint4* gv = reinterpret_cast<uint4*>(g + cut.head) + v0;
    for (int v = tid; v < n; v += NT) __stcs(gv + v, make_uint4(0, 0, 0, 0));
    const int ends = ends_of(cut);
    if (tid < ends) g[tid < cut.head ? tid : in.V - ends + tid] = Vec<T>::put(0.f);
  }
  // A row that does not count.
  __device__ __forceinline__ void skip(int64_t row) const {
    if constexpr (MODE != kBwd) {
      if (rank == 0 && tid == 0) {
        out.logprob[row] = 0.f;
        if (out.entropy) out.entropy[row] = 0.f;
        if (out.stats) out.stats[2 * row] = out.stats[2 * row + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
    if (MODE != kFwd && gr.g) zeros(row);
  }
  // The next row to work on, or -1; the same in all threads of the team.
  __device__ __forceinline__ int64_t advance() {
    if (in.order) {
      // The rows that count come first, so that every team gets as many of them; the others are
      // taken in between, as many to each.
      const int64_t at = next;
      next += teams;
      const int64_t other = in.rows - 1 - at;  // from the far end
      if (other >= kept) skip(in.order[1 + other]);
      if (at < kept) return in.order[1 + at];
      for (int64_t more = in.rows - 1 - next; more >= kept; more -= teams) {
        skip(in.order[1 + more]);
        next += teams;
      }
      return -1;
    }
    for (;;) {
      if (next >= in.rows) return -1;
      if (left == 0) {
        window = __ballot_sync(0xffffffffu, wanted(next + (tid & 31) * teams));
        left = 32;
      }
      const bool yes = window & 1u;
      const int64_t row = next;
      window >>= 1;
      --left;
      next += teams;
      if (yes) return row;
      skip(row);
    }
  }
  __device__ __forceinline__ const T* row_at(int64_t row) const { return in.x + in.at(row); }
  // The CTA's stretch begins v0 vectors into the row and has as many.
  __device__ __forceinline__ int stretch(const Cut& cut, int& v0) const {
    if constexpr (!CL) {
      v0 = 0;
      return cut.nvec;
    }
    const int per = (cut.nvec + (int)size - 1) >> log_size;
    v0 = per * (int)rank;
    const int n = cut.nvec - v0;
    return n < 0 ? 0 : n < per ? n : per;
  }
  // Vectors a CTA has of any row, at most.
  __device__ __forceinline__ int most() const {
    return ((in.V + N - 1) / N + (int)size - 1) >> log_size;
  }

  struct Place {
    int64_t row;
    const uint4* at;  // this thread's first vector
    int n, mid;       // vectors of the stretch, and from the thread's first to its end
  };
  __device__ __forceinline__ Place place(int64_t row) const {
    const T* x = row_at(row);
    const Cut cut = cut_row(x, in.V);
    int v0;
    const int n = stretch(cut, v0);
    return Place{row, reinterpret_cast<const uint4*>(x + cut.head) + v0 + tid, n, n - tid};
  }
  // What the row's one-off steps need, asked for a row ahead.
  struct Extra {
    int64_t tok;
    float end, xt;              // the thread's end element; the token's logit
    float old_lp, adv, ref, w;  // the policy loss's inputs
    float a, b;                 // incoming gradients of a backward call
    float4 stats;
  };
  __device__ __forceinline__ Extra extra(int64_t row) const {
    Extra p;
    const T* x = row_at(row);
    const Cut cut = cut_row(x, in.V);
    const int ends = ends_of(cut);
    p.tok = in.tokens[row];
    p.end = tid < ends ? Vec<T>::get(x + (tid < cut.head ? tid : in.V - ends + tid)) : 0.f;
    if constexpr (Src::kPolicy) {
      const int64_t env = in.env(row);
      p.w = policy_weight(src.p, env);
      if constexpr (MODE != kBwd) {
        p.old_lp = src.p.old_lp[row];
        p.adv = src.p.adv[src.p.adv_row ? env : row];
        p.ref = src.p.ref ? src.p.ref[row] : 0.f;
      }
    }
    if constexpr (MODE == kBwd) {
      p.stats = out.stats[2 * row];
      if constexpr (Src::kPolicy) p.a = out.stats[2 * row + 1].x;
      else p.a = src.g_lp ? src.g_lp[row] : 0.f;
      if constexpr (ENT && !Src::kPolicy) p.b = src.g_ent[row];
    }
    return p;
  }
  // The token's logit, asked for once the token itself is there.
  __device__ __forceinline__ void token_logit(int64_t row, Extra& p) const {
    p.xt = p.tok >= 0 && p.tok < in.V ? Vec<T>::get(row_at(row) + p.tok) : NAN;
  }
  // Elements outside the row's vectors: the first CTA's threads take one each.
  __device__ __forceinline__ int ends_of(const Cut& cut) const { return rank == 0 ? (int)(cut.head + cut.tail) : 0; }

  // How far the token's vector lies from the thread's first, and the element there; the
  // thread has it where that is a multiple of NT.  Far below 0: not in the stretch.
  __device__ __forceinline__ int token_vector(int64_t row, const Extra& ex, int& e) const {
    const Cut cut = cut_row(row_at(row), in.V);
    int v0;
    const int n = stretch(cut, v0);
    const int rel = (int)ex.tok - cut.head - v0 * N;
    e = rel & (N - 1);
    return ex.tok >= 0 && ex.tok < in.V && rel >= 0 && rel < n * N ? rel / N - tid : -(1 << 30);
  }

  // The statistics of the row from every thread's share of the vectors, the token
  // left out (the ends are added here, and the token last); the same in all
  // threads of the team.
  template <bool ASYNC>
  __device__ __forceinline__ RowStats join(Run<ENT>& run, int64_t row, const Extra& ex, Table<NT, CL, ASYNC>& table,
                                           Turns& turn) const {
    const int lane = tid & 31;
    const float c = in.c;
    const T* x = row_at(row);
    const Cut cut = cut_row(x, in.V);
    const int ends = ends_of(cut);
    if (tid < ends && ex.tok != (tid < cut.head ? tid : in.V - ends + tid)) {
      const float f[1] = {ex.end};
      run.add(f, c);
    }
    gather<32>(run.m, run.s0, run.s1, c);
    {
      const float4* tab = exchange(table, turn, make_float4(run.m, run.s0, run.s1, 0.f), rank, size);
      if (turn.broken) return no_stats();
      // every group of lanes reads all of the table
      constexpr int kWarps = NT / 32;
      if constexpr (!CL) {
        const float4 q = tab[lane & (kWarps - 1)];
        run.m = q.x; run.s0 = q.y; run.s1 = q.z;
        gather<kWarps>(run.m, run.s0, run.s1, c);
      } else {
        const int n = (int)size * kWarps;
        float4 q = lane < n ? tab[lane] : make_float4(-kFar, 0.f, 0.f, 0.f);
        if (lane + 32 < n) {
          const float4 q2 = tab[lane + 32];
          const float top = fmaxf(q.x, q2.x);
          const float to = offset_of(top, c), d0 = offset_of(q.x, c) - to, d1 = offset_of(q2.x, c) - to;
          const float k0 = ex2(d0), k1 = ex2(d1);
          q.z = fmaf(q.y, fmaxf(d0, kDeep), q.z) * k0 + fmaf(q2.y, fmaxf(d1, kDeep), q2.z) * k1;
          q.y = q.y * k0 + q2.y * k1;
          q.x = top;
        }
        run.m = q.x; run.s0 = q.y; run.s1 = q.z;
        gather<32>(run.m, run.s0, run.s1, c);
      }
    }
    {
      const float others = run.s0, by_others = run.s1;
      run.off = offset_of(run.m, c);
      if (ex.xt > run.m) run.raise(ex.xt, c);
      const float d = fmaf(ex.xt, c, -run.off), e = ex2(d);
      const float s0 = run.s0 + e, s1 = fmaf(e, fmaxf(d, kDeep), run.s1);
      if (s0 >= kLeast && s0 <= kMost) {
        const bool alone = ENT && others == 0.f && by_others == 0.f;
        return RowStats{run.m, s0, alone ? d : s1 / s0, false, alone, run.s0,
                        run.s0 > 0.f ? __fdividef(run.s1, run.s0) : 0.f};
      }
    }
    // The far form, from global memory (what the row was read into may hold the
    // next one).  All threads of the team come here or none.
    int v0;
    const int64_t n = (int64_t)stretch(cut, v0) * N;
    const T* xs = x + cut.head + (int64_t)v0 * N;
    float m = tid < ends ? ex.end : -INFINITY;
    for (int64_t i = tid; i < n; i += NT) m = fmaxf(m, Vec<T>::get(xs + i));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float4* tab = exchange(table, turn, make_float4(m, 0.f, 0.f, 0.f), rank, size);
    if (turn.broken) return no_stats();
    for (int w = 0; w < (int)size * (NT / 32); ++w) m = fmaxf(m, tab[w].x);
    float s0 = 0.f, s1 = 0.f;
    auto add = [&](float y) {
      const float d = (y - m) * c;
      const float e = ex2(d);
      s0 += e;
      s1 = fmaf(e, fmaxf(d, kDeep), s1);
    };
    for (int64_t i = tid; i < n; i += NT) add(Vec<T>::get(xs + i));
    if (tid < ends) add(ex.end);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
    tab = exchange(table, turn, make_float4(s0, s1, 0.f, 0.f), rank, size);
    if (turn.broken) return no_stats();
    s0 = s1 = 0.f;
    for (int w = 0; w < (int)size * (NT / 32); ++w) { s0 += tab[w].x; s1 += tab[w].y; }
    return RowStats{m, s0, s1 / s0, true, s0 == 1.f && s1 == 0.f, -1.f, 0.f};
  }

  // What a row gives besides its gradient; one warp of a CTA calls these.  The
  // incoming gradients come first: the other warps wait for them.
  struct Result {
    double lp;
    float ent;
    PolicyTerm o;
  };
  __device__ __forceinline__ Result result(const RowStats& r, const Extra& ex, float& a, float& b) const {
    Result q{};
    q.lp = logprob_of(ex.xt, r, in.c, in.c64, in.c_off);
    if constexpr (Src::kPolicy) {
      q.o = policy_term(src.p, diff(q.lp, ex.old_lp), ex.adv, diff(q.lp, ex.ref));
      a = ex.w * q.o.d;
      b = ENT ? -ex.w * src.p.ent_coef : 0.f;
    }
    return q;
  }
  __device__ __forceinline__ void outputs(int64_t row, const RowStats& r, const Extra& ex, const Result& q, float a) const {
    if (rank != 0 || tid != 0) return;
    float ent = 0.f;
    if constexpr (ENT) ent = entropy_of(r);
    int flags = kFlagKept;
    if constexpr (Src::kPolicy) {
      const float term = ENT && src.p.ent_coef != 0.f ? q.o.loss - src.p.ent_coef * ent : q.o.loss;
      if (q.o.clipped) flags |= kFlagClipped;
      out.stats[2 * row + 1] = make_float4(a, ex.w * term, q.o.kl, drift_of(diff(q.lp, ex.old_lp)));
    }
    out.logprob[row] = (float)q.lp;
    if (out.entropy) out.entropy[row] = ent;
    if (out.stats) out.stats[2 * row] = stats_word(r, flags);
  }

  // Writing a row's gradient.
  struct Writer {
    T* g;             // null: nothing to write
    T* gs;            // this thread's first vector's place
    Shift sh;
    RowGrad rg;
  };
  // (a, b) as the loss's scale and a token outside the vocabulary leave them.
  __device__ __forceinline__ void scaled(const Extra& ex, float& a, float& b) const {
    if constexpr (Src::kPolicy) { a *= src.up(); b *= src.up(); }
    if (ex.tok < 0 || ex.tok >= in.V) a = NAN;
  }
  __device__ __forceinline__ Writer writer(int64_t row, const RowStats& r, float a, float b) const {
    Writer w;
    w.g = gr.g ? gr.g + gr.at(row, in) : nullptr;
    if (w.g && a == 0.f && b == 0.f) {
      zeros(row);
      w.g = nullptr;
    }
    w.sh = shift_of(r, in.c);
    w.rg = row_grad(a, b, r, in.inv_temp);
    const T* x = row_at(row);
    const Cut cut = cut_row(x, in.V);
    int v0;
    stretch(cut, v0);
    w.gs = w.g + cut.head + (int64_t)(v0 + tid) * N;
    return w;
  }
  // The gradient of the vector v places after the thread's first, stored where
  // `inside` (the token's element is put right by finish()).
  __device__ __forceinline__ void write(const Writer& w, int v, uint4 u, bool inside) const {
    constexpr int P = N / 2;
    F2 f[P];
    const F2 cc = f2(in.c, in.c), no = f2(-w.sh.off, -w.sh.off), nA = f2(-w.rg.A, -w.rg.A);
    if constexpr (ENT) u = Vec<T>::bound(u);
#pragma unroll
    for (int q = 0; q < P; ++q) {
      const F2 d = fma2(Vec<T>::pair(u, q), cc, no);
      f[q] = mul2(ex2(d), ENT ? fma2(f2(-w.rg.B, -w.rg.B), d, nA) : nA);
    }
    const uint4 o = Vec<T>::join(f);
    if (inside) __stcs(reinterpret_cast<uint4*>(w.gs) + v, o);
  }
  // The same for all of the thread's vectors of a row in the far form, read again.
  __device__ __forceinline__ void write_far(const Writer& w, const Place& p) const {
    const T* x = reinterpret_cast<const T*>(p.at);
#pragma unroll 1
    for (int v = 0; v < p.mid; v += NT)
#pragma unroll 1
      for (int e = v * N; e < v * N + N; ++e) w.gs[e] = Vec<T>::put(grad_at<ENT>(Vec<T>::get(x + e), w.sh, w.rg));
  }
  // The row's end elements, and the token's by the thread that wrote its place;
  // incoming() gives (a, b, S0, t) to that one.
  template <class F>
  __device__ __forceinline__ void finish(const Writer& w, int64_t row, const Extra& ex, F&& incoming) const {
    const Cut cut = cut_row(row_at(row), in.V);
    const int ends = ends_of(cut);
    const int end = tid < ends ? (tid < cut.head ? tid : in.V - ends + tid) : -1;
    if (end >= 0) w.g[end] = Vec<T>::put(grad_at<ENT>(ex.end, w.sh, w.rg));
    if (ex.tok < 0 || ex.tok >= in.V) return;
    int v0;
    const int n = stretch(cut, v0);
    const int tok = (int)ex.tok, rel = tok - cut.head - v0 * N;
    if (rel >= 0 && rel < n * N ? rel / N % NT == tid : tok == end) {
      const float4 q = incoming();
      w.g[tok] = Vec<T>::put(token_grad(ex.xt, w.sh, q.x, q.y, q.z, q.w, in.inv_temp));
    }
  }
};

// ---- forward alone, and gradient alone: rows stream through registers --------------
// Every element is used once, so nothing is kept: each thread has U vectors of
// loads in flight and refills each as soon as it is used.  Bound by DRAM: 1.07 GB of bf16 logits
// in rows of 131072 take 189 us forward (0.88 of the measured copy bandwidth) and, read and
// written, 372 us backward (0.89); fp32 rows of 50021 164 us (1.01) and 385 us (0.86).  Short rows
// go to one warp each, which needs no barrier (2048 bf16: 0.55 forward, by
// instruction issue, 0.92 backward); few rows to a cluster of CTAs each (one row of 131072: 5 us).
__device__ __forceinline__ uint4 load_once(const uint4* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}


template <class T, bool ENT, int MODE, class Src, int NT, int U, bool CL>
__global__ void __launch_bounds__(NT, (MODE == kFwd ? 768 : 1024) / NT)
    stream_rows_kernel(Rows<T> in, RowOut out, GradRows<T> gr, Src src) {
  if constexpr (Src::kPolicy && MODE == kBwd) {
    if (src.skip()) return;
  }
  constexpr int M = 2;  // vectors taken at a time
  static_assert(MODE != kBoth && U % M == 0, "streams");
  __shared__ Table<NT, CL, false> table;
  Turns turn{0, nullptr, 0, false};
  using W = Walk<T, ENT, MODE, Src, NT, CL>;
  W walk(in, out, gr, src);
  const unsigned low = Vec<T>::kLowest;
  uint4 u[U];
  // Vectors j .. j + M - 1 of the round that begins at `base`; `full`: all threads have them.
  auto fetch = [&](const typename W::Place& p, int base, bool full, int j) {
    if (full) {
#pragma unroll
      for (int k = j; k < j + M; ++k) u[k] = load_once(p.at + base + k * NT);
    } else {
#pragma unroll
      for (int k = j; k < j + M; ++k) {
        u[k] = make_uint4(low, low, low, low);
        if (base + k * NT < p.mid) u[k] = load_once(p.at + base + k * NT);
      }
    }
  };
  const int rounds = (walk.most() + NT * U - 1) / (NT * U);
  const int64_t first = walk.advance();
  if (first < 0) return;  // the same for every CTA of the team
  typename W::Place now = walk.place(first);
  typename W::Extra ex = walk.extra(first);
#pragma unroll
  for (int j = 0; j < U; j += M) fetch(now, 0, NT * U <= now.n, j);
  walk.token_logit(first, ex);
  if constexpr (CL && MODE == kFwd) cluster_barrier();  // the others' tables exist
  for (;;) {
    typename W::Place next{-1, nullptr, 0, 0};
    typename W::Extra nx{};
    const int64_t row = walk.advance();
    if (row >= 0) {
      next = walk.place(row);
      nx = walk.extra(row);
    }
    Run<ENT> run(in.c);
    int token_e = 0;
    const int token_v = MODE == kFwd ? walk.token_vector(now.row, ex, token_e) : 0;
    typename W::Writer wr{};
    float a = 0.f, b = 0.f;
    if constexpr (MODE == kBwd) {
      a = ex.a;
      b = ENT ? incoming_entropy(src, ex.w, ex.b) : 0.f;
      walk.scaled(ex, a, b);
      wr = walk.writer(now.row, stats_of(ex.stats), a, b);
    }
    const bool near = MODE == kBwd && wr.g && !wr.sh.far;
    if (MODE == kBwd && wr.g && !near) walk.write_far(wr, now);
    for (int round = 0; round < rounds; ++round) {
      const int base = round * (NT * U);
      const bool over = round + 1 == rounds;
      const typename W::Place& then = over ? next : now;
      const int from = over ? 0 : base + NT * U;
      const bool then_full = from + NT * U <= then.n;
#pragma unroll
      for (int j = 0; j < U; j += M) {
        if constexpr (MODE == kFwd) {
          uint4 t[M];
#pragma unroll
          for (int k = 0; k < M; ++k) t[k] = u[j + k];
          run.template add_vectors<T, M, NT>(t, in.c, token_v - (base + j * NT), token_e);
        } else if (near) {
#pragma unroll
          for (int k = 0; k < M; ++k) {
            const int v = base + (j + k) * NT;
            walk.write(wr, v, u[j + k], v < now.mid);
          }
        }
        fetch(then, from, then_full, j);
      }
    }
    if constexpr (MODE == kFwd) {
      const RowStats r = walk.join(run, now.row, ex, table, turn);
      if (walk.rank == 0 && threadIdx.x < 32) {
        const typename W::Result q = walk.result(r, ex, a, b);
        walk.outputs(now.row, r, ex, q, a);
      }
    } else if (wr.g) {
      walk.finish(wr, now.row, ex, [&] { return make_float4(a, b, ex.stats.y, ex.stats.z); });
    }
    if (next.row < 0) break;
    walk.token_logit(next.row, nx);
    now = next;
    ex = nx;
  }
}

// ---- both in one pass: a row waits in shared memory for its gradient ---------------
// The policy loss's incoming gradient of a row follows from its own
// log-probability (and the mask's counts), so the row is read once and its
// gradient written while it is on chip: two thirds of the traffic of separate passes.
// Each thread's vectors of the row, at most K, have slots of its own, filled by
// cp.async (all K in flight at once): no barrier, only the thread's own wait.
// 64 KB a CTA, three CTAs an SM: while one adds up, another stores and a third waits.
// 1.07 GB of logits read and written: 131072 bf16 (four CTAs a row) 454 us, 0.73 of the copy
// bandwidth, 32768 bf16 (one) 425 us, 0.78, 8192 fp32 376 us, 0.88.  Bound by latency,
// the row's serial steps between its passes (half of the issue slots and 46 % of DRAM's
// peak are used at 1024 rows of 131072 bf16).
template <class T, bool ENT, class Src, int NT, int K, bool CL>
__global__ void __launch_bounds__(NT, 768 / NT) both_rows_kernel(Rows<T> in, RowOut out, GradRows<T> gr, Src src) {
  constexpr int M = 2;
  static_assert(K % M == 0, "whole groups");
  extern __shared__ uint4 slots[];  // [K][NT]
  __shared__ Table<NT, CL, true> table;
  __shared__ float4 incoming;       // (a, b, S0, t) of the row, from the warp that formed them
  Turns turn{0, src.error, src.tries, false};
  using W = Walk<T, ENT, kBoth, Src, NT, CL>;
  W walk(in, out, gr, src);
  uint4* mine = slots + threadIdx.x;
  const unsigned low = Vec<T>::kLowest;
  auto fetch = [&](const typename W::Place& p, int j) {
    if (j * NT < p.mid) copy16(mine + j * NT, p.at + j * NT);
    copy_commit();
  };
  const int64_t first = walk.advance();
  if (first < 0) return;  // the same for every CTA of the team
  typename W::Place now = walk.place(first);
  typename W::Extra ex = walk.extra(first);
#pragma unroll
  for (int j = 0; j < K; ++j) fetch(now, j);
  walk.token_logit(first, ex);
  if constexpr (CL) {  // the others' tables exist, their barriers are set
    if (threadIdx.x == 0) {
      bar_init(&table.bar[0]);
      bar_init(&table.bar[1]);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_barrier();
  }
  for (;;) {
    Run<ENT> run(in.c);
    int token_e = 0;
    const int token_v = walk.token_vector(now.row, ex, token_e);
#pragma unroll
    for (int j = 0; j < K; j += M) {
      copy_wait_upto<K - M>(K - M - j);
      uint4 u[M];
#pragma unroll
      for (int k = 0; k < M; ++k) {
        u[k] = make_uint4(low, low, low, low);
        if ((j + k) * NT < now.mid) u[k] = mine[(j + k) * NT];
      }
      run.template add_vectors<T, M, NT>(u, in.c, token_v - j * NT, token_e);
    }
    RowStats r = walk.join(run, now.row, ex, table, turn);
    typename W::Result q;
    float own = 0.f;
    if (threadIdx.x < 32) {
      float b = 0.f;
      q = walk.result(r, ex, own, b);
      float a = own;
      walk.scaled(ex, a, b);
      if (threadIdx.x == 0) incoming = make_float4(a, b, r.s0, r.t);
    }
    typename W::Place next{-1, nullptr, 0, 0};
    typename W::Extra nx{};
    const int64_t row = walk.advance();
    if (row >= 0) {
      next = walk.place(row);
      nx = walk.extra(row);
    }
    if constexpr (CL) {
      turn.broken = __syncthreads_or(turn.broken);
      if (turn.broken) {
        r = no_stats();
        q.lp = q.o.loss = own = NAN;
      }
    } else {
      __syncthreads();
    }
    if (threadIdx.x < 32) walk.outputs(now.row, r, ex, q, own);
    const typename W::Writer wr = walk.writer(now.row, r, turn.broken ? NAN : incoming.x, incoming.y);
    if (wr.g && !wr.sh.far) {
#pragma unroll
      for (int j = 0; j < K; ++j) {
        walk.write(wr, j * NT, mine[j * NT], j * NT < now.mid);
        fetch(next, j);
      }
    } else {
      if (wr.g) walk.write_far(wr, now);
#pragma unroll
      for (int j = 0; j < K; ++j) fetch(next, j);
    }
    if (wr.g) walk.finish(wr, now.row, ex, [&] { return incoming; });
    if (next.row < 0) break;
    walk.token_logit(next.row, nx);
    now = next;
    ex = nx;
  }
  // No CTA leaves while another might still store to it.  Where every wait succeeded all that was
  // sent here has come; after one that ran out the rest, all sent by now, is on its way.
  if constexpr (CL) {
    cluster_barrier();
    if (turn.broken)
      for (int k = 0; k < 64; ++k) __nanosleep(1000);
  }
}

// ---- short rows in tiles ---------------------------------------------------------
// Rows that lie one after the other, each of few logits: a CTA copies a tile of R whole rows
// (R a power of two, the tile 16-byte aligned) to shared memory as one
// stretch, G = 256 / R lanes (at most 32) sum up each row, one thread a row then forms its
// log-probability, loss term and coefficients -- the fp64 and the transcendental steps
// that would cost a whole warp's time with a warp a row -- and the gradient is
// written over the stretch again, by vectors that need not respect the rows.
// Bound by instruction issue (73 % of the slots, 39 % of DRAM's peak): 1.07 GB in rows of 18 fp32 take 281 us forward
// (0.59 of the copy bandwidth) and 652 us with the gradient (0.51), where a warp's lanes
// in groups of 8 took 887 and 2211; rows of 64 bf16 279 us (0.60), of 512 bf16 252 us
// (0.66), of 200 fp32 201 us (0.83).  More CTAs an SM are faster at any unrolling (5
// of 256 threads: 48 registers).
// ACC: how a lane reads a row: 0 one element, 1 two (V even), 2 a 16-byte vector (rows are whole vectors).
constexpr int kTileThreads = 256;
constexpr int kTileCtas = 5;  // an SM: 48 registers a thread

struct TileShape {
  int rows, log_lanes; // R, log2 G
  int turn;            // a row's lanes start `turn` rounds further than the last row's do (bank conflicts), ...
  int rounds;          // ... of so many that all lanes take part in
  Divide by_vocab;     // an element's row
};

template <class T, bool ENT, int MODE, class Src, int ACC>
__global__ void __launch_bounds__(kTileThreads, kTileCtas) tile_rows_kernel(Rows<T> in, RowOut out, GradRows<T> gr, Src src,
                                                                    TileShape shape) {
  if constexpr (Src::kPolicy && MODE == kBwd) {
    if (src.skip()) return;
  }
  constexpr int N = Vec<T>::N;
  constexpr bool kTerms = Src::kPolicy && MODE != kBwd;
  extern __shared__ uint4 tile[];
  __shared__ float4 found[kTileThreads];  // a row's m, S0, S1; then its m, A, B and whether it has a gradient
  const T* elems = reinterpret_cast<const T*>(tile);
  const int tid = threadIdx.x, V = in.V, R = shape.rows, G = 1 << shape.log_lanes;
  const float c = in.c;
  double sum[kTerms ? kSums : 1] = {};
  const int r = tid >> shape.log_lanes, lane = tid & (G - 1);
  const int first = lane + (shape.turn && shape.rounds ? r % shape.rounds * G : 0);
  const int64_t tiles = (in.rows + R - 1) / R;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t row0 = t * R;
    const int rows = (int)(in.rows - row0 < R ? in.rows - row0 : R);
    const int count = rows * V, vecs = count / N;
    const T* x = in.x + row0 * V;
    for (int v = tid; v < vecs; v += kTileThreads) copy16(tile + v, reinterpret_cast<const uint4*>(x) + v);
    copy_commit();
    for (int i = vecs * N + tid; i < count; i += kTileThreads) reinterpret_cast<T*>(tile)[i] = x[i];
    // what the row's thread needs, asked for meanwhile
    const int64_t row = row0 + tid;
    const bool own = tid < rows;
    bool kept = false;
    int64_t tok = 0;
    float old_lp = 0.f, adv = 0.f, ref = 0.f, w = 0.f, a = 0.f, b = 0.f;
    if (own) {
      kept = mask_at(in.mask, row);
      if (kept) tok = in.tokens[row];
      if constexpr (Src::kPolicy) {
        const int64_t env = in.env(row);
        old_lp = src.p.old_lp[row];
        adv = src.p.adv[src.p.adv_row ? env : row];
        if (src.p.ref) ref = src.p.ref[row];
        if (kept) w = policy_weight(src.p, env);
      } else if constexpr (MODE == kBwd) {
        if (src.g_lp) a = src.g_lp[row];
        if constexpr (ENT) b = src.g_ent[row];
      }
    }
    copy_wait<0>();
    __syncthreads();
    // ---- a row's sums, by its lanes
    if (r < R) {  // whole warps
      const bool there = r < rows;
      const T* line = elems + r * V;
      constexpr int W = ACC == 2 ? N : ACC == 1 ? 2 : 1;
      const int n = there ? V / W : 0;         // accesses of the row, lane, lane + G, ... of which are this lane's
      auto load = [&](int k, F2 (&f)[ACC == 2 ? N / 2 : 1]) {
        if constexpr (ACC == 2) {
          const uint4 u = reinterpret_cast<const uint4*>(line)[k];
#pragma unroll
          for (int q = 0; q < N / 2; ++q) f[q] = Vec<T>::pair(u, q);
        } else if constexpr (ACC == 1) {
          f[0] = Vec<T>::two(line + 2 * k);
        } else {
          f[0] = f2(Vec<T>::get(line + k), -INFINITY);
        }
      };
      // the lane's accesses; with a turn from `first` on, around the end of the whole
      // rounds, then the rest (always going round costs 8 % where no turn is needed)
      auto each = [&](auto&& f) {
        if (!shape.turn) {
          for (int k = lane; k < n; k += G) f(k);
        } else {
          const int whole = there ? shape.rounds : 0, wrap = shape.rounds * G;
          int k = first;
          for (int i = 0; i < whole; ++i) {
            f(k);
            k += G;
            if (k >= wrap) k -= wrap;
          }
          if (lane + wrap < n) f(lane + wrap);
        }
      };
      float m = -INFINITY;
      each([&](int k) {
        F2 f[ACC == 2 ? N / 2 : 1];
        load(k, f);
#pragma unroll
        for (int q = 0; q < (ACC == 2 ? N / 2 : 1); ++q) {
          float y, z;
          split(f[q], y, z);
          m = fmaxf(m, fmaxf(y, z));
        }
      });
      for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      F2 s0 = f2(0.f, 0.f), s1 = s0;
      const F2 nm = f2(-m, -m), cc = f2(c, c);
      each([&](int k) {
        F2 f[ACC == 2 ? N / 2 : 1];
        load(k, f);
#pragma unroll
        for (int q = 0; q < (ACC == 2 ? N / 2 : 1); ++q) {
          const F2 d = mul2(add2(f[q], nm), cc);
          float y, z;
          split(d, y, z);
          const F2 e = f2(ex2(y), ex2(z));
          s0 = add2(s0, e);
          s1 = fma2(e, f2(fmaxf(y, kDeep), fmaxf(z, kDeep)), s1);
        }
      });
      float p0, p1, y;
      split(s0, p0, y);
      p0 += y;
      split(s1, p1, y);
      p1 += y;
      for (int o = G / 2; o > 0; o >>= 1) {
        p0 += __shfl_xor_sync(0xffffffffu, p0, o);
        p1 += __shfl_xor_sync(0xffffffffu, p1, o);
      }
      if (lane == 0) found[r] = make_float4(m, p0, p1, 0.f);
    }
    __syncthreads();
    // ---- a row's results, by its thread
    float at_token = 0.f;
    bool has = false;
    if (own) {
      const float4 q = found[tid];
      const RowStats st{q.x, q.y, q.z / q.y, true, q.y == 1.f && q.z == 0.f};
      const bool ok = tok >= 0 && tok < V;
      const float xt = ok ? Vec<T>::get(elems + tid * V + (int)tok) : NAN;
      double lp = 0.0;
      float ent = 0.f;
      if (kept) {
        if constexpr (Src::kPolicy || MODE != kBwd) lp = logprob_of(xt, st, c, in.c64, in.c_off);
        if constexpr (ENT && MODE != kBwd) ent = entropy_of(st);
        if constexpr (Src::kPolicy) {
          const Policy& p = src.p;
          const PolicyTerm o = policy_term(p, diff(lp, old_lp), adv, diff(lp, ref));
          a = w * o.d;
          if constexpr (ENT) b = -w * p.ent_coef;
          if constexpr (kTerms) {
            const float term = ENT && p.ent_coef != 0.f ? o.loss - p.ent_coef * ent : o.loss;
            sum[0] += (double)w * (double)term;
            if (src.sums.stats) {
              sum[1] += o.kl; sum[2] += drift_of(diff(lp, old_lp)); sum[3] += o.clipped ? 1.0 : 0.0; sum[4] += ent;
              sum[5] += 1.0;
            }
          }
          a *= src.up();
          b *= src.up();
        }
        if (!ok) a = NAN;
      } else {
        a = b = 0.f;
      }
      if constexpr (MODE != kBwd) {
        out.logprob[row] = (float)lp;
        if (out.entropy) out.entropy[row] = ent;
      }
      if constexpr (MODE != kFwd) {
        has = a != 0.f || b != 0.f;
        const RowGrad rg = row_grad(a, b, st, in.inv_temp);
        found[tid] = make_float4(st.m, -rg.A, -rg.B, has ? 1.f : 0.f);
        has = has && ok;
        if (has) at_token = token_grad(xt, Shift{c, st.m, true}, a, b, st.s0, st.t, in.inv_temp);
      }
    }
    // ---- the gradient over the stretch
    if constexpr (MODE != kFwd) {
      __syncthreads();
      T* g = gr.g;
      if (g) {
        g += row0 * V;
        auto at = [&](float y, const float4& q) {
          const float d = (y - q.x) * c, e = ex2(d);
          const float v = ENT ? e * fmaf(q.z, fmaxf(d, kDeep), q.y) : e * q.y;
          return q.w != 0.f ? v : 0.f;
        };
        for (int v = tid; v < vecs; v += kTileThreads) {
          const uint4 u = tile[v];
          float f[N];
          Vec<T>::unpack(u, f);
          int line = (int)shape.by_vocab(v * N);
          float4 q = found[line];
          if constexpr (ACC == 2) {
#pragma unroll
            for (int e = 0; e < N; ++e) f[e] = at(f[e], q);
          } else {
            int left = (line + 1) * V - v * N;  // elements to the end of the row
#pragma unroll
            for (int e = 0; e < N; ++e) {
              if (left == 0) {
                q = found[++line];
                left = V;
              }
              f[e] = at(f[e], q);
              --left;
            }
          }
          __stcs(reinterpret_cast<uint4*>(g) + v, Vec<T>::pack(f));
        }
        for (int i = vecs * N + tid; i < count; i += kTileThreads)
          g[i] = Vec<T>::put(at(Vec<T>::get(elems + i), found[(int)shape.by_vocab(i)]));
        __syncthreads();  // the token's element goes over what its vector holds
        if (has) g[(int64_t)tid * V + tok] = Vec<T>::put(at_token);
      }
    }
    __syncthreads();  // the tile is read
  }
  if constexpr (kTerms) finish_sums<kTileThreads>(sum, src.sums);
}

// ---- short rows anywhere: G lanes a row, E elements a lane, the row in registers -----
// For rows that do not lie one after the other from a 16-byte boundary on.  The fixed steps of a row cost
// the whole group's time: 14.9 million rows of 18 fp32 in 887 us forward (0.19 of the copy
// bandwidth), 1024 fp32 in 194 us (0.86).
// Each CTA takes tiles of 256 / G rows in strides of the grid; with the policy
// loss it adds up its own rows' terms on the way.
template <class T, bool ENT, int MODE, class Src, int G, int E>
__global__ void __launch_bounds__(256) lane_rows_kernel(Rows<T> in, RowOut out, GradRows<T> gr, Src src) {
  if constexpr (Src::kPolicy && MODE == kBwd) {
    if (src.skip()) return;
  }
  constexpr bool kTerms = Src::kPolicy && MODE != kBwd;
  constexpr int kPer = 256 / G;
  const int lane = threadIdx.x & (G - 1);
  const int V = (int)in.V;
  double sum[kTerms ? kSums : 1] = {};
  const int64_t tiles = (in.rows + kPer - 1) / kPer;
  for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const int64_t row_raw = tile * kPer + threadIdx.x / G;
    const bool live = row_raw < in.rows;
    const int64_t row = live ? row_raw : in.rows - 1;  // idle lanes shuffle along on the last row
    const T* x = in.x + in.at(row);
    T* g = MODE == kFwd || !gr.g ? nullptr : gr.g + gr.at(row, in);
    const bool kept = mask_at(in.mask, row);
    const int64_t tok = kept ? in.tokens[row] : 0;
    const bool ok = tok >= 0 && tok < V;
    float f[E];
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const int i = lane + k * G;
      f[k] = i < V && kept ? Vec<T>::get(x + i) : -INFINITY;
    }
    const float xt = kept && ok ? Vec<T>::get(x + tok) : NAN;
    float m = f[0];
#pragma unroll
    for (int k = 1; k < E; ++k) m = fmaxf(m, f[k]);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const Shift sh{in.c, m, true};
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int k = 0; k < E; ++k) {
      const float d = lane + k * G < V ? sh(f[k]) : -INFINITY;
      const float e = ex2(d);
      s0 += e;
      s1 = fmaf(e, fmaxf(d, kDeep), s1);
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) {
      s0 += __shfl_xor_sync(0xffffffffu, s0, o);
      s1 += __shfl_xor_sync(0xffffffffu, s1, o);
    }
    const RowStats r{m, s0, s1 / s0, true, ENT && s0 == 1.f && s1 == 0.f};
    double lp = 0.0;
    float ent = 0.f;
    if (Src::kPolicy || MODE != kBwd) lp = logprob_of(xt, r, in.c, in.c64, in.c_off);
    if constexpr (ENT) ent = entropy_of(r);
    if (!kept) { lp = 0.0; ent = 0.f; }
    float a = 0.f, b = 0.f;
    if (kept) {
      if constexpr (Src::kPolicy) {
        const int64_t env = in.env(row);
        const Policy& p = src.p;
        const PolicyTerm o = policy_term(p, diff(lp, p.old_lp[row]), p.adv[p.adv_row ? env : row],
                                         diff(lp, p.ref ? p.ref[row] : 0.f));
        const float w = policy_weight(p, env);
        a = w * o.d;
        if constexpr (ENT) b = -w * p.ent_coef;
        if constexpr (kTerms) {
          if (live && lane == 0) {
            const float term = ENT && p.ent_coef != 0.f ? o.loss - p.ent_coef * ent : o.loss;
            sum[0] += (double)w * (double)term;
            sum[1] += o.kl; sum[2] += drift_of(diff(lp, p.old_lp[row])); sum[3] += o.clipped ? 1.0 : 0.0; sum[4] += ent; sum[5] += 1.0;
          }
        }
        a *= src.up();
        b *= src.up();
      } else {
        a = src.g_lp ? src.g_lp[row] : 0.f;
        if constexpr (ENT && MODE == kBwd) b = src.g_ent[row];
      }
      if (!ok) a = NAN;
    }
    if constexpr (MODE != kBwd) {
      if (live && lane == 0) {
        out.logprob[row] = (float)lp;
        if (out.entropy) out.entropy[row] = ent;
      }
    }
    if (g && live) {
      const bool none = a == 0.f && b == 0.f;
      const RowGrad rg = row_grad(a, b, r, in.inv_temp);
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int i = lane + k * G;
        if (i < V) {
          const float o = i == tok ? token_grad(f[k], sh, a, b, r.s0, r.t, in.inv_temp) : grad_at<ENT>(f[k], sh, rg);
          g[i] = Vec<T>::put(none ? 0.f : o);
        }
      }
    }
  }
  if constexpr (kTerms) finish_sums<256>(sum, src.sums);
}

}  // namespace tok
}  // namespace rls
