// preference.cu -- the paired preference loss over token log-probabilities
// (rlscan.h has the formulas).  Forward: one CTA a pair sums both responses;
// the last CTA to finish adds the pairs' losses in their order.  The forward
// call writes one coefficient a response, from which the backward call writes
// the gradient: nothing per token is kept between them.
#include <cmath>
#include <cstdint>
#include <mutex>

#include "host_shared.h"
#include "token_kernels.cuh"

using namespace rls;
using namespace rls::tok;

namespace {

struct Side {
  const float* lp;
  const float* ref;  // may be null
  Mask mask;
  int64_t T;
};

struct PrefArgs {
  Side side[2];      // chosen, rejected
  bool ref_pair;
  int64_t B;
  float beta, smoothing;
  int kind;
  bool normalized;
  float* loss;
  float* rewards;    // [2, B]
  float* coef;       // [2, B] or null
  double* terms;     // [B]
  unsigned* ticket;
};

template <int NT>
__device__ __forceinline__ double2 block_sum2(double a, double b) {
  __shared__ double2 part[NT / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a += __shfl_xor_sync(0xffffffffu, a, o);
    b += __shfl_xor_sync(0xffffffffu, b, o);
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_double2(a, b);
  __syncthreads();
  double2 s = part[0];
  for (int w = 1; w < NT / 32; ++w) { s.x += part[w].x; s.y += part[w].y; }
  return s;
}

// A response's sum and count, over the CTA.  Sums are fp64: a sum over 10^5
// steps of differences near 0 keeps the accuracy of its terms.
template <int NT>
__device__ __forceinline__ double2 side_sum(const Side& d, bool ref_pair, int64_t b) {
  double sum = 0, n = 0;
  const bool ref = d.ref && !ref_pair;
  for (int64_t t = threadIdx.x; t < d.T; t += NT) {
    const int64_t i = b * d.T + t;
    if (mask_at(d.mask, i)) {
      sum += (double)d.lp[i] - (ref ? (double)d.ref[i] : 0.0);
      n += 1.0;
    }
  }
  double2 s = block_sum2<NT>(sum, n);
  if (d.ref && ref_pair) s.x -= (double)d.ref[b];
  return s;
}

template <int NT>
__global__ void __launch_bounds__(NT) preference_kernel(PrefArgs p) {
  __shared__ bool last;
  const int64_t b = blockIdx.x;
  double s[2], n[2];
  for (int k = 0; k < 2; ++k) {
    const double2 q = side_sum<NT>(p.side[k], p.ref_pair, b);
    n[k] = p.normalized ? fmax(q.y, 1.0) : 1.0;
    s[k] = q.x / n[k];
  }
  if (threadIdx.x == 0) {
    const double beta = p.beta, gap = s[0] - s[1], x = beta * gap, e = p.smoothing;
    double term, d;  // d: by gap
    if (p.kind == RLS_PREFERENCE_SIGMOID) {
      const double z = exp(-fabs(x)), l = log1p(z);
      term = (1.0 - e) * (l + fmax(-x, 0.0)) + e * (l + fmax(x, 0.0));
      const double sig = x >= 0 ? 1.0 / (1.0 + z) : z / (1.0 + z);
      d = beta * (sig - (1.0 - e));
      if (isnan(x)) term = d = x;
    } else if (p.kind == RLS_PREFERENCE_IPO) {
      const double y = gap - 0.5 / beta;
      term = y * y;
      d = 2.0 * y;
    } else {
      term = 1.0 - x > 0.0 ? 1.0 - x : isnan(x) ? x : 0.0;
      d = x < 1.0 ? -beta : isnan(x) ? x : 0.0;
    }
    p.rewards[b] = (float)(beta * s[0]);
    p.rewards[p.B + b] = (float)(beta * s[1]);
    if (p.coef) {
      p.coef[b] = (float)(d / (n[0] * (double)p.B));
      p.coef[p.B + b] = (float)(-d / (n[1] * (double)p.B));
    }
    p.terms[b] = term;
    __threadfence();
    last = atomicAdd(p.ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double sum = 0;
  for (int64_t i = threadIdx.x; i < p.B; i += NT) sum += __ldcg(&p.terms[i]);
  const double2 all = block_sum2<NT>(sum, 0.0);
  if (threadIdx.x == 0) {
    *p.loss = (float)(all.x / (double)p.B);
    *p.ticket = 0u;
  }
}

constexpr int kSpread = 256;

struct SpreadArgs {
  const float* coef;
  const float* g;
  Mask mask[2];
  float* grad[2];
  int64_t T[2];
  int64_t B, chunks[2];  // chunks of kSpread * 4 steps in a response
};

// grad = coefficient of the response where its step counts.
__global__ void __launch_bounds__(kSpread) preference_spread_kernel(SpreadArgs a) {
  int64_t id = blockIdx.x;
  const int k = id >= a.B * a.chunks[0] ? 1 : 0;
  if (k) id -= a.B * a.chunks[0];
  const int64_t b = id / a.chunks[k], c = id - b * a.chunks[k];
  const int64_t T = a.T[k], t0 = c * (kSpread * 4);
  const float w = a.coef[k * a.B + b] * *a.g;
  const int64_t t1 = t0 + kSpread * 4 < T ? t0 + kSpread * 4 : T;
  for (int64_t t = t0 + threadIdx.x; t < t1; t += kSpread) {
    const int64_t i = b * T + t;
    a.grad[k][i] = mask_at(a.mask[k], i) ? w : 0.f;
  }
}

bool al(const void* p, size_t a) { return p == nullptr || ((uintptr_t)p % a) == 0; }
size_t mask_align(int kind) {
  return kind == RLS_MASK_I64 ? 8 : kind == RLS_MASK_F32 || kind == RLS_MASK_I32 ? 4 : kind == RLS_MASK_BF16 ? 2 : 1;
}
bool sizes_ok(int64_t B, int64_t T0, int64_t T1) {
  if (B < 0 || T0 < 0 || T1 < 0) return false;
  const int64_t T = T0 > T1 ? T0 : T1;
  return T == 0 || B <= INT64_MAX / (8 * T);
}
Mask mask_of(const void* p, int kind) { return Mask{p, p ? kind : RLS_MASK_NONE}; }

}  // namespace

extern "C" int rls_preference_loss(const float* chosen, const float* rejected, const float* ref_chosen,
                                   const float* ref_rejected, int ref_per_pair, const void* chosen_mask,
                                   const void* rejected_mask, int mask_kind, int64_t pairs, int64_t chosen_len,
                                   int64_t rejected_len, float beta, float smoothing, int kind,
                                   int length_normalized, float* loss, float* rewards, float* coef, void* ws,
                                   size_t ws_bytes, void* stream) {
  if (!sizes_ok(pairs, chosen_len, rejected_len) || !loss) return RLS_EINVAL;
  if (kind < RLS_PREFERENCE_SIGMOID || kind > RLS_PREFERENCE_HINGE) return RLS_EINVAL;
  if (mask_kind < RLS_MASK_NONE || mask_kind > RLS_MASK_I64) return RLS_EINVAL;
  if ((chosen_mask || rejected_mask) && mask_kind == RLS_MASK_NONE) return RLS_EINVAL;
  if (!std::isfinite(beta) || (kind == RLS_PREFERENCE_IPO && beta == 0.f)) return RLS_EINVAL;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (pairs == 0) {
    DeviceGuard guard{loss};
    if (guard.status()) return guard.status();
    return cudaMemsetAsync(loss, 0, sizeof(float), s) == cudaSuccess ? RLS_OK : RLS_ECUDA;
  }
  if (pairs > 0x7fffffffLL) return RLS_EINVAL;
  if ((chosen_len > 0 && !chosen) || (rejected_len > 0 && !rejected) || !rewards || !ws) return RLS_EINVAL;
  if (!al(chosen, 16) || !al(rejected, 16) || !al(ref_chosen, ref_per_pair ? 4 : 16) ||
      !al(ref_rejected, ref_per_pair ? 4 : 16) || !al(rewards, 4) || !al(coef, 4) || !al(loss, 4) || !al(ws, 16) ||
      !al(chosen_mask, mask_align(mask_kind)) || !al(rejected_mask, mask_align(mask_kind)))
    return RLS_EALIGN;
  if (64 + (size_t)pairs * sizeof(double) > ws_bytes) return RLS_EWORKSPACE;
  DeviceGuard guard{chosen_len ? chosen : nullptr, rejected_len ? rejected : nullptr, ref_chosen, ref_rejected,
                    chosen_mask, rejected_mask, loss, rewards, coef, ws};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  if (int st = prepare_layout(ws, ws_bytes, kLayoutScratch, s)) return st;
  PrefArgs p{};
  p.side[0] = Side{chosen, ref_chosen, mask_of(chosen_mask, mask_kind), chosen_len};
  p.side[1] = Side{rejected, ref_rejected, mask_of(rejected_mask, mask_kind), rejected_len};
  p.ref_pair = ref_per_pair != 0;
  p.B = pairs;
  p.beta = beta;
  p.smoothing = smoothing;
  p.kind = kind;
  p.normalized = length_normalized != 0;
  p.loss = loss;
  p.rewards = rewards;
  p.coef = coef;
  p.terms = reinterpret_cast<double*>(static_cast<char*>(ws) + 64);
  p.ticket = &static_cast<WsHeader*>(ws)->pad[4];
  preference_kernel<512><<<(unsigned)pairs, 512, 0, s>>>(p);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

extern "C" int rls_preference_loss_backward(const float* coef, const float* grad_loss, const void* chosen_mask,
                                            const void* rejected_mask, int mask_kind, float* grad_chosen,
                                            float* grad_rejected, int64_t pairs, int64_t chosen_len,
                                            int64_t rejected_len, void* stream) {
  if (!sizes_ok(pairs, chosen_len, rejected_len)) return RLS_EINVAL;
  if (mask_kind < RLS_MASK_NONE || mask_kind > RLS_MASK_I64) return RLS_EINVAL;
  if ((chosen_mask || rejected_mask) && mask_kind == RLS_MASK_NONE) return RLS_EINVAL;
  const int64_t per = kSpread * 4;
  // a side without a gradient takes no blocks
  const int64_t c0 = grad_chosen ? (chosen_len + per - 1) / per : 0;
  const int64_t c1 = grad_rejected ? (rejected_len + per - 1) / per : 0;
  const int64_t blocks = pairs * (c0 + c1);
  if (blocks == 0) return RLS_OK;
  if (blocks > 0x7fffffffLL) return RLS_EINVAL;
  if (!coef || !grad_loss) return RLS_EINVAL;
  if (!al(coef, 4) || !al(grad_loss, 4) || !al(grad_chosen, 16) || !al(grad_rejected, 16) ||
      !al(chosen_mask, mask_align(mask_kind)) || !al(rejected_mask, mask_align(mask_kind)))
    return RLS_EALIGN;
  DeviceGuard guard{coef, grad_loss, chosen_mask, rejected_mask, grad_chosen, grad_rejected};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  SpreadArgs a{};
  a.coef = coef;
  a.g = grad_loss;
  a.mask[0] = mask_of(chosen_mask, mask_kind);
  a.mask[1] = mask_of(rejected_mask, mask_kind);
  a.grad[0] = grad_chosen;
  a.grad[1] = grad_rejected;
  a.T[0] = chosen_len;
  a.T[1] = rejected_len;
  a.B = pairs;
  a.chunks[0] = c0;
  a.chunks[1] = c1;
  preference_spread_kernel<<<(unsigned)blocks, kSpread, 0, reinterpret_cast<cudaStream_t>(stream)>>>(a);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}
