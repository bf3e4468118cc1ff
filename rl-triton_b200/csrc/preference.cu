// preference.cu -- the paired preference loss over token log-probabilities
// (rlscan.h has the formulas).  Forward: one CTA a pair sums both responses;
// the last CTA to finish adds the pairs' losses in their order.  The forward
// call writes one coefficient a response, from which the backward call writes
// the gradient: nothing per token is kept between them.  9 bytes a step forward, 5
// backward; 512 pairs x 4096 take 18 us (2.1 TB/s: a CTA's loads, then its one thread's
// loss) and 9 us (2.4 TB/s), 4 x 257 take 6 us and 2 us, all latency.
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
  float* rewards[2]; // [B] each
  float* coef;       // [2, B] or null
  double* terms;     // [B]
  unsigned* ticket;
};

template <int NT, int K>
__device__ __forceinline__ void block_sums(double (&v)[K]) {
  __shared__ double part[NT / 32][K];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) part[threadIdx.x >> 5][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    v[k] = part[0][k];
    for (int w = 1; w < NT / 32; ++w) v[k] += part[w][k];
  }
}

// A thread's share of a response's sum and count.  Differences are fp32, of four steps
// at a time; their sums fp64: a sum over 10^5 steps of differences near 0 keeps the
// accuracy of its terms.
template <int NT>
__device__ __forceinline__ void side_sum(const Side& d, bool ref_pair, int64_t b, double& sum, double& n) {
  const float* ref = ref_pair ? nullptr : d.ref;
  const int64_t i0 = b * d.T;
  unsigned count = 0;
  sum = 0;
  if (d.T % 4 == 0 && (((uintptr_t)d.lp | (uintptr_t)ref) & 15) == 0) {
#pragma unroll 2
    for (int64_t t = threadIdx.x * 4; t < d.T; t += NT * 4) {
      const unsigned m = mask_four(d.mask, i0 + t, i0 + d.T);
      const float4 x = __ldcs(reinterpret_cast<const float4*>(d.lp + i0 + t));
      const float4 y = ref ? __ldcs(reinterpret_cast<const float4*>(ref + i0 + t)) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float a = (m & 1u ? x.x - y.x : 0.f) + (m & 2u ? x.y - y.y : 0.f);
      const float c = (m & 4u ? x.z - y.z : 0.f) + (m & 8u ? x.w - y.w : 0.f);
      sum += (double)(a + c);
      count += __popc(m);
    }
  } else {
#pragma unroll 4
    for (int64_t t = threadIdx.x; t < d.T; t += NT)
      if (mask_at(d.mask, i0 + t)) {
        sum += (double)(d.lp[i0 + t] - (ref ? ref[i0 + t] : 0.f));
        ++count;
      }
  }
  n = count;
}

template <int NT>
__global__ void __launch_bounds__(NT) preference_kernel(PrefArgs p) {
  __shared__ bool last;
  const int64_t b = blockIdx.x;
  double s[2], n[2], v[4];
  side_sum<NT>(p.side[0], p.ref_pair, b, v[0], v[1]);
  side_sum<NT>(p.side[1], p.ref_pair, b, v[2], v[3]);
  block_sums<NT>(v);
  for (int k = 0; k < 2; ++k) {
    if (p.side[k].ref && p.ref_pair) v[2 * k] -= (double)p.side[k].ref[b];
    n[k] = p.normalized ? fmax(v[2 * k + 1], 1.0) : 1.0;
    s[k] = v[2 * k] / n[k];
  }
  if (threadIdx.x == 0) {
    const double beta = p.beta, gap = s[0] - s[1], x = beta * gap, e = p.smoothing;
    double term, d;  // d: by gap
    if (p.kind == RLS_PREFERENCE_SIGMOID) {
      // the parts of size 1 in fp32, as one thread forms them while the CTA waits
      const float z = expf(-fabsf((float)x)), l = log1pf(z);
      term = (double)l + (1.0 - e) * fmax(-x, 0.0);
      if (e > 0.0) term += e * fmax(x, 0.0);  // x may be +inf: a rejected token of log-probability -inf
      const float less = z / (1.f + z);  // the smaller of sig(x) and sig(-x)
      d = beta * (x >= 0 ? e - (double)less : (double)less - (1.0 - e));
      if (isnan(x)) term = d = x;
    } else if (p.kind == RLS_PREFERENCE_IPO) {
      const double y = gap - 0.5 / beta;
      term = y * y;
      d = 2.0 * y;
    } else {
      term = 1.0 - x > 0.0 ? 1.0 - x : isnan(x) ? x : 0.0;
      d = x < 1.0 ? -beta : isnan(x) ? x : 0.0;
    }
    p.rewards[0][b] = (float)(beta * s[0]);
    p.rewards[1][b] = (float)(beta * s[1]);
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
  double all[1] = {0};
  for (int64_t i = threadIdx.x; i < p.B; i += NT) all[0] += __ldcg(&p.terms[i]);
  block_sums<NT>(all);
  if (threadIdx.x == 0) {
    *p.loss = (float)(all[0] / (double)p.B);
    *p.ticket = 0u;
  }
}

constexpr int kSpread = 256;
constexpr int64_t kSpreadSteps = kSpread * 16;  // of a response, a CTA's

struct SpreadArgs {
  const float* coef;
  const float* g;
  Mask mask[2];
  float* grad[2];
  int64_t T[2];
  int64_t B, chunks[2];  // CTAs of a response
};

// grad = coefficient of the response where its step counts.
__global__ void __launch_bounds__(kSpread) preference_spread_kernel(SpreadArgs a) {
  int64_t id = blockIdx.x;
  const int k = id >= a.B * a.chunks[0] ? 1 : 0;
  if (k) id -= a.B * a.chunks[0];
  const int64_t b = id / a.chunks[k], c = id - b * a.chunks[k];
  const int64_t T = a.T[k], t0 = c * kSpreadSteps, i0 = b * T;
  const float w = a.coef[k * a.B + b] * *a.g;
  const int64_t t1 = t0 + kSpreadSteps < T ? t0 + kSpreadSteps : T;
  if (T % 4 == 0 && ((uintptr_t)a.grad[k] & 15) == 0) {
#pragma unroll 4
    for (int64_t t = t0 + threadIdx.x * 4; t < t1; t += kSpread * 4) {
      const unsigned m = mask_four(a.mask[k], i0 + t, i0 + T);
      __stcs(reinterpret_cast<float4*>(a.grad[k] + i0 + t),
             make_float4(m & 1u ? w : 0.f, m & 2u ? w : 0.f, m & 4u ? w : 0.f, m & 8u ? w : 0.f));
    }
  } else {
#pragma unroll 4
    for (int64_t t = t0 + threadIdx.x; t < t1; t += kSpread) a.grad[k][i0 + t] = mask_at(a.mask[k], i0 + t) ? w : 0.f;
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
                                   int length_normalized, float* loss, float* chosen_rewards, float* rejected_rewards, float* coef, void* ws,
                                   size_t ws_bytes, void* stream) {
  if (!sizes_ok(pairs, chosen_len, rejected_len) || !loss) return RLS_EINVAL;
  if (kind < RLS_PREFERENCE_SIGMOID || kind > RLS_PREFERENCE_HINGE) return RLS_EINVAL;
  if (mask_kind < RLS_MASK_NONE || mask_kind > RLS_MASK_I64) return RLS_EINVAL;
  if ((chosen_mask || rejected_mask) && mask_kind == RLS_MASK_NONE) return RLS_EINVAL;
  if (!std::isfinite(beta) || (kind == RLS_PREFERENCE_IPO && beta == 0.f)) return RLS_EINVAL;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (pairs == 0) {
    TokenGuard guard{loss};
    if (guard.status()) return guard.status();
    return cudaMemsetAsync(loss, 0, sizeof(float), s) == cudaSuccess ? RLS_OK : RLS_ECUDA;
  }
  if (pairs > 0x7fffffffLL) return RLS_EINVAL;
  if ((chosen_len > 0 && !chosen) || (rejected_len > 0 && !rejected) || !chosen_rewards ||
      !rejected_rewards || !ws) return RLS_EINVAL;
  if (!al(chosen, 4) || !al(rejected, 4) || !al(ref_chosen, 4) || !al(ref_rejected, 4) || !al(chosen_rewards, 4) ||
      !al(rejected_rewards, 4) || !al(coef, 4) || !al(loss, 4) || !al(ws, 16) ||
      !al(chosen_mask, mask_align(mask_kind)) || !al(rejected_mask, mask_align(mask_kind)))
    return RLS_EALIGN;
  if (64 + (size_t)pairs * sizeof(double) > ws_bytes) return RLS_EWORKSPACE;
  TokenGuard guard{chosen_len ? chosen : nullptr, rejected_len ? rejected : nullptr, ref_chosen, ref_rejected,
                    chosen_mask, rejected_mask, loss, chosen_rewards, rejected_rewards, coef, ws};
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
  p.rewards[0] = chosen_rewards;
  p.rewards[1] = rejected_rewards;
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
  const int64_t per = kSpreadSteps;
  // a side without a gradient takes no blocks
  const int64_t c0 = grad_chosen ? (chosen_len + per - 1) / per : 0;
  const int64_t c1 = grad_rejected ? (rejected_len + per - 1) / per : 0;
  const int64_t blocks = pairs * (c0 + c1);
  if (blocks == 0) return RLS_OK;
  if (blocks > 0x7fffffffLL) return RLS_EINVAL;
  if (!coef || !grad_loss) return RLS_EINVAL;
  if (!al(coef, 4) || !al(grad_loss, 4) || !al(grad_chosen, 4) || !al(grad_rejected, 4) ||
      !al(chosen_mask, mask_align(mask_kind)) || !al(rejected_mask, mask_align(mask_kind)))
    return RLS_EALIGN;
  TokenGuard guard{coef, grad_loss, chosen_mask, rejected_mask, grad_chosen, grad_rejected};
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
