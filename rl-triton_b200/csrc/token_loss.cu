// token_loss.cu -- C ABI of the token-level policy operators: log-probabilities
// from logits with their gradient, and the clipped policy loss from
// log-probabilities or from the logits (rlscan.h has the formulas).
#include <cmath>
#include <cstdint>
#include <mutex>

#include "host_shared.h"
#include "token_launch.h"

using namespace rls;
using namespace rls::tok;

namespace {

constexpr int kThreads = 256;

// Tries of a wait of a row's CTAs on one another, each suspended for a while by the hardware.
constexpr unsigned kTeamWait = 1u << 16;
thread_local int g_wait_tries = -1;  // rls_wait_tries

// The ticket and the counts lie in words of the workspace header that the
// estimators do not use; every launch leaves them zero.
unsigned* ticket_of(void* ws) { return &static_cast<WsHeader*>(ws)->pad[4]; }
static_assert(offsetof(WsHeader, pad) % 8 == 0, "the total is 8-byte aligned");

// ---- the mask once over -------------------------------------------------------------
// norm (may be null): norm[1 + n] = steps of env n that count; norm[0] = 1 / (all of
// them), or 1 / (envs that have any) for the mean by sequence.  order (may be null):
// order[0] = all of them, order[1 ..] = those rows, then the others; which row comes
// where depends on timing, nothing that a row gives does.  A CTA an env, or a warp where there are
// many (4096 x 2048 bytes: 9 us; an order of 16 x 512: 5 us, all latency).  Counts are whole numbers: their
// atomics give the same sum in any order.
struct CountWords {
  unsigned long long* total;
  unsigned *some, *front, *back, *ticket;
};
// A thread's share (of NT) of the steps that count among T from i0 on.
template <int NT>
__device__ __forceinline__ unsigned count_steps(const Mask& mask, int64_t i0, int64_t T, int tid) {
  unsigned c = 0;
  int64_t t = 0;
  if (mask.kind == RLS_MASK_U8) {  // 16 bytes at a time from the first boundary on
    const uint8_t* p = reinterpret_cast<const uint8_t*>(mask.p) + i0;
    const int64_t head = (int64_t)((16 - ((uintptr_t)p & 15)) & 15), lead = head < T ? head : T;
    if (tid < lead) c += p[tid] != 0;
    const int64_t vecs = (T - lead) / 16;
#pragma unroll 4
    for (int64_t v = tid; v < vecs; v += NT) {
      const uint4 w = *reinterpret_cast<const uint4*>(p + lead + v * 16);
      c += __popc(__vsetne4(w.x, 0u)) + __popc(__vsetne4(w.y, 0u)) + __popc(__vsetne4(w.z, 0u)) +
           __popc(__vsetne4(w.w, 0u));
    }
    t = lead + vecs * 16;
  }
  for (t += tid; t < T; t += NT) c += mask_at(mask, i0 + t) ? 1u : 0u;
  return c;
}

__global__ void __launch_bounds__(kThreads) count_kernel(Mask mask, int64_t N, int64_t T, int reduction, float* norm,
                                                         int* order, bool warps, CountWords words) {
  __shared__ unsigned part[kThreads / 32], base[2];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long sum = 0;
  unsigned rows = 0;
  if (warps) {  // many envs: a warp each
    for (int64_t n = (int64_t)blockIdx.x * (kThreads / 32) + warp; n < N; n += (int64_t)gridDim.x * (kThreads / 32)) {
      const unsigned c = __reduce_add_sync(0xffffffffu, count_steps<32>(mask, n * T, T, lane));
      if (lane == 0 && norm) norm[1 + n] = (float)c;
      sum += c;
      rows += c > 0;
    }
    __syncthreads();
    if (lane == 0) {
      part[warp] = rows;
      atomicAdd(words.total, sum);
    }
    __syncthreads();
    sum = 0;
    rows = 0;
    for (int w = 0; w < kThreads / 32; ++w) rows += part[w];
    N = 0;
  }
  for (int64_t n = blockIdx.x; n < N; n += gridDim.x) {
    const int64_t i0 = n * T;
    unsigned c = count_steps<kThreads>(mask, i0, T, tid);
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if (lane == 0) part[warp] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < kThreads / 32; ++w) c += part[w];
    sum += c;
    rows += c > 0;
    if (tid == 0) {
      if (norm) norm[1 + n] = (float)c;
      if (order) {
        base[0] = atomicAdd(words.front, c);
        base[1] = atomicAdd(words.back, (unsigned)T - c);
      }
    }
    if (order) {
      const int64_t last = N * T;  // order's last place
      unsigned yes_before = 0;     // of the env, before the chunk
      for (int64_t t0 = 0; t0 < T; t0 += kThreads) {
        const int64_t u = t0 + tid;
        const bool there = u < T, yes = there && mask_at(mask, i0 + u);
        const unsigned votes = __ballot_sync(0xffffffffu, yes);
        __syncthreads();
        if (lane == 0) part[warp] = __popc(votes);
        __syncthreads();
        unsigned before = yes_before;
        for (int w = 0; w < kThreads / 32; ++w) {
          if (w < warp) before += part[w];
          yes_before += part[w];
        }
        const unsigned rank = before + __popc(votes & ((1u << lane) - 1u));
        if (there) order[yes ? 1 + (int64_t)(base[0] + rank) : last - (int64_t)(base[1] + (unsigned)u - rank)] = (int)(i0 + u);
      }
    }
  }
  if (tid == 0) {
    atomicAdd(words.total, sum);
    atomicAdd(words.some, rows);
    __threadfence();
    if (atomicAdd(words.ticket, 1u) == gridDim.x - 1) {
      __threadfence();
      const unsigned long long all = atomicExch(words.total, 0ull);
      const unsigned envs = atomicExch(words.some, 0u);
      atomicExch(words.front, 0u);
      atomicExch(words.back, 0u);
      const double by = reduction == RLS_REDUCE_SEQUENCE ? (double)envs : (double)all;
      if (norm) norm[0] = by > 0.0 ? (float)(1.0 / by) : 0.f;
      if (order) order[0] = (int)all;
      *words.ticket = 0u;
    }
  }
}

// ---- the loss over log-probabilities ----------------------------------------------
struct Terms {
  const float* lp;
  Policy p;
  Mask mask;
  int64_t M, T;
  Divide env;
};

__device__ __forceinline__ void load4(const float* p, int64_t i, int64_t M, float (&o)[4]) {
  if (i + 4 <= M) {
    const float4 v = *reinterpret_cast<const float4*>(p + i);
    o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = i + e < M ? p[i + e] : 0.f;
  }
}

// One pass over the steps: the sums of the loss and the statistics (SUMS) and
// the gradient (GRAD).  17 bytes read and 4 written a step; bound by instruction issue (71 % of
// the slots, 30 % of DRAM's peak: two exponentials, two two-float differences): 4096 x 2048
// steps in 59 us, 3.0 TB/s.  A batch of at most kAlone steps is one CTA's, which then counts
// the steps itself first (COUNT; norm is written as count_kernel does): one launch instead of two, where
// the launches are most of the time.
constexpr int kAlone = 8192, kAloneThreads = 1024;

template <int NT>
__device__ __forceinline__ void count_alone(const Mask& mask, int N, int T, int reduction, float* norm) {
  __shared__ unsigned total, some;
  if (threadIdx.x == 0) total = some = 0u;
  __syncthreads();
  // a warp a row
  for (int n = threadIdx.x >> 5; n < N; n += NT / 32) {
    unsigned c = 0;
    for (int t = threadIdx.x & 31; t < T; t += 32) c += mask_at(mask, (int64_t)n * T + t) ? 1u : 0u;
    c = __reduce_add_sync(0xffffffffu, c);
    if ((threadIdx.x & 31) == 0) {
      norm[1 + n] = (float)c;
      atomicAdd(&total, c);
      if (c) atomicAdd(&some, 1u);
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    const double by = reduction == RLS_REDUCE_SEQUENCE ? (double)some : (double)total;
    norm[0] = by > 0.0 ? (float)(1.0 / by) : 0.f;
  }
  __syncthreads();
}

constexpr int kPolicyCtas = 5;  // an SM
template <bool SUMS, bool GRAD, bool COUNT, int NT>
__global__ void __launch_bounds__(NT, NT == kThreads ? kPolicyCtas : 1) policy_kernel(Terms t, float scale, const float* g, int force, float* grad,
                                                    float* norm, SumOut out) {
  if constexpr (!SUMS) {
    if (g && !force && *g == scale) return;
  }
  if constexpr (COUNT) count_alone<NT>(t.mask, (int)(t.M / t.T), (int)t.T, t.p.reduction, norm);
  const float up = g ? *g : scale;
  double sum[kSums] = {0, 0, 0, 0, 0, 0};
  const int64_t step = (int64_t)gridDim.x * NT * 4;
  for (int64_t i = ((int64_t)blockIdx.x * NT + threadIdx.x) * 4; i < t.M; i += step) {
    float lp[4], old_lp[4], adv[4], ref[4], d[4];
    const unsigned mask = mask_four(t.mask, i, t.M);
    load4(t.lp, i, t.M, lp);
    load4(t.p.old_lp, i, t.M, old_lp);
    if (!t.p.adv_row) load4(t.p.adv, i, t.M, adv);
    if (t.p.ref) load4(t.p.ref, i, t.M, ref);
    int64_t env = t.env(i), col = i - env * t.T;
    float w = policy_weight(t.p, env), a_row = t.p.adv_row ? t.p.adv[env] : 0.f;
    float loss = 0.f;  // of the four
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      d[e] = 0.f;
      if (mask >> e & 1u) {
        const Diff lr = diff(lp[e], old_lp[e]);
        const PolicyTerm o = policy_term(t.p, lr, t.p.adv_row ? a_row : adv[e], diff(lp[e], t.p.ref ? ref[e] : 0.f));
        d[e] = w * o.d * up;
        if constexpr (SUMS) {
          loss = fmaf(w, o.loss, loss);
          if (out.stats) {
            sum[1] += o.kl; sum[2] += drift_of(lr); sum[3] += o.clipped ? 1.0 : 0.0;
            sum[5] += 1.0;
          }
        }
      }
      if (++col == t.T && e < 3 && i + e + 1 < t.M) {
        col = 0;
        ++env;
        w = policy_weight(t.p, env);
        if (t.p.adv_row) a_row = t.p.adv[env];
      }
    }
    if constexpr (SUMS) sum[0] += (double)loss;
    if constexpr (GRAD) {
      if (i + 4 <= t.M) {
        *reinterpret_cast<float4*>(grad + i) = make_float4(d[0], d[1], d[2], d[3]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (i + e < t.M) grad[i + e] = d[e];
      }
    }
  }
  if constexpr (SUMS) finish_sums<NT>(sum, out);
}

// The policy loss over long rows: their records' terms (8192 rows: 5 us, latency).
__global__ void __launch_bounds__(kThreads) row_sums_kernel(const float4* stats, const float* entropy, int64_t rows,
                                                       SumOut o) {
  double sum[kSums] = {0, 0, 0, 0, 0, 0};
  for (int64_t row = (int64_t)blockIdx.x * kThreads + threadIdx.x; row < rows; row += (int64_t)gridDim.x * kThreads) {
    const int flags = __float_as_int(stats[2 * row].w);
    if (!(flags & kFlagKept)) continue;
    const float4 q = stats[2 * row + 1];
    sum[0] += q.y; sum[1] += q.z; sum[2] += q.w;
    sum[3] += flags & kFlagClipped ? 1.0 : 0.0;
    if (entropy) sum[4] += entropy[row];
    sum[5] += 1.0;
  }
  finish_sums<kThreads>(sum, o);
}

bool aligned(const void* p, size_t a = 16) { return p == nullptr || ((uintptr_t)p % a) == 0; }

bool policy_ok(const rls_policy_t* q) {
  return q && q->kl_kind >= RLS_KL_K1 && q->kl_kind <= RLS_KL_K3 && q->reduction >= RLS_REDUCE_TOKEN &&
         q->reduction <= RLS_REDUCE_SUM;
}
bool mask_ok(const void* mask, int kind) {
  return kind >= RLS_MASK_NONE && kind <= RLS_MASK_I64 && (mask == nullptr) == (kind == RLS_MASK_NONE);
}
size_t mask_align(int kind) {
  return kind == RLS_MASK_I64 ? 8 : kind == RLS_MASK_F32 || kind == RLS_MASK_I32 ? 4 : kind == RLS_MASK_BF16 ? 2 : 1;
}

Policy make_policy(const rls_policy_t& q, const float* old_lp, const float* adv, int per_env, const float* ref,
                   const float* norm, bool masked, int64_t N, int64_t T) {
  Policy p{};
  p.old_lp = old_lp;
  p.adv = adv;
  p.adv_row = per_env != 0;
  p.ref = ref;
  // The bounds are the caller's numbers: what the ratio is compared with (their
  // logarithms) and what the clip holds it at (rounded once) come from the same ones.
  const double lo = 1.0 - q.clip_low, hi = 1.0 + q.clip_high;
  p.lo = (float)lo;
  p.hi = (float)hi;
  p.dual = (float)q.dual_clip;
  auto two = [](double x) {
    const float a = (float)x;
    return make_float2(a, std::isfinite(x) ? (float)(x - (double)a) : 0.f);
  };
  p.log_lo = two(lo > 0.0 ? std::log(lo) : -INFINITY);
  p.log_hi = two(std::log(hi));
  p.log_dual = two(q.dual_clip > 0.0 ? std::log(q.dual_clip) : INFINITY);
  p.kl_coef = q.kl_coef;
  p.kl_kind = q.kl_kind;
  p.ent_coef = q.entropy_coef;
  p.reduction = q.reduction;
  p.norm = masked && q.reduction != RLS_REDUCE_SUM ? norm : nullptr;
  // Without a mask both means weigh every step alike.
  p.w = q.reduction == RLS_REDUCE_SUM ? 1.f : (float)(1.0 / ((double)N * (double)T));
  return p;
}

CountWords count_words(void* ws) {
  unsigned* pad = static_cast<WsHeader*>(ws)->pad;
  return CountWords{reinterpret_cast<unsigned long long*>(&pad[6]), &pad[8], &pad[9], &pad[10], ticket_of(ws)};
}

// norm and order may be null.
int launch_count(int reduction, const Mask& mask, float* norm, int* order, int64_t N, int64_t T, void* ws,
                 cudaStream_t s) {
  if (!norm && !order) return RLS_OK;
  int64_t blocks = N < 8LL * num_sms() ? N : 8LL * num_sms();
  const bool warps = !order && N > 16 * num_sms();
  if (warps && (N + 7) / 8 < blocks) blocks = (N + 7) / 8;
  count_kernel<<<(unsigned)blocks, kThreads, 0, s>>>(mask, N, T, reduction, norm, order, warps, count_words(ws));
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

int64_t policy_blocks(int64_t M) {
  const int64_t need = (M + kThreads * 4 - 1) / (kThreads * 4), most = (int64_t)kPolicyCtas * num_sms();
  return need < most ? need : most;
}

// Where a call of `blocks` CTAs leaves its sums.
int sums_in(void* ws, size_t wsb, int64_t blocks, float* loss, float* stats, cudaStream_t s, SumOut* o) {
  if (64 + (size_t)blocks * kSums * sizeof(double) > wsb) return RLS_EWORKSPACE;
  if (int st = prepare_layout(ws, wsb, kLayoutScratch, s)) return st;
  *o = SumOut{reinterpret_cast<double*>(static_cast<char*>(ws) + 64), ticket_of(ws), loss, stats};
  return RLS_OK;
}

// No steps at all: loss and statistics 0.
int clear_loss(float* loss, float* stats, cudaStream_t s) {
  TokenGuard guard{loss, stats};
  if (guard.status()) return guard.status();
  if (cudaMemsetAsync(loss, 0, sizeof(float), s) != cudaSuccess) return RLS_ECUDA;
  if (stats && cudaMemsetAsync(stats, 0, (kSums - 1) * sizeof(float), s) != cudaSuccess) return RLS_ECUDA;
  return RLS_OK;
}

// ---- logits -----------------------------------------------------------------------
struct LogitsCall {
  const void* x;
  int64_t es, ss;
  const int64_t* tokens;
  Mask mask;
  const int* order;
  void* g;
  int64_t ges, gss;
  int64_t N, T, V;
  double temperature;
  int dtype;
};

constexpr int64_t kMostVocab = 0x7fffff00;  // a row's elements are counted in 32 bits

int check_logits(const LogitsCall& c) {
  if (c.N < 0 || c.T < 0 || c.V < 1 || c.V > kMostVocab) return RLS_EINVAL;
  if (c.dtype != RLS_F32 && c.dtype != RLS_BF16) return RLS_EINVAL;
  if (!(c.temperature > 0.0) || !std::isfinite(c.temperature)) return RLS_EINVAL;
  if (!mask_ok(c.mask.p, c.mask.kind)) return RLS_EINVAL;
  if (c.T > 0 && c.N > INT64_MAX / c.T) return RLS_EINVAL;
  if (c.N == 0 || c.T == 0) return RLS_OK;
  if (!c.x || !c.tokens) return RLS_EINVAL;
  if (c.order && (!c.mask.p || c.N * c.T > 0x7ffffffe)) return RLS_EINVAL;
  if (c.es < 0 || c.ss < 0 || c.ges < 0 || c.gss < 0) return RLS_EINVAL;
  // a gradient's rows may not overlap, in whichever order they lie
  if (c.g) {
    const bool steps_in = (c.T == 1 || c.gss >= c.V) && (c.N == 1 || c.ges >= (c.T - 1) * c.gss + c.V);
    const bool envs_in = (c.N == 1 || c.ges >= c.V) && (c.T == 1 || c.gss >= (c.N - 1) * c.ges + c.V);
    if (!steps_in && !envs_in) return RLS_EINVAL;
  }
  const size_t e = c.dtype == RLS_BF16 ? 2 : 4;
  if (!aligned(c.x, e) || !aligned(c.g, e) || !aligned(c.tokens, 8) || !aligned(c.mask.p, mask_align(c.mask.kind)) || !aligned(c.order, 4))
    return RLS_EALIGN;
  return RLS_OK;
}

template <class T>
Rows<T> rows_of_call(const LogitsCall& c) {
  Rows<T> r{};
  r.x = static_cast<const T*>(c.x);
  r.es = c.es;
  r.ss = c.ss;
  r.rows = c.N * c.T;
  r.seq = c.T;
  r.env = Divide::of(c.T, c.N * c.T);
  r.V = (int)c.V;
  r.tokens = c.tokens;
  r.mask = c.mask;
  r.order = c.order;
  r.c64 = 1.4426950408889634074 / c.temperature;
  r.c = (float)r.c64;
  r.c_off = r.c64 / (double)r.c - 1.0;
  r.inv_temp = (float)(1.0 / c.temperature);
  r.flat = c.N == 1 || (c.T == 1 ? false : c.es == c.T * c.ss);
  if (c.T == 1 && c.N > 1) { r.ss = c.es; r.flat = true; }
  return r;
}
template <class T>
GradRows<T> grad_of_call(const LogitsCall& c) {
  GradRows<T> r{};
  r.g = static_cast<T*>(c.g);
  r.es = c.ges;
  r.ss = c.gss;
  r.flat = c.N == 1 || c.ges == c.T * c.gss;
  auto off = [](int64_t elements) { return (elements * (int64_t)sizeof(T)) & 15; };
  r.alike = (((uintptr_t)c.x ^ (uintptr_t)c.g) & 15) == 0 && (c.N == 1 || off(c.es) == off(c.ges)) &&
            (c.T == 1 || off(c.ss) == off(c.gss));
  if (c.T == 1 && c.N > 1) { r.ss = c.ges; r.flat = true; }
  return r;
}

template <class T, bool ENT, int MODE, class Src>
int launch_rows(const LogitsCall& c, const RowOut& out, const Src& src, cudaStream_t s) {
  const Rows<T> in = rows_of_call<T>(c);
  const GradRows<T> gr = grad_of_call<T>(c);
  if (c.V <= kLaneVocab) return launch_lane_rows<T, ENT, MODE, Src>(in, out, gr, src, s);
  return launch_cta_rows<T, ENT, MODE, Src>(in, out, gr, src, s);
}
template <int MODE, class Src>
int launch_logits(const LogitsCall& c, bool ent, const RowOut& out, const Src& src, cudaStream_t s) {
  if (c.dtype == RLS_F32)
    return ent ? launch_rows<float, true, MODE>(c, out, src, s) : launch_rows<float, false, MODE>(c, out, src, s);
  return ent ? launch_rows<__nv_bfloat16, true, MODE>(c, out, src, s)
             : launch_rows<__nv_bfloat16, false, MODE>(c, out, src, s);
}

}  // namespace

int rls::tok::num_sms() {
  static int sms[64] = {0};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
    sms[dev] = n;
  }
  return sms[dev];
}

int64_t rls::tok::sum_blocks(int64_t need) {
  const int64_t most = 8LL * num_sms();
  return need < most ? need : most;
}

extern "C" int rls_wait_tries(int tries) {
  const int before = g_wait_tries;
  g_wait_tries = tries < 0 ? -1 : tries;
  return before;
}

extern "C" int rls_row_order(const void* mask, int mask_kind, int64_t num_envs, int64_t seq_len, int32_t* order,
                             void* ws, size_t ws_bytes, void* stream) {
  if (num_envs < 0 || seq_len < 0 || !mask_ok(mask, mask_kind)) return RLS_EINVAL;
  if (num_envs == 0 || seq_len == 0) return RLS_OK;
  if (!mask || !order || !ws || num_envs > 0x7ffffffe / seq_len) return RLS_EINVAL;
  if (ws_bytes < sizeof(WsHeader)) return RLS_EWORKSPACE;
  if (!aligned(order, 4) || !aligned(ws) || !aligned(mask, mask_align(mask_kind))) return RLS_EALIGN;
  TokenGuard guard{mask, order, ws};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  return launch_count(RLS_REDUCE_TOKEN, Mask{mask, mask_kind}, nullptr, order, num_envs, seq_len, ws,
                      reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int rls_token_logprobs(const void* logits, int64_t env_stride, int64_t step_stride, const int64_t* tokens,
                                  const void* mask, int mask_kind, const int32_t* order, float* logprobs, float* entropy, float* row_stats,
                                  int64_t num_envs, int64_t seq_len, int64_t vocab, double temperature, int in_dtype,
                                  void* stream) {
  LogitsCall c{logits, env_stride, step_stride, tokens, Mask{mask, mask_kind}, order, nullptr, 0, 0, num_envs, seq_len,
               vocab, temperature, in_dtype};
  if (int st = check_logits(c)) return st;
  if (num_envs == 0 || seq_len == 0) return RLS_OK;
  if (!logprobs) return RLS_EINVAL;
  if (!aligned(logprobs) || !aligned(entropy) || !aligned(row_stats)) return RLS_EALIGN;
  TokenGuard guard{logits, tokens, order, mask, logprobs, entropy, row_stats};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  return launch_logits<kFwd>(c, entropy != nullptr, RowOut{logprobs, entropy, reinterpret_cast<float4*>(row_stats)},
                             GivenGrad{nullptr, nullptr}, reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int rls_token_logprobs_backward(const void* logits, int64_t env_stride, int64_t step_stride,
                                           const int64_t* tokens, const void* mask, int mask_kind, const int32_t* order,
                                           const float* row_stats, const float* grad_logprobs,
                                           const float* grad_entropy, void* grad_logits, int64_t grad_env_stride,
                                           int64_t grad_step_stride, int64_t num_envs, int64_t seq_len, int64_t vocab,
                                           double temperature, int in_dtype, void* stream) {
  LogitsCall c{logits, env_stride, step_stride, tokens, Mask{mask, mask_kind}, order, grad_logits, grad_env_stride,
               grad_step_stride, num_envs, seq_len, vocab, temperature, in_dtype};
  if (int st = check_logits(c)) return st;
  if (num_envs == 0 || seq_len == 0) return RLS_OK;
  if ((!row_stats && vocab > kLaneVocab) || !grad_logits) return RLS_EINVAL;
  if (!aligned(row_stats) || !aligned(grad_logprobs, 4) || !aligned(grad_entropy, 4)) return RLS_EALIGN;
  TokenGuard guard{logits, tokens, order, mask, row_stats, grad_logprobs, grad_entropy, grad_logits};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  const RowOut out{nullptr, nullptr, reinterpret_cast<float4*>(const_cast<float*>(row_stats))};
  return launch_logits<kBwd>(c, grad_entropy != nullptr, out, GivenGrad{grad_logprobs, grad_entropy},
                             reinterpret_cast<cudaStream_t>(stream));
}

extern "C" int rls_policy_loss(const float* logprobs, const float* old_logprobs, const float* advantages,
                               int advantages_per_env, const float* ref_logprobs, const void* mask, int mask_kind,
                               const rls_policy_t* policy, float grad_scale, float* norm, float* loss,
                               float* stats, float* grad_logprobs, int64_t num_envs, int64_t seq_len, void* ws, size_t ws_bytes,
                               void* stream) {
  if (num_envs < 0 || seq_len < 0 || !loss || !policy_ok(policy) || !mask_ok(mask, mask_kind)) return RLS_EINVAL;
  if (seq_len > 0 && num_envs > INT64_MAX / seq_len) return RLS_EINVAL;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t M = num_envs * seq_len;
  if (M == 0) {
    return clear_loss(loss, stats, s);
  }
  if (!logprobs || !old_logprobs || !advantages || !ws) return RLS_EINVAL;
  if (mask && policy->reduction != RLS_REDUCE_SUM && !norm) return RLS_EINVAL;
  if (!aligned(logprobs) || !aligned(old_logprobs) || !aligned(advantages) || !aligned(ref_logprobs) ||
      !aligned(grad_logprobs) || !aligned(ws) || !aligned(norm, 4) || !aligned(loss, 4) || !aligned(stats, 4) ||
      !aligned(mask, mask_align(mask_kind)))
    return RLS_EALIGN;
  TokenGuard guard{logprobs, old_logprobs, advantages, ref_logprobs, mask, norm, loss, stats, grad_logprobs, ws};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  Terms t{logprobs,
          make_policy(*policy, old_logprobs, advantages, advantages_per_env, ref_logprobs, norm, mask != nullptr,
                      num_envs, seq_len),
          Mask{mask, mask_kind}, M, seq_len, Divide::of(seq_len, M)};
  SumOut sums;
  const bool alone = M <= kAlone;
  const int64_t blocks = alone ? 1 : policy_blocks(M);
  if (int st = sums_in(ws, ws_bytes, blocks, loss, stats, s, &sums)) return st;
  if (alone) {
    const bool count = t.p.norm != nullptr;
    auto kern = grad_logprobs ? (count ? policy_kernel<true, true, true, kAloneThreads>
                                       : policy_kernel<true, true, false, kAloneThreads>)
                              : (count ? policy_kernel<true, false, true, kAloneThreads>
                                       : policy_kernel<true, false, false, kAloneThreads>);
    kern<<<1, kAloneThreads, 0, s>>>(t, grad_scale, nullptr, 0, grad_logprobs, norm, sums);
  } else {
    if (int st = launch_count(t.p.reduction, t.mask, t.p.norm ? norm : nullptr, nullptr, num_envs, seq_len, ws, s))
      return st;
    auto kern = grad_logprobs ? policy_kernel<true, true, false, kThreads> : policy_kernel<true, false, false, kThreads>;
    kern<<<(unsigned)blocks, kThreads, 0, s>>>(t, grad_scale, nullptr, 0, grad_logprobs, nullptr, sums);
  }
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

extern "C" int rls_policy_loss_backward(const float* logprobs, const float* old_logprobs, const float* advantages,
                                        int advantages_per_env, const float* ref_logprobs, const void* mask,
                                        int mask_kind, const rls_policy_t* policy, float grad_scale,
                                        const float* grad_loss, int force, const float* norm, float* grad_logprobs,
                                        int64_t num_envs, int64_t seq_len, void* stream) {
  if (num_envs < 0 || seq_len < 0 || !policy_ok(policy) || !mask_ok(mask, mask_kind)) return RLS_EINVAL;
  if (seq_len > 0 && num_envs > INT64_MAX / seq_len) return RLS_EINVAL;
  const int64_t M = num_envs * seq_len;
  if (M == 0) return RLS_OK;
  if (!logprobs || !old_logprobs || !advantages || !grad_loss || !grad_logprobs) return RLS_EINVAL;
  if (mask && policy->reduction != RLS_REDUCE_SUM && !norm) return RLS_EINVAL;
  if (!aligned(logprobs) || !aligned(old_logprobs) || !aligned(advantages) || !aligned(ref_logprobs) ||
      !aligned(grad_logprobs) || !aligned(norm, 4) || !aligned(grad_loss, 4) || !aligned(mask, mask_align(mask_kind)))
    return RLS_EALIGN;
  TokenGuard guard{logprobs, old_logprobs, advantages, ref_logprobs, mask, norm, grad_loss, grad_logprobs};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  Terms t{logprobs,
          make_policy(*policy, old_logprobs, advantages, advantages_per_env, ref_logprobs, norm, mask != nullptr,
                      num_envs, seq_len),
          Mask{mask, mask_kind}, M, seq_len, Divide::of(seq_len, M)};
  policy_kernel<false, true, false, kThreads>
      <<<(unsigned)policy_blocks(M), kThreads, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
          t, grad_scale, grad_loss, force, grad_logprobs, nullptr, SumOut{});
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

extern "C" int rls_policy_loss_logits(const void* logits, int64_t env_stride, int64_t step_stride,
                                      const int64_t* tokens, const float* old_logprobs, const float* advantages,
                                      int advantages_per_env, const float* ref_logprobs, const void* mask,
                                      int mask_kind, int32_t* order, const rls_policy_t* policy, float grad_scale, float* norm,
                                      float* logprobs, float* entropy, float* row_stats, float* loss, float* stats,
                                      void* grad_logits, int64_t grad_env_stride, int64_t grad_step_stride,
                                      int64_t num_envs, int64_t seq_len, int64_t vocab, double temperature,
                                      int in_dtype, void* ws, size_t ws_bytes, void* stream) {
  LogitsCall c{logits, env_stride, step_stride, tokens, Mask{mask, mask_kind}, order, grad_logits, grad_env_stride,
               grad_step_stride, num_envs, seq_len, vocab, temperature, in_dtype};
  if (!policy_ok(policy) || !loss) return RLS_EINVAL;
  if (int st = check_logits(c)) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const int64_t M = num_envs * seq_len;
  if (M == 0) {
    return clear_loss(loss, stats, s);
  }
  if (!old_logprobs || !advantages || !logprobs || (!row_stats && vocab > kLaneVocab) || !ws) return RLS_EINVAL;
  if (policy->entropy_coef != 0.f && !entropy) return RLS_EINVAL;
  if (mask && policy->reduction != RLS_REDUCE_SUM && !norm) return RLS_EINVAL;
  if (!aligned(old_logprobs) || !aligned(advantages) || !aligned(ref_logprobs) || !aligned(logprobs) ||
      !aligned(entropy) || !aligned(row_stats) || !aligned(ws) || !aligned(norm, 4) || !aligned(loss, 4) || !aligned(stats, 4))
    return RLS_EALIGN;
  TokenGuard guard{logits, tokens, order, old_logprobs, advantages, ref_logprobs, mask, norm, logprobs, entropy, row_stats,
                    loss, stats, grad_logits, ws};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  const Policy p = make_policy(*policy, old_logprobs, advantages, advantages_per_env, ref_logprobs, norm,
                               mask != nullptr, num_envs, seq_len);
  PolicyGrad src{p, grad_scale, nullptr, false, SumOut{}, &static_cast<WsHeader*>(ws)->error,
                 g_wait_tries < 0 ? kTeamWait : (unsigned)g_wait_tries};
  const int64_t blocks = sum_blocks((M + kThreads - 1) / kThreads);
  if (int st = sums_in(ws, ws_bytes, sum_blocks(M), loss, stats, s, &src.sums)) return st;
  if (vocab <= kLaneVocab) order = nullptr;
  if (int st = launch_count(p.reduction, c.mask, p.norm ? norm : nullptr, order, num_envs, seq_len, ws, s)) return st;
  c.order = order;
  const RowOut ro{logprobs, entropy, reinterpret_cast<float4*>(row_stats)};
  if (int st = launch_logits<kBoth>(c, entropy != nullptr, ro, src, s)) return st;
  if (vocab <= kLaneVocab) return RLS_OK;  // its kernel added up the terms itself
  row_sums_kernel<<<(unsigned)blocks, kThreads, 0, s>>>(ro.stats, entropy, M, src.sums);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

extern "C" int rls_policy_loss_logits_backward(const void* logits, int64_t env_stride, int64_t step_stride,
                                               const int64_t* tokens, const float* old_logprobs,
                                               const float* advantages, int advantages_per_env,
                                               const float* ref_logprobs, const void* mask, int mask_kind, const int32_t* order,
                                               const rls_policy_t* policy, float grad_scale, const float* grad_loss,
                                               int force, const float* norm,
                                               const float* row_stats, void* grad_logits, int64_t grad_env_stride,
                                               int64_t grad_step_stride, int64_t num_envs, int64_t seq_len,
                                               int64_t vocab, double temperature, int in_dtype, void* stream) {
  LogitsCall c{logits, env_stride, step_stride, tokens, Mask{mask, mask_kind}, order, grad_logits, grad_env_stride,
               grad_step_stride, num_envs, seq_len, vocab, temperature, in_dtype};
  if (!policy_ok(policy)) return RLS_EINVAL;
  if (int st = check_logits(c)) return st;
  if (num_envs == 0 || seq_len == 0) return RLS_OK;
  if (!old_logprobs || !advantages || !grad_loss || (!row_stats && vocab > kLaneVocab) || !grad_logits) return RLS_EINVAL;
  if (mask && policy->reduction != RLS_REDUCE_SUM && !norm) return RLS_EINVAL;
  if (!aligned(old_logprobs) || !aligned(advantages) || !aligned(ref_logprobs) || !aligned(row_stats) ||
      !aligned(norm, 4) || !aligned(grad_loss, 4))
    return RLS_EALIGN;
  TokenGuard guard{logits, tokens, order, old_logprobs, advantages, ref_logprobs, mask, norm, grad_loss, row_stats,
                    grad_logits};
  if (guard.status()) return guard.status();
  std::lock_guard<std::recursive_mutex> lock(launch_mutex());
  const Policy p = make_policy(*policy, old_logprobs, advantages, advantages_per_env, ref_logprobs, norm,
                               mask != nullptr, num_envs, seq_len);
  const RowOut ro{nullptr, nullptr, reinterpret_cast<float4*>(const_cast<float*>(row_stats))};
  return launch_logits<kBwd>(c, policy->entropy_coef != 0.f, ro, PolicyGrad{p, grad_scale, grad_loss, force != 0, SumOut{}, nullptr, 0},
                             reinterpret_cast<cudaStream_t>(stream));
}
