// token_launch.h -- launchers of the logits kernels (token_kernels.cuh), one
// translation unit for each family.
#pragma once
#include "rlscan.h"
#include "token_kernels.cuh"

namespace rls {
namespace tok {

constexpr int64_t kLaneVocab = RLS_SHORT_VOCAB;  // short rows (token_lanes.cu) have at most so many logits

int num_sms();  // of the current device

// CTAs of the kernels that sum: at most this many, whatever the batch.
int64_t sum_blocks(int64_t need);

template <class T, bool ENT, int MODE, class Src>
int launch_lane_rows(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s);
template <class T, bool ENT, int MODE, class Src>
int launch_cta_rows(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s);

#define RLS_TOKEN_INSTANTIATE(FN)                                                                                    \
  RLS_TOKEN_INST1(FN, float, false) RLS_TOKEN_INST1(FN, float, true) RLS_TOKEN_INST1(FN, __nv_bfloat16, false)        \
  RLS_TOKEN_INST1(FN, __nv_bfloat16, true)
#define RLS_TOKEN_INST1(FN, T, ENT)                                                                                  \
  template int FN<T, ENT, kFwd, GivenGrad>(const Rows<T>&, const RowOut&, const GradRows<T>&, const GivenGrad&,       \
                                           cudaStream_t);                                                            \
  template int FN<T, ENT, kBwd, GivenGrad>(const Rows<T>&, const RowOut&, const GradRows<T>&, const GivenGrad&,       \
                                           cudaStream_t);                                                            \
  template int FN<T, ENT, kBwd, PolicyGrad>(const Rows<T>&, const RowOut&, const GradRows<T>&, const PolicyGrad&,     \
                                            cudaStream_t);                                                           \
  template int FN<T, ENT, kBoth, PolicyGrad>(const Rows<T>&, const RowOut&, const GradRows<T>&, const PolicyGrad&,    \
                                             cudaStream_t);

}  // namespace tok
}  // namespace rls
