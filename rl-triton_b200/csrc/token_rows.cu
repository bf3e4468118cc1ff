// token_rows.cu -- the logits kernels for long rows: one CTA a row.
#include "token_launch.h"

namespace rls {
namespace tok {
namespace {

template <class T, bool ENT, int MODE, class Src, int NT>
int go(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int64_t blocks = in.rows < 0x7fffffffLL ? in.rows : 0x7fffffffLL;
  cta_rows_kernel<T, ENT, MODE, Src, NT, 4><<<(unsigned)blocks, NT, 0, s>>>(in, out, gr, src);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

}  // namespace

template <class T, bool ENT, int MODE, class Src>
int launch_cta_rows(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int64_t nvec = in.V / Vec<T>::N;
  if (nvec <= 512) return go<T, ENT, MODE, Src, 128>(in, out, gr, src, s);
  return go<T, ENT, MODE, Src, 512>(in, out, gr, src, s);
}

RLS_TOKEN_INSTANTIATE(launch_cta_rows)

}  // namespace tok
}  // namespace rls
