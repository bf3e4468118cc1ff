// token_rows.cu -- the logits kernels for long rows: a pipeline over rows, and one CTA a row beyond
// its reach.
#include "token_launch.h"

namespace rls {
namespace tok {
namespace {

// A kernel over teams of `size` CTAs.
template <class T, class Src, int NT, size_t smem, bool CL>
int launch(void (*kern)(Rows<T>, RowOut, GradRows<T>, Src), const Rows<T>& in, const RowOut& out,
           const GradRows<T>& gr, const Src& src, int size, int (&resident)[64][4], cudaStream_t s) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return RLS_ECUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = size;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CL ? 1 : 0;
  // Teams that fit on the device at once, asked once per device and cluster size
  // (under the launch lock): a team that had to wait for another would double
  // the time.
  int& most = resident[dev][size == 1 ? 0 : size == 2 ? 1 : size == 4 ? 2 : 3];
  if (!most) {
    int n = 0;
    if (smem > 32 * 1024 &&
        cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return RLS_ECUDA;
    if (CL) {
      cfg.gridDim = dim3((unsigned)size);
      if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n < 1) return RLS_ECUDA;
    } else {
      if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, NT, smem) != cudaSuccess || n < 1) return RLS_ECUDA;
      n *= num_sms();
    }
    most = n;
  }
  int64_t teams = most;
  if (teams > in.rows) teams = in.rows;
  cfg.gridDim = dim3((unsigned)(teams * size));
  return cudaLaunchKernelEx(&cfg, kern, in, out, gr, src) == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

template <class T, bool ENT, int MODE, class Src, int NT, int U, bool CL>
int stream(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, int size, cudaStream_t s) {
  static int resident[64][4] = {{0}};
  return launch<T, Src, NT, 0, CL>(stream_rows_kernel<T, ENT, MODE, Src, NT, U, CL>, in, out, gr, src, size, resident,
                                   s);
}
template <class T, bool ENT, class Src, int NT, int K, bool CL>
int both(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, int size, cudaStream_t s) {
  static int resident[64][4] = {{0}};
  return launch<T, Src, NT, (size_t)NT * K * 16, CL>(both_rows_kernel<T, ENT, Src, NT, K, CL>, in, out, gr, src, size,
                                                     resident, s);
}

// Rows beyond the slots of a full cluster: one CTA a row, the second pass from L2.
template <class T, bool ENT, int MODE, class Src>
int plain(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int64_t blocks = in.rows < 0x7fffffffLL ? in.rows : 0x7fffffffLL;
  cta_rows_kernel<T, ENT, MODE, Src, 512, 4><<<(unsigned)blocks, 512, 0, s>>>(in, out, gr, src);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

}  // namespace

template <class T, bool ENT, int MODE, class Src>
int launch_cta_rows(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int64_t nvec = in.V / Vec<T>::N;
  // Vector stores need rows that lie alike (the operators see to it where they can).
  if (MODE != kFwd && gr.g && !gr.alike) return plain<T, ENT, MODE, Src>(in, out, gr, src, s);
  int size = 1;
  // With the gradient a row stays in the slots (64 KB a CTA).
  if (MODE == kBoth)
    while (size < kMostCtas && nvec > (int64_t)size * 4096) size *= 2;
  // few rows: more CTAs for each, down to 1024 vectors a CTA
  while (size < kMostCtas && in.rows * size < 2 * num_sms() && nvec > (int64_t)size * 1024) size *= 2;
  const int64_t each = (nvec + size - 1) / size;
  if constexpr (MODE == kBoth) {
    if (each > 4096) return plain<T, ENT, MODE, Src>(in, out, gr, src, s);
    if (size > 1) {
      if (each <= 1024) return both<T, ENT, Src, 256, 4, true>(in, out, gr, src, size, s);
      return both<T, ENT, Src, 256, 16, true>(in, out, gr, src, size, s);
    }
    if (each <= 256) return both<T, ENT, Src, 32, 8, false>(in, out, gr, src, 1, s);
    if (each <= 512) return both<T, ENT, Src, 32, 16, false>(in, out, gr, src, 1, s);
    if (each <= 1024) return both<T, ENT, Src, 64, 16, false>(in, out, gr, src, 1, s);
    if (each <= 2048) return both<T, ENT, Src, 128, 16, false>(in, out, gr, src, 1, s);
    return both<T, ENT, Src, 256, 16, false>(in, out, gr, src, 1, s);
  } else {
    if (size > 1) return stream<T, ENT, MODE, Src, 256, 4, true>(in, out, gr, src, size, s);
    if (each <= 1024) return stream<T, ENT, MODE, Src, 32, 8, false>(in, out, gr, src, 1, s);
    if (each <= 4096) return stream<T, ENT, MODE, Src, 128, 8, false>(in, out, gr, src, 1, s);
    return stream<T, ENT, MODE, Src, 256, 8, false>(in, out, gr, src, 1, s);
  }
}

RLS_TOKEN_INSTANTIATE(launch_cta_rows)

}  // namespace tok
}  // namespace rls
