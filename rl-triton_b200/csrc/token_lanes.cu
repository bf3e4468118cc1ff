// token_lanes.cu -- the logits kernels for short rows (discrete actions, small
// vocabularies): a group of lanes holds a row in registers, so the gradient
// pass needs no second read and no statistics from an earlier call.
#include "token_launch.h"

namespace rls {
namespace tok {
namespace {

template <class T, bool ENT, int MODE, class Src, int G, int E>
int go(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  constexpr int64_t per = 256 / G;
  int64_t blocks = (in.rows + per - 1) / per;
  if (blocks > 0x7fffffffLL) blocks = 0x7fffffffLL;
  if (Src::kPolicy && MODE != kBwd) blocks = sum_blocks(blocks);
  lane_rows_kernel<T, ENT, MODE, Src, G, E><<<(unsigned)blocks, 256, 0, s>>>(in, out, gr, src);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

}  // namespace

template <class T, bool ENT, int MODE, class Src>
int launch_lane_rows(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int64_t V = in.V;
  if (V <= 4) return go<T, ENT, MODE, Src, 1, 4>(in, out, gr, src, s);
  if (V <= 8) return go<T, ENT, MODE, Src, 2, 4>(in, out, gr, src, s);
  if (V <= 16) return go<T, ENT, MODE, Src, 4, 4>(in, out, gr, src, s);
  if (V <= 32) return go<T, ENT, MODE, Src, 8, 4>(in, out, gr, src, s);
  if (V <= 64) return go<T, ENT, MODE, Src, 16, 4>(in, out, gr, src, s);
  if (V <= 128) return go<T, ENT, MODE, Src, 32, 4>(in, out, gr, src, s);
  if (V <= 256) return go<T, ENT, MODE, Src, 32, 8>(in, out, gr, src, s);
  if (V <= 512) return go<T, ENT, MODE, Src, 32, 16>(in, out, gr, src, s);
  return go<T, ENT, MODE, Src, 32, 32>(in, out, gr, src, s);
}

RLS_TOKEN_INSTANTIATE(launch_lane_rows)

}  // namespace tok
}  // namespace rls
