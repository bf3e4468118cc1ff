// token_lanes.cu -- the logits kernels for short rows (discrete actions, small
// vocabularies): tiles of rows in shared memory, or, where the rows do not lie one after the
// other, a group of lanes holds a row in registers.  Either way the gradient
// needs no statistics from an earlier call.
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

// The most lanes that one phase of a shared-memory access (`words` 4-byte words a lane,
// 32 words a phase) brings to the same banks, rows of `pitch` words, `lanes` a row.
int conflicts(int lanes, int words, int pitch, int turn) {
  int at[32] = {0}, most = 0;
  const int slots = 32 / words;
  for (int l = 0; l < slots; ++l) {
    const int word = (l / lanes) * pitch + (l % lanes + (l / lanes) * turn * lanes) * words;
    const int n = ++at[word / words % slots];
    if (n > most) most = n;
  }
  return most;
}

template <class T, bool ENT, int MODE, class Src, int ACC>
int tiles(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int line = in.V * (int)sizeof(T);
  // Up to 40 KB a tile (512 bf16: 250 us against 324 with 20 KB for 1.07 GB: more rows share
  // a tile's serial steps), five tiles an SM; at least 8 rows, which are whole vectors
  // for any V.
  TileShape sh{};
  sh.rows = 8;
  while (sh.rows < kTileThreads && 2 * sh.rows * line <= 40 * 1024) sh.rows *= 2;
  const int lanes = kTileThreads / sh.rows < 32 ? kTileThreads / sh.rows : 32;
  while ((1 << sh.log_lanes) < lanes) ++sh.log_lanes;
  const int size = (ACC == 2 ? 16 : ACC == 1 ? 2 * (int)sizeof(T) : (int)sizeof(T));  // bytes of an access
  if (size >= 4)
    sh.turn = conflicts(lanes, size / 4, line / 4, 1) < conflicts(lanes, size / 4, line / 4, 0);
  sh.rounds = line / (size * lanes);
  sh.by_vocab = Divide::of(in.V, 0);
  const size_t smem = ((size_t)sh.rows * line + 15) / 16 * 16;  // at most 40 KB
  auto kern = tile_rows_kernel<T, ENT, MODE, Src, ACC>;
  const int64_t all = (in.rows + sh.rows - 1) / sh.rows, fit = (int64_t)num_sms() * kTileCtas;
  const int64_t blocks = all < fit ? all : fit;
  kern<<<(unsigned)blocks, kTileThreads, smem, s>>>(in, out, gr, src, sh);
  return cudaPeekAtLastError() == cudaSuccess ? RLS_OK : RLS_ECUDA;
}

}  // namespace

template <class T, bool ENT, int MODE, class Src>
int launch_lane_rows(const Rows<T>& in, const RowOut& out, const GradRows<T>& gr, const Src& src, cudaStream_t s) {
  const int64_t V = in.V;
  // Rows (and their gradients) one after the other from a 16-byte boundary on.
  const bool whole = in.flat && in.ss == V && ((uintptr_t)in.x & 15) == 0;
  if (whole && (MODE == kFwd || !gr.g || (gr.flat && gr.ss == V && ((uintptr_t)gr.g & 15) == 0))) {
    if (V * sizeof(T) % 16 == 0) return tiles<T, ENT, MODE, Src, 2>(in, out, gr, src, s);
    if (V % 2 == 0) return tiles<T, ENT, MODE, Src, 1>(in, out, gr, src, s);
    return tiles<T, ENT, MODE, Src, 0>(in, out, gr, src, s);
  }
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
