// reorder.hip -- state[b, k] <- state[b, parent[b, k]] in place, for all states of a model in one launch.
//
// A thread owns one piece (16, 4 or 1 bytes) of the same place in all beams of a sequence: it reads the pieces that
// some other beam wants, then writes the beams that change.  No other thread touches them, so no copy of the state
// is needed, whatever the parents are.  A beam that stays is neither read for itself nor written.
//
// Bound by HBM.  1.43 GB of moves among 8 beams (caches of 3001 tokens) take 236 to 252 us on different cards, 5.7 to
// 6.1 TB/s.  How it got there, timed in one way on one card (277 us, 16 beams 289): the pieces go past the caches
// (362 us without: nothing of a long state is read again before it is gone), and a workgroup is one wave with one
// piece to a thread (four waves 310 us, four pieces 332).  Each piece read is stored to its children one by one:
// choosing every beam's piece among the registers cost 435 us for 16 beams.
#include "device.h"

namespace tl_ops {
namespace {

constexpr int kThreads = 64;  // one wave: it finds the children by ballot
constexpr int64_t kBytes = 16 * kThreads;  // of a row, for a workgroup
static_assert(kReorderStates <= 128);

template <typename P, int BEAMS>
__device__ inline void reorder_row(const ReorderState& st, const int64_t* parents, int64_t b, int beams,
                                   int64_t block) {
  uint8_t* base = st.data + b * beams * st.stride;
  // children[j]: the beams that j's piece goes to.  A parent that is none leaves its beam as it is.
  const int lane = threadIdx.x;
  const int64_t parent = lane < beams ? parents[b * beams + lane] : -1;
  uint32_t children[BEAMS];
#pragma unroll
  for (int j = 0; j < BEAMS; ++j) children[j] = j < beams ? uint32_t(__ballot(parent == j && lane != j)) : 0;
  const int64_t pieces = st.bytes / int64_t(sizeof(P)), at = block * (kBytes / int64_t(sizeof(P)));
  const int64_t end = min(pieces, at + kBytes / int64_t(sizeof(P)));
  for (int64_t i = at + lane; i < end; i += kThreads) {
    P v[BEAMS];
#pragma unroll
    for (int j = 0; j < BEAMS; ++j)
      if (children[j]) v[j] = __builtin_nontemporal_load(reinterpret_cast<const P*>(base + j * st.stride) + i);
#pragma unroll
    for (int j = 0; j < BEAMS; ++j)
      for (uint32_t m = children[j]; m; m &= m - 1)
        __builtin_nontemporal_store(v[j], reinterpret_cast<P*>(base + __builtin_ctz(m) * st.stride) + i);
  }
}

template <int BEAMS>
__global__ __launch_bounds__(kThreads) void reorder_kernel(ReorderArgs a) {
  int at = 0;  // the last state whose workgroups begin no later than this one
  for (int step = 64; step > 0; step >>= 1)
    if (at + step < a.states && a.state[at + step].first <= int64_t(blockIdx.x)) at += step;
  const ReorderState st = a.state[at];
  const int64_t b = blockIdx.y, block = int64_t(blockIdx.x) - st.first;
  const uint64_t all = reinterpret_cast<uint64_t>(st.data) | uint64_t(st.stride) | uint64_t(st.bytes);
  if (all % 16 == 0)
    reorder_row<u32x4, BEAMS>(st, a.parents, b, a.beams, block);
  else if (all % 4 == 0)
    reorder_row<uint32_t, BEAMS>(st, a.parents, b, a.beams, block);
  else
    reorder_row<uint8_t, BEAMS>(st, a.parents, b, a.beams, block);
}

}  // namespace

void reorder_hip(ReorderArgs a, Stream s) {
  if (a.batch == 0) return;
  const auto k = a.beams <= 4    ? reorder_kernel<4>
                 : a.beams <= 8  ? reorder_kernel<8>
                 : a.beams <= 16 ? reorder_kernel<16>
                                 : reorder_kernel<32>;
  // States whose rows are larger together than a launch takes go into several.
  constexpr int64_t kMost = kReorderMaxBytes / kBytes;
  static_assert((kMost + 1) * kThreads == int64_t(1) << 32);
  ReorderArgs part = a;
  for (int i = 0; i < a.states;) {
    int64_t blocks = 0;
    for (part.states = 0; i < a.states; ++i, ++part.states) {
      const int64_t more = ceil_div(a.state[i].bytes, kBytes);
      if (blocks + more > kMost) break;
      part.state[part.states] = a.state[i];
      part.state[part.states].first = blocks;
      blocks += more;
    }
    launch(k, dim3(unsigned(blocks), unsigned(a.batch)), kThreads, part, s, "reorder_states");
  }
}

}  // namespace tl_ops
