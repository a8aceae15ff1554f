// reorder.hip -- state[b, k] <- state[b, parent[b, k]] in place, for all states of a model in one launch.
//
// A thread owns one piece (16, 4 or 1 bytes) of the same place in all beams of a sequence: it reads the pieces that
// some other beam wants, then writes the beams that change.  No other thread touches them, so no copy of the state
// is needed, whatever the parents are.  A beam that stays is neither read for itself nor written.
#include "device.h"

namespace tl_ops {
namespace {

constexpr int kThreads = 256;

template <typename P, int BEAMS>
__device__ inline void reorder_row(const ReorderState& st, const int64_t* parents, int64_t b, int beams) {
  uint8_t* base = st.data + b * beams * st.stride;
  int parent[BEAMS];
#pragma unroll
  for (int k = 0; k < BEAMS; ++k) {
    const int64_t p = k < beams ? parents[b * beams + k] : k;
    parent[k] = p < 0 || p >= beams ? k : int(p);  // a parent that is none leaves its beam as it is
  }
  uint32_t wanted = 0;
#pragma unroll
  for (int k = 0; k < BEAMS; ++k) wanted |= parent[k] != k ? 1u << parent[k] : 0u;
  const int64_t pieces = st.bytes / int64_t(sizeof(P));
  for (int64_t i = int64_t(blockIdx.x) * kThreads + threadIdx.x; i < pieces; i += int64_t(gridDim.x) * kThreads) {
    P v[BEAMS];
#pragma unroll
    for (int k = 0; k < BEAMS; ++k)
      if (wanted >> k & 1) v[k] = reinterpret_cast<const P*>(base + k * st.stride)[i];
#pragma unroll
    for (int k = 0; k < BEAMS; ++k) {
      if (parent[k] == k) continue;
      P w = v[0];
#pragma unroll
      for (int j = 1; j < BEAMS; ++j) w = parent[k] == j ? v[j] : w;
      reinterpret_cast<P*>(base + k * st.stride)[i] = w;
    }
  }
}

template <int BEAMS>
__global__ __launch_bounds__(kThreads) void reorder_kernel(ReorderArgs a) {
  const ReorderState st = a.state[blockIdx.y];
  const int64_t b = blockIdx.z;
  const uint64_t all = reinterpret_cast<uint64_t>(st.data) | uint64_t(st.stride) | uint64_t(st.bytes);
  if (all % 16 == 0)
    reorder_row<u32x4, BEAMS>(st, a.parents, b, a.beams);
  else if (all % 4 == 0)
    reorder_row<uint32_t, BEAMS>(st, a.parents, b, a.beams);
  else
    reorder_row<uint8_t, BEAMS>(st, a.parents, b, a.beams);
}

}  // namespace

void reorder_hip(const ReorderArgs& a, Stream s) {
  if (a.batch == 0 || a.states == 0) return;
  int64_t most = 0;
  for (int i = 0; i < a.states; ++i) most = a.state[i].bytes > most ? a.state[i].bytes : most;
  int64_t blocks = ceil_div(most, 16 * kThreads);
  if (blocks == 0) return;
  if (blocks > 4096) blocks = 4096;
  const dim3 grid(unsigned(blocks), a.states, unsigned(a.batch));
  const auto k = a.beams <= 4    ? reorder_kernel<4>
                 : a.beams <= 8  ? reorder_kernel<8>
                 : a.beams <= 16 ? reorder_kernel<16>
                                 : reorder_kernel<32>;
  launch(k, grid, kThreads, a, s, "reorder_states");
}

}  // namespace tl_ops
