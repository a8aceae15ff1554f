// beam_select.hip -- the `take` best continuations of a batch of beams.
//
//   value[k, t] = score[k] + x[k, t] - logsumexp_t x[k, :];  largest first, ties to the lowest k * vocab + t
//
// Two launches, the logits are read once.  beam_scan_kernel: a workgroup holds one chunk of a row in registers and
// writes its softmax statistics (maximum, sum of exponentials) and its `take` best logits in order, each as one
// 64-bit key (logit's order in the upper half, ~token in the lower), so that ties go to the lowest token by
// themselves.  Within a row the values have the logits' order, whatever the logarithm rounds to.
// beam_merge_kernel: a workgroup per sequence joins the statistics, forms the values of the heads of all lists in
// float64 (where two beams' values tie only if they are equal) and takes the best head `take` times.
#include "device.h"

namespace tl_ops {
namespace {

constexpr int kThreads = 256;
constexpr int kPer = 16;  // logits of a thread
constexpr int kChunk = kThreads * kPer;

// The order of floats as that of unsigned integers; -0 counts as 0.
__device__ inline uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ inline float from_order(uint32_t k) {
  return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}

__device__ inline uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, m);
    v = w > v ? w : v;
  }
  return v;
}

template <Type TYPE>
__global__ __launch_bounds__(kThreads) void beam_scan_kernel(BeamArgs a) {
  using T = typename Scalar<TYPE>::type;
  __shared__ float f_lds[2][kThreads / 64];
  __shared__ uint64_t best_lds[2][kThreads / 64];
  const int tid = threadIdx.x, chunk = blockIdx.x;
  const int64_t row = blockIdx.y;
  const T* x = static_cast<const T*>(a.logits) + row * a.stride;
  const int begin = int(int64_t(a.vocab) * chunk / a.chunks), end = int(int64_t(a.vocab) * (chunk + 1) / a.chunks);
  float v[kPer];
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int t = begin + i * kThreads + tid;
    v[i] = t < end ? float(x[t]) : -INFINITY;
    nan |= v[i] != v[i];
    top = fmaxf(top, v[i]);
  }
  top = block_reduce<kThreads>(top, f_lds[0], Max());
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) sum += begin + i * kThreads + tid < end ? expf(v[i] - top) : 0.0f;
  sum = block_reduce<kThreads>(nan ? NAN : sum, f_lds[1], Add());
  const int64_t at = row * a.chunks + chunk;
  if (tid == 0) a.part_stat[2 * at] = top, a.part_stat[2 * at + 1] = top == -INFINITY ? 0.0f : sum;

  uint64_t key[kPer], mine = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int t = begin + i * kThreads + tid;
    key[i] = t < end ? uint64_t(order_of(v[i])) << 32 | uint32_t(~t) : 0;
    mine = key[i] > mine ? key[i] : mine;
  }
  for (int n = 0; n < a.take; ++n) {
    uint64_t best = wave_max(mine);
    if ((tid & 63) == 0) best_lds[n & 1][tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) best = best_lds[n & 1][w] > best ? best_lds[n & 1][w] : best;
    if (tid == 0) a.part_list[at * a.take + n] = best;  // 0: the chunk has no more
    if (mine == best && best) {
      mine = 0;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        if (key[i] == best) key[i] = 0;
        mine = key[i] > mine ? key[i] : mine;
      }
    }
  }
}

struct Candidate {
  double value;
  int64_t at;  // beam * vocab + token; INT64_MAX: none
};
__device__ inline bool before(const Candidate& a, const Candidate& b) {
  return a.value > b.value || (a.value == b.value && a.at < b.at);
}
__device__ inline Candidate shuffle(const Candidate& c, int m) {
  return {__shfl_xor(c.value, m), (int64_t)__shfl_xor((long long)c.at, m)};
}

__global__ __launch_bounds__(kThreads) void beam_merge_kernel(BeamArgs a) {
  __shared__ double lse_lds[kBeamMaxBeams];
  __shared__ Candidate best_lds[2][kThreads / 64];
  const int tid = threadIdx.x;
  const int64_t b = blockIdx.x;
  const double inf = INFINITY;
  for (int k = tid; k < a.beams; k += kThreads) {
    const float* stat = a.part_stat + (b * a.beams + k) * a.chunks * 2;
    float top = -INFINITY;
    for (int c = 0; c < a.chunks; ++c) top = fmaxf(top, stat[2 * c]);
    double sum = 0.0;
    for (int c = 0; c < a.chunks; ++c) sum += double(stat[2 * c + 1]) * exp(double(stat[2 * c]) - double(top));
    lse_lds[k] = double(top) + log(sum);
  }
  __syncthreads();

  // List j belongs to beam j / chunks.  A beam without a finite score or logsumexp has only -inf to offer, a
  // finished one its eos token and -inf: their tokens are counted off by the beam's first list.
  const int lists = a.beams * a.chunks;
  const auto head = [&](int j, int nth) -> Candidate {
    const int k = j / a.chunks, c = j - k * a.chunks;
    const int64_t none = INT64_MAX, first = int64_t(k) * a.vocab;
    if (nth >= a.take) return {-inf, none};
    const float score = a.scores[b * a.beams + k];
    const double lse = lse_lds[k];
    const bool live = fabsf(score) < INFINITY, done = a.finished && a.finished[b * a.beams + k];
    if (done && live) {
      if (c || nth >= a.vocab) return {-inf, none};
      if (nth == 0) return {double(score), first + a.eos};
      return {-inf, first + (nth - 1 < a.eos ? nth - 1 : nth)};
    }
    if (!live || !(fabs(lse) < inf)) {
      if (c || nth >= a.vocab) return {-inf, none};
      return {-inf, first + nth};
    }
    const uint64_t key = a.part_list[((b * a.beams + k) * a.chunks + c) * a.take + nth];
    if (key == 0) return {-inf, none};
    const double x = from_order(uint32_t(key >> 32));
    return {double(score) + (x - lse), first + uint32_t(~uint32_t(key))};
  };
  Candidate mine{-inf, INT64_MAX};
  int mine_list = -1;
  // a list's position is the number of its candidates that won so far; kept by the thread that owns it
  constexpr int kOwn = kBeamMaxLists / kThreads;
  int taken[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) taken[i] = 0;
  const auto look = [&] {
    mine = {-inf, INT64_MAX};
    mine_list = -1;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const int j = i * kThreads + tid;
      if (j < lists) {
        const Candidate h = head(j, taken[i]);
        if (before(h, mine)) mine = h, mine_list = i;
      }
    }
  };
  look();
  for (int n = 0; n < a.take; ++n) {
    Candidate best = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const Candidate other = shuffle(best, m);
      if (before(other, best)) best = other;
    }
    if ((tid & 63) == 0) best_lds[n & 1][tid >> 6] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w)
      if (before(best_lds[n & 1][w], best)) best = best_lds[n & 1][w];
    if (tid == 0) {
      a.out_scores[b * a.take + n] = float(best.value);
      a.out_parents[b * a.take + n] = best.at / a.vocab;
      a.out_tokens[b * a.take + n] = best.at % a.vocab;
    }
    if (mine_list >= 0 && mine.at == best.at) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) taken[i] += i == mine_list;
      look();
    }
  }
}

}  // namespace

int beam_select_chunks(int64_t, int vocab) { return int(ceil_div(vocab, kChunk)); }

void beam_select_hip(const BeamArgs& a, Stream s) {
  if (a.batch == 0) return;
  const dim3 grid(a.chunks, unsigned(a.batch * a.beams));
  const auto scan = a.type == kF32   ? beam_scan_kernel<kF32>
                    : a.type == kF16 ? beam_scan_kernel<kF16>
                                     : beam_scan_kernel<kBF16>;
  launch(scan, grid, kThreads, a, s, "beam_select");
  launch(beam_merge_kernel, dim3(unsigned(a.batch)), kThreads, a, s, "beam_select");
}

}  // namespace tl_ops
