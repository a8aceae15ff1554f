// beam_select.hip -- the `take` best continuations of a batch of beams.
//
//   value[k, t] = score[k] + x[k, t] - logsumexp_t x[k, :];  largest first, ties to the lowest k * vocab + t
//
// Two launches; the logits are read once, and what is sorted is only what can win.
//
// beam_scan_kernel: a workgroup holds one chunk of a row in registers.  Its waves write the chunk's softmax
// statistics (maximum, sum of exponentials), and the workgroup its `take` best logits in order, each as one 64-bit
// key (the logit's order in the upper half, ~token in the lower), so that ties go to the lowest token by themselves.
// If q lanes of a wave hold a logit of at least T, the chunk's q best are no less: with T the `take`-th largest of
// the lanes' maxima, found bit by bit with one ballot each, few logits reach T.  Those go to LDS, and each finds its
// place by counting the larger ones.
// beam_merge_kernel: a workgroup per sequence joins the statistics and does the same with the lists' values, which
// are float64: within a beam they have the logits' order.  A beam's logsumexp comes from float32 exponentials and
// sums of each wave, joined in float64: off by less than 2^-19 (a term 2^-d of the largest by d 2^-23 of itself, and d
// is 20 on average at most), which can decide between two beams' values that are as close; float64 exponentials of
// every logit would cost more than the scan does.
//
// 8 x 8 beams over 129280 fp32 logits (33 MB), 16 taken: 14 + 8 us; 4 beams over 32002 in fp16, 8 taken: 6 + 5 us.
// The scan is one wave of workgroups, whose latency (load, threshold, exponentials, places) bounds it, not HBM.
//
// Where ties let too many candidates through (a constant row, say), the best one is taken `take` times instead.
#include "device.h"

namespace tl_ops {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kMergeThreads = 512, kMergeWaves = kMergeThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKept = 512;        // candidates of a chunk that LDS takes
constexpr int kMergeKept = 2048;  // and of a sequence

// The order of floats as that of unsigned integers; -0 counts as 0.
__device__ inline uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ inline float from_order(uint32_t k) {
  return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
// The upper half of a double's order: a <= b gives order_of(a) <= order_of(b).
__device__ inline uint32_t order_of(double x) {
  const uint32_t u = uint32_t(__double2hiint(x + 0.0));
  return u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}

// A value that at least `want` of the wave's lanes reach (the largest one, up to its last BITS left out).
template <int BITS>
__device__ inline uint32_t reached_by(uint32_t key, int want) {
  uint32_t t = 0;
#pragma unroll 1
  for (uint32_t bit = 0x80000000u; bit >= 1u << BITS; bit >>= 1)
    if (__popcll(__ballot(key >= (t | bit))) >= want) t |= bit;
  return t;
}

__device__ inline uint64_t wave_max(uint64_t v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, m);
    v = w > v ? w : v;
  }
  return v;
}
__device__ inline double wave_sum(double v) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
  return v;
}

// A slot of `count` for every lane that keeps something, in lane order within the wave.
__device__ inline int slot_for(bool keep, int* count) {
  const uint64_t mask = __ballot(keep);
  if (mask == 0) return 0;
  const int lane = threadIdx.x & 63, first = __ffsll((unsigned long long)mask) - 1;
  int base = 0;
  if (lane == first) base = atomicAdd(count, __popcll(mask));
  base = __shfl(base, first);
  return base + int(__builtin_amdgcn_mbcnt_hi(uint32_t(mask >> 32), __builtin_amdgcn_mbcnt_lo(uint32_t(mask), 0)));
}

// The place of a candidate among n: eight lanes count the larger ones together.
template <typename C, typename F>
__device__ inline int place_of(const C* kept, int n, const C& mine, F before) {
  int place = 0;
  for (int j = threadIdx.x & 7; j < n; j += 8) place += before(kept[j], mine);
#pragma unroll
  for (int m = 1; m < 8; m <<= 1) place += __shfl_xor(place, m);
  return place;
}

// (eight waves to a SIMD: 2048 chunks, 8 rows of 129280 tokens for each of 8 beams, are in flight at once)
template <Type TYPE, int PER>
__global__ __launch_bounds__(kThreads, PER == 16 ? 8 : 1) void beam_scan_kernel(BeamArgs a) {
  using T = typename Scalar<TYPE>::type;
  constexpr int VEC = 16 / sizeof(T), VECS = PER / VEC, CHUNK = kThreads * PER;
  __shared__ uint32_t t_lds[kWaves];
  __shared__ uint64_t best_lds[2][kWaves];
  __shared__ uint64_t kept[kKept];
  __shared__ int count;
  const int tid = threadIdx.x, wave = tid >> 6, chunk = blockIdx.x;
  const int64_t row = blockIdx.y;
  const int begin = chunk * CHUNK, left = a.vocab - begin;  // tokens from the chunk on
  const T* x = static_cast<const T*>(a.logits) + row * a.stride + begin;
  if (tid == 0) count = 0;

  // vector i of the thread: tokens at(i, 0) .. at(i, VEC - 1) of the chunk
  const auto at = [&](int i, int e) { return (i * kThreads + tid) * VEC + e; };
  float v[PER];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    if (at(i, VEC) <= left) {
      T r[VEC];
      __builtin_memcpy(r, x + at(i, 0), 16);  // rows begin anywhere
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = float(r[e]);
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i * VEC + e] = at(i, e) < left ? float(x[at(i, e)]) : -INFINITY;
    }
  }
  float top = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    nan |= v[j] != v[j];
    top = fmaxf(top, v[j]);
  }
  // the lane's largest key; 0 (less than any logit's) where it has no logit at all
  const uint32_t mine = at(0, 0) < left ? order_of(top) : 0;
  const uint32_t t = reached_by<12>(mine, a.take < 64 ? a.take : 64);
  if ((tid & 63) == 0) t_lds[wave] = t;
  top = wave_reduce(top, Max());
  float sum = 0.0f;
  if (top > -INFINITY) {
#pragma unroll
    for (int j = 0; j < PER; ++j) sum += __builtin_amdgcn_exp2f((v[j] - top) * kLog2e);
  }
  sum = wave_reduce(nan ? NAN : sum, Add());
  const int64_t list = row * a.chunks + chunk;
  if ((tid & 63) == 0) {
    float* stat = a.part_stat + (list * kWaves + wave) * 2;
    stat[0] = top;
    stat[1] = sum;
  }
  __syncthreads();
  uint32_t limit = order_of(-INFINITY);
#pragma unroll
  for (int w = 0; w < kWaves; ++w) limit = t_lds[w] > limit ? t_lds[w] : limit;
  const float least = from_order(limit);

  const auto key_of = [&](int j) -> uint64_t {
    const int token = at(j / VEC, j % VEC);
    return token < left ? uint64_t(order_of(v[j])) << 32 | uint32_t(~(begin + token)) : 0;
  };
#pragma unroll
  for (int j = 0; j < PER; ++j) {
    const bool keep = v[j] >= least && at(j / VEC, j % VEC) < left;
    if (__any(keep)) {
      const int s = slot_for(keep, &count);
      if (keep && s < kKept) kept[s] = key_of(j);
    }
  }
  __syncthreads();
  const int n = count;
  uint64_t* out = a.part_list + list * a.take;
  if (n <= kKept) {
    for (int i = tid >> 3; i < n; i += kThreads / 8) {
      const uint64_t key = kept[i];
      const int place = place_of(kept, n, key, [](uint64_t x, uint64_t y) { return x > y; });
      if ((tid & 7) == 0 && place < a.take) out[place] = key;
    }
    for (int i = n + tid; i < a.take; i += kThreads) out[i] = 0;  // the chunk has no more
    return;
  }
  uint64_t taken = ~0ull, best_of = 0;  // what the thread has left: its keys below the last one taken
  const auto look = [&] {
    best_of = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const uint64_t key = key_of(j);
      if (key < taken && key > best_of) best_of = key;
    }
  };
  look();
  for (int k = 0; k < a.take; ++k) {
    uint64_t best = wave_max(best_of);
    if ((tid & 63) == 0) best_lds[k & 1][wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) best = best_lds[k & 1][w] > best ? best_lds[k & 1][w] : best;
    if (tid == 0) out[k] = best;
    if (best_of == best && best) {
      taken = best;
      look();
    }
  }
}

constexpr int kNone = INT32_MAX;

struct Candidate {
  double value;
  int at;  // beam * vocab + token, less than 2^26; kNone: no candidate
};
__device__ inline bool before(const Candidate& a, const Candidate& b) {
  return a.value > b.value || (a.value == b.value && a.at < b.at);
}
__device__ inline Candidate shuffle(const Candidate& c, int m) { return {__shfl_xor(c.value, m), __shfl_xor(c.at, m)}; }

// A beam's chunk: its candidates are in order.  A beam without a finite score or logsumexp has only -inf to offer, a
// finished one its eos token and -inf: their tokens are counted off by the beam's first list.
struct List {
  const uint64_t* keys;  // null: there is no such list
  int beam, chunk;
  float score;
  bool done;
};

__global__ __launch_bounds__(kMergeThreads) void beam_merge_kernel(BeamArgs a) {
  __shared__ double lse_lds[kBeamMaxBeams];
  __shared__ Candidate kept[kMergeKept];
  __shared__ Candidate best_lds[2][kMergeWaves];
  __shared__ uint32_t t_lds[kMergeWaves];
  __shared__ int count;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int64_t b = blockIdx.x;
  if (tid == 0) count = 0;

  // The first keys of the thread's first list are on their way while the statistics are joined.
  const int lists = a.beams * a.chunks;
  const auto list_of = [&](int j) -> List {
    if (j >= lists) return {nullptr, 0, 0, 0.0f, false};
    const int k = j / a.chunks;
    const int64_t row = b * a.beams + k;
    return {a.part_list + (row * a.chunks + (j - k * a.chunks)) * a.take, k, j - k * a.chunks, a.scores[row],
            a.finished && a.finished[row]};
  };
  const auto key_of = [&](const List& l, int nth) { return l.keys && nth < a.take ? l.keys[nth] : 0; };
  const int lanes = lists < 64 ? lists : 64, nth = (a.take - 1) / lanes, q = (a.take + nth) / (nth + 1);
  constexpr int kAhead = 4;
  const List own = list_of(tid);
  uint64_t own_keys[kAhead];
#pragma unroll
  for (int e = 0; e < kAhead; ++e) own_keys[e] = key_of(own, e);
  const uint64_t own_nth = key_of(own, nth);

  constexpr int kStats = 64 * kWaves / 64;  // a row has at most 64 chunks
  for (int k = wave; k < a.beams; k += kMergeWaves) {
    const int n = a.chunks * kWaves;
    const float* stat = a.part_stat + (b * a.beams + k) * n * 2;
    float m[kStats], l[kStats], top = -INFINITY;
#pragma unroll
    for (int i = 0; i < kStats; ++i) {
      const bool mine = 64 * i + lane < n;
      m[i] = mine ? stat[2 * (64 * i + lane)] : -INFINITY;
      l[i] = mine ? stat[2 * (64 * i + lane) + 1] : 0.0f;
      top = fmaxf(top, m[i]);
    }
    top = wave_reduce(top, Max());
    double sum = 0.0;  // not-a-number where a wave's is, or where the maximum is infinite: such a beam is dead
#pragma unroll
    for (int i = 0; i < kStats; ++i) sum += double(l[i]) * double(__builtin_amdgcn_exp2f((m[i] - top) * kLog2e));
    sum = wave_sum(sum);
    if (lane == 0) lse_lds[k] = double(top) + log(sum);
  }
  __syncthreads();

  const auto candidate = [&](const List& l, uint64_t key, int nth) -> Candidate {
    const double none = -INFINITY;
    const int first = l.beam * a.vocab;
    if (!l.keys || nth >= a.take) return {none, kNone};
    const double lse = lse_lds[l.beam];
    const bool finite = fabsf(l.score) < INFINITY, done = l.done && finite;
    if (done || !finite || !(fabs(lse) < double(INFINITY))) {
      if (l.chunk || nth >= a.vocab) return {none, kNone};
      if (done && nth == 0) return {double(l.score), first + int(a.eos)};
      return {none, first + (done && nth - 1 < a.eos ? nth - 1 : nth)};
    }
    if (key == 0) return {none, kNone};
    return {double(l.score) + (double(from_order(uint32_t(key >> 32))) - lse), first + int(~uint32_t(key))};
  };
  const auto order = [&](const Candidate& c) { return c.at == kNone ? 0u : order_of(c.value); };

  // If q lists' candidates number `nth` (from 0) reach T, the best q (nth + 1) do: T is such that this is `take`.
  if (wave * 64 < lists) {
    const uint32_t t = reached_by<8>(order(candidate(own, own_nth, nth)), q);
    if (lane == 0) t_lds[wave] = t;
  } else if (lane == 0) {
    t_lds[wave] = 0;
  }
  __syncthreads();
  uint32_t limit = 1;
#pragma unroll
  for (int w = 0; w < kMergeWaves; ++w) limit = t_lds[w] > limit ? t_lds[w] : limit;
  // Lists are in order: each is read up to its first candidate below T
  for (int j0 = 0; j0 < lists; j0 += kMergeThreads) {
    const List l = j0 ? list_of(j0 + tid) : own;
    bool open = true;
    for (int i = 0; i < a.take && __any(open); i += kAhead) {
      uint64_t key[kAhead];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) key[e] = j0 + i ? key_of(l, i + e) : own_keys[e];
#pragma unroll
      for (int e = 0; e < kAhead; ++e) {
        const Candidate c = candidate(l, key[e], i + e);
        open = open && order(c) >= limit;
        if (!__any(open)) break;
        const int s = slot_for(open, &count);
        if (open && s < kMergeKept) kept[s] = c;
      }
    }
  }
  __syncthreads();
  const auto write = [&](int place, const Candidate& c) {
    a.out_scores[b * a.take + place] = float(c.value);
    a.out_parents[b * a.take + place] = c.at / a.vocab;
    a.out_tokens[b * a.take + place] = c.at % a.vocab;
  };
  const int n = count;
  if (n <= kMergeKept) {
    for (int i = tid >> 3; i < n; i += kMergeThreads / 8) {
      const Candidate c = kept[i];
      const int place = place_of(kept, n, c, before);
      if ((tid & 7) == 0 && place < a.take) write(place, c);
    }
    return;
  }
  // The best head of all lists, `take` times; a list's position is kept by the thread that owns it.
  constexpr int kOwn = kBeamMaxLists / kMergeThreads;
  uint8_t taken[kOwn];
#pragma unroll
  for (int i = 0; i < kOwn; ++i) taken[i] = 0;
  Candidate mine{-double(INFINITY), kNone};
  int mine_list = -1;
  const auto look = [&] {
    mine = {-double(INFINITY), kNone};
    mine_list = -1;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const List l = list_of(i * kMergeThreads + tid);
      const Candidate h = candidate(l, key_of(l, taken[i]), taken[i]);
      if (before(h, mine)) mine = h, mine_list = i;
    }
  };
  look();
  for (int k = 0; k < a.take; ++k) {
    Candidate best = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
      const Candidate other = shuffle(best, m);
      if (before(other, best)) best = other;
    }
    if (lane == 0) best_lds[k & 1][wave] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w)
      if (before(best_lds[k & 1][w], best)) best = best_lds[k & 1][w];
    if (tid == 0) write(k, best);
    if (mine_list >= 0 && mine.at == best.at) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) taken[i] += i == mine_list;
      look();
    }
  }
}

// Logits of a thread: 16, or 64 where a row would have more than 64 chunks.
int per_thread(int vocab) { return vocab <= 64 * 16 * kThreads ? 16 : 64; }

template <Type TYPE>
void launch_scan(const BeamArgs& a, Stream s) {
  const dim3 grid(a.chunks, unsigned(a.batch * a.beams));
  launch(per_thread(a.vocab) == 16 ? beam_scan_kernel<TYPE, 16> : beam_scan_kernel<TYPE, 64>, grid, kThreads, a, s,
         "beam_select");
}

}  // namespace

int beam_select_chunks(int vocab) { return int(ceil_div(vocab, per_thread(vocab) * kThreads)); }

int64_t beam_select_scratch(int64_t rows, int chunks, int take) { return rows * chunks * (take + kWaves); }

void beam_select_hip(BeamArgs a, uint64_t* scratch, Stream s) {
  if (a.batch == 0) return;
  a.part_list = scratch;
  a.part_stat = reinterpret_cast<float*>(scratch + a.batch * a.beams * a.chunks * a.take);
  if (a.type == kF32)
    launch_scan<kF32>(a, s);
  else if (a.type == kF16)
    launch_scan<kF16>(a, s);
  else
    launch_scan<kBF16>(a, s);
  launch(beam_merge_kernel, dim3(unsigned(a.batch)), kMergeThreads, a, s, "beam_select");
}

}  // namespace tl_ops
