// kv_append.hip -- new tokens into the e4m3 cache, with one scale per page and head.
//
//   s_new = pow2ceil(max |new tokens of the page| / 448);  s = s_new if the page begins with them, else
//   max(s_old, s_new);  codes = e4m3(x / s), and the page's older codes c become e4m3(c s_old / s) if s grew.
//
// Scales are powers of two: dividing by one rounds nothing, so a code that is scaled again keeps its value but for
// what falls below e4m3's smallest step.  One workgroup owns one (page, head) of K or of V: no two write one scale.
#include "device.h"

namespace tl_ops {
namespace {

constexpr int kThreads = 256;

// Where a workgroup's new tokens go: slots [slot0, slot0 + n) of the page, token `first` onwards.
struct Span {
  int64_t page;
  int slot0, n, first;
};

// The nth page that sequence b's new tokens reach; n = 0 if there is none, or its id is outside the pool.
__device__ inline Span span_of(const Cache& c, int b, int new_tokens, int nth) {
  const int page = 1 << c.page_shift;
  const int64_t end = c.lengths[b], begin = end - new_tokens;  // the new tokens' positions
  const int64_t from = begin < 0 ? 0 : begin;
  const int64_t at = (from >> c.page_shift) + nth;
  Span s{0, 0, 0, 0};
  if (at >= c.table_width) return s;
  const int64_t lo = at * page > from ? at * page : from;
  const int64_t hi = (at + 1) * page < end ? (at + 1) * page : end;
  if (hi <= lo) return s;
  const int id = c.table[b * c.table_stride + at];
  if (id < 0 || id >= c.pages) return s;
  s.page = id;
  s.slot0 = int(lo - at * page);
  s.n = int(hi - lo);
  s.first = int(lo - begin);
  return s;
}

template <Type TYPE>
__global__ __launch_bounds__(kThreads) void kv_append_kernel(AppendArgs a) {
  using T = typename Scalar<TYPE>::type;
  __shared__ float lds[kThreads / 64];
  const Cache& c = a.cache;
  const int head = blockIdx.x, b = blockIdx.z >> 1, which = blockIdx.z & 1, tid = threadIdx.x;
  const Span s = span_of(c, b, a.new_tokens, blockIdx.y);
  if (s.n == 0) return;
  const T* x = static_cast<const T*>(a.x[which]) + b * a.stride_b[which] + head * a.stride_h[which];
  const int64_t st = a.stride_t[which];
  // non-finite values do not set a scale: infinities are stored as the largest code, not-a-number as itself
  float amax = 0.0f;
  for (int i = tid; i < s.n * c.dim; i += kThreads) {
    const int t = i / c.dim, d = i - t * c.dim;
    const float v = fabsf(float(x[(s.first + t) * st + d]));
    amax = v < INFINITY ? fmaxf(amax, v) : amax;
  }
  amax = block_reduce<kThreads>(amax, lds, Max());
  float* scale_at = (which ? c.v_scale : c.k_scale) + s.page * c.heads + head;
  const float fresh = pow2_scale(fmaxf(amax, kAmaxFloor)), before = s.slot0 ? *scale_at : 0.0f;
  const float scale = fmaxf(fresh, before), inv = 1.0f / scale;
  __syncthreads();
  if (tid == 0) *scale_at = scale;
  const int page = 1 << c.page_shift;
  uint8_t* pool = (which ? c.v : c.k) + (s.page * c.heads + head) * int64_t(page) * c.wide;
  const auto code = [&](float v) { return uint8_t(pack_fp8(v, 0.0f, 0.0f, 0.0f)); };
  const auto clamped = [&](float v) { return v > kFp8Max ? kFp8Max : v < -kFp8Max ? -kFp8Max : v; };
  const int upto = s.slot0 + s.n, old = scale > before ? 0 : s.slot0;  // slots that are written: [old, upto)
  for (int i = tid; i < (upto - old) * c.wide; i += kThreads) {
    const int row = i / c.wide, d = i - row * c.wide, slot = old + row;
    uint8_t* p = pool + (which ? d * page + slot : slot * c.wide + d);
    if (slot < s.slot0) {
      const float v = __builtin_amdgcn_cvt_f32_fp8(int(*p), 0);
      *p = code(v * (before * inv));
    } else {
      const float v = d < c.dim ? float(x[(s.first + slot - s.slot0) * st + d]) : 0.0f;
      *p = code(clamped(v * inv));
    }
  }
}

}  // namespace

void kv_append_hip(const AppendArgs& a, Stream s) {
  if (a.batch == 0 || a.new_tokens == 0 || a.cache.heads == 0 || a.cache.table_width == 0) return;
  const int page = 1 << a.cache.page_shift;
  int64_t pages = (a.new_tokens - 1) / page + 2;
  if (pages > a.cache.table_width) pages = a.cache.table_width;
  const dim3 grid(a.cache.heads, unsigned(pages), 2 * a.batch);
  const auto k = a.type == kF32   ? kv_append_kernel<kF32>
                 : a.type == kF16 ? kv_append_kernel<kF16>
                                  : kv_append_kernel<kBF16>;
  launch(k, grid, kThreads, a, s, "kv_cache_append");
}

}  // namespace tl_ops
