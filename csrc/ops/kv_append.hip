// kv_append.hip -- new tokens into the e4m3 cache, with one scale per page and head.
//
//   s_new = pow2ceil(max |new tokens of the page| / 448);  s = s_new if the page begins with them, else
//   max(s_old, s_new);  codes = e4m3(x / s), and the page's older codes c become e4m3(c s_old / s) if s grew.
//
// Scales are powers of two: a code that is scaled again keeps its value unless it becomes subnormal.  Then it is
// rounded once more, to a multiple of 2^-9 of the new scale: off by up to 2^-10 of it, each time.  One workgroup owns
// one (page, head) of K or of V: no two write one scale.
//
// Bound by HBM: 3 bytes an element in 16 bits.  8 prompts of 4001 tokens, 8 heads of 128 (197 MB): 40 us, 4.9 TB/s;
// pages of over 512 items (KEEP = false) read their tokens a second time: heads of 256 in pages of 128 2.5 times a
// copy's time, pages of 1024 2.2 times.
//
// Codes that are scaled again take a read and a write of one byte for each thread in turn, which bounds the calls that
// reach it: one token for 32 sequences, 8 heads of 128, pages of 64 that are nearly full, in a graph, 48 us where every
// scale grows against 5.7 where none does; pages of 1024 tokens of 256 1.4 ms.
#include "device.h"

namespace tl_ops {
namespace {

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

// A thread's item: 4 slots of the page (one dword of a V row) by 8 dims (16 bytes of a 16-bit token).
constexpr int kSlots = 4, kDims = 8;

// KEEP: the items fit the threads, and a token is read once; else a second time for its codes.
// VEC: every 8 elements of a token are a vector on a 16-byte boundary (fp32: two).
template <Type TYPE, int THREADS, bool KEEP, bool VEC>
__global__ __launch_bounds__(THREADS) void kv_append_kernel(AppendArgs a) {
  using T = typename Scalar<TYPE>::type;
  constexpr bool TILE = KEEP && THREADS >= 256;
  __shared__ float lds[THREADS / 64];
  const Cache& c = a.cache;
  const int head = blockIdx.x, b = blockIdx.z >> 1, which = blockIdx.z & 1, tid = threadIdx.x;
  const Span s = span_of(c, b, a.new_tokens, blockIdx.y);
  if (s.n == 0) return;
  const int page = 1 << c.page_shift, upto = s.slot0 + s.n;
  const T* x = static_cast<const T*>(a.x[which]) + b * a.stride_b[which] + head * a.stride_h[which];
  const int64_t st = a.stride_t[which];
  uint8_t* pool = (which ? c.v : c.k) + (s.page * c.heads + head) * int64_t(page) * c.wide;
  float* scale_at = (which ? c.v_scale : c.k_scale) + s.page * c.heads + head;
  const float before = s.slot0 ? *scale_at : 0.0f;

  const int octs = c.wide / kDims, quad0 = s.slot0 / kSlots, items = ((upto - 1) / kSlots - quad0 + 1) * octs;
  float v[kSlots][kDims];
  const auto load = [&](int item) {
    const int slot = (quad0 + item / octs) * kSlots, d = item % octs * kDims;
#pragma unroll
    for (int t = 0; t < kSlots; ++t) {
      const bool mine = slot + t >= s.slot0 && slot + t < upto;
      const T* p = x + (s.first + slot + t - s.slot0) * st + d;
      if (VEC) {
        typedef T V __attribute__((ext_vector_type(kDims)));
        V r{};
        if (mine && d < c.dim) r = __builtin_nontemporal_load(reinterpret_cast<const V*>(p));
#pragma unroll
        for (int e = 0; e < kDims; ++e) v[t][e] = float(r[e]);
      } else {
        load8_anywhere(p, mine ? c.dim - d : 0, v[t]);
      }
    }
  };
  // non-finite values do not set a scale: infinities are stored as the largest code, not-a-number as itself
  float amax = 0.0f;
  for (int i = tid; i < items; i += THREADS) {
    load(i);
#pragma unroll
    for (int t = 0; t < kSlots; ++t)
#pragma unroll
      for (int e = 0; e < kDims; ++e) amax = fabsf(v[t][e]) < INFINITY ? fmaxf(amax, fabsf(v[t][e])) : amax;
  }
  amax = block_reduce<THREADS>(amax, lds, Max());
  const float scale = fmaxf(pow2_scale(fmaxf(amax, kAmaxFloor)), before), inv = 1.0f / scale;
  if (THREADS > 64) __syncthreads();  // everybody has read the scale
  if (tid == 0) *scale_at = scale;

  // A whole page of V turns around in LDS and is written in its own order (up to 256 rows, padded by a dword
  // against bank conflicts): 40 us for 8 x 4001 tokens in 8 heads of 128, 48 with each thread's dwords straight to
  // memory.
  __shared__ uint32_t tile[TILE ? THREADS * kDims + 256 : 1];
  const bool whole = TILE && which && s.n == page;
  const int pitch = page / kSlots + 1;
  for (int i = tid; i < items; i += THREADS) {
    if (!KEEP) load(i);
    const int slot = (quad0 + i / octs) * kSlots, d = i % octs * kDims;
    uint32_t code[kSlots][2];  // of a token's 8 dims
#pragma unroll
    for (int t = 0; t < kSlots; ++t) {
#pragma unroll
      for (int e = 0; e < kDims; ++e) {
        const float w = v[t][e] * inv;
        v[t][e] = w > kFp8Max ? kFp8Max : w < -kFp8Max ? -kFp8Max : w;
      }
      code[t][0] = pack_fp8(v[t][0], v[t][1], v[t][2], v[t][3]);
      code[t][1] = pack_fp8(v[t][4], v[t][5], v[t][6], v[t][7]);
    }
    if (which == 0) {
#pragma unroll
      for (int t = 0; t < kSlots; ++t)
        if (slot + t >= s.slot0 && slot + t < upto)
          *reinterpret_cast<u32x2*>(pool + (slot + t) * c.wide + d) = u32x2{code[t][0], code[t][1]};
    } else {
      const bool all = slot >= s.slot0 && slot + kSlots <= upto;
#pragma unroll
      for (int e = 0; e < kDims; ++e) {
        const uint32_t at = 8 * (e & 3);
        uint32_t w = 0;
#pragma unroll
        for (int t = 0; t < kSlots; ++t) w |= (code[t][e >> 2] >> at & 0xff) << (8 * t);
        uint8_t* p = pool + (d + e) * page + slot;
        if (whole) {
          tile[(d + e) * pitch + slot / kSlots] = w;
        } else if (all) {
          *reinterpret_cast<uint32_t*>(p) = w;
        } else {
#pragma unroll
          for (int t = 0; t < kSlots; ++t)
            if (slot + t >= s.slot0 && slot + t < upto) p[t] = uint8_t(w >> (8 * t));
        }
      }
    }
  }
  if (whole) {
    __syncthreads();
    for (int i = tid; i < c.wide * (page / kSlots); i += THREADS) {
      const int row = i >> (c.page_shift - 2), word = i & (page / kSlots - 1);
      reinterpret_cast<uint32_t*>(pool)[i] = tile[row * pitch + word];
    }
  }
  if (scale > before) {  // the page's older tokens
    for (int i = tid; i < s.slot0 * c.wide; i += THREADS) {
      const int slot = i / c.wide, d = i - slot * c.wide;
      uint8_t* p = pool + (which ? d * page + slot : i);
      *p = uint8_t(pack_fp8(__builtin_amdgcn_cvt_f32_fp8(int(*p), 0) * (before * inv), 0.0f, 0.0f, 0.0f));
    }
  }
}

template <Type TYPE>
void launch_type(const AppendArgs& a, Stream s) {
  using T = typename Scalar<TYPE>::type;
  const int page = 1 << a.cache.page_shift;
  int64_t pages = (a.new_tokens - 1) / page + 2;
  if (pages > a.cache.table_width) pages = a.cache.table_width;
  const dim3 grid(a.cache.heads, unsigned(pages), 2 * a.batch);
  bool vec = a.cache.dim % kDims == 0;
  for (int w = 0; w < 2; ++w)
    vec = vec && (reinterpret_cast<uintptr_t>(a.x[w]) | uintptr_t(a.stride_b[w] * sizeof(T)) |
                  uintptr_t(a.stride_t[w] * sizeof(T)) | uintptr_t(a.stride_h[w] * sizeof(T))) % 16 == 0;
  // the items of a page: a few tokens touch two quads at most for every four of them, and no more than the page has
  const int quads = a.new_tokens < page ? (a.new_tokens + kSlots - 2) / kSlots + 1 : page / kSlots;
  const int items = quads * (a.cache.wide / kDims);
  const char* what = "kv_cache_append";
  if (items <= 64)
    launch(vec ? kv_append_kernel<TYPE, 64, true, true> : kv_append_kernel<TYPE, 64, true, false>, grid, 64, a, s,
           what);
  else if (items <= 256)
    launch(vec ? kv_append_kernel<TYPE, 256, true, true> : kv_append_kernel<TYPE, 256, true, false>, grid, 256, a, s,
           what);
  else if (items <= 512)
    launch(vec ? kv_append_kernel<TYPE, 512, true, true> : kv_append_kernel<TYPE, 512, true, false>, grid, 512, a, s,
           what);
  else
    launch(vec ? kv_append_kernel<TYPE, 256, false, true> : kv_append_kernel<TYPE, 256, false, false>, grid, 256, a, s,
           what);
}

}  // namespace

void kv_append_hip(const AppendArgs& a, Stream s) {
  if (a.batch == 0 || a.new_tokens == 0 || a.cache.table_width == 0) return;
  if (a.type == kF32) return launch_type<kF32>(a, s);
  if (a.type == kF16) return launch_type<kF16>(a, s);
  launch_type<kBF16>(a, s);
}

}  // namespace tl_ops
