// kv_attention.hip -- attention over the e4m3 paged cache (flash-decoding form, any number of new tokens).
//
//   o = sum_j softmax_j(scale ks_j q.k_j) vs_j v_j over the keys j <= position of the query
//
// The (new token, query head) pairs that share a key head are the rows of its two products, 16 NR at a time; a wave
// takes 64 keys at a time through both without leaving its registers:
//
//   S^T = K Q^T   mfma 16x16x32, A = K (16 keys), B = Q (16 rows): a lane then holds scores of ONE row
//   O^T = V^T P^T A = V^T (16 dims), B = P: the scores' own registers, since the contraction's order is free
//
// Key tile kt's row r stands for key 16 (r / 4) + 4 kt + r % 4, so the lane group g = lane / 16 ends up with the 16
// keys 16 g .. 16 g + 15 of its row, and V's matching operand is 16 consecutive bytes of V's [dim][token] page.
// K's contraction goes over d = 64 chunk + 16 g + 0..15 for the same reason: both operands come from memory in
// 16-byte loads and the softmax needs one exchange over the four lane groups.  e4m3 widens to bf16 and fp16 exactly;
// the products run on 16-bit operands and accumulate in float32.  P is rounded to bf16 (V's scale folded in, whose
// range only bf16 has): a weight is off by up to 2^-8 of itself, as the output's own rounding to bf16 is of it.  The
// largest weight is 1 and exact here, which leaves the error against float64 that of the output's rounding (0.0017 in
// the root mean square, 32 sequences of up to 8192 keys); for the chunks see SLACK.  For fp16 the rounding's rest goes
// through a second product, which keeps the error that of the output's own rounding there too.
//
// The waves of a workgroup take tiles in turn and join in LDS; `splits` workgroups share a long key axis and
// kv_join_kernel joins them (3 us for 32 rows in 7 parts).
//
// Single tokens are bound by HBM: no byte of the cache is read twice, and two workgroups on a CU (heads up to 128;
// wider ones have registers for one) keep 128 KB in flight.
// 32 sequences of 4096 to 8192 tokens, 32 heads on 8 of 128: 75 us, 5.4 TB/s; one of 777 tokens: 6.4 us and the join.
#include <algorithm>
#include <type_traits>

#include "device.h"

namespace tl_ops {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 64;  // keys of one wave's step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// The weighted sums of V are kept 2^32 times smaller than they are: of values up to float32's largest, 2^24 weights
// of 2^SLACK can be summed.
constexpr float kLogUnit = 32.0f, kUnit = 0x1p32f;

// The operands of the first product: Q's type, into which e4m3 widens exactly.  (The matrix cores' own e4m3 product
// needs no widening, with Q split into e4m3 parts; but it aligns its summands in few bits: sums of 128 were off by up
// to 2^-12 of the largest summand, which a softmax statistic may not be.)
template <Type TYPE> struct Half;
template <> struct Half<kBF16> {
  using X8 = bf16x8;
  static __device__ f32x4 mfma(X8 a, X8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ X8 widen(uint32_t lo, uint32_t hi) {
    union { X8 x; bf16x2 h[4]; } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return r.x;
  }
};
template <> struct Half<kF16> {
  using X8 = f16x8;
  static __device__ f32x4 mfma(X8 a, X8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ X8 widen(uint32_t lo, uint32_t hi) {
    union { X8 x; f16x2 h[4]; } r;
    r.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
    r.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    r.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
    r.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return r.x;
  }
};
using Wide = Half<kBF16>;  // the second product's operands

__device__ inline float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // results under 2^-126 are zero

// The lanes that hold a row's keys are 16 and 32 apart; a swap of a register with itself leaves both halves of each
// pair in both lanes, without a trip through LDS.
template <typename F>
__device__ inline float across_groups(float v, F f) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// e4m3 bytes that are not-a-number (0x7f, 0xff): bit 7 of each such byte
__device__ inline uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// the first n bytes of four
__device__ inline uint32_t first_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u; }

// One row's Q as operands of the first product; the scores' scale may be negative, and its sign goes here, so that
// the largest product is the largest score.
template <Type TYPE, int DC>
__device__ inline void load_q(const AttentionArgs& a, int b, int head, int row, int rows, int grp,
                              typename Half<TYPE>::X8 (&q)[2 * DC]) {
  using T = typename Scalar<TYPE>::type;
  using X8 = typename Half<TYPE>::X8;
  const Cache& c = a.cache;
  const int per = a.heads / c.heads, i = row / per, h = head * per + row % per;
  const T* p = static_cast<const T*>(a.q) + b * a.stride_b + i * a.stride_t + h * a.stride_h;
  const bool whole = row < rows && c.dim == c.wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
#pragma unroll
  for (int k = 0; k < 2 * DC; ++k) {
    const int d = 64 * (k >> 1) + 16 * grp + 8 * (k & 1);
    if (whole) {
      q[k] = *reinterpret_cast<const X8*>(p + d);
    } else if (row < rows && d + 8 <= c.dim) {
      __builtin_memcpy(&q[k], p + d, sizeof(X8));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) q[k][j] = row < rows && d + j < c.dim ? p[d + j] : T(0.0f);
    }
    if (a.scale < 0.0f) q[k] = -q[k];
  }
}

// Scores of keys behind the row's position, or of a page that is not there, become -inf.
__device__ inline void hide(f32x4 (&s)[4], bool there, int key, int pos) {
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (!there || key + 4 * t + i > pos) s[t][i] = -INFINITY;
}

// A row that sees one of the not-a-numbers that `is` marks becomes one, a row that does not stays as it is.
__device__ inline void poison(bf16x8 is, bool there, int key, int pos, f32x4& o) {
  bf16x8 seen;
#pragma unroll
  for (int e = 0; e < 8; ++e) seen[e] = __bf16(there && key + e <= pos ? 1.0f : 0.0f);
  const f32x4 count = Wide::mfma(is, seen, f32x4{});
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = count[i] > 0.0f ? NAN : o[i];
}

// The weights of 16 scores of each of NR rows (in units of 1 / ks), with V's scale, as operands of the second
// product; a page that is not `there` has none.  The sums are relative to m, which moves when the scores outgrow it by
// more than a factor of 2^SLACK.  With 0 the largest weight is 1 and rounds to itself; a larger one saves most of the
// sums' rescaling where that counts, and rounds the largest weight too.  2 x 509 tokens on up to 4096 keys in the chunk
// form: 82.0 us and an error against float64 of 0.0021 with 8, 86.7 us and 0.0018 with 0, of which the output's
// rounding is 0.0017.
template <Type TYPE, int NR, int DT, int SLACK>
__device__ inline void softmax_step(const f32x4 (&s)[NR][4], float ks, float vs, bool there, float (&m)[NR],
                                    float (&l)[NR], f32x4 (&o)[NR][DT], bf16x8 (&hi)[NR][2], bf16x8 (&lo)[NR][2]) {
  float top[NR];
  bool grown = false;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    top[r] = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top[r] = fmaxf(top[r], s[r][t][i]);
    top[r] = across_groups(there ? top[r] * ks : -INFINITY, Max());
    grown |= top[r] > m[r] + float(SLACK);
  }
  if (__any(grown)) {
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float next = fmaxf(m[r], top[r]), alpha = next == -INFINITY ? 1.0f : exp2_of(m[r] - next);
      m[r] = next;
      l[r] *= alpha;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[r][d] *= alpha;
    }
  }
  // V's scale goes into the exponent; it is taken as 2^-68 where it is less (an append's are 2^-22 at least)
  vs = fmaxf(vs, 0x1p-68f);
  const float log_vs = __builtin_amdgcn_logf(vs) - kLogUnit, inv_vs = kUnit / vs;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const float base = there ? log_vs - (m[r] == -INFINITY ? 0.0f : m[r]) : -INFINITY;
    float sum = 0.0f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float w = exp2_of(fmaf(s[r][t][i], ks, base));
        sum += w;
        hi[r][t >> 1][4 * (t & 1) + i] = __bf16(w);
        if (TYPE == kF16) lo[r][t >> 1][4 * (t & 1) + i] = __bf16(w - float(__bf16(w)));
      }
    l[r] += sum * inv_vs;
  }
}

// Values at .. at + 3 of a row of `dim` (at % 4 == 0); at once where every row begins on such a boundary.
template <typename T>
__device__ inline void store4(T* row, f32x4 v, int at, int dim) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  if (dim % 4 == 0) {
    if (at < dim) *reinterpret_cast<T4*>(row + at) = T4{T(v[0]), T(v[1]), T(v[2]), T(v[3])};
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + i < dim) row[at + i] = T(v[i]);
  }
}

// STREAM: past the caches.  For what they could not keep until it is read again: 32 sequences of 4096 to 8192 tokens
// (400 MB) take 74.7 us with it and 80.9 without, 16 of 1024 to 2048 in heads of 100 (206 MB) 40.3 and 34.6.
template <bool STREAM>
__device__ inline u32x4 load16(const uint8_t* p) {
  const u32x4* q = reinterpret_cast<const u32x4*>(p);
  return STREAM ? __builtin_nontemporal_load(q) : *q;
}

// The pages of a lane's K row and of its 16 keys in one tile, and where they are.  Pages of 64 tokens and more hold
// WHOLE tiles: then both are one page for all lanes, and its id, address and scales stay in scalar registers.
struct Pages {
  int k, v;
};
struct Place {
  const uint8_t *k, *v;
  float ks, vs;
  bool there;  // whether the page of its 16 keys is in the pool
};

template <Type TYPE, int DC, int NR, bool WHOLE, bool STREAM>
__global__ __launch_bounds__(kThreads) void kv_attention_kernel(AttentionArgs a) {
  using T = typename Scalar<TYPE>::type;
  constexpr int ROWS = 16 * NR, DT = 4 * DC;  // rows of the workgroup, 16-wide slices of the head
  using H = Half<TYPE>;
  using X8 = typename H::X8;
  constexpr int WIDTH = DC * 64, PITCH = WIDTH + 4;
  __shared__ float o_lds[kWaves][ROWS][PITCH];
  __shared__ float m_lds[kWaves][ROWS], l_lds[kWaves][ROWS];

  const Cache& c = a.cache;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int split = blockIdx.y, b = blockIdx.z;
  const int head = int(blockIdx.x) % c.heads, row0 = int(blockIdx.x) / c.heads * ROWS;
  const int per = a.heads / c.heads, rows = a.new_tokens * per;  // query heads of a key head
  const int page = 1 << c.page_shift;

  const int past = max(c.lengths[b], 0) - a.new_tokens;  // query i sees the keys up to past + i
  const int last = (row0 + ROWS < rows ? row0 + ROWS : rows) - 1;
  // one behind the last key that a row of this workgroup sees and the table can name
  const int end = min(past + last / per + 1, c.table_width << c.page_shift);
  const int tiles = end > 0 ? (end + kTile - 1) / kTile : 0;
  const int tile0 = int(int64_t(tiles) * split / a.splits) + wave;
  const int tile1 = int(int64_t(tiles) * (split + 1) / a.splits);

  const int* table = c.table + b * c.table_stride;
  const uint32_t head_bytes = uint32_t(page) * c.wide;
  const auto pages_of = [&](int tile) {
    // a group of keys behind the end reads the last page
    const auto page_of = [&](int key) { return table[(key < end ? key : end - 1) >> c.page_shift]; };
    if (WHOLE) return Pages{page_of(tile * kTile), page_of(tile * kTile)};
    return Pages{page_of(tile * kTile + 16 * (col >> 2)), page_of(tile * kTile + 16 * grp)};
  };
  const auto place_of = [&](int tile, Pages id) {
    const auto in_pool = [&](int i) { return i >= 0 && i < c.pages; };
    const int key_k = tile * kTile + 16 * (col >> 2), key_v = tile * kTile + 16 * grp;
    const uint32_t page_k = uint32_t(in_pool(id.k) ? id.k : 0) * c.heads + head;
    const uint32_t page_v = uint32_t(in_pool(id.v) ? id.v : 0) * c.heads + head;
    Place p;
    p.there = in_pool(id.v);
    p.k = c.k + uint64_t(page_k) * head_bytes + ((key_k & (page - 1)) + (col & 3)) * c.wide + 16 * grp;
    p.v = c.v + uint64_t(page_v) * head_bytes + (key_v & (page - 1));
    p.ks = c.k_scale[page_v];
    p.vs = c.v_scale[page_v];
    return p;
  };
  u32x4 kx[4][DC], vx[DT];
  const auto load_k = [&](const Place& p) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < DC; ++k) kx[t][k] = load16<STREAM>(p.k + 4 * t * c.wide + 64 * k);
  };
  // What a tile needs is asked for a tile ahead (its pages' ids two ahead), and V behind K: no wait is for a load
  // that has just been issued.  Behind the last tile the loads repeat it.
  const auto ahead = [&](int tile) { return tile < tile1 ? tile : tile1 - 1; };
  Place at{};
  Pages next{};
  if (tile0 < tile1) {
    const Pages first = pages_of(tile0);
    next = pages_of(ahead(tile0 + kWaves));
    at = place_of(tile0, first);
    load_k(at);
  }

  X8 q[NR][2 * DC];
  int pos[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = row0 + 16 * r + col;
    pos[r] = row < rows ? min(past + row / per, end - 1) : -1;
    load_q<TYPE, DC>(a, b, head, row, rows, grp, q[r]);
  }
  const float to_log2 = fabsf(a.scale) * kLog2e;
  f32x4 o[NR][DT] = {};
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.0f;

  for (int tile = tile0; tile < tile1; tile += kWaves) {
    const int key0 = tile * kTile, key_v = key0 + 16 * grp;
    const Place now = at;
#pragma unroll
    for (int d = 0; d < DT; ++d)  // a padded row is not read: another one stands in, its result is not written
      vx[d] = load16<STREAM>(now.v + (16 * d + col < c.dim ? 16 * d + col : c.dim - 1) * page);
    at = place_of(ahead(tile + kWaves), next);
    next = pages_of(ahead(tile + 2 * kWaves));

    f32x4 s[NR][4] = {};
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < 2 * DC; ++k) {
        const u32x4 x = kx[t][k >> 1];
        const X8 k8 = k & 1 ? H::widen(x.z, x.w) : H::widen(x.x, x.y);
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][t] = H::mfma(k8, q[r][k], s[r][t]);
      }
    load_k(at);

    // some row does not see some key, or a page is absent
    const bool masked = key0 + kTile > min(past + row0 / per + 1, end) || __any(!now.there);
    if (masked) {
      const int n = now.there ? end - key_v : 0;
      uint32_t found = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          vx[d][j] &= first_bytes(n - 4 * j);  // what lies behind the sequence must not count, not even times zero
          found |= nan_bytes(vx[d][j]);
        }
#pragma unroll
      for (int r = 0; r < NR; ++r) hide(s[r], now.there, key_v, pos[r]);
      if (__any(found != 0)) {
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t n0 = nan_bytes(vx[d][2 * u]) >> 7, n1 = nan_bytes(vx[d][2 * u + 1]) >> 7;
            vx[d][2 * u] &= ~(n0 * 0xff);
            vx[d][2 * u + 1] &= ~(n1 * 0xff);
            const bf16x8 is = Wide::widen(n0 * 0x38, n1 * 0x38);  // 0x38: 1.0
#pragma unroll
            for (int r = 0; r < NR; ++r) poison(is, now.there, key_v + 8 * u, pos[r], o[r][d]);
          }
      }
    }

    const float ks = fmaxf(now.ks * to_log2, 1e-30f);  // never zero: a hidden score stays -inf
    const float vs = now.there ? now.vs : 0.0f;
    bf16x8 hi[NR][2], lo[NR][2];
    softmax_step<TYPE, NR, DT, 0>(s, ks, vs, now.there, m, l, o, hi, lo);
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bf16x8 v = Wide::widen(vx[d][2 * u], vx[d][2 * u + 1]);
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          o[r][d] = Wide::mfma(v, hi[r][u], o[r][d]);
          if (TYPE == kF16) o[r][d] = Wide::mfma(v, lo[r][u], o[r][d]);
        }
      }
  }

  // join the waves: sums relative to the largest maximum
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] = across_groups(l[r], Add());
    if (grp == 0) m_lds[wave][16 * r + col] = m[r], l_lds[wave][16 * r + col] = l[r];
  }
  const int here = rows - row0 < ROWS ? rows - row0 : ROWS;
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int d = 0; d < DT; ++d)
      *reinterpret_cast<f32x4*>(&o_lds[wave][16 * r + col][16 * d + 4 * grp]) = o[r][d];
  __syncthreads();
  for (int i = threadIdx.x; i < here * (WIDTH / 4); i += kThreads) {
    const int r = i / (WIDTH / 4), d0 = i % (WIDTH / 4) * 4, row = row0 + r;
    float top = m_lds[0][r], sum = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w][r]);
    f32x4 v = {};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = m_lds[w][r] == -INFINITY ? 0.0f : exp2_of(m_lds[w][r] - top);
      sum += l_lds[w][r] * f;
      v += *reinterpret_cast<const f32x4*>(&o_lds[w][r][d0]) * f;
    }
    const int64_t out = (int64_t(b) * a.new_tokens + row / per) * a.heads + head * per + row % per;
    if (a.splits == 1) {
      const float inv = sum == 0.0f ? 0.0f : kUnit / sum;
      store4(static_cast<T*>(a.out) + out * c.dim, v * inv, d0, c.dim);
      if (d0 == 0 && a.lse) a.lse[out] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    } else {
      const int64_t part = out * a.splits + split;
      store4(a.part_o + part * c.dim, v, d0, c.dim);
      if (d0 == 0) a.part_ml[part * 2] = top, a.part_ml[part * 2 + 1] = sum;
    }
  }
}

// Keeps what stands before it before what stands behind it: reads of operands from LDS stay a group ahead of the
// products that use them (4 % of the chunks' time).
__device__ inline void in_order() { __builtin_amdgcn_sched_barrier(0); }

// The form for many rows (chunks of prompts): arithmetic bounds it, not the cache, so the keys of a step are widened
// once for all rows.  A workgroup holds 128 rows, 32 to a wave; waves 0-3 take the even tiles, waves 4-7 the odd ones,
// two waves to a SIMD so that one's softmax runs beside the other's products.  Each step's two tiles lie in LDS as the
// operands that the products read (16 bytes a lane, in lane order: no bank conflict), in two buffers: the next step is
// loaded during the products and written behind them, with one barrier a step.  2 x 509 tokens on up to 4096 keys, 32
// heads on 8 of 128: 82 us, 675 TFLOP/s; what bounds it is the softmax beside the products.
constexpr int kChunkWaves = 8, kChunkThreads = kChunkWaves * 64, kChunkRows = 128;

template <Type TYPE, int DC, bool WHOLE>
__global__ __launch_bounds__(kChunkThreads, 2) void kv_attention_chunk_kernel(AttentionArgs a) {
  using T = typename Scalar<TYPE>::type;
  using H = Half<TYPE>;
  using X8 = typename H::X8;
  constexpr int DT = 4 * DC, NR = 2, PITCH = DC * 64 + 4;
  struct Tile {
    X8 k[4][2 * DC][64];
    bf16x8 v[DT][2][64];
  };
  struct Scales {
    float ks, vs;
    int there;
  };
  union Lds {
    Tile tile[2][2];
    float o[kChunkRows][PITCH];
  };
  __shared__ Lds lds;
  __shared__ Scales scales[2][2][4];
  // V's not-a-numbers go as zeros into the product and reach the rows that see them by `poison`: whether what a wave
  // wrote holds any (a byte for each), and where (bit e: key 16 grp + e of the lane).  Only where some row does not
  // see all of the tile: elsewhere they may spread by themselves
  __shared__ uint32_t nan[2][2];
  __shared__ uint16_t nan_marks[2][2][DT][64];
  __shared__ float m_lds[kChunkRows], l_lds[kChunkRows];

  const Cache& c = a.cache;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 15, grp = lane >> 4;
  const int part = wave >> 2, mine = wave & 3;  // the tile of a step, and what of it this wave loads
  const int split = blockIdx.y, b = blockIdx.z;
  const int head = int(blockIdx.x) % c.heads, row0 = int(blockIdx.x) / c.heads * kChunkRows;
  const int per = a.heads / c.heads, rows = a.new_tokens * per;
  const int page = 1 << c.page_shift;
  const int past = max(c.lengths[b], 0) - a.new_tokens;
  const int last = min(row0 + kChunkRows, rows) - 1;
  const int end = min(past + last / per + 1, c.table_width << c.page_shift);
  const int steps = end > 0 ? (end + 2 * kTile - 1) / (2 * kTile) : 0;
  const int step0 = int(int64_t(steps) * split / a.splits), step1 = int(int64_t(steps) * (split + 1) / a.splits);
  const int* table = c.table + b * c.table_stride;
  const uint32_t head_bytes = uint32_t(page) * c.wide;

  // This wave's share of a tile: K rows of slice `mine`, V's slices `mine`, `mine` + 4, ..  A step's loads are issued
  // a step before they are written to LDS (its pages' ids another step before); behind the last step they repeat it.
  u32x4 kx[DC], vx[DC];
  Scales sc{};
  bool k_there = true;
  const auto ahead = [&](int step) { return step < step1 ? step : step1 - 1; };
  const auto pages_of = [&](int step) {
    const int key0 = (2 * ahead(step) + part) * kTile;
    // a group of keys behind the end reads the last page
    const auto page_of = [&](int key) { return table[(key < end ? key : end - 1) >> c.page_shift]; };
    if (WHOLE) return Pages{page_of(key0), page_of(key0)};
    return Pages{page_of(key0 + 16 * (col >> 2)), page_of(key0 + 16 * grp)};
  };
  const auto load = [&](int step, Pages id) {
    const int key0 = (2 * ahead(step) + part) * kTile, key_k = key0 + 16 * (col >> 2), key_v = key0 + 16 * grp;
    const auto in_pool = [&](int i) { return i >= 0 && i < c.pages; };
    const uint32_t page_k = uint32_t(in_pool(id.k) ? id.k : 0) * c.heads + head;
    const uint32_t page_v = uint32_t(in_pool(id.v) ? id.v : 0) * c.heads + head;
    const uint8_t* kp = c.k + uint64_t(page_k) * head_bytes + ((key_k & (page - 1)) + (col & 3) + 4 * mine) * c.wide +
                        16 * grp;
    const uint8_t* vp = c.v + uint64_t(page_v) * head_bytes + (16 * mine + col) * page + (key_v & (page - 1));
#pragma unroll
    for (int k = 0; k < DC; ++k) kx[k] = *reinterpret_cast<const u32x4*>(kp + 64 * k);
#pragma unroll
    for (int d = 0; d < DC; ++d) vx[d] = *reinterpret_cast<const u32x4*>(vp + 64 * d * page);
    sc = {c.k_scale[page_v], c.v_scale[page_v], in_pool(id.v)};
    k_there = in_pool(id.k);
  };
  const auto write = [&](int step, int buf) {
    if (__any(!k_there)) {  // the scores of a page that is not there stay finite, and its weights become zero
#pragma unroll
      for (int k = 0; k < DC; ++k) kx[k] = k_there ? kx[k] : u32x4{};
    }
#pragma unroll
    for (int k = 0; k < DC; ++k) {
      lds.tile[buf][part].k[mine][2 * k][lane] = H::widen(kx[k].x, kx[k].y);
      lds.tile[buf][part].k[mine][2 * k + 1][lane] = H::widen(kx[k].z, kx[k].w);
    }
    const int key0 = (2 * ahead(step) + part) * kTile;
    if (key0 + kTile > end || __any(!sc.there)) {
      // what lies behind the sequence must not count, not even times zero
      const int n = sc.there ? end - key0 - 16 * grp : 0;
#pragma unroll
      for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) vx[d][j] &= first_bytes(n - 4 * j);
    }
    uint32_t found = 0;
    if (key0 + kTile > past + row0 / per + 1) {
#pragma unroll
      for (int d = 0; d < DC; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= nan_bytes(vx[d][j]);
      found = __any(found != 0);
    }
    if (lane == 0) reinterpret_cast<uint8_t*>(&nan[buf][part])[mine] = uint8_t(found);
    if (mine == 0 && col == 0) scales[buf][part][grp] = sc;
#pragma unroll
    for (int d = 0; d < DC; ++d) {
      if (found) {
        uint32_t marks = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t n = nan_bytes(vx[d][j]) >> 7;
          marks |= ((n | n >> 7 | n >> 14 | n >> 21) & 15) << (4 * j);
          vx[d][j] &= ~(n * 0xff);
        }
        nan_marks[buf][part][mine + 4 * d][lane] = uint16_t(marks);
      }
      lds.tile[buf][part].v[mine + 4 * d][0][lane] = Wide::widen(vx[d].x, vx[d].y);
      lds.tile[buf][part].v[mine + 4 * d][1][lane] = Wide::widen(vx[d].z, vx[d].w);
    }
  };

  X8 q[NR][2 * DC];
  int pos[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = row0 + 32 * mine + 16 * r + col;
    pos[r] = row < rows ? min(past + row / per, end - 1) : -1;
    load_q<TYPE, DC>(a, b, head, row, rows, grp, q[r]);
  }
  const float to_log2 = fabsf(a.scale) * kLog2e;
  f32x4 o[NR][DT] = {};
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.0f;

  Pages next{};
  if (step0 < step1) {
    load(step0, pages_of(step0));
    next = pages_of(step0 + 1);
    write(step0, step0 & 1);
    load(step0 + 1, next);
    next = pages_of(step0 + 2);
  }
  __syncthreads();
  const auto run = [&](int step, auto masked) {
    constexpr bool MASKED = decltype(masked)::value;  // whether some row does not see some key
    const int buf = step & 1, key_v = (2 * step + part) * kTile + 16 * grp;
    const Tile& t = lds.tile[buf][part];
    f32x4 s[NR][4] = {};
    X8 k8[2][4];
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) k8[0][kt] = t.k[kt][0][lane];
#pragma unroll
    for (int k = 0; k < 2 * DC; ++k) {
      if (k + 1 < 2 * DC) {
#pragma unroll
        for (int kt = 0; kt < 4; ++kt) k8[(k + 1) & 1][kt] = t.k[kt][k + 1][lane];
      }
      in_order();
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int r = 0; r < NR; ++r) s[r][kt] = H::mfma(k8[k & 1][kt], q[r][k], s[r][kt]);
      in_order();
    }
    const Scales now = scales[buf][part][grp];
    if (MASKED) {
#pragma unroll
      for (int r = 0; r < NR; ++r) hide(s[r], now.there, key_v, pos[r]);
    }
    bf16x8 hi[NR][2], lo[NR][2];
    bf16x8 v8[2][4];
#pragma unroll
    for (int d = 0; d < 4; ++d) v8[0][d] = t.v[d][0][lane];
    in_order();
    softmax_step<TYPE, NR, DT, 8>(s, fmaxf(now.ks * to_log2, 1e-30f), now.vs, now.there, m, l, o, hi, lo);
    in_order();
#pragma unroll
    for (int i = 0; i < 2 * DC; ++i) {  // slices 4 (i / 2) to 4 (i / 2) + 3, half i % 2 of their keys
      if (i + 1 < 2 * DC) {
#pragma unroll
        for (int d = 0; d < 4; ++d) v8[(i + 1) & 1][d] = t.v[4 * ((i + 1) >> 1) + d][(i + 1) & 1][lane];
      }
      in_order();
#pragma unroll
      for (int d = 0; d < 4; ++d)
#pragma unroll
        for (int r = 0; r < NR; ++r) {
          f32x4& to = o[r][4 * (i >> 1) + d];
          to = Wide::mfma(v8[i & 1][d], hi[r][i & 1], to);
          if (TYPE == kF16) to = Wide::mfma(v8[i & 1][d], lo[r][i & 1], to);
        }
      in_order();
    }
    const uint32_t bad = MASKED ? __builtin_amdgcn_readfirstlane(nan[buf][part]) : 0;
    if (bad) {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        if (!(bad >> (8 * (d & 3)) & 1)) continue;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t marks = nan_marks[buf][part][d][lane] >> (8 * u);
          bf16x8 is;
#pragma unroll
          for (int e = 0; e < 8; ++e) is[e] = __bf16(marks >> e & 1 ? 1.0f : 0.0f);
#pragma unroll
          for (int r = 0; r < NR; ++r) poison(is, now.there, key_v + 8 * u, pos[r], o[r][d]);
        }
      }
    }
    if (step + 1 < step1) {
      write(step + 1, buf ^ 1);
      load(step + 2, next);
      next = pages_of(step + 3);
    }
    __syncthreads();
  };
  // the steps whose keys all rows see
  const int clean = max(step0, min(step1, min(past + row0 / per + 1, end) / (2 * kTile)));
  int step = step0;
  for (; step < clean; ++step) run(step, std::false_type());
  for (; step < step1; ++step) run(step, std::true_type());

  // waves 4-7 hand their sums to waves 0-3, which hold the same rows
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] = across_groups(l[r], Add());
    const int at = 32 * mine + 16 * r + col;
    if (part == 1) {
      if (grp == 0) m_lds[at] = m[r], l_lds[at] = l[r];
#pragma unroll
      for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(&lds.o[at][16 * d + 4 * grp]) = o[r][d];
    }
  }
  __syncthreads();
  if (part == 1) return;
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int at = 32 * mine + 16 * r + col, row = row0 + at;
    if (row >= rows) continue;
    const float top = fmaxf(m[r], m_lds[at]);
    const float f0 = m[r] == -INFINITY ? 0.0f : exp2_of(m[r] - top);
    const float f1 = m_lds[at] == -INFINITY ? 0.0f : exp2_of(m_lds[at] - top);
    const float sum = l[r] * f0 + l_lds[at] * f1, inv = sum == 0.0f ? 0.0f : kUnit / sum;
    const int64_t out = (int64_t(b) * a.new_tokens + row / per) * a.heads + head * per + row % per;
    const int64_t part_at = out * a.splits + split;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      const f32x4 v = o[r][d] * f0 + *reinterpret_cast<const f32x4*>(&lds.o[at][16 * d + 4 * grp]) * f1;
      if (a.splits == 1)
        store4(static_cast<T*>(a.out) + out * c.dim, v * inv, 16 * d + 4 * grp, c.dim);
      else
        store4(a.part_o + part_at * c.dim, v, 16 * d + 4 * grp, c.dim);
    }
    if (grp == 0) {
      if (a.splits > 1)
        a.part_ml[part_at * 2] = top, a.part_ml[part_at * 2 + 1] = sum;
      else if (a.lse)
        a.lse[out] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    }
  }
}

constexpr int kJoinMost = 128;  // parts of one row

// One wave joins one row's parts: weights 2^(m_s - max m), the sum of the weighted sums below.  A lane holds the
// statistics of parts lane and lane + 64, and the loads of eight parts are in flight together.
template <Type TYPE, int DC>
__global__ __launch_bounds__(64) void kv_join_kernel(AttentionArgs a) {
  using T = typename Scalar<TYPE>::type;
  const int64_t at = blockIdx.x;
  const int lane = threadIdx.x, dim = a.cache.dim, splits = a.splits;
  const float* ml = a.part_ml + at * splits * 2;
  const float* part = a.part_o + at * splits * dim;
  float m[2], l[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = 64 * j + lane;
    m[j] = s < splits ? ml[2 * s] : -INFINITY;
    l[j] = s < splits ? ml[2 * s + 1] : 0.0f;
  }
  const float top = wave_reduce(fmaxf(m[0], m[1]), Max());
#pragma unroll
  for (int j = 0; j < 2; ++j) m[j] = m[j] == -INFINITY ? 0.0f : exp2_of(m[j] - top);  // a part without keys: 0
  const float sum = wave_reduce(l[0] * m[0] + l[1] * m[1], Add());
  float o[DC] = {};
  constexpr int BATCH = 8;  // parts whose loads are in flight together; behind the last one they repeat it
  for (int s0 = 0; s0 < splits; s0 += BATCH) {
    float v[BATCH][DC];
#pragma unroll
    for (int k = 0; k < BATCH; ++k)
#pragma unroll
      for (int j = 0; j < DC; ++j)
        v[k][j] = part[int64_t(min(s0 + k, splits - 1)) * dim + min(64 * j + lane, dim - 1)];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int s = s0 + k;
      const float w = s < splits ? __shfl(s < 64 ? m[0] : m[1], s & 63) : 0.0f;  // a part without keys holds zeros
#pragma unroll
      for (int j = 0; j < DC; ++j) o[j] += s < splits ? w * v[k][j] : 0.0f;
    }
  }
#pragma unroll
  for (int j = 0; j < DC; ++j)
    if (64 * j + lane < dim)
      static_cast<T*>(a.out)[at * dim + 64 * j + lane] = T(sum == 0.0f ? 0.0f : o[j] / sum * kUnit);
  if (lane == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

template <Type TYPE, int DC>
void launch_dim(const AttentionArgs& a, Stream s) {
  const int rows = a.new_tokens * (a.heads / a.cache.heads), tile = a.tile;
  const dim3 grid(unsigned(a.cache.heads * ceil_div(rows, tile)), a.splits, a.batch);
  const bool whole = 1 << a.cache.page_shift >= kTile;
  const char* what = "kv_cache_attention";
  // what one call reads of the cache at most, against the 256 MB of the last cache
  const int64_t pages = std::min(int64_t(a.batch) * a.cache.table_width, a.cache.pages);
  const bool stream = (pages * a.cache.heads * a.cache.wide << (a.cache.page_shift + 1)) > (int64_t(256) << 20);
  if (tile == 16 && stream)
    launch(whole ? kv_attention_kernel<TYPE, DC, 1, true, true> : kv_attention_kernel<TYPE, DC, 1, false, true>, grid,
           kThreads, a, s, what);
  else if (tile == 16)
    launch(whole ? kv_attention_kernel<TYPE, DC, 1, true, false> : kv_attention_kernel<TYPE, DC, 1, false, false>,
           grid, kThreads, a, s, what);
  else if (tile == 32)
    launch(whole ? kv_attention_kernel<TYPE, DC, 2, true, false> : kv_attention_kernel<TYPE, DC, 2, false, false>,
           grid, kThreads, a, s, what);
  else if constexpr (DC == 2)
    launch(whole ? kv_attention_chunk_kernel<TYPE, DC, true> : kv_attention_chunk_kernel<TYPE, DC, false>, grid,
           kChunkThreads, a, s, what);
  if (a.splits > 1)
    launch(kv_join_kernel<TYPE, DC>, dim3(unsigned(a.batch * a.new_tokens * a.heads)), 64, a, s, what);
}

template <Type TYPE>
void launch_type(const AttentionArgs& a, Stream s) {
  switch (a.cache.wide / 64) {
    case 1: return launch_dim<TYPE, 1>(a, s);
    case 2: return launch_dim<TYPE, 2>(a, s);
    case 3: return launch_dim<TYPE, 3>(a, s);
    default: return launch_dim<TYPE, 4>(a, s);
  }
}

}  // namespace

// Rows of a workgroup: 16 where a key head has no more, else 32, or the 128 of the chunk kernel for heads of 65 to 128
// with enough rows and keys to fill the chip.  Its start costs 13 us against 6; measured (us, bf16, 32 heads on 8,
// 128 rows / 32 rows, by groups of 32 rows x keys):
//   8 x 32 tokens, 1024 keys (0.25 M) 27 / 15;   1 x 509, 2048 (1 M) 45 / 43;    4 x 509, 512 (1 M) 41 / 80
//   2 x 509, 4096 (4 M) 88 / 123;                64 x 16, 2048 (2 M, 64 rows) 90 / 88
// and for heads of 64, where a 32-row tile leaves room for two workgroups on a CU, 32 rows were never slower by a
// tenth and up to 1.7 times faster.  Heads of 129 to 256 have no other form for many rows; it fills the registers (at
// 256 wide 63 to 81 go to scratch memory): 2 x 509 tokens on up to 4096 keys take 170 us at 192 wide and 349 at 256.
// Rows and parts come from what the table can hold, since the lengths are the device's: 20 tokens on 777 keys take
// 13.5 us, and 20.3 with a table for 65536.
//
// Parts of the key axis: one workgroup for each of the 256 CUs, and no less than 128 keys (two waves' tiles) for each.
// Measured (us, heads of 128, one new token, 32 on 8 heads):
//   1 x 8192 keys: 1 part 47, 8 13.9, 32 11.3, 64 13.7;      1 x 65536: 1 344, 16 35, 32 29, 64 32
//   4 x 8192: 1 48, 4 21, 8 17, 32 22;                       32 x 8192: 1 82, 4 80, 16 107
void kv_attention_plan(AttentionArgs& a, int64_t longest) {
  const int rows = a.new_tokens * (a.heads / a.cache.heads);
  const int64_t heads = int64_t(a.batch) * a.cache.heads;
  a.tile = rows <= 16 ? 16 : 32;
  if (a.cache.wide == 128 && rows > 64 && heads * ceil_div(rows, 32) * longest >= 1 << 20) a.tile = kChunkRows;
  const int64_t parts = std::min(ceil_div(256, heads * ceil_div(rows, a.tile)), ceil_div(longest, 2 * kTile));
  a.splits = int(std::clamp(parts, int64_t(1), int64_t(kJoinMost)));
}

void kv_attention_hip(const AttentionArgs& a, Stream s) {
  if (a.batch == 0 || a.new_tokens == 0 || a.heads == 0) return;
  if (a.type == kF16) return launch_type<kF16>(a, s);
  launch_type<kBF16>(a, s);
}

}  // namespace tl_ops
