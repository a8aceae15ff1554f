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
// range only bf16 has); for fp16 the rounding's rest goes through a second product, which keeps the error that of
// the output's own rounding.
//
// The waves of a workgroup take tiles in turn and join in LDS; `splits` workgroups share a long key axis and
// kv_join_kernel joins them.
#include "device.h"

namespace tl_ops {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kTile = 64;  // keys of one wave's step
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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

__device__ inline float across_groups_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float across_groups_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// e4m3 bytes that are not-a-number (0x7f, 0xff): bit 7 of each such byte
__device__ inline uint32_t nan_bytes(uint32_t x) { return ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// the first n bytes of four
__device__ inline uint32_t first_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1u; }

// The keys of one tile: where this lane's K rows and V columns begin, and its 16 keys' scales.
struct Place {
  const uint8_t *k, *v;
  float ks, vs;
  bool there;  // whether the page of its 16 keys is in the pool
};

template <Type TYPE, int DC, int NR>
__global__ __launch_bounds__(kThreads) void kv_attention_kernel(AttentionArgs a) {
  using T = typename Scalar<TYPE>::type;
  constexpr int ROWS = 16 * NR, DT = 4 * DC;  // rows of the workgroup, 16-wide slices of the head
  using H = Half<TYPE>;
  using X8 = typename H::X8;
  constexpr int PASSES = NR > 2 ? 2 : 1;  // the waves join in so many passes over the head
  constexpr int PITCH = DC * 64 / PASSES + 4;
  __shared__ float o_lds[kWaves][ROWS][PITCH];
  __shared__ float m_lds[kWaves][ROWS], l_lds[kWaves][ROWS];

  const Cache& c = a.cache;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
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
  const int64_t head_bytes = int64_t(page) * c.wide;
  const auto place_of = [&](int tile) {
    // a group of keys behind the end reads the last page
    const auto page_of = [&](int key, bool& there) {
      const int id = table[(key < end ? key : end - 1) >> c.page_shift];
      there = id >= 0 && id < c.pages;
      return (there ? int64_t(id) : int64_t(0)) * c.heads + head;
    };
    Place p;
    const int key_k = tile * kTile + 16 * (col >> 2), key_v = tile * kTile + 16 * grp;
    const int64_t page_k = page_of(key_k, p.there), page_v = page_of(key_v, p.there);
    p.k = c.k + page_k * head_bytes + int64_t((key_k & (page - 1)) + (col & 3)) * c.wide + 16 * grp;
    p.v = c.v + page_v * head_bytes + int64_t(col) * page + (key_v & (page - 1));
    p.ks = c.k_scale[page_v];
    p.vs = c.v_scale[page_v];
    return p;
  };
  u32x4 kx[4][DC], vx[DT];
  const auto load_k = [&](const Place& p) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < DC; ++k) kx[t][k] = *reinterpret_cast<const u32x4*>(p.k + 4 * t * c.wide + 64 * k);
  };
  Place at;
  if (tile0 < tile1) {
    at = place_of(tile0);
    load_k(at);
  }

  X8 q[NR][2 * DC];
  int pos[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = row0 + 16 * r + col, i = row / per, h = head * per + row % per;
    pos[r] = row < rows ? min(past + i, end - 1) : -1;
    const T* p = static_cast<const T*>(a.q) + b * a.stride_b + i * a.stride_t + h * a.stride_h;
    const bool whole = row < rows && c.dim == c.wide && reinterpret_cast<uintptr_t>(p) % 16 == 0;
#pragma unroll
    for (int k = 0; k < 2 * DC; ++k) {
      const int d = 64 * (k >> 1) + 16 * grp + 8 * (k & 1);
      if (whole) {
        q[r][k] = *reinterpret_cast<const X8*>(p + d);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[r][k][j] = row < rows && d + j < c.dim ? p[d + j] : T(0.0f);
      }
      // the scores' scale may be negative; its sign goes here, so that the largest product is the largest score
      if (a.scale < 0.0f) q[r][k] = -q[r][k];
    }
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
    for (int d = 0; d < DT; ++d) vx[d] = *reinterpret_cast<const u32x4*>(now.v + 16 * d * page);
    const bool more = tile + kWaves < tile1;
    if (more) at = place_of(tile + kWaves);

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
    if (more) load_k(at);

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
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!now.there || key_v + 4 * t + i > pos[r]) s[r][t][i] = -INFINITY;
      if (__any(found != 0)) {
        // a row that sees a not-a-number becomes one, a row that does not stays as it is: count the seen ones
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          uint32_t bad[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            bad[j] = nan_bytes(vx[d][j]) >> 7;  // 1 where not-a-number
            vx[d][j] &= ~(bad[j] * 0xff);
          }
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            f32x4 count = {};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              bf16x8 seen;
#pragma unroll
              for (int e = 0; e < 8; ++e) seen[e] = __bf16(now.there && key_v + 8 * u + e <= pos[r] ? 1.0f : 0.0f);
              count = Wide::mfma(Wide::widen(bad[2 * u] * 0x38, bad[2 * u + 1] * 0x38), seen, count);  // 0x38: 1.0
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) o[r][d][i] = count[i] > 0.0f ? NAN : o[r][d][i];
          }
        }
      }
    }

    const float vs = now.there ? now.vs : 0.0f;
    bf16x8 hi[NR][2], lo[NR][2];
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      const float ks = fmaxf(now.ks * to_log2, 1e-30f);  // never zero: a hidden score stays -inf
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = fmaxf(top, s[r][t][i]);
      top = across_groups_max(top * ks);
      // The sums are relative to m.  It moves only when the scores outgrow it by more than 2^8: weights up to
      // 2^8 lose nothing in bf16 and float32.
      if (__any(top > m[r] + 8.0f)) {
        const float next = fmaxf(m[r], top), alpha = next == -INFINITY ? 1.0f : exp2_of(m[r] - next);
        m[r] = next;
        l[r] *= alpha;
#pragma unroll
        for (int d = 0; d < DT; ++d) o[r][d] *= alpha;
      }
      const float base = m[r] == -INFINITY ? 0.0f : m[r];
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = exp2_of(fmaf(s[r][t][i], ks, -base));
          sum += p;
          const float w = p * vs;
          hi[r][t >> 1][4 * (t & 1) + i] = __bf16(w);
          if (TYPE == kF16) lo[r][t >> 1][4 * (t & 1) + i] = __bf16(w - float(__bf16(w)));
        }
      l[r] += sum;
    }
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
    l[r] = across_groups_sum(l[r]);
    if (grp == 0) m_lds[wave][16 * r + col] = m[r], l_lds[wave][16 * r + col] = l[r];
  }
  constexpr int WIDTH = DC * 64 / PASSES;
  const int here = rows - row0 < ROWS ? rows - row0 : ROWS;
#pragma unroll
  for (int pass = 0; pass < PASSES; ++pass) {
    if (pass) __syncthreads();
#pragma unroll
    for (int r = 0; r < NR; ++r)
#pragma unroll
      for (int d = 0; d < DT / PASSES; ++d)
        *reinterpret_cast<f32x4*>(&o_lds[wave][16 * r + col][16 * d + 4 * grp]) = o[r][pass * (DT / PASSES) + d];
    __syncthreads();
    for (int i = threadIdx.x; i < here * (WIDTH / 4); i += kThreads) {
      const int r = i / (WIDTH / 4), d4 = i % (WIDTH / 4) * 4, d0 = pass * WIDTH + d4, row = row0 + r;
      float top = m_lds[0][r], sum = 0.0f;
#pragma unroll
      for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w][r]);
      f32x4 v = {};
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        const float f = m_lds[w][r] == -INFINITY ? 0.0f : exp2_of(m_lds[w][r] - top);
        sum += l_lds[w][r] * f;
        v += *reinterpret_cast<const f32x4*>(&o_lds[w][r][d4]) * f;
      }
      const int64_t out = (int64_t(b) * a.new_tokens + row / per) * a.heads + head * per + row % per;
      if (a.splits == 1) {
        const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d0 + j < c.dim) static_cast<T*>(a.out)[out * c.dim + d0 + j] = T(v[j] * inv);
        if (d0 == 0 && a.lse) a.lse[out] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
      } else {
        const int64_t part = out * a.splits + split;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d0 + j < c.dim) a.part_o[part * c.dim + d0 + j] = v[j];
        if (d0 == 0) a.part_ml[part * 2] = top, a.part_ml[part * 2 + 1] = sum;
      }
    }
  }
}

// One wave joins one row's parts: weights 2^(m_s - max m), the sum of the weighted sums below.
template <Type TYPE>
__global__ __launch_bounds__(64) void kv_join_kernel(AttentionArgs a) {
  using T = typename Scalar<TYPE>::type;
  const int64_t at = blockIdx.x;
  const int lane = threadIdx.x, dim = a.cache.dim;
  const float* ml = a.part_ml + at * a.splits * 2;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[2 * s]);
  float sum = 0.0f, o[4] = {};
  for (int s = 0; s < a.splits; ++s) {
    if (ml[2 * s + 1] == 0.0f) continue;  // it had no keys
    const float w = exp2_of(ml[2 * s] - (top == -INFINITY ? 0.0f : top));
    sum += ml[2 * s + 1] * w;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (64 * j + lane < dim) o[j] += w * a.part_o[(at * a.splits + s) * dim + 64 * j + lane];
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (64 * j + lane < dim)
      static_cast<T*>(a.out)[at * dim + 64 * j + lane] = T(sum == 0.0f ? 0.0f : o[j] / sum);
  if (lane == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
}

template <Type TYPE, int DC, int NR>
void launch_rows(const AttentionArgs& a, Stream s) {
  const int rows = a.new_tokens * (a.heads / a.cache.heads);
  const dim3 grid(unsigned(a.cache.heads * ceil_div(rows, 16 * NR)), a.splits, a.batch);
  launch(kv_attention_kernel<TYPE, DC, NR>, grid, kThreads, a, s, "kv_cache_attention");
  if (a.splits > 1)
    launch(kv_join_kernel<TYPE>, dim3(unsigned(a.batch * a.new_tokens * a.heads)), 64, a, s, "kv_cache_attention");
}

// Rows that a workgroup takes: as few 16-row tiles as hold a key head's rows, up to what the registers hold.
template <Type TYPE, int DC>
void launch_dim(const AttentionArgs& a, Stream s) {
  const int rows = a.new_tokens * (a.heads / a.cache.heads);
  if (rows <= 16) return launch_rows<TYPE, DC, 1>(a, s);
  if (rows <= 32 || DC > 2) return launch_rows<TYPE, DC, 2>(a, s);
  if constexpr (DC <= 2) launch_rows<TYPE, DC, 4>(a, s);
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

int kv_attention_splits(int batch, int new_tokens, int heads, int kv_heads, int wide, int64_t longest) {
  const int rows = new_tokens * (heads / kv_heads), tile = rows <= 16 ? 16 : rows <= 32 || wide > 128 ? 32 : 64;
  const int64_t groups = int64_t(batch) * kv_heads * ceil_div(rows, tile);
  const int64_t most = ceil_div(longest, kTile * kWaves);  // a tile for every wave
  int64_t want = ceil_div(1024, groups);
  if (want > most) want = most;
  return int(want < 1 ? 1 : want > 128 ? 128 : want);
}

void kv_attention_hip(const AttentionArgs& a, Stream s) {
  if (a.batch == 0 || a.new_tokens == 0 || a.heads == 0) return;
  if (a.type == kF16) return launch_type<kF16>(a, s);
  launch_type<kBF16>(a, s);
}

}  // namespace tl_ops
