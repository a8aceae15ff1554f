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

template <Type TYPE, int DC, int NR>
__global__ __launch_bounds__(kThreads) void kv_attention_kernel(AttentionArgs a) {
  using T = typename Scalar<TYPE>::type;
  using H = Half<TYPE>;
  using X8 = typename H::X8;
  constexpr int ROWS = 16 * NR, DT = 4 * DC;  // rows of the workgroup, 16-wide slices of the head
  __shared__ float o_lds[ROWS][DC * 64 + 4];
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

  X8 q[NR][2 * DC];
  int pos[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    const int row = row0 + 16 * r + col, i = row / per, h = head * per + row % per;
    pos[r] = row < rows ? min(past + i, end - 1) : -1;
    const T* p = static_cast<const T*>(a.q) + b * a.stride_b + i * a.stride_t + h * a.stride_h;
#pragma unroll
    for (int k = 0; k < 2 * DC; ++k)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = 64 * (k >> 1) + 16 * grp + 8 * (k & 1) + j;
        q[r][k][j] = row < rows && d < c.dim ? p[d] : T(0.0f);
      }
  }
  f32x4 o[NR][DT] = {};
  float m[NR], l[NR];
#pragma unroll
  for (int r = 0; r < NR; ++r) m[r] = -INFINITY, l[r] = 0.0f;

  const int tiles = end > 0 ? (end + kTile - 1) / kTile : 0;
  const int tile1 = int(int64_t(tiles) * (split + 1) / a.splits);
  const int* table = c.table + b * c.table_stride;
  const int64_t head_bytes = int64_t(page) * c.wide;
  const float to_log2 = a.scale * kLog2e;

  for (int tile = int(int64_t(tiles) * split / a.splits) + wave; tile < tile1; tile += kWaves) {
    const int key0 = tile * kTile;
    // the pages of the lane's K row and of its 16 keys; a group of keys behind the end reads the last page
    const auto page_of = [&](int key, bool& there) {
      const int id = table[(key < end ? key : end - 1) >> c.page_shift];
      there = id >= 0 && id < c.pages;
      return there ? int64_t(id) : int64_t(0);
    };
    bool there;
    const int key_k = key0 + 16 * (col >> 2), key_v = key0 + 16 * grp;
    const int64_t page_k = page_of(key_k, there) * c.heads + head;
    const int64_t page_v = page_of(key_v, there) * c.heads + head;
    const uint8_t* kp = c.k + page_k * head_bytes + int64_t((key_k & (page - 1)) + (col & 3)) * c.wide + 16 * grp;
    const uint8_t* vp = c.v + page_v * head_bytes + int64_t(col) * page + (key_v & (page - 1));
    const float ks = c.k_scale[page_v] * to_log2, vs = c.v_scale[page_v];
    u32x4 kx[4][DC], vx[DT];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int k = 0; k < DC; ++k) kx[t][k] = *reinterpret_cast<const u32x4*>(kp + 4 * t * c.wide + 64 * k);
#pragma unroll
    for (int d = 0; d < DT; ++d) vx[d] = *reinterpret_cast<const u32x4*>(vp + 16 * d * page);

    // what the slots behind the sequence hold must not reach the product, not even times zero
    if (key0 + kTile > end || !there) {
      const int n = there ? end - key_v : 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) vx[d][j] &= first_bytes(n - 4 * j);
    }
    const bool diagonal = key0 + kTile > past + row0 / per + 1;  // some row does not see some key
    bool bad = false;
    if (diagonal) {
      uint32_t found = 0;
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) found |= nan_bytes(vx[d][j]);
      bad = __any(found != 0);
    }

#pragma unroll
    for (int r = 0; r < NR; ++r) {
      f32x4 s[4] = {};
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < DC; ++k) {
          s[t] = H::mfma(H::widen(kx[t][k].x, kx[t][k].y), q[r][2 * k], s[t]);
          s[t] = H::mfma(H::widen(kx[t][k].z, kx[t][k].w), q[r][2 * k + 1], s[t]);
        }
      float top = -INFINITY;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool seen = there && key_v + 4 * t + i <= pos[r];
          s[t][i] = seen ? s[t][i] * ks : -INFINITY;
          top = fmaxf(top, s[t][i]);
        }
      top = fmaxf(m[r], across_groups_max(top));
      const float base = top == -INFINITY ? 0.0f : top;
      const float alpha = exp2f(m[r] - base);
      m[r] = top;
      float sum = 0.0f;
      bf16x8 hi[2], lo[2];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = exp2f(s[t][i] - base);
          sum += p;
          const float w = there ? p * vs : 0.0f;
          hi[t >> 1][4 * (t & 1) + i] = __bf16(w);
          if (TYPE == kF16) lo[t >> 1][4 * (t & 1) + i] = __bf16(w - float(__bf16(w)));
        }
      l[r] = l[r] * alpha + sum;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        o[r][d] *= alpha;
        u32x4 x = vx[d];
        if (bad) {
          // a row that sees a not-a-number becomes one, a row that does not stays as it is: count the seen ones
          bf16x8 seen[2];
          f32x4 count = {};
#pragma unroll
          for (int e = 0; e < 16; ++e) seen[e >> 3][e & 7] = __bf16(there && key_v + e <= pos[r] ? 1.0f : 0.0f);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t n0 = nan_bytes(x[2 * u]) >> 7, n1 = nan_bytes(x[2 * u + 1]) >> 7;  // 1 where not-a-number
            const bf16x8 is = Half<kBF16>::widen(n0 * 0x38, n1 * 0x38);                       // 0x38: 1.0
            count = Half<kBF16>::mfma(is, seen[u], count);
            x[2 * u] &= ~(n0 * 0xff);
            x[2 * u + 1] &= ~(n1 * 0xff);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) o[r][d][i] = count[i] > 0.0f ? NAN : o[r][d][i];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const bf16x8 v8 = Half<kBF16>::widen(x[2 * u], x[2 * u + 1]);
          o[r][d] = Half<kBF16>::mfma(v8, hi[u], o[r][d]);
          if (TYPE == kF16) o[r][d] = Half<kBF16>::mfma(v8, lo[u], o[r][d]);
        }
      }
    }
  }

  // join the waves: the largest maximum, then the sums relative to it, one wave after the other
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    l[r] = across_groups_sum(l[r]);
    if (grp == 0) m_lds[wave][16 * r + col] = m[r], l_lds[wave][16 * r + col] = l[r];
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < NR; ++r) {
    float top = m_lds[0][16 * r + col];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w][16 * r + col]);
    const float f = exp2f(m[r] - (top == -INFINITY ? 0.0f : top));
#pragma unroll
    for (int d = 0; d < DT; ++d) o[r][d] *= f;
  }
  for (int w = 0; w < kWaves; ++w) {
    if (wave == w) {
#pragma unroll
      for (int r = 0; r < NR; ++r)
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          f32x4* p = reinterpret_cast<f32x4*>(&o_lds[16 * r + col][16 * d + 4 * grp]);
          *p = w == 0 ? o[r][d] : *p + o[r][d];
        }
    }
    __syncthreads();
  }

  for (int i = threadIdx.x; i < ROWS * c.dim; i += kThreads) {
    const int r = i / c.dim, d = i - r * c.dim, row = row0 + r;
    if (row >= rows) break;
    float top = m_lds[0][r], sum = 0.0f;
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_lds[w][r]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) sum += l_lds[w][r] * exp2f(m_lds[w][r] - (top == -INFINITY ? 0.0f : top));
    const int64_t at = (int64_t(b) * a.new_tokens + row / per) * a.heads + head * per + row % per;
    if (a.splits == 1) {
      static_cast<T*>(a.out)[at * c.dim + d] = T(sum == 0.0f ? 0.0f : o_lds[r][d] / sum);
      if (d == 0 && a.lse) a.lse[at] = sum == 0.0f ? -INFINITY : (top + log2f(sum)) * kLn2;
    } else {
      a.part_o[(at * a.splits + split) * c.dim + d] = o_lds[r][d];
      if (d == 0) a.part_ml[(at * a.splits + split) * 2] = top, a.part_ml[(at * a.splits + split) * 2 + 1] = sum;
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
    const float w = exp2f(ml[2 * s] - (top == -INFINITY ? 0.0f : top));
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
