// norm_quant.hip -- residual addition + RMS norm + e4m3 output with scales, one pass over the row.
//
//   h = x + residual;  y_j = h_j w_j / sqrt(mean(h^2) + eps);  s_g = max(max_g |y|, 1e-4) / 448;  q = e4m3(y / s)
//
// Everything between the loads and the stores is float32: h and y are rounded only where they are written, and
// the codes come from the unrounded y.  A row whose squares' sum is beyond float32 has zeros for norms (not-a-number
// where it is infinite).  One workgroup owns a row and keeps it in registers (NV vectors of 8 elements per thread), so
// every input byte is read once.  A vector belongs to one scale group; the lanes that hold a group are neighbours and
// reduce its maximum among themselves.
//
// Bound by HBM: 7 bytes an element with a residual in 16 bits.  8192 x 7168 bf16: 79 us, 5.2 TB/s.  (Times here and
// in the other kernels' files are of calls one behind the other, each with other inputs.)
#include "device.h"

namespace tl_ops {
namespace {

template <typename T>
__device__ inline void load8(const T* p, bool whole, int n, float (&v)[8]) {
  if (whole) {
    typedef T V __attribute__((ext_vector_type(8)));
    const V r = *reinterpret_cast<const V*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = float(r[j]);
  } else {
    load8_anywhere(p, n, v);
  }
}

template <typename T>
__device__ inline void store8(T* p, bool whole, int n, const float (&v)[8]) {
  if (whole) {
    typedef T V __attribute__((ext_vector_type(8)));
    V r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = T(v[j]);
    *reinterpret_cast<V*>(p) = r;
  } else if (n >= 8) {
    T r[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = T(v[j]);
    __builtin_memcpy(p, r, sizeof(r));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = T(v[j]);
  }
}

// WHOLE: the rows are vectors of 8 elements on 16-byte boundaries; else they begin and end anywhere.
template <Type TYPE, int THREADS, int NV, bool WHOLE>
__global__ __launch_bounds__(THREADS) void norm_quant_kernel(NormQuantArgs a) {
  using T = typename Scalar<TYPE>::type;
  __shared__ float lds[2][THREADS / 64];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, width = a.width;
  const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
  const T* res = static_cast<const T*>(a.residual) + row * a.residual_stride;
  const T* w = static_cast<const T*>(a.weight);
  float v[NV][8];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * THREADS + tid) * 8, n = width - at;
    if (n > 0) {
      load8(x + at, WHOLE, n, v[i]);
      if (a.residual) {
        float r[8];
        load8(res + at, WHOLE, n, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] += r[j];
      }
      if (a.h) store8(static_cast<T*>(a.h) + row * width + at, WHOLE, n, v[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
  }
  ss = block_reduce<THREADS>(ss, lds[0], Add());
  const float r = 1.0f / sqrtf(ss / float(width) + a.eps);
  float amax[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * THREADS + tid) * 8, n = width - at;
    amax[i] = 0.0f;
    if (n > 0) {
      float g[8];
      load8(w + at, WHOLE, n, g);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        v[i][j] *= r * g[j];
        amax[i] = fmaxf(amax[i], fabsf(v[i][j]));
      }
      if (a.y) store8(static_cast<T*>(a.y) + row * width + at, WHOLE, n, v[i]);
    }
  }
  const bool per_row = a.group == width;
  if (per_row) {
    float m = amax[0];
#pragma unroll
    for (int i = 1; i < NV; ++i) m = fmaxf(m, amax[i]);
    m = block_reduce<THREADS>(m, lds[1], Max());
#pragma unroll
    for (int i = 0; i < NV; ++i) amax[i] = m;
  } else {
    for (int m = 1; m < a.group / 8; m <<= 1) {
#pragma unroll
      for (int i = 0; i < NV; ++i) amax[i] = fmaxf(amax[i], __shfl_xor(amax[i], m));
    }
  }
  const int groups = width / a.group;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int at = (i * THREADS + tid) * 8, n = width - at;
    if (n <= 0) continue;
    const float m = fmaxf(amax[i], kAmaxFloor);
    const float s = a.pow2 ? pow2_scale(m) : m / kFp8Max;
    if (at % a.group == 0) a.scale[row * groups + at / a.group] = s;
    // y / s as IEEE division rounds it, by two corrections of y r with r = 1 / s (Markstein: where r is the rounded
    // reciprocal and q within one last place, q + (y - q s) r rounds to the quotient; what underflows in it has the
    // code 0).  A product with 448 / m puts 0.1 % of the codes of 16-bit rows on the other side of a tie; 8192 x 7168
    // take 78.5 us with it, 78.9 with this and 82.0 with the compiler's division.  |y| / s rounds to 448 at most.
    const float r = 1.0f / s, d = s < INFINITY ? s : 0.0f;  // infinite: finite values become 0, others not-a-number
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float y = v[i][j];
      float q = y * r;
      q = fmaf(fmaf(-q, d, y), r, q);
      q = fmaf(fmaf(-q, d, y), r, q);
      v[i][j] = copysignf(q, y);
    }
    u32x2 c;
    c.x = pack_fp8(v[i][0], v[i][1], v[i][2], v[i][3]);
    c.y = pack_fp8(v[i][4], v[i][5], v[i][6], v[i][7]);
    uint8_t* q = a.q + row * width + at;
    if (WHOLE) {
      *reinterpret_cast<u32x2*>(q) = c;
    } else if (n >= 8) {
      __builtin_memcpy(q, &c, 8);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) q[j] = uint8_t((j < 4 ? c.x : c.y) >> (8 * (j & 3)));
    }
  }
}

// A launch has fewer than 2^32 threads: more rows than kLaunchRows take another.
constexpr int64_t kLaunchRows = 1 << 21;

template <Type TYPE, int THREADS, int NV>
void launch_rows(const NormQuantArgs& a, bool whole, Stream s) {
  using T = typename Scalar<TYPE>::type;
  for (int64_t row = 0; row < a.rows; row += kLaunchRows) {
    NormQuantArgs part = a;
    part.rows = a.rows - row < kLaunchRows ? a.rows - row : kLaunchRows;
    part.x = static_cast<const T*>(a.x) + row * a.x_stride;
    if (a.residual) part.residual = static_cast<const T*>(a.residual) + row * a.residual_stride;
    part.q = a.q + row * a.width;
    part.scale = a.scale + row * (a.width / a.group);
    if (a.h) part.h = static_cast<T*>(a.h) + row * a.width;
    if (a.y) part.y = static_cast<T*>(a.y) + row * a.width;
    launch(whole ? norm_quant_kernel<TYPE, THREADS, NV, true> : norm_quant_kernel<TYPE, THREADS, NV, false>,
           dim3(unsigned(part.rows)), THREADS, part, s, "add_rms_norm_quant");
  }
}

template <Type TYPE>
void launch_type(const NormQuantArgs& a, Stream s) {
  const size_t bytes = sizeof(typename Scalar<TYPE>::type);
  const auto on16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool whole = a.width % 8 == 0 && on16(a.x) && on16(a.residual) && on16(a.weight) &&
                     a.x_stride * bytes % 16 == 0 && a.residual_stride * bytes % 16 == 0;
  // Few vectors to a thread keep rows in flight; 7168 wide, 8192 rows: 512 threads by 2 79.2 us, 256 by 4 85.6, 1024
  // by 1 85.1; 64 rows: 5.7, 6.8, 6.0.
  const int vectors = int(ceil_div(a.width, 8));
  if (vectors <= 64) return launch_rows<TYPE, 64, 1>(a, whole, s);
  if (vectors <= 256) return launch_rows<TYPE, 256, 1>(a, whole, s);
  if (vectors <= 512) return launch_rows<TYPE, 256, 2>(a, whole, s);
  if (vectors <= 1024) return launch_rows<TYPE, 512, 2>(a, whole, s);
  if (vectors <= 2048) return launch_rows<TYPE, 512, 4>(a, whole, s);
  launch_rows<TYPE, 1024, 8>(a, whole, s);
}

}  // namespace

void norm_quant_hip(const NormQuantArgs& a, Stream s) {
  if (a.rows == 0) return;
  if (a.type == kF32) return launch_type<kF32>(a, s);
  if (a.type == kF16) return launch_type<kF16>(a, s);
  launch_type<kBF16>(a, s);
}

}  // namespace tl_ops
