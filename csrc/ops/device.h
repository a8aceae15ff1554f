// device.h -- what the kernels of the serving operators share: types, conversions, wave reductions, launches.
#pragma once

#include <hip/hip_runtime.h>

#include <sstream>
#include <stdexcept>

#include "ops.h"

namespace tl_ops {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr float kFp8Max = 448.0f;    // largest e4m3 value
constexpr float kAmaxFloor = 1e-4f;  // below it a group of values is scaled as if it held this one

template <Type> struct Scalar;
template <> struct Scalar<kF32> { using type = float; };
template <> struct Scalar<kF16> { using type = _Float16; };
template <> struct Scalar<kBF16> { using type = __bf16; };

// The smallest power of two that is no smaller than amax / 448, from the bits: 448 = 1.75 * 2^8.
__device__ inline float pow2_scale(float amax) {
  const uint32_t bits = __float_as_uint(amax);
  const int e = int(bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
  return __uint_as_float(uint32_t(e < 1 ? 1 : e) << 23);
}

// Four values as e4m3, rounded to nearest even.  |x| <= 464 (or not-a-number, which stays one).
__device__ inline uint32_t pack_fp8(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true));
}

// Eight elements that begin anywhere, as one load for 16-bit types (the memory takes any alignment), or the n that
// there are and zeros.
template <typename T>
__device__ inline void load8_anywhere(const T* p, int n, float (&v)[8]) {
  if (n >= 8) {
    T r[8];
    __builtin_memcpy(r, p, sizeof(r));
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = float(r[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = j < n ? float(p[j]) : 0.0f;
  }
}

template <typename F>
__device__ inline float wave_reduce(float v, F f) {
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) v = f(v, __shfl_xor(v, m));
  return v;
}

struct Add {
  __device__ float operator()(float a, float b) const { return a + b; }
};
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};

// The reduction of `v` over a workgroup of THREADS; `lds` holds THREADS / 64 floats and is free afterwards
// only behind another barrier.
template <int THREADS, typename F>
__device__ inline float block_reduce(float v, float* lds, F f) {
  v = wave_reduce(v, f);
  if constexpr (THREADS > 64) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = lds[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) v = f(v, lds[w]);
  }
  return v;
}

template <typename Args>
inline void launch(void (*kernel)(Args), dim3 grid, int threads, const Args& args, Stream stream, const char* what) {
  void* p[] = {const_cast<Args*>(&args)};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), p, 0, stream);
  if (e != hipSuccess) {
    std::ostringstream os;
    os << "HIP error " << hipGetErrorName(e) << " (" << hipGetErrorString(e) << ") at " << what;
    throw std::runtime_error(os.str());
  }
}

}  // namespace tl_ops
