// RMS norm whose output is in 8 bits, with the residual's addition before it, in one pass:
//     h <- h + y (rounded to h's type; where y is given)
//     n = h rsqrt(mean h^2 + eps) w                      (norm 0: n = h, the quantiser)
//     a = max(max |n|, 2^-100),  scale = a / 448,  q = n (448 / a) rounded to e4m3
// n stays in fp32 until it is rounded to 8 bits (and to h's type, where n is asked for as well).
// 2^-100 keeps 448 / a finite; a row of zeros gives zeros.  A NaN or infinity in a row makes its
// scale NaN or leaves NaN in its place, as in torch.
//
// Bound: bytes (7 a value with the residual in 16 bits).  A row stays in the registers of its
// group of threads: a warp for up to 1024 values, 128, 512 or 1024 threads beyond, 32 values a
// thread; two reductions (squares, then magnitudes) by shuffles and, above a warp, one exchange
// through shared memory each.  Rows of a width that is no multiple of 8, or not 16-byte aligned,
// are read value by value, neighbouring threads at neighbouring places.
#include "common.cuh"

#include <cuda_fp8.h>

namespace verace {
namespace {

__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct NormArgs {
  const void *h, *y, *w;
  void *sum, *n;
  uint8_t* q;
  float* scale;
  long long rows;
  int cols, norm;
  float eps;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float* x) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    unpack8<T>(*reinterpret_cast<const uint4*>(p), x);
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* x) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4*>(p) = pack8<T>(x);
  }
}
template <typename T>
__device__ __forceinline__ float rounded(float x) {
  return to_f32(from_f32<T>(x));
}

// A group of G threads holds a row of up to 32 G values: VEC (8 or 1) neighbouring ones at VEC (g + G i).
template <typename T, int G, int VEC>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_fp8_kernel(NormArgs a) {
  constexpr int NT = G < 128 ? 128 : G, NV = 32 / VEC, W = G / 32;
  __shared__ float part[2][W > 1 ? W : 1];
  const int g = threadIdx.x % G;
  const long long row = (long long)blockIdx.x * (NT / G) + threadIdx.x / G;
  if (G < 128 && row >= a.rows) return;   // (whole warps; larger groups are one row a CTA)
  const long long off = row * a.cols;
  const T* h = static_cast<const T*>(a.h) + off;
  const T* y = a.y ? static_cast<const T*>(a.y) + off : nullptr;
  const T* w = static_cast<const T*>(a.w);
  float v[NV][VEC];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = VEC * (g + G * i);
    if (c < a.cols) {
      if constexpr (VEC == 8) load8<T>(h + c, v[i]);
      else v[i][0] = to_f32(h[c]);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
    }
  }
  if (y) {
    T* sum = static_cast<T*>(a.sum) + off;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = VEC * (g + G * i);
      if (c < a.cols) {
        if constexpr (VEC == 8) {
          float t[8];
          load8<T>(y + c, t);
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = rounded<T>(v[i][j] + t[j]);
          store8<T>(sum + c, v[i]);
        } else {
          v[i][0] = rounded<T>(v[i][0] + to_f32(y[c]));
          sum[c] = from_f32<T>(v[i][0]);
        }
      }
    }
  }
  if (a.norm) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VEC; ++j) ss = fmaf(v[i][j], v[i][j], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (W > 1) {
      if (g % 32 == 0) part[0][g / 32] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) ss += part[0][i];
    }
    const float rs = rsqrtf(ss / (float)a.cols + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = VEC * (g + G * i);
      if (c < a.cols) {
        float t[VEC];
        if (w) {
          if constexpr (VEC == 8) load8<T>(w + c, t);
          else t[0] = to_f32(w[c]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = w ? v[i][j] * rs * t[j] : v[i][j] * rs;
      }
    }
  }
  float top = 0x1p-100f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VEC; ++j) top = max_nan(top, fabsf(v[i][j]));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if constexpr (W > 1) {
    if (g % 32 == 0) part[1][g / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max_nan(top, part[1][i]);
  }
  const float inv = 448.f / top;
  if (g == 0) a.scale[row] = top / 448.f;
  uint8_t* q = a.q + off;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = VEC * (g + G * i);
    if (c < a.cols) {
      if constexpr (VEC == 8) {
        uint32_t o[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[i][4 * j] * inv, v[i][4 * j + 1] * inv),
                                                       __NV_SATFINITE, __NV_E4M3);
          const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[i][4 * j + 2] * inv, v[i][4 * j + 3] * inv),
                                                       __NV_SATFINITE, __NV_E4M3);
          o[j] = lo | hi << 16;
        }
        *reinterpret_cast<uint2*>(q + c) = make_uint2(o[0], o[1]);
        if (a.n) store8<T>(static_cast<T*>(a.n) + off + c, v[i]);
      } else {
        q[c] = __nv_cvt_float_to_fp8(v[i][0] * inv, __NV_SATFINITE, __NV_E4M3);
        if (a.n) static_cast<T*>(a.n)[off + c] = from_f32<T>(v[i][0]);
      }
    }
  }
}

template <typename T, int VEC>
int launch(const NormArgs& a, cudaStream_t st) {
  if (a.cols <= 1024) norm_fp8_kernel<T, 32, VEC><<<(unsigned)((a.rows + 3) / 4), 128, 0, st>>>(a);
  else if (a.cols <= 4096) norm_fp8_kernel<T, 128, VEC><<<(unsigned)a.rows, 128, 0, st>>>(a);
  else if (a.cols <= 16384) norm_fp8_kernel<T, 512, VEC><<<(unsigned)a.rows, 512, 0, st>>>(a);
  else norm_fp8_kernel<T, 1024, VEC><<<(unsigned)a.rows, 1024, 0, st>>>(a);
  return check_launch("norm_fp8_kernel");
}

template <typename T>
int launch(const NormArgs& a, cudaStream_t st) {
  const size_t all = (size_t)a.h | (size_t)a.y | (size_t)a.w | (size_t)a.sum | (size_t)a.n;
  return a.cols % 8 == 0 && all % 16 == 0 && (size_t)a.q % 8 == 0 ? launch<T, 8>(a, st) : launch<T, 1>(a, st);
}

}  // namespace
}  // namespace verace

using namespace verace;

extern "C" int verace_rmsnorm_fp8(const void* h, const void* y, void* sum, const void* weight, float eps, int norm,
                                  void* q, float* scale, void* n, long long rows, int cols, int dtype, void* stream) {
  VERACE_REQUIRE(rows >= 0 && cols >= 1, VERACE_ERR_INVALID, "verace_rmsnorm_fp8: invalid sizes rows=%lld cols=%d", rows,
                 cols);
  VERACE_REQUIRE(dtype == VERACE_F32 || dtype == VERACE_BF16 || dtype == VERACE_F16, VERACE_ERR_INVALID,
                 "verace_rmsnorm_fp8: dtype %d", dtype);
  VERACE_REQUIRE(cols <= 32768 && rows < 1LL << 31, VERACE_ERR_UNSUPPORTED,
                 "verace_rmsnorm_fp8: rows %lld, cols %d unsupported (at most 32768 columns)", rows, cols);
  if (rows == 0) return VERACE_OK;
  VERACE_REQUIRE(h && q && scale && (y == nullptr) == (sum == nullptr), VERACE_ERR_INVALID,
                 "verace_rmsnorm_fp8: NULL pointer, or one of y and sum without the other");
  const NormArgs a{h, y, weight, sum, n, static_cast<uint8_t*>(q), scale, rows, cols, norm, eps};
  cudaStream_t st = (cudaStream_t)stream;
  switch (dtype) {
    case VERACE_F32: return launch<float>(a, st);
    case VERACE_BF16: return launch<__nv_bfloat16>(a, st);
    default: return launch<__half>(a, st);
  }
}
