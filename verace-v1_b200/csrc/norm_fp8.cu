// RMS norm whose output is in 8 bits, with the residual's addition before it, in one pass:
//     h <- h + y (rounded to h's type; where y is given)
//     n = h rsqrt(mean h^2 + eps) w                      (norm 0: n = h, the quantiser)
//     a = max(max |n|, 2^-100),  scale = a / 448,  q = n (448 / a) rounded to e4m3
// n stays in fp32 until it is rounded to 8 bits (and to h's type, where n is asked for as well).
// 2^-100 keeps 448 / a finite; a row of zeros gives zeros.  A NaN or infinity in a row makes its
// scale NaN or leaves NaN in its place, as in torch.
//
// Bound: bytes (7 a value with the residual in 16 bits; 16384 x 4096 bf16 with the residual 71.5 us, 6.55 TB/s, the
// rate of a copy).  A row stays in the registers of its group of 8 to 1024 threads, 32 values a thread (8 for up to 256
// values: 56541 x 70 bf16 with the residual 19.0 us, with a warp a row 50), all loads of a row in flight before its first
// store; two reductions (squares, then magnitudes) by shuffles and, above a warp, one exchange through shared memory each.
// A group has the warps that a row fills (16384 x 5120 bf16: 51 us; with 256 threads instead of 160, 67).
// Rows whose width is no multiple of 8 start anywhere in a 16-byte word: their words are those of the whole
// tensor, the first and last one masked, so that all is read and written a word at a time all the same; the weights,
// which start at another place in their words, are shifted there (8888 x 5001 bf16: 42 us, with weights read value by
// value and 256 threads 70; whole words, 8888 x 5000, take 30).
#include "linear_tc.cuh"

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

// VEC neighbouring values (16 bytes, or 32 of fp32), as loaded
template <typename T, int VEC>
struct Lot {
  static constexpr int WORDS = VEC * (int)sizeof(T) / 16;
  uint4 w[WORDS];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void values(float (&v)[VEC]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        v[4 * i] = __uint_as_float(w[i].x); v[4 * i + 1] = __uint_as_float(w[i].y);
        v[4 * i + 2] = __uint_as_float(w[i].z); v[4 * i + 3] = __uint_as_float(w[i].w);
      }
    } else {
      unpack8<T>(w[0], v);
    }
  }
};
template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const float (&v)[VEC]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      reinterpret_cast<float4*>(p)[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
    *reinterpret_cast<uint4*>(p) = pack8<T>(v);
  }
}
template <typename T>
__device__ __forceinline__ float rounded(float x) {
  return to_f32(from_f32<T>(x));
}

// The VEC values (16 bytes) from column c of a row of `cols` on, wherever it starts: the aligned words around them, those
// that hold a value of the row.  Values outside of the row are whatever lies there.
template <typename T, int VEC>
__device__ __forceinline__ void unaligned(const T* p, int c, int cols, float (&v)[VEC]) {
  static_assert(VEC * sizeof(T) == 16, "a word");
  const int off = (int)((size_t)(p + c) & 15), first = c - off / (int)sizeof(T);
  const uint4* w = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(p + c) - off);
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (first + VEC > 0 && first < cols) a = w[0];
  if (off && first + 2 * VEC > 0 && first + VEC < cols) b = w[1];
  uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int j = 0; j < 6; ++j) x[j] = off & 8 ? x[j + 2] : x[j];
#pragma unroll
  for (int j = 0; j < 5; ++j) x[j] = off & 4 ? x[j + 1] : x[j];
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = off & 2 ? __funnelshift_r(x[j], x[j + 1], 16) : x[j];
  }
  Lot<T, VEC> l;
  l.w[0] = make_uint4(x[0], x[1], x[2], x[3]);
  l.values(v);
}

// A group of G threads (of a block of 128, or a block) holds a row of up to 32 G values: VEC neighbouring ones from column
// VEC (g + G i) on, less `shift`, the row's place in its first word, where rows are not WHOLE words.
template <typename T, int G, bool WHOLE, bool ADD>
__global__ void __launch_bounds__(G < 128 ? 128 : G) norm_fp8_kernel(NormArgs a) {
  constexpr int NT = G < 128 ? 128 : G, VEC = WHOLE ? 8 : 16 / (int)sizeof(T), NV = 32 / VEC, W = G > 32 ? G / 32 : 1;
  __shared__ float part[2][NT / G][W > 1 ? W : 1];
  const int g = threadIdx.x % G, mine = threadIdx.x / G;
  long long row = (long long)blockIdx.x * (NT / G) + mine;
  lin::depend();
  // a group behind the last row goes along with the others' reductions: a row of no columns
  const bool act = NT == G || row < a.rows;
  const int cols = act ? a.cols : 0;
  if (!act) row = 0;
  const long long off = row * a.cols;
  const T* h = static_cast<const T*>(a.h) + off;
  const T* w = static_cast<const T*>(a.w);
  const int shift = WHOLE ? 0 : (int)(((size_t)h & 15) / sizeof(T));
  auto column = [&](int i) { return VEC * (g + G * i) - shift; };
  auto any = [&](int i) { return VEC * G * i < cols + shift && column(i) < cols; };
  auto in = [&](int c) { return WHOLE || (c >= 0 && c < cols); };
  auto inner = [&](int c) { return WHOLE || (c >= 0 && c + VEC <= cols); };   // all but the first and the last vector
  // whether a vector of p may be moved as one: inside of the row, and p's words where h's are
  auto as_one = [&](const T* p, int c) {
    return WHOLE || (inner(c) && ((size_t)(p + off + c) & 15) == 0);
  };
  auto put = [&](void* to, int c, const float (&v)[VEC]) {
    T* p = static_cast<T*>(to);
    if (as_one(p, c)) {
      store<T, VEC>(p + off + c, v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (in(c + j)) p[off + c + j] = from_f32<T>(v[j]);
    }
  };
  float v[NV][VEC];
  {
    // h and y on their way together, before the first store (sum may be either)
    Lot<T, VEC> lh[NV], ly[ADD ? NV : 1];
    const T* y = static_cast<const T*>(a.y);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (any(i)) {
        lh[i].load(h + column(i));
        if constexpr (ADD) {
          if constexpr (WHOLE) {
            ly[i].load(y + off + column(i));
          } else {
            float t[VEC];
            unaligned<T, VEC>(y + off, column(i), cols, t);
            store<T, VEC>(reinterpret_cast<T*>(ly[i].w), t);
          }
        }
      }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[i][j] = 0.f;
      if (any(i)) {
        lh[i].values(v[i]);
        if (!inner(column(i))) {
#pragma unroll
          for (int j = 0; j < VEC; ++j)
            if (!in(column(i) + j)) v[i][j] = 0.f;
        }
        if constexpr (ADD) {
          float t[VEC];
          ly[i].values(t);
#pragma unroll
          for (int j = 0; j < VEC; ++j) v[i][j] = rounded<T>(v[i][j] + (in(column(i) + j) ? t[j] : 0.f));
          put(a.sum, column(i), v[i]);
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
    for (int o = G < 32 ? G / 2 : 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if constexpr (W > 1) {
      if (g % 32 == 0) part[0][mine][g / 32] = ss;
      __syncthreads();
      ss = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) ss += part[0][mine][i];
    }
    const float rs = rsqrtf(ss / (float)a.cols + a.eps);
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (any(i)) {
        float t[VEC];
        if (w) {
          if constexpr (WHOLE) {
            Lot<T, VEC> lw;
            lw.load(w + column(i));
            lw.values(t);
          } else {
            unaligned<T, VEC>(w, column(i), cols, t);
          }
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[i][j] = w ? v[i][j] * rs * t[j] : v[i][j] * rs;
      }
  }
  float top = 0x1p-100f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (!any(i)) continue;
    if (inner(column(i))) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) top = max_nan(top, fabsf(v[i][j]));
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (in(column(i) + j)) top = max_nan(top, fabsf(v[i][j]));
    }
  }
#pragma unroll
  for (int o = G < 32 ? G / 2 : 16; o > 0; o >>= 1) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  if constexpr (W > 1) {
    if (g % 32 == 0) part[1][mine][g / 32] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < W; ++i) top = max_nan(top, part[1][mine][i]);
  }
  const float inv = 448.f / top;
  if (g == 0 && act) a.scale[row] = top / 448.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (any(i)) {
      const int c = column(i);
      uint32_t o[VEC / 4];
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[i][4 * j] * inv, v[i][4 * j + 1] * inv), __NV_SATFINITE,
                                                     __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[i][4 * j + 2] * inv, v[i][4 * j + 3] * inv),
                                                     __NV_SATFINITE, __NV_E4M3);
        o[j] = lo | hi << 16;
      }
      uint8_t* q = a.q + off + c;
      if (WHOLE || (inner(c) && (size_t)q % VEC == 0)) {
        if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q) = make_uint2(o[0], o[1]);
        else *reinterpret_cast<uint32_t*>(q) = o[0];
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (in(c + j)) q[j] = (uint8_t)(o[j / 4] >> (8 * (j & 3)));
      }
      if (a.n) put(a.n, c, v[i]);
    }
}

template <typename T, bool WHOLE, bool ADD>
int launch(const NormArgs& a, cudaStream_t st) {
  const int cols = a.cols + (WHOLE ? 0 : 7);   // (a row may start in the middle of a word)
  auto go = [&](auto group) {
    constexpr int G = decltype(group)::value, NT = G < 128 ? 128 : G;
    const dim3 grid((unsigned)((a.rows + NT / G - 1) / (NT / G)));
    return lin::launch_after("norm_fp8_kernel", norm_fp8_kernel<T, G, WHOLE, ADD>, grid, NT, 0, st, 1, a);
  };
#define VERACE_GROUP(G) \
  if (cols <= 32 * G) return go(std::integral_constant<int, G>())
  VERACE_GROUP(8); VERACE_GROUP(16); VERACE_GROUP(32); VERACE_GROUP(64); VERACE_GROUP(128);
  VERACE_GROUP(160); VERACE_GROUP(192); VERACE_GROUP(224); VERACE_GROUP(256); VERACE_GROUP(320); VERACE_GROUP(384);
  VERACE_GROUP(512); VERACE_GROUP(640); VERACE_GROUP(768);
#undef VERACE_GROUP
  return go(std::integral_constant<int, 1024>());
}

template <typename T>
int launch(const NormArgs& a, cudaStream_t st) {
  const size_t all = (size_t)a.h | (size_t)a.y | (size_t)a.w | (size_t)a.sum | (size_t)a.n;
  const bool whole = a.cols % 8 == 0 && all % 16 == 0 && (size_t)a.q % 8 == 0;
  VERACE_REQUIRE(whole || a.cols <= 32761, VERACE_ERR_UNSUPPORTED,
                 "verace_rmsnorm_fp8: rows of %d columns that are not whole 16-byte words (at most 32761)", a.cols);
  if (a.y) return whole ? launch<T, true, true>(a, st) : launch<T, false, true>(a, st);
  return whole ? launch<T, true, false>(a, st) : launch<T, false, false>(a, st);
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
