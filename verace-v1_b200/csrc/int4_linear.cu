// Product of a few tokens with 4-bit weights:
//     y[i][n] = sum_k x[i][k] W[n][k] (+ bias[n]),   W[n][k] = s[k/G][n] (q[n][k] - z[k/G][n])
// q in [0, 15], two to a byte along k (the even k in the low half); z in [0, 15], 8 when no
// zeros are given.  One group's terms are summed with the integers q - z, exact in every
// type, and scaled once: y = sum_g s_g (sum_{k in g} x_k (q_k - z_g)), all in fp32.
#include "common.cuh"

namespace verace {
namespace {

constexpr int NT = 128;
constexpr int TOK = 8;   // tokens per warp
// A group's unscaled sum reaches 128 * 15 times its largest input: inputs are brought down by
// 2^12 (exact) and the result back up, so that sums of any finite inputs stay finite.
constexpr float DOWN = 1.f / 4096.f, UP = 4096.f;

// One warp per output row and TOK tokens: lanes step along k in words of 8 codes.
template <typename T, typename O>
__global__ void __launch_bounds__(NT)
int4_linear_rows(const T* __restrict__ x, long long ldx, const uint32_t* __restrict__ q, const T* __restrict__ s,
                 const uint8_t* __restrict__ z, const T* __restrict__ bias, O* __restrict__ y, long long m, int n,
                 int k, int group) {
  const int row = blockIdx.x * (NT / 32) + threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const long long m0 = (long long)blockIdx.y * TOK;
  if (row >= n) return;
  const int mt = (int)(m - m0 < TOK ? m - m0 : TOK);
  float acc[TOK];
#pragma unroll
  for (int i = 0; i < TOK; ++i) acc[i] = 0.f;
  for (int w = lane; w < k / 8; w += 32) {
    const uint32_t c = q[(long long)row * (k / 8) + w];
    const int g = w * 8 / group;
    const float sc = to_f32(s[(long long)g * n + row]);
    const float zero = z ? (float)z[(long long)g * n + row] : 8.f;
#pragma unroll
    for (int i = 0; i < TOK; ++i) {
      if (i < mt) {
        const T* xp = x + (m0 + i) * ldx + w * 8;
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) part = fmaf(to_f32(xp[j]) * DOWN, (float)((c >> (4 * j)) & 15u) - zero, part);
        acc[i] = fmaf(part, sc, acc[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TOK; ++i) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
    if (lane == 0 && i < mt) y[(m0 + i) * n + row] = from_f32<O>(acc[i] * UP + (bias ? to_f32(bias[row]) : 0.f));
  }
}

template <typename T, typename O>
int run(const void* x, long long ldx, const void* q, const void* s, const void* z, const void* bias, void* y,
        long long m, int n, int k, int group, cudaStream_t st) {
  dim3 grid((n + NT / 32 - 1) / (NT / 32), (unsigned)((m + TOK - 1) / TOK));
  int4_linear_rows<T, O><<<grid, NT, 0, st>>>(
      static_cast<const T*>(x), ldx, static_cast<const uint32_t*>(q), static_cast<const T*>(s),
      static_cast<const uint8_t*>(z), static_cast<const T*>(bias), static_cast<O*>(y), m, n, k, group);
  return check_launch("int4_linear");
}

}  // namespace
}  // namespace verace

using namespace verace;

extern "C" int verace_int4_linear(const void* x, long long ldx, const void* qweight, const void* scales,
                                  const void* zeros, const void* bias, void* y, long long m, int n, int k,
                                  int group, int dtype, int out_dtype, void* stream) {
  VERACE_REQUIRE(m >= 0 && n >= 0 && k >= 0, VERACE_ERR_INVALID, "int4_linear: negative size");
  VERACE_REQUIRE(dtype == VERACE_F32 || dtype == VERACE_BF16 || dtype == VERACE_F16, VERACE_ERR_INVALID,
                 "int4_linear: dtype %d", dtype);
  VERACE_REQUIRE(out_dtype == dtype || out_dtype == VERACE_F32, VERACE_ERR_INVALID,
                 "int4_linear: out_dtype %d (the input's or fp32)", out_dtype);
  VERACE_REQUIRE(group == 32 || group == 64 || group == 128, VERACE_ERR_UNSUPPORTED,
                 "int4_linear: group size %d (32, 64 or 128)", group);
  VERACE_REQUIRE(k % 32 == 0, VERACE_ERR_UNSUPPORTED, "int4_linear: k %d is not a multiple of 32", k);
  VERACE_REQUIRE(ldx >= k, VERACE_ERR_INVALID, "int4_linear: row stride %lld < k %d", ldx, k);
  if (m == 0 || n == 0) return VERACE_OK;
  VERACE_REQUIRE(y && (k == 0 || (x && qweight && scales)), VERACE_ERR_INVALID, "int4_linear: NULL pointer");
  const size_t esz = dtype == VERACE_F32 ? 4 : 2;
  VERACE_REQUIRE((size_t)x % 16 == 0 && ldx * esz % 16 == 0 && (size_t)qweight % 16 == 0, VERACE_ERR_INVALID,
                 "int4_linear: x rows and qweight must be 16-byte aligned");
  VERACE_REQUIRE(m <= 65535LL * TOK, VERACE_ERR_UNSUPPORTED, "int4_linear: m %lld too large", m);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f32o = out_dtype == VERACE_F32;
  if (dtype == VERACE_F32) return run<float, float>(x, ldx, qweight, scales, zeros, bias, y, m, n, k, group, st);
  if (dtype == VERACE_BF16)
    return f32o ? run<__nv_bfloat16, float>(x, ldx, qweight, scales, zeros, bias, y, m, n, k, group, st)
                : run<__nv_bfloat16, __nv_bfloat16>(x, ldx, qweight, scales, zeros, bias, y, m, n, k, group, st);
  return f32o ? run<__half, float>(x, ldx, qweight, scales, zeros, bias, y, m, n, k, group, st)
              : run<__half, __half>(x, ldx, qweight, scales, zeros, bias, y, m, n, k, group, st);
}
