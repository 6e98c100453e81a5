// Choice of a token per row of logits l (NaN counts as -inf).  z = (l - max l) / T, which no T
// sends above 0; kept are the tokens with l at least the k-th largest, then (over those) with
// less than p of the mass exp(z) above them, and with exp(z) >= min_p.  Equal values stand or fall together, so the kept
// set depends on no order.  token = argmax over the kept of z - log(noise), the lowest index
// on ties: with noise drawn from Exp(1) this is a draw from the softmax over the kept (the
// smallest of exponentials with rates w_i is i with probability w_i / sum w).  T = 0 takes
// the largest logit.  logprob = log softmax(z)[token] over the whole row (T = 0: of l).
//
// The thresholds come from a radix selection on the values' order-preserving 32-bit keys,
// eight bits at a time: by count for k, by mass for p.  Mass is summed in 2^-40 fixed point,
// so that the order of the atomics changes nothing.
#include "common.cuh"

namespace verace {
namespace {

constexpr int NT = 1024;

struct SampleArgs {
  const void* logits;
  long long ld;
  const float* noise;
  long long noise_ld;
  int b, v;
  const float* t_rows;
  const int* k_rows;
  const float* p_rows;
  const float* minp_rows;
  float t, p, minp;
  int k;
  long long* tokens;
  float* logprobs;
};

__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

template <typename T>
__device__ __forceinline__ float value(T l) {
  const float x = to_f32(l);
  return x != x ? -INFINITY : x + 0.f;   // -0 -> +0: equal values, equal keys
}

// z of a value against the row's largest (equal infinities: 0)
__device__ __forceinline__ float scaled(float x, float top, float t) { return x == top ? 0.f : (x - top) / t; }

template <typename F>
__device__ __forceinline__ float block_reduce(float x, float* s, F f) {
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  if (lane == 0) s[w] = x;
  __syncthreads();
  x = s[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

template <typename T>
__global__ void __launch_bounds__(NT) sample_kernel(SampleArgs a) {
  __shared__ float red[32];
  __shared__ unsigned long long hist[256];
  __shared__ uint32_t s_prefix;
  __shared__ unsigned long long s_left;
  __shared__ unsigned long long s_best;
  const int row = blockIdx.x, tid = threadIdx.x;
  const T* l = static_cast<const T*>(a.logits) + row * a.ld;
  const float* noise = a.noise + row * a.noise_ld;
  const float t = a.t_rows ? a.t_rows[row] : a.t;
  const bool greedy = !(t > 0.f);
  const float ts = greedy ? 1.f : t;
  const int k = a.k_rows ? a.k_rows[row] : a.k;
  const float p = a.p_rows ? a.p_rows[row] : a.p;
  const float minp = a.minp_rows ? a.minp_rows[row] : a.minp;

  float top = -INFINITY;
  for (int i = tid; i < a.v; i += NT) top = fmaxf(top, value(l[i]));
  top = block_reduce(top, red, [](float x, float y) { return fmaxf(x, y); });
  if (top == -INFINITY) {
    if (tid == 0) a.tokens[row] = -1, a.logprobs[row] = -INFINITY;
    return;
  }
  float ties = 0.f, rest = 0.f;
  for (int i = tid; i < a.v; i += NT) {
    const float x = value(l[i]);
    if (x == top) ties += 1.f;
    else rest += expf(scaled(x, top, ts));
  }
  ties = block_reduce(ties, red, [](float x, float y) { return x + y; });
  rest = block_reduce(rest, red, [](float x, float y) { return x + y; });
  const float lse = logf(ties) + log1pf(rest / ties);

  // the smallest kept key: every key above key_of(-inf), then by count, then by mass
  uint32_t least = key_of(-INFINITY) + 1;
  if (!greedy) {
    for (int by_mass = 0; by_mass < 2; ++by_mass) {
      if (by_mass ? !(p < 1.f) : (k <= 0 || k >= a.v)) continue;
      unsigned long long left = (unsigned long long)(by_mass ? 0 : k);
      uint32_t prefix = 0;
      for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = tid; i < a.v; i += NT) {
          const float x = value(l[i]);
          const uint32_t key = key_of(x);
          if (key >= least && (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))))
            atomicAdd(&hist[(key >> shift) & 255],
                      by_mass ? (unsigned long long)(expf(scaled(x, top, ts)) * 1099511627776.f + 0.5f) : 1ull);
        }
        __syncthreads();
        if (tid == 0) {
          if (by_mass && shift == 24) {
            unsigned long long total = 0;
            for (int i = 0; i < 256; ++i) total += hist[i];
            left = (unsigned long long)ceil((double)p * (double)total);
            if (left < 1) left = 1;
          }
          int bin = 255;
          while (bin > 0 && hist[bin] < left) left -= hist[bin--];
          s_prefix = prefix | ((uint32_t)bin << shift);
          s_left = left;
        }
        __syncthreads();
        prefix = s_prefix;
        left = s_left;
      }
      if (prefix > least) least = prefix;
    }
  }
  if (tid == 0) s_best = 0;
  __syncthreads();
  unsigned long long best = 0;
  for (int i = tid; i < a.v; i += NT) {
    const float x = value(l[i]);
    if (key_of(x) < least) continue;
    const float z = scaled(x, top, ts);
    if (!greedy && x != top && !(expf(z) >= minp)) continue;
    float key = greedy ? x : z - logf(noise[i]);
    if (!(key > -INFINITY)) continue;
    const unsigned long long c = ((unsigned long long)key_of(key + 0.f) << 32) | (0xffffffffu - (uint32_t)i);
    if (c > best) best = c;
  }
  atomicMax(&s_best, best);
  __syncthreads();
  if (tid == 0) {
    if (s_best == 0) {
      a.tokens[row] = -1, a.logprobs[row] = -INFINITY;
    } else {
      const int i = (int)(0xffffffffu - (uint32_t)s_best);
      a.tokens[row] = i;
      a.logprobs[row] = scaled(value(l[i]), top, ts) - lse;
    }
  }
}

}  // namespace
}  // namespace verace

using namespace verace;

extern "C" int verace_sample(const void* logits, long long ld, const float* noise, long long noise_ld, int b, int v,
                             int dtype, const float* t_rows, float t, const int* k_rows, int k,
                             const float* p_rows, float p, const float* minp_rows, float minp, long long* tokens,
                             float* logprobs, void* stream) {
  VERACE_REQUIRE(b >= 0 && v >= 0, VERACE_ERR_INVALID, "sample: negative size");
  VERACE_REQUIRE(dtype == VERACE_F32 || dtype == VERACE_BF16 || dtype == VERACE_F16, VERACE_ERR_INVALID,
                 "sample: dtype %d", dtype);
  if (b == 0) return VERACE_OK;
  VERACE_REQUIRE(v > 0, VERACE_ERR_INVALID, "sample: empty vocabulary");
  VERACE_REQUIRE(logits && tokens && logprobs, VERACE_ERR_INVALID, "sample: NULL pointer");
  VERACE_REQUIRE(ld >= v && (!noise || noise_ld >= v), VERACE_ERR_INVALID,
                 "sample: row stride below the vocabulary size");
  VERACE_REQUIRE(noise || (!t_rows && !(t > 0.f)), VERACE_ERR_INVALID,
                 "sample: noise is needed unless every row has temperature 0");
  SampleArgs a{logits, ld, noise, noise_ld, b, v, t_rows, k_rows, p_rows, minp_rows, t, p, minp, k, tokens, logprobs};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == VERACE_F32) sample_kernel<float><<<b, NT, 0, st>>>(a);
  else if (dtype == VERACE_BF16) sample_kernel<__nv_bfloat16><<<b, NT, 0, st>>>(a);
  else sample_kernel<__half><<<b, NT, 0, st>>>(a);
  return check_launch("sample");
}
