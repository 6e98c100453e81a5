// Penalties for repeated tokens, biases and a grammar's mask on a batch of logits, one pass.
// Per row, with c[v] the count of v among the generated tokens of the row's history and
// seen[v] any occurrence, the prompt's included:
//     l <- l / r if l > 0 else l r      where seen
//     l <- l - f c - p                  where c > 0
//     l <- l + bias[v]                  where the row's list names v
//     l <- -inf                         where the mask's bit is 0
#include "common.cuh"

namespace verace {
namespace {

constexpr int NT = 256;
constexpr int CHUNK = 4096;   // vocabulary entries per CTA

struct LogitsArgs {
  const void* logits;
  long long ld;
  void* out;
  long long out_ld;
  int b, v;
  const void* tokens;
  long long tokens_ld;
  int tokens_i64, length;
  const int* lengths;
  const int* prompt_lengths;
  const float* rep_rows;
  const float* pres_rows;
  const float* freq_rows;
  float rep, pres, freq;
  const void* bias_ids;
  const float* bias_values;
  int n_bias, bias_i64;
  const uint32_t* allowed;
  long long allowed_ld;
};

__device__ __forceinline__ long long id_at(const void* p, int i64, long long i) {
  return i64 ? static_cast<const long long*>(p)[i] : (long long)static_cast<const int*>(p)[i];
}

// The CTA's CHUNK entries: counts (bit 31: seen in the prompt; below it the generated count)
// and the last bias entry per token, in shared memory, from one pass over the row's lists.
template <typename T, typename O>
__global__ void __launch_bounds__(NT) logits_kernel(LogitsArgs a) {
  __shared__ uint32_t cnt[CHUNK];
  __shared__ uint32_t slot[CHUNK];
  const int row = blockIdx.y, v0 = blockIdx.x * CHUNK;
  const int nv = min(CHUNK, a.v - v0);
  for (int i = threadIdx.x; i < CHUNK; i += NT) cnt[i] = 0, slot[i] = 0;
  __syncthreads();
  if (a.tokens) {
    const int len = a.lengths ? min(a.lengths[row], a.length) : a.length;
    const int prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    for (int i = threadIdx.x; i < len; i += NT) {
      const long long t = id_at(a.tokens, a.tokens_i64, row * a.tokens_ld + i) - v0;
      if (t >= 0 && t < nv) {
        if (i < prompt) atomicOr(&cnt[t], 0x80000000u);
        else atomicAdd(&cnt[t], 1u);
      }
    }
  }
  for (int i = threadIdx.x; i < a.n_bias; i += NT) {
    const long long t = id_at(a.bias_ids, a.bias_i64, (long long)row * a.n_bias + i) - v0;
    if (t >= 0 && t < nv) atomicMax(&slot[t], (uint32_t)i + 1);
  }
  __syncthreads();
  const float r = a.rep_rows ? a.rep_rows[row] : a.rep;
  const float p = a.pres_rows ? a.pres_rows[row] : a.pres;
  const float f = a.freq_rows ? a.freq_rows[row] : a.freq;
  const T* in = static_cast<const T*>(a.logits) + row * a.ld + v0;
  O* out = static_cast<O*>(a.out) + row * a.out_ld + v0;
  for (int i = threadIdx.x; i < nv; i += NT) {
    float l = to_f32(in[i]);
    const uint32_t c = cnt[i];
    if (c) l = l > 0.f ? l / r : l * r;
    const uint32_t made = c & 0x7fffffffu;
    if (made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(f, (float)made)), p);
    if (slot[i]) l += a.bias_values[(long long)row * a.n_bias + slot[i] - 1];
    if (a.allowed && !((a.allowed[row * a.allowed_ld + (v0 + i) / 32] >> (i % 32)) & 1u)) l = -INFINITY;
    out[i] = from_f32<O>(l);
  }
}

template <typename T, typename O>
int run(const LogitsArgs& a, cudaStream_t st) {
  logits_kernel<T, O><<<dim3((a.v + CHUNK - 1) / CHUNK, a.b), NT, 0, st>>>(a);
  return check_launch("logits_process");
}

}  // namespace
}  // namespace verace

using namespace verace;

extern "C" int verace_logits_process(const void* logits, long long ld, void* out, long long out_ld, int b, int v,
                                     int dtype, int out_dtype, const void* tokens, long long tokens_ld,
                                     int tokens_i64, int length, const int* lengths, const int* prompt_lengths,
                                     const float* rep_rows, float rep, const float* pres_rows, float pres,
                                     const float* freq_rows, float freq, const void* bias_ids,
                                     const float* bias_values, int n_bias, int bias_i64,
                                     const uint32_t* allowed, long long allowed_ld, void* stream) {
  VERACE_REQUIRE(b >= 0 && v >= 0 && length >= 0 && n_bias >= 0, VERACE_ERR_INVALID, "logits_process: negative size");
  VERACE_REQUIRE(dtype == VERACE_F32 || dtype == VERACE_BF16 || dtype == VERACE_F16, VERACE_ERR_INVALID,
                 "logits_process: dtype %d", dtype);
  VERACE_REQUIRE(out_dtype == dtype || out_dtype == VERACE_F32, VERACE_ERR_INVALID,
                 "logits_process: out_dtype %d (the input's or fp32)", out_dtype);
  VERACE_REQUIRE(b <= 65535, VERACE_ERR_UNSUPPORTED, "logits_process: %d rows (at most 65535)", b);
  if (b == 0 || v == 0) return VERACE_OK;
  VERACE_REQUIRE(logits && out, VERACE_ERR_INVALID, "logits_process: NULL pointer");
  VERACE_REQUIRE(ld >= v && out_ld >= v, VERACE_ERR_INVALID, "logits_process: row stride below the vocabulary size");
  VERACE_REQUIRE(logits != out || (dtype == out_dtype && ld == out_ld), VERACE_ERR_INVALID,
                 "logits_process: in place needs one type and row stride");
  VERACE_REQUIRE(!tokens || tokens_ld >= length, VERACE_ERR_INVALID, "logits_process: token row stride below length");
  VERACE_REQUIRE(n_bias == 0 || (bias_ids && bias_values), VERACE_ERR_INVALID, "logits_process: NULL bias list");
  VERACE_REQUIRE(!allowed || allowed_ld == 0 || allowed_ld >= (v + 31) / 32, VERACE_ERR_INVALID,
                 "logits_process: mask row stride below its words");
  LogitsArgs a{logits, ld, out, out_ld, b, v, length > 0 ? tokens : nullptr, tokens_ld, tokens_i64, length, lengths,
               prompt_lengths, rep_rows, pres_rows, freq_rows, rep, pres, freq, bias_ids, bias_values, n_bias,
               bias_i64, allowed, allowed_ld};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == VERACE_F32) return run<float, float>(a, st);
  if (dtype == VERACE_BF16)
    return out_dtype == VERACE_F32 ? run<__nv_bfloat16, float>(a, st) : run<__nv_bfloat16, __nv_bfloat16>(a, st);
  return out_dtype == VERACE_F32 ? run<__half, float>(a, st) : run<__half, __half>(a, st);
}
