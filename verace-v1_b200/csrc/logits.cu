// Penalties for repeated tokens, biases and a grammar's mask on a batch of logits, one pass.
// Per row, with c[v] the count of v among the generated tokens of the row's history and
// seen[v] any occurrence, the prompt's included:
//     l <- l / r if l > 0 else l r      where seen
//     l <- l - f c - p                  where c > 0
//     l <- l + bias[v]                  where the row's list names v
//     l <- -inf                         where the mask's bit is 0
//
// Bound: the bytes of the logits in and out.  A cluster of CTAs takes a row, each CTA a range of
// the vocabulary with a 32-bit counter per token in shared memory.  The cluster reads the row's
// history once, a share to each CTA, and counts a token in the counters of the CTA that owns it
// (distributed shared memory; equal tokens of a warp are added as one, since text repeats a few
// tokens most).  Then each CTA streams its range, eight values a thread: most have no count, no
// bias and a full mask, and are copied.  Biased tokens are marked in their counters and looked up
// in a short list.  Without history and biases there are no counters and no cluster.
#include "common.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace verace {
namespace {

namespace cg = cooperative_groups;

constexpr int NT = 512;
constexpr int CHUNK = 4096;   // vocabulary entries per CTA of logits_chunks
constexpr int LIST = 1024;    // biases of a CTA's range held in shared memory
constexpr uint32_t PROMPT = 0x80000000u, BIASED = 0x40000000u, COUNT = 0x3fffffffu;

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

struct Controls {
  float r, p, f;
};
__device__ __forceinline__ Controls controls(const LogitsArgs& a, int row) {
  return {a.rep_rows ? a.rep_rows[row] : a.rep, a.pres_rows ? a.pres_rows[row] : a.pres,
          a.freq_rows ? a.freq_rows[row] : a.freq};
}
__device__ __forceinline__ int history(const LogitsArgs& a, int row) {
  return !a.tokens ? 0 : a.lengths ? max(0, min(a.lengths[row], a.length)) : a.length;
}
// A logit of a token with counter c (not 0).
__device__ __forceinline__ float penalised(float l, uint32_t c, const Controls& k) {
  if (c & ~BIASED) l = l > 0.f ? l / k.r : l * k.r;
  if (c & COUNT) l = __fsub_rn(__fsub_rn(l, __fmul_rn(k.f, (float)(c & COUNT))), k.p);
  return l;
}

struct Biases {
  int n;                          // entries of the CTA's range; beyond LIST the global list is searched
  int id[LIST], order[LIST];
  float value[LIST];
};

// The last of the row's biases for a token.
__device__ __noinline__ float bias_of(const LogitsArgs& a, const Biases& s, int row, int v0, int token) {
  float value = 0.f;
  if (s.n <= LIST) {
    int last = -1;
    for (int i = 0; i < s.n; ++i)
      if (s.id[i] == token && s.order[i] > last) last = s.order[i], value = s.value[i];
  } else {
    for (int i = a.n_bias - 1; i >= 0; --i)
      if (id_at(a.bias_ids, a.bias_i64, (long long)row * a.n_bias + i) == v0 + token)
        return a.bias_values[(long long)row * a.n_bias + i];
  }
  return value;
}

// Rows in clusters of `ctas` (COUNTED: with counters; else the CTAs of a row have nothing in
// common), `range` tokens a CTA.
template <typename T, typename O, bool COUNTED>
__global__ void __launch_bounds__(NT, 2) logits_ranges(LogitsArgs a, int ctas, int range) {
  extern __shared__ __align__(16) uint32_t cnt[];
  __shared__ Biases s;
  const int tid = threadIdx.x, lane = tid % 32, rank = blockIdx.x % ctas, row = blockIdx.x / ctas;
  const int v0 = rank * range, nv = max(0, min(range, a.v - v0));
  const Controls k = controls(a, row);
  if constexpr (COUNTED) {
    cg::cluster_group cl = cg::this_cluster();
    for (int i = 4 * tid; i < range; i += 4 * NT) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
    if (tid == 0) s.n = 0;
    const int len = history(a, row), prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    if (ctas > 1) cl.sync();
    else __syncthreads();
    for (int i = tid; i < a.n_bias; i += NT) {
      const long long id = id_at(a.bias_ids, a.bias_i64, (long long)row * a.n_bias + i) - v0;
      if (id >= 0 && id < nv) {
        const int at = atomicAdd(&s.n, 1);
        if (at < LIST) s.id[at] = (int)id, s.order[at] = i, s.value[at] = a.bias_values[(long long)row * a.n_bias + i];
        atomicOr(&cnt[id], BIASED);
      }
    }
    const int share = (len + ctas - 1) / ctas, first = rank * share, last = min(len, first + share);
    const long long base = row * a.tokens_ld;
    for (int i0 = first; i0 < last; i0 += 4 * NT) {
      long long t[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + e * NT + tid;
        t[e] = i < last ? id_at(a.tokens, a.tokens_i64, base + i) : -1;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (i0 + e * NT >= last) break;
        const int i = i0 + e * NT + tid;
        const bool ok = t[e] >= 0 && t[e] < a.v, made = i >= prompt;
        const int token = ok ? (int)t[e] : -1;
        const uint32_t same = __match_any_sync(0xffffffffu, ok ? 2 * token + (made ? 1 : 0) : -1);
        if (ok && lane == __ffs(same) - 1) {
          const int owner = token / range;
          uint32_t* c = ctas > 1 ? cl.map_shared_rank(cnt, owner) : cnt;
          if (made) atomicAdd(c + (token - owner * range), (uint32_t)__popc(same));
          else atomicOr(c + (token - owner * range), PROMPT);
        }
      }
    }
    if (ctas > 1) cl.sync();
    else __syncthreads();
  }

  const T* in = static_cast<const T*>(a.logits) + row * a.ld + v0;
  O* out = static_cast<O*>(a.out) + row * a.out_ld + v0;
  const uint8_t* mask = a.allowed ? reinterpret_cast<const uint8_t*>(a.allowed + row * a.allowed_ld) + v0 / 8 : nullptr;
  auto one = [&](float l, int j) {
    if constexpr (COUNTED) {
      const uint32_t c = cnt[j];
      if (c) {
        l = penalised(l, c, k);
        if (c & BIASED) l += bias_of(a, s, row, v0, j);
      }
    }
    return l;
  };
  int done = 0;
  if ((reinterpret_cast<size_t>(in) | reinterpret_cast<size_t>(out)) % 16 == 0) {
    done = nv / 8 * 8;
#pragma unroll 2
    for (int j = 8 * tid; j < done; j += 8 * NT) {
      uint4 u[sizeof(T) / 2];
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) u[i] = reinterpret_cast<const uint4*>(in + j)[i];
      const uint32_t bits = mask ? __ldg(mask + j / 8) : 255u;
      float l[8];
      if constexpr (sizeof(T) == 4) {
        l[0] = __uint_as_float(u[0].x); l[1] = __uint_as_float(u[0].y);
        l[2] = __uint_as_float(u[0].z); l[3] = __uint_as_float(u[0].w);
        l[4] = __uint_as_float(u[1].x); l[5] = __uint_as_float(u[1].y);
        l[6] = __uint_as_float(u[1].z); l[7] = __uint_as_float(u[1].w);
      } else {
        unpack8<T>(u[0], l);
      }
      if constexpr (COUNTED) {
        const uint4 c = *reinterpret_cast<const uint4*>(cnt + j), d = *reinterpret_cast<const uint4*>(cnt + j + 4);
        if (c.x | c.y | c.z | c.w | d.x | d.y | d.z | d.w) {
#pragma unroll
          for (int i = 0; i < 8; ++i) l[i] = one(l[i], j + i);
        }
      }
      if (bits != 255u) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (!(bits >> i & 1u)) l[i] = -INFINITY;
      }
      if constexpr (sizeof(O) == 4) {
        reinterpret_cast<float4*>(out + j)[0] = make_float4(l[0], l[1], l[2], l[3]);
        reinterpret_cast<float4*>(out + j)[1] = make_float4(l[4], l[5], l[6], l[7]);
      } else {
        *reinterpret_cast<uint4*>(out + j) = pack8<O>(l);
      }
    }
  }
#pragma unroll 4
  for (int j = done + tid; j < nv; j += NT) {
    float l = one(to_f32(in[j]), j);
    if (mask && !(__ldg(mask + j / 8) >> (j % 8) & 1u)) l = -INFINITY;
    out[j] = from_f32<O>(l);
  }
}

// One CTA per CHUNK of a row's vocabulary, each over the whole history: for vocabularies whose
// counters no cluster holds.
template <typename T, typename O>
__global__ void __launch_bounds__(NT) logits_chunks(LogitsArgs a) {
  __shared__ uint32_t cnt[CHUNK];
  __shared__ uint32_t slot[CHUNK];        // the last bias entry per token
  const int row = blockIdx.y, v0 = blockIdx.x * CHUNK;
  const int nv = min(CHUNK, a.v - v0);
  for (int i = threadIdx.x; i < CHUNK; i += NT) cnt[i] = 0, slot[i] = 0;
  __syncthreads();
  const int len = history(a, row), prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
  for (int i = threadIdx.x; i < len; i += NT) {
    const long long t = id_at(a.tokens, a.tokens_i64, row * a.tokens_ld + i) - v0;
    if (t >= 0 && t < nv) {
      if (i < prompt) atomicOr(&cnt[t], PROMPT);
      else atomicAdd(&cnt[t], 1u);
    }
  }
  for (int i = threadIdx.x; i < a.n_bias; i += NT) {
    const long long t = id_at(a.bias_ids, a.bias_i64, (long long)row * a.n_bias + i) - v0;
    if (t >= 0 && t < nv) atomicMax(&slot[t], (uint32_t)i + 1);
  }
  __syncthreads();
  const Controls k = controls(a, row);
  const T* in = static_cast<const T*>(a.logits) + row * a.ld + v0;
  O* out = static_cast<O*>(a.out) + row * a.out_ld + v0;
  for (int i = threadIdx.x; i < nv; i += NT) {
    float l = to_f32(in[i]);
    if (cnt[i]) l = penalised(l, cnt[i], k);
    if (slot[i]) l += a.bias_values[(long long)row * a.n_bias + slot[i] - 1];
    if (a.allowed && !((a.allowed[row * a.allowed_ld + (v0 + i) / 32] >> (i % 32)) & 1u)) l = -INFINITY;
    out[i] = from_f32<O>(l);
  }
}

constexpr int RANGE_MAX = 49152;       // counters of a CTA at most (192 KB)
constexpr int RANGE_HALF = 24576;      // and where two CTAs share an SM

template <typename T, typename O, bool COUNTED>
int launch_ranges(const LogitsArgs& a, int ctas, int range, cudaStream_t st) {
  auto kern = logits_ranges<T, O, COUNTED>;
  if (!COUNTED) {
    kern<<<(unsigned)((long long)a.b * ctas), NT, 0, st>>>(a, ctas, range);
    return check_launch("logits_process");
  }
  static std::atomic<uint64_t> ready{0};      // devices whose limits are raised
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, RANGE_MAX * 4));
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)a.b * ctas));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = (size_t)range * 4;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ctas > 1 ? 1 : 0;
  VERACE_CUDA(cudaLaunchKernelEx(&cfg, kern, a, ctas, range));
  return check_launch("logits_process");
}

template <typename T, typename O>
int run(const LogitsArgs& a, cudaStream_t st) {
  auto range_of = [&](int c) { return ((a.v + c - 1) / c + 31) / 32 * 32; };
  if (!a.tokens && a.n_bias == 0) {
    // 4096 values a CTA, or more where the rows alone fill the device several times over
    int c = (a.v + 4095) / 4096;
    if ((long long)a.b * c > 4096) c = (a.v + 16383) / 16384;
    return launch_ranges<T, O, false>(a, c, range_of(c), st);
  }
  // as few CTAs a row as hold its counters two to an SM, more (of 2048 tokens at least) while the
  // rows alone leave the device empty
  int c = 1;
  while (c < 8 && range_of(c) > RANGE_HALF) c *= 2;
  if (range_of(c) > RANGE_HALF) c = 16;
  while (c < 8 && (long long)a.b * c * 2 <= 296 && range_of(2 * c) >= 2048) c *= 2;
  if (range_of(c) > RANGE_MAX || (long long)a.b * c > 0x7fffffffLL) {
    logits_chunks<T, O><<<dim3((a.v + CHUNK - 1) / CHUNK, a.b), NT, 0, st>>>(a);
    return check_launch("logits_process");
  }
  return launch_ranges<T, O, true>(a, c, range_of(c), st);
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
