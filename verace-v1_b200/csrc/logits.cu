// Penalties for repeated tokens, biases and a grammar's mask on a batch of logits, one pass.
// Per row, with c[v] the count of v among the generated tokens of the row's history and
// seen[v] any occurrence, the prompt's included:
//     l <- l / r if l > 0 else l r      where seen
//     l <- l - f c - p                  where c > 0
//     l <- l + bias[v]                  where the row's list names v
//     l <- -inf                         where the mask's bit is 0
//
// Bound: the bytes of the logits in and out.  Each CTA takes a range of a row's vocabulary, with a
// counter per token in shared memory, and reads the whole history of the row (from L2 after the
// first), counting what falls into its range.  (Sharing the history out over a cluster and counting
// in distributed shared memory was slower: 23 k clocks for 8192 tokens a CTA, remote atomics being
// the slower ones.)  Then it streams its range, eight values a thread: most have no count, no bias
// and a full mask, and are copied.
//
// Measured on the device: a row of 32000 with 200 tokens of history 3.7 us; 64 rows of 163840, bf16
// to fp32, 63 MB: mask alone 12.9 us (4.9 TB/s), with 4096 tokens of history 19.5, with 300 biases too
// 22.0 (2.9 TB/s; 28 before the listed form: the counting went before the stream, not beside it; what
// is left is the counting's chain of loads under the stream's, 10 us); 8 rows of 32000 with 65536
// tokens of history 12.3, in which every CTA of a row reads its history from L2.  (0.5 to 0.8 us of
// both last ones are the repetition penalty's division, beside a product with 1 / r.)
#include "common.cuh"

#include <atomic>

namespace verace {
namespace {

constexpr int NT = 512;
constexpr int CHUNK = 4096;   // vocabulary entries per CTA of logits_chunks
constexpr int LIST = 512;     // biases of a CTA's range held in shared memory
// A counter: seen in the prompt, biased, the bias's place in the list, the generated count.
constexpr uint32_t PROMPT = 0x80000000u, BIASED = 0x40000000u, PLACE = 20, COUNT = 0xfffffu;
constexpr int LENGTH_MAX = 1 << 20, LENGTH_LISTED = 1 << 14;   // histories below these fit the counters
constexpr int RANGE = 11264, RANGE_LONG = 24576, RANGE_LISTED = 18432;   // tokens of a CTA at most
constexpr int TOUCHED = 2048; // touched tokens listed

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
// A logit of a token seen, `made` of its occurrences being generated.
__device__ __forceinline__ float penalised(float l, uint32_t made, const Controls& k) {
  l = l > 0.f ? l / k.r : l * k.r;       // (the quotient itself: few tokens are touched)
  if (made) l = __fsub_rn(__fsub_rn(l, __fmul_rn(k.f, (float)made)), k.p);
  return l;
}

struct Biases {
  int n;                          // entries of the CTA's range; beyond LIST the global list is searched
  int id[LIST], order[LIST];
  float value[LIST];
};

// Eight values from 16 or 32 bytes, and eight to the output, those left out by the mask as -inf.
template <typename T>
__device__ __forceinline__ void values8(const uint4* u, float* l) {
  if constexpr (sizeof(T) == 4) {
    l[0] = __uint_as_float(u[0].x); l[1] = __uint_as_float(u[0].y);
    l[2] = __uint_as_float(u[0].z); l[3] = __uint_as_float(u[0].w);
    l[4] = __uint_as_float(u[1].x); l[5] = __uint_as_float(u[1].y);
    l[6] = __uint_as_float(u[1].z); l[7] = __uint_as_float(u[1].w);
  } else {
    unpack8<T>(u[0], l);
  }
}
template <typename O>
__device__ __forceinline__ void store8(O* out, float* l, uint32_t bits) {
  if (bits != 255u) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (!(bits >> i & 1u)) l[i] = -INFINITY;
  }
  if constexpr (sizeof(O) == 4) {
    reinterpret_cast<float4*>(out)[0] = make_float4(l[0], l[1], l[2], l[3]);
    reinterpret_cast<float4*>(out)[1] = make_float4(l[4], l[5], l[6], l[7]);
  } else {
    *reinterpret_cast<uint4*>(out) = pack8<O>(l);
  }
}

// The last of the row's biases for a token.
__device__ __noinline__ float bias_of(const void* ids, int i64, const float* values, long long first, int n, int token) {
  for (int i = n - 1; i >= 0; --i)
    if (id_at(ids, i64, first + i) == token) return values[first + i];
  return 0.f;
}

// `ctas` CTAs a row, `range` tokens each; COUNTED: with counters; LONG: for long histories, whose
// time is the pass over them: twice the threads, and twice the loads in flight for each.
template <typename T, typename O, bool COUNTED, bool LONG>
__global__ void __launch_bounds__(LONG ? 2 * NT : NT, LONG ? 1 : 4) logits_ranges(LogitsArgs a, int ctas, int range) {
  constexpr int NTH = LONG ? 2 * NT : NT;
  extern __shared__ __align__(16) uint32_t cnt[];
  __shared__ Biases s;
  const int tid = threadIdx.x, rank = blockIdx.x % ctas, row = blockIdx.x / ctas;
  const int v0 = rank * range, nv = max(0, min(range, a.v - v0));
  const Controls k = controls(a, row);
  const T* in = static_cast<const T*>(a.logits) + row * a.ld + v0;
  O* out = static_cast<O*>(a.out) + row * a.out_ld + v0;
  const uint8_t* mask = a.allowed ? reinterpret_cast<const uint8_t*>(a.allowed + row * a.allowed_ld) + v0 / 8 : nullptr;
  if constexpr (COUNTED) {
    // the range comes into L2 while the history is counted
    constexpr int LINE = 128 / sizeof(T);
    for (int i = tid * LINE; i < nv; i += NTH * LINE) asm volatile("prefetch.global.L2 [%0];" ::"l"(in + i));
    if (mask && tid * 1024 < nv) asm volatile("prefetch.global.L2 [%0];" ::"l"(mask + tid * 128));
    for (int i = 4 * tid; i < range; i += 4 * NTH) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
    if (tid == 0) s.n = 0;
    const int len = history(a, row), prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    __syncthreads();
    for (int i = tid; i < a.n_bias; i += NTH) {
      const long long id = id_at(a.bias_ids, a.bias_i64, (long long)row * a.n_bias + i) - v0;
      if (id >= 0 && id < nv) {
        const int at = atomicAdd(&s.n, 1);
        if (at < LIST) s.id[at] = (int)id, s.order[at] = i, s.value[at] = a.bias_values[(long long)row * a.n_bias + i];
        else atomicOr(&cnt[id], BIASED);
      }
    }
    auto count = [&](long long token, int i) {
      // (in 32-bit halves: this runs for every token of the history)
      const uint32_t t = (uint32_t)token - (uint32_t)v0;
      if (t < (uint32_t)nv && (uint32_t)((unsigned long long)token >> 32) == 0u) {
        if (i >= prompt) atomicAdd(&cnt[t], 1u);
        else atomicOr(&cnt[t], PROMPT);
      }
    };
    const long long base = row * a.tokens_ld;
    int done = 0;
    if (a.tokens_i64) {
      const long long* tk = static_cast<const long long*>(a.tokens) + base;
      if (reinterpret_cast<size_t>(tk) % 16 == 0) {
        constexpr int FLY = LONG ? 8 : 4;
        done = len / 2 * 2;
        for (int i = 2 * tid; i < done; i += 2 * NTH * FLY) {
          longlong2 u[FLY];
#pragma unroll
          for (int e = 0; e < FLY; ++e) {
            const int j = i + e * 2 * NTH;
            u[e] = j < done ? __ldg(reinterpret_cast<const longlong2*>(tk + j)) : make_longlong2(-1, -1);
          }
#pragma unroll
          for (int e = 0; e < FLY; ++e) {
            count(u[e].x, i + e * 2 * NTH);
            count(u[e].y, i + e * 2 * NTH + 1);
          }
        }
      }
    } else {
      const int* tk = static_cast<const int*>(a.tokens) + base;
      if (reinterpret_cast<size_t>(tk) % 16 == 0) {
        constexpr int FLY = LONG ? 8 : 2;
        done = len / 4 * 4;
        for (int i = 4 * tid; i < done; i += 4 * NTH * FLY) {
          int4 u[FLY];
#pragma unroll
          for (int e = 0; e < FLY; ++e) {
            const int j = i + e * 4 * NTH;
            u[e] = j < done ? __ldg(reinterpret_cast<const int4*>(tk + j)) : make_int4(-1, -1, -1, -1);
          }
#pragma unroll
          for (int e = 0; e < FLY; ++e) {
            const int j = i + e * 4 * NTH;
            count(u[e].x, j);
            count(u[e].y, j + 1);
            count(u[e].z, j + 2);
            count(u[e].w, j + 3);
          }
        }
      }
    }
#pragma unroll 4
    for (int i = done + tid; i < len; i += NTH) count(id_at(a.tokens, a.tokens_i64, base + i), i);
    __syncthreads();
    if (a.n_bias) {
      // of the list's entries for one token the last in the row's order holds
      const int listed = min(s.n, LIST);
      for (int i = tid; i < listed; i += NTH) {
        const int id = s.id[i], order = s.order[i];
        bool last = true;
        for (int j = 0; j < listed; ++j) last = last && !(s.id[j] == id && s.order[j] > order);
        if (last) atomicOr(&cnt[id], BIASED | (uint32_t)i << PLACE);
      }
      __syncthreads();
    }
  }

  auto one = [&](float l, uint32_t c, int j) {
    if (c & (PROMPT | COUNT)) l = penalised(l, c & COUNT, k);
    if (c & BIASED) l += s.n <= LIST ? s.value[c >> PLACE & (LIST - 1)] : bias_of(a.bias_ids, a.bias_i64, a.bias_values, (long long)row * a.n_bias, a.n_bias, v0 + j);
    return l;
  };
  int done = 0;
  if ((reinterpret_cast<size_t>(in) | reinterpret_cast<size_t>(out)) % 16 == 0) {
    done = nv / 8 * 8;
#pragma unroll 2
    for (int j = 8 * tid; j < done; j += 8 * NTH) {
      uint4 u[sizeof(T) / 2];
#pragma unroll
      for (int i = 0; i < (int)(sizeof(T) / 2); ++i) u[i] = reinterpret_cast<const uint4*>(in + j)[i];
      const uint32_t bits = mask ? __ldg(mask + j / 8) : 255u;
      float l[8];
      values8<T>(u, l);
      if constexpr (COUNTED) {
        const uint4 c = *reinterpret_cast<const uint4*>(cnt + j), d = *reinterpret_cast<const uint4*>(cnt + j + 4);
        if (c.x | c.y | c.z | c.w | d.x | d.y | d.z | d.w) {
          const uint32_t e[8] = {c.x, c.y, c.z, c.w, d.x, d.y, d.z, d.w};
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (e[i]) l[i] = one(l[i], e[i], j + i);
        }
      }
      store8<O>(out + j, l, bits);
    }
  }
#pragma unroll 4
  for (int j = done + tid; j < nv; j += NTH) {
    float l = to_f32(in[j]);
    if constexpr (COUNTED) {
      if (cnt[j]) l = one(l, cnt[j], j);
    }
    if (mask && !(__ldg(mask + j / 8) >> (j % 8) & 1u)) l = -INFINITY;
    out[j] = from_f32<O>(l);
  }
}

struct Places {      // places in the row's list of biases whose tokens are in the CTA's range, in any order
  int n;
  int2 entry[LIST];  // token, place
};

// The same for many wide rows, in which history and bias touch few tokens.  Half the threads count,
// list each token at its first time and compute the listed ones' logits; the other half, and then
// all, stream the range as though nothing touched it; the listed logits are stored last.  (In place
// too: a value that the mask leaves is stored as it was read.)  The counters are of 16 bits, a pair
// to a word, so that four CTAs' fit an SM and the rows one wave.
template <typename T, typename O>
__global__ void __launch_bounds__(NT, 4) logits_listed(LogitsArgs a, int ctas, int range) {
  constexpr int CT = NT / 2;
  constexpr uint32_t SEEN = 0x8000u, NAMED = 0x4000u, MADE = NAMED - 1;
  extern __shared__ __align__(16) uint32_t cnt[];
  __shared__ Places s;
  __shared__ uint16_t list[TOUCHED];
  __shared__ float value[TOUCHED];
  __shared__ int touched, next;                                  // tokens listed; the first piece that no warp has
  const int tid = threadIdx.x, lane = tid % 32, rank = blockIdx.x % ctas, row = blockIdx.x / ctas;
  const int v0 = rank * range, nv = max(0, min(range, a.v - v0));
  const T* in = static_cast<const T*>(a.logits) + row * a.ld + v0;
  O* out = static_cast<O*>(a.out) + row * a.out_ld + v0;
  const uint8_t* mask = a.allowed ? reinterpret_cast<const uint8_t*>(a.allowed + row * a.allowed_ld) + v0 / 8 : nullptr;
  const long long first = row * (long long)a.n_bias;
  auto counter = [&](int j) { return cnt[j / 2] >> 16 * (j & 1) & 0xffffu; };
  auto bias_at = [&](int j) {
    const int listed = s.n;
    if (listed > LIST) return bias_of(a.bias_ids, a.bias_i64, a.bias_values, first, a.n_bias, v0 + j);
    int place = 0;                                               // the last of equal tokens holds
    for (int e = 0; e < listed; ++e) {
      const int2 entry = s.entry[e];
      if (entry.x == j) place = max(place, entry.y);
    }
    return a.bias_values[first + place];
  };
  auto final_of = [&](int j, const Controls& k) {
    const uint32_t c = counter(j);
    float l = to_f32(in[j]);
    if (c & (SEEN | MADE)) l = penalised(l, c & MADE, k);
    return c & NAMED ? l + bias_at(j) : l;
  };
  if (tid == 0) s.n = 0, touched = 0, next = 0;
  __syncthreads();

  if (tid < CT) {
    auto together = [] { asm volatile("bar.sync 1, %0;" ::"n"(CT) : "memory"); };
    // the first tokens and biases are asked for before all else (within the rows' strides, whatever
    // the lengths): under the stream's loads each step of such a chain waits for microseconds
    constexpr int FLY = 4;
    const long long base = row * a.tokens_ld;
    const char* tk = static_cast<const char*>(a.tokens) + base * (a.tokens_i64 ? 8 : 4);
    const int per = a.tokens_i64 ? 2 : 4;                        // tokens in 16 bytes
    const int fast = a.tokens && reinterpret_cast<size_t>(tk) % 16 == 0 ? a.length / per * per : 0;
    uint4 u[FLY];
    auto fetch = [&](int i0) {
#pragma unroll
      for (int e = 0; e < FLY; ++e) {
        const int i = i0 + (e * CT + tid) * per;
        if (i < fast) u[e] = __ldg(reinterpret_cast<const uint4*>(tk + (long long)i * (16 / per)));
      }
    };
    fetch(0);
    const long long bias0 = tid < a.n_bias ? id_at(a.bias_ids, a.bias_i64, first + tid) : -1;
    const int len = history(a, row), prompt = a.prompt_lengths ? a.prompt_lengths[row] : 0;
    for (int i = 4 * tid; i < range / 2; i += 4 * CT) *reinterpret_cast<uint4*>(cnt + i) = make_uint4(0, 0, 0, 0);
    together();
    const Controls k = controls(a, row);
    auto mark = [&](uint32_t t, uint32_t bits, bool add) {
      const int at = 16 * (t & 1);
      const uint32_t old = add ? atomicAdd(cnt + t / 2, bits << at) : atomicOr(cnt + t / 2, bits << at);
      if (old >> at & 0xffffu) return;
      const int n = atomicAdd(&touched, 1);                      // the token's first time
      if (n < TOUCHED) list[n] = (uint16_t)t;
    };
    auto count = [&](uint32_t low, uint32_t high, int i) {
      const uint32_t t = low - (uint32_t)v0;
      if (t < (uint32_t)nv && high == 0u) mark(t, i >= prompt ? 1u : SEEN, i >= prompt);
    };
    for (int i = tid; i < a.n_bias; i += CT) {
      const long long id = (i == tid ? bias0 : id_at(a.bias_ids, a.bias_i64, first + i)) - v0;
      if (id >= 0 && id < nv) {
        const int at = atomicAdd(&s.n, 1);
        if (at < LIST) s.entry[at] = make_int2((int)id, i);
        mark((uint32_t)id, NAMED, false);
      }
    }
    const int done = min(fast, len / per * per);
    for (int i0 = 0; i0 < done; i0 += FLY * CT * per) {
      if (i0 > 0) fetch(i0);
#pragma unroll
      for (int e = 0; e < FLY; ++e) {
        const int i = i0 + (e * CT + tid) * per;
        if (i < done) {
          if (a.tokens_i64) {
            count(u[e].x, u[e].y, i);
            count(u[e].z, u[e].w, i + 1);
          } else {                                               // (a negative one's high half is not 0)
            count(u[e].x, u[e].x >> 31, i);
            count(u[e].y, u[e].y >> 31, i + 1);
            count(u[e].z, u[e].z >> 31, i + 2);
            count(u[e].w, u[e].w >> 31, i + 3);
          }
        }
      }
    }
    for (int i = done + tid; i < len; i += CT) {
      const long long t = id_at(a.tokens, a.tokens_i64, base + i);
      count((uint32_t)t, (uint32_t)((unsigned long long)t >> 32), i);
    }
    together();
    if (touched <= TOUCHED)
      for (int i = tid; i < touched; i += CT) value[i] = final_of(list[i], k);
    __syncwarp();
  }

  // the range, in pieces of a warp's 512 values
  const bool wide = (reinterpret_cast<size_t>(in) | reinterpret_cast<size_t>(out)) % 16 == 0;
  while (true) {
    int at = 0;
    if (lane == 0) at = atomicAdd(&next, 1);
    const int j0 = __shfl_sync(~0u, at, 0) * 512;
    if (j0 >= nv) break;
    if (wide && j0 + 512 <= nv) {
      uint4 u[2][sizeof(T) / 2];
      uint32_t bits[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + 8 * (32 * e + lane);
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) u[e][i] = reinterpret_cast<const uint4*>(in + j)[i];
        bits[e] = mask ? __ldg(mask + j / 8) : 255u;
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float l[8];
        values8<T>(u[e], l);
        store8<O>(out + j0 + 8 * (32 * e + lane), l, bits[e]);
      }
    } else {
      for (int j = j0 + lane; j < min(j0 + 512, nv); j += 32) {
        const bool kept = !mask || __ldg(mask + j / 8) >> (j % 8) & 1u;
        out[j] = from_f32<O>(kept ? to_f32(in[j]) : -INFINITY);
      }
    }
  }
  __syncthreads();
  auto put = [&](int j, float l) {
    if (!mask || __ldg(mask + j / 8) >> (j % 8) & 1u) out[j] = from_f32<O>(l);
  };
  if (touched <= TOUCHED) {
    for (int i = tid; i < touched; i += NT) put(list[i], value[i]);
  } else {                                                       // more than the list holds
    const Controls k = controls(a, row);
    for (int j = tid; j < nv; j += NT)
      if (counter(j)) put(j, final_of(j, k));
  }
}

// The same with a counter and a bias slot of 32 bits each: for histories that the counters above
// do not hold.
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
    if (cnt[i]) l = penalised(l, cnt[i] & ~PROMPT, k);
    if (slot[i]) l += a.bias_values[(long long)row * a.n_bias + slot[i] - 1];
    if (a.allowed && !((a.allowed[row * a.allowed_ld + (v0 + i) / 32] >> (i % 32)) & 1u)) l = -INFINITY;
    out[i] = from_f32<O>(l);
  }
}

// Raises a kernel's limit of shared memory, once on each device.
int raise_limit(const void* kern, std::atomic<uint64_t>& ready, int bytes) {
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return VERACE_OK;
}

template <typename T, typename O, bool COUNTED, bool LONG>
int launch_ranges(const LogitsArgs& a, int ctas, int range, cudaStream_t st) {
  auto kern = logits_ranges<T, O, COUNTED, LONG>;
  const size_t smem = COUNTED ? (size_t)range * 4 : 0;
  if (COUNTED) {
    static std::atomic<uint64_t> ready{0};
    if (int rc = raise_limit(reinterpret_cast<const void*>(kern), ready, 4 * RANGE_LONG)) return rc;
  }
  VERACE_REQUIRE((long long)a.b * ctas <= 0x7fffffffLL, VERACE_ERR_UNSUPPORTED, "logits_process: %d rows of %d", a.b,
                 a.v);
  kern<<<(unsigned)((long long)a.b * ctas), LONG ? 2 * NT : NT, smem, st>>>(a, ctas, range);
  return check_launch("logits_process");
}

template <typename T, typename O>
int run(const LogitsArgs& a, cudaStream_t st) {
  auto range_of = [&](int c) { return ((a.v + c - 1) / c + 31) / 32 * 32; };
  int c;
  if (!a.tokens && a.n_bias == 0) {
    // 4096 values a CTA, or more where the rows alone fill the device several times over
    c = (a.v + 4095) / 4096;
    if ((long long)a.b * c > 4096) c = (a.v + 16383) / 16384;
    return launch_ranges<T, O, false, false>(a, c, range_of(c), st);
  }
  if (a.length >= LENGTH_MAX) {
    logits_chunks<T, O><<<dim3((a.v + CHUNK - 1) / CHUNK, a.b), NT, 0, st>>>(a);
    return check_launch("logits_process");
  }
  // Many wide rows of 16 bits with short histories: listed (256 rows of 32000 with 512 tokens 15.0 us,
  // by ranges 18.0; 64 of 163840 with 4096 and 300 biases 20.9, by ranges 28; but 64 of 163840 with
  // 16000 44 against 36, 16 of 163840 with 1024 8.3 against 7.8, and fp32 rows are no faster).
  if constexpr (sizeof(T) == 2) {
    if (a.length < LENGTH_LISTED && a.length <= a.v / 16 && (long long)a.b * a.v >= 1LL << 22) {
      c = (a.v + RANGE_LISTED - 1) / RANGE_LISTED;
      while ((long long)a.b * c * 2 <= 592 && range_of(2 * c) >= 2048) c *= 2;
      VERACE_REQUIRE((long long)a.b * c <= 0x7fffffffLL, VERACE_ERR_UNSUPPORTED, "logits_process: %d rows of %d", a.b, a.v);
      auto kern = logits_listed<T, O>;
      static std::atomic<uint64_t> ready{0};
      if (int rc = raise_limit(reinterpret_cast<const void*>(kern), ready, 2 * RANGE_LISTED)) return rc;
      kern<<<(unsigned)((long long)a.b * c), NT, range_of(c) * 2, st>>>(a, c, range_of(c));
      return check_launch("logits_process");
    }
  }
  // long histories, which every CTA of a row reads: fewer and larger ranges; otherwise more of
  // them (of 2048 tokens at least) while the rows leave the device empty
  const bool long_history = a.length > 16384;
  const int most = long_history ? RANGE_LONG : RANGE;
  c = (a.v + most - 1) / most;
  while ((long long)a.b * c * 2 <= 296 && range_of(2 * c) >= 2048) c *= 2;
  return long_history ? launch_ranges<T, O, true, true>(a, c, range_of(c), st)
                      : launch_ranges<T, O, true, false>(a, c, range_of(c), st);
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
  // (indices run a stride past the end in 32 bits)
  VERACE_REQUIRE(v <= 1 << 30 && length <= 1 << 30 && n_bias <= 1 << 30, VERACE_ERR_UNSUPPORTED,
                 "logits_process: %d tokens, histories of %d, %d biases (at most 2^30 of each)", v, length, n_bias);
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
