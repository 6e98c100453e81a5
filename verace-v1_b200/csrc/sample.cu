// Choice of a token per row of logits l (NaN counts as -inf).  z = (l - max l) / T, which no T
// sends above 0; kept are the tokens with l at least the k-th largest, then (over those) with
// less than p of the mass exp(z) above them, and with exp(z) >= min_p.  Equal values stand or fall together, so the kept
// set depends on no order.  token = argmax over the kept of z - log(noise), the lowest index
// on ties: with noise drawn from Exp(1) this is a draw from the softmax over the kept (the
// smallest of exponentials with rates w_i is i with probability w_i / sum w).  T = 0 takes
// the largest logit.  logprob = log softmax(z)[token] over the whole row (T = 0: of l).
//
// Two kernels.  sample_cluster: a cluster of CTAs per row, the row read once and kept in shared
// memory, where the passes after the first run.  The cuts by count (k) and by mass (p) come from
// histograms in shared memory, joined over the cluster: first 512 bins linear in z (values
// near the top spread over many bins; bins of the float's bits would put most of a row into a
// handful), then within the bin of the cut 512 bins of the values' order-preserving keys, until
// a bin holds one value or one key: two or three levels for most rows, five at worst.
// sample_rows: one CTA per row that reads it again for every pass; for rows that no cluster
// holds.  Mass is summed in 2^-40 fixed point, so that the order of the atomics changes nothing.
#include "common.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace verace {
namespace {

namespace cg = cooperative_groups;

constexpr int NT = 1024;       // threads of sample_rows
constexpr int CT = 512;        // threads of sample_cluster's CTAs: two or three of them share an SM
constexpr int BINS = 512;

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

template <int WARPS = NT / 32, typename F>
__device__ __forceinline__ float block_reduce(float x, float* s, F f) {
  const int lane = threadIdx.x % 32, w = threadIdx.x / 32;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  __syncthreads();
  if (lane == 0) s[w] = x;
  __syncthreads();
  x = s[lane % WARPS];
#pragma unroll
  for (int o = WARPS / 2; o > 0; o >>= 1) x = f(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}

template <typename T>
__global__ void __launch_bounds__(NT) sample_rows(SampleArgs a) {
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

// ------------------------------------------------------------------ a cluster per row
// A histogram over a CTA's part of the row: how many values a bin has, and by how much their
// weights fall short of the bin's largest (exp(-bin / 16), less than a sixteenth), in 2^-20 of it:
// 16 bits a value, so that no sum over 65536 of them overflows.
struct Hist {
  uint32_t count[BINS], lack[BINS];
};
constexpr int LIST = 4096;             // values kept by the first level that a CTA lists
struct Shared {
  Hist hist[2];                        // of alternate levels: a level clears the next one's
  float top, ties, rest;
  unsigned long long best;
  float red[32];
  unsigned long long red64[32];
  uint32_t list[LIST];
  uint32_t listed;
  int bin;
  uint32_t found;                      // the values in it
  unsigned long long left;             // of the target, before that bin
};

// Every CTA's copy of one field, combined in rank order.
template <typename V, typename F>
__device__ __forceinline__ V over_cluster(cg::cluster_group& cl, V* field, F f) {
  const int n = cl.num_blocks();
  V v = *cl.map_shared_rank(field, 0);
#pragma unroll 8
  for (int i = 1; i < n; ++i) v = f(v, *cl.map_shared_rank(field, i));
  return v;
}

// Adds a value of weight `part` times its first-level bin's largest (the last bin's weights, below
// exp(-31), are left out).
__device__ __forceinline__ void add_to(Hist& h, int b, bool by_mass, float part) {
  atomicAdd(&h.count[b], 1u);
  if (by_mass) {
    const uint32_t lack = (uint32_t)fminf(fmaxf((1.f - part) * 1048576.f + 0.5f, 0.f), 65535.f);
    if (lack) atomicAdd(&h.lack[b], lack);
  }
}

// The cluster's histogram h: the first bin at which the running count (or mass) reaches `left`,
// the last one if none does.  Thread i has bin i.  Masses are in
// units of exp(-bin / 16) (`first`) or of `weight`.  Sets s.bin, s.found and s.left.
__device__ void find_bin(cg::cluster_group& cl, Shared& s, int h, bool by_mass, bool first, float p,
                         unsigned long long left, float weight) {
  static_assert(BINS == CT, "a bin a thread");
  const int tid = threadIdx.x, lane = tid % 32, w = tid / 32, n = cl.num_blocks();
  uint32_t count = 0;
  unsigned long long lack = 0;
#pragma unroll 8
  for (int i = 0; i < n; ++i) {
    const Hist* r = &cl.map_shared_rank(&s, i)->hist[h];
    count += r->count[tid];
    if (by_mass) lack += r->lack[tid];
  }
  // in 2^-40 of the largest weight
  const float unit = !first ? weight : tid == BINS - 1 ? 0.f : expf(-0.0625f * tid);
  const unsigned long long mine =
      by_mass ? (unsigned long long)((double)(((unsigned long long)count << 20) - lack) * (1048576.0 * unit)) : count;
  unsigned long long run = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long v = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += v;
  }
  if (lane == 31) s.red64[w] = run;
  __syncthreads();
  unsigned long long before = 0, total = 0;
#pragma unroll
  for (int i = 0; i < CT / 32; ++i) {
    const unsigned long long v = s.red64[i];
    before += i < w ? v : 0;
    total += v;
  }
  run += before;
  if (by_mass && first) {
    // a token is kept while the mass strictly above it is below p * total
    left = (unsigned long long)ceil((double)p * (double)total);
    if (left < 1) left = 1;
  }
  if ((run >= left && run - mine < left) || (tid == BINS - 1 && run < left)) {
    s.bin = tid;
    s.found = count;
    s.left = left - (run - mine);
  }
  __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(CT, 2) sample_cluster(SampleArgs a, int chunk) {
  extern __shared__ __align__(16) uint8_t raw[];
  __shared__ __align__(16) Shared s;
  T* xs = reinterpret_cast<T*>(raw);
  cg::cluster_group cl = cg::this_cluster();
  const int tid = threadIdx.x, lane = tid % 32, rank = cl.block_rank();
  const int row = blockIdx.x / cl.num_blocks();
  const T* l = static_cast<const T*>(a.logits) + row * a.ld;
  const float t = a.t_rows ? a.t_rows[row] : a.t;
  const bool greedy = !(t > 0.f);
  const float ts = greedy ? 1.f : t;
  const int k = a.k_rows ? a.k_rows[row] : a.k;
  const float p = a.p_rows ? a.p_rows[row] : a.p;
  const float minp = a.minp_rows ? a.minp_rows[row] : a.minp;
  const float log_minp = minp > 0.f ? logf(minp) : -INFINITY;

  // ---- this CTA's part of the row
  const int i0 = rank * chunk, n = max(0, min(chunk, a.v - i0));
  const T* src = l + i0;
  float top = -INFINITY;
  constexpr int E = 16 / sizeof(T);
  const T none = from_f32<T>(-INFINITY);
  int done = 0;
  if (reinterpret_cast<size_t>(src) % 16 == 0) {
    done = n / E * E;
#pragma unroll 4
    for (int j = tid * E; j < done; j += CT * E) {
      uint4 u = __ldg(reinterpret_cast<const uint4*>(src + j));
      float f[E];
      if constexpr (E == 4) {
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y);
        f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
      } else {
        unpack8<T>(u, f);
      }
      float most = f[0];                        // (fmaxf passes over a NaN)
      bool nan = f[0] != f[0];
#pragma unroll
      for (int e = 1; e < E; ++e) most = fmaxf(most, f[e]), nan |= f[e] != f[e];
      *reinterpret_cast<uint4*>(xs + j) = u;
      if (nan) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (f[e] != f[e]) xs[j + e] = none;
      }
      top = fmaxf(top, most);
    }
  }
#pragma unroll 8
  for (int j = done + tid; j < n; j += CT) {
    const T u = src[j];
    const float f = to_f32(u);
    xs[j] = f != f ? none : u;
    top = fmaxf(top, f);
  }
  const int n8 = (n + 7) / 8;
  if (tid < n8 * 8 - n) xs[n + tid] = none;
  // f(eight values, the first one's index in the CTA's part)
  auto each = [&](auto f) {
    for (int j = tid; j < n8; j += CT) {
      float v[8];
      if constexpr (sizeof(T) == 4) {
        const float4 u = reinterpret_cast<const float4*>(xs)[2 * j], g = reinterpret_cast<const float4*>(xs)[2 * j + 1];
        v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
        v[4] = g.x; v[5] = g.y; v[6] = g.z; v[7] = g.w;
      } else {
        unpack8<T>(reinterpret_cast<const uint4*>(xs)[j], v);
      }
      f(v, 8 * j);
    }
  };
  for (int i = tid; i < BINS; i += CT) s.hist[0].count[i] = 0, s.hist[0].lack[i] = 0;
  if (tid == 0) s.best = 0, s.listed = 0;
  top = block_reduce<CT / 32>(top, s.red, [](float u, float v) { return fmaxf(u, v); });
  if (tid == 0) s.top = top;
  cl.sync();
  top = over_cluster(cl, &s.top, [](float u, float v) { return fmaxf(u, v); });
  if (top == -INFINITY) {              // (the same for every CTA of the cluster)
    if (rank == 0 && tid == 0) a.tokens[row] = -1, a.logprobs[row] = -INFINITY;
    cl.sync();
    return;
  }

  // ---- log sum, and the first histogram
  const bool cut_k = !greedy && k > 0 && k < a.v, cut_p = !greedy && p < 1.f;
  const float inv = 1.f / ts, per = 16.f * inv;         // bins of 1/16 in z
  auto below = [&](float x) { return x == top ? 0.f : top - x; };
  // the first-level bin of a value, not yet cut to a whole number
  auto place = [&](float x) { return fminf(below(x) * per, (float)(BINS - 1)); };
  auto weight = [&](float d) { return __expf(-d * inv); };
  // a weight in units of its first-level bin's largest
  auto part_of = [&](float d, int b) { return __expf(0.0625f * b - d * inv); };
  // keys: order-preserving, without the bits that a 16-bit type leaves empty
  constexpr int EMPTY = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  auto key = [&](float x) { return key_of(x + 0.f) >> EMPTY; };
  float ties = 0.f, rest = 0.f;
  const bool cuts = cut_k || cut_p, mass = cut_p && !cut_k;
  each([&](const float (&v)[8], int) {
    float d[8], e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      d[i] = below(v[i]);
      e[i] = weight(d[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      ties += d[i] == 0.f ? 1.f : 0.f;
      rest += d[i] == 0.f ? 0.f : e[i];
    }
    if (cuts) {
      int b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) b[i] = (int)place(v[i]);
      if (mass) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = part_of(d[i], b[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] > -INFINITY) add_to(s.hist[0], b[i], mass, e[i]);
    }
  });
  {
    // both sums at once
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      ties += __shfl_xor_sync(0xffffffffu, ties, o);
      rest += __shfl_xor_sync(0xffffffffu, rest, o);
    }
    __syncthreads();
    if (lane == 0) s.red[tid / 32] = ties, s.red[16 + tid / 32] = rest;
    __syncthreads();
    if (tid == 0) {
      ties = rest = 0.f;
      for (int i = 0; i < CT / 32; ++i) ties += s.red[i], rest += s.red[16 + i];
      s.ties = ties, s.rest = rest;
    }
  }
  cl.sync();
  ties = over_cluster(cl, &s.ties, [](float u, float v) { return u + v; });
  rest = over_cluster(cl, &s.rest, [](float u, float v) { return u + v; });
  const float lse = logf(ties) + log1pf(rest / ties);

  // ---- the cuts: what is kept is every value in a bin before `edge`, and in it the keys from
  // `least` on
  int edge = BINS;
  uint32_t least = 0;
  int h = 0;
  bool listing = false;
  // f(value, index) for what the first level kept, from the list where that holds it all
  auto visit = [&](auto f) {
    if (listing) {
      for (int i = tid; i < (int)s.listed; i += CT) f(to_f32(xs[s.list[i]]), (int)s.list[i]);
    } else {
      each([&](const float (&v)[8], int j) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (v[i] > -INFINITY) f(v[i], j + i);
      });
    }
  };
  for (int by_mass = 0; by_mass < 2; ++by_mass) {
    if (by_mass ? !cut_p : !cut_k) continue;
    const int kept_edge = edge;
    const uint32_t kept_least = least;
    auto kept = [&](float x) {
      const float f = place(x);
      return f < (float)kept_edge || (f < (float)(kept_edge + 1) && key(x) >= kept_least);
    };
    if (by_mass && cut_k) {            // the mass of what k kept
      h ^= 1;
      for (int i = tid; i < BINS; i += CT) s.hist[h].count[i] = 0, s.hist[h].lack[i] = 0;
      __syncthreads();
      visit([&](float x, int) {
        if (kept(x)) {
          const int b = (int)place(x);
          add_to(s.hist[h], b, true, part_of(below(x), b));
        }
      });
      cl.sync();
    }
    find_bin(cl, s, h, by_mass, true, p, (unsigned long long)k, 1.f);
    const int cut = s.bin;
    uint32_t from = 0;
    unsigned long long left = s.left;
    bool more = s.found > 1 && !(!by_mass && left >= s.found);
    if (!listing) {
      // from here on only the values up to this bin matter
      each([&](const float (&v)[8], int j) {
        uint32_t in = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) in |= (v[i] > -INFINITY && place(v[i]) < (float)(cut + 1) ? 1u : 0u) << i;
        if (in) {
          uint32_t at = atomicAdd(&s.listed, (uint32_t)__popc(in));
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (in >> i & 1u) {
              if (at < LIST) s.list[at] = (uint32_t)(j + i);
              ++at;
            }
        }
      });
      __syncthreads();
      listing = s.listed <= LIST;
    }
    if (more) {
      // the keys that bin `cut` can hold (its bounds, widened by the roundings of place)
      const float wide = 1.f / per, slack = (fabsf(top) + (cut + 1) * wide) * 1e-6f;
      uint32_t lo = cut == BINS - 1 ? key_of(-INFINITY) + 1 : key_of(value(top - (cut + 1) * wide - slack));
      uint32_t hi = key_of(fminf(top, top - cut * wide + slack));
      if (!(fabsf(top) <= 3.4028235e38f)) lo = key_of(-INFINITY) + 1, hi = key_of(top);
      lo >>= EMPTY;
      hi >>= EMPTY;
      if (lo > hi) lo = hi;
      const float unit = cut == BINS - 1 ? 0.f : expf(-0.0625f * cut);
      while (more) {
        const int bits = 32 - __clz(hi - lo), shift = bits > 9 ? bits - 9 : 0;
        h ^= 1;
        // (this histogram was last read before the cluster's last barrier but one)
        for (int i = tid; i < BINS; i += CT) s.hist[h].count[i] = 0, s.hist[h].lack[i] = 0;
        __syncthreads();
        visit([&](float x, int) {
          const float f = place(x);
          if (f >= (float)cut && f < (float)(cut + 1)) {
            const uint32_t q = key(x);
            if (q >= lo && q <= hi && (cut < kept_edge || q >= kept_least))
              add_to(s.hist[h], BINS - 1 - (int)((q - lo) >> shift), by_mass, part_of(below(x), cut));   // descending
          }
        });
        cl.sync();
        find_bin(cl, s, h, by_mass, false, p, left, unit);
        const uint32_t b = BINS - 1 - s.bin;
        left = s.left;
        from = lo + (b << shift);
        more = shift > 0 && s.found > 1 && !(!by_mass && left >= s.found);
        if (shift > 0) hi = min(hi, from + ((1u << shift) - 1));
        lo = from;
        __syncthreads();
      }
    }
    if (cut < edge) edge = cut, least = from;
    else if (cut == edge) least = max(least, from);
    cl.sync();                         // before the histograms are used again
  }

  // ---- the choice
  // The score is l / T - log(noise) where that is in range, z - log(noise) where it is not.  Most
  // values are far from the best so far: fast arithmetic (off by less than 1e-4 and 1e-5 of its
  // terms) passes over them.
  const float* noise = a.noise + row * a.noise_ld + i0;
  const float shift = top * inv;
  const bool direct = fabsf(top / ts) <= 3.4028235e38f;
  float best = -INFINITY;
  int at = -1;
  if (greedy) {
    each([&](const float (&v)[8], int j) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] > best) best = v[i], at = j + i;
    });
  } else if (listing) {
    visit([&](float x, int j) {
      const float f = place(x), d = below(x);
      if (f > (float)edge && (f >= (float)(edge + 1) || key(x) < least)) return;
      if (f >= (float)edge && key(x) < least) return;
      if (minp > 0.f && d != 0.f && !(-d * inv >= log_minp)) return;
      const float score = (direct ? x / ts : -(d / ts)) - logf(__ldg(noise + j));
      if (score > best || (score == best && score > -INFINITY && j < at)) best = score, at = j;
    });
  } else {
    const bool wide = reinterpret_cast<size_t>(noise) % 16 == 0;
    float bound = -INFINITY;             // no score of the warp's that counts is below this
    for (int j0 = 0; j0 < n8; j0 += CT) {
      // (whole warps: the bound is the warp's)
      const int j8 = j0 + tid, j = 8 * j8;
      const bool live = j8 < n8;
      float v[8];
      if (live) {
        if constexpr (sizeof(T) == 4) {
          const float4 u = reinterpret_cast<const float4*>(xs)[2 * j8], g = reinterpret_cast<const float4*>(xs)[2 * j8 + 1];
          v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
          v[4] = g.x; v[5] = g.y; v[6] = g.z; v[7] = g.w;
        } else {
          unpack8<T>(reinterpret_cast<const uint4*>(xs)[j8], v);
        }
      }
      uint32_t in = 0;
      float r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        bool ok = live && v[i] > -INFINITY;
        if (edge < BINS) {
          const float f = place(v[i]);
          ok = ok && (f < (float)edge || (f < (float)(edge + 1) && key(v[i]) >= least));
        }
        const float d = below(v[i]);
        if (minp > 0.f) ok = ok && (d == 0.f || -d * inv >= log_minp);
        in |= (ok ? 1u : 0u) << i;
        r[i] = 1.f;
      }
      // all noise first: one trip to memory for the eight
      if (wide && in == 255u) {
        const float4 u = __ldg(reinterpret_cast<const float4*>(noise + j));
        const float4 g = __ldg(reinterpret_cast<const float4*>(noise + j + 4));
        r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
        r[4] = g.x; r[5] = g.y; r[6] = g.z; r[7] = g.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (in >> i & 1u) r[i] = __ldg(noise + j + i);
      }
      float high[8], sure = -INFINITY;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = -below(v[i]) * inv, l = __logf(r[i]), near = (direct ? shift + z : z) - l;
        const float off = 1e-4f + 1e-5f * (fabsf(shift) + fabsf(z) + fabsf(l));
        high[i] = near + off;
        if (in >> i & 1u) sure = fmaxf(sure, near - off);
      }
      const uint32_t most = __reduce_max_sync(0xffffffffu, key_of(sure + 0.f));
      bound = fmaxf(bound, __uint_as_float(most ^ (most >> 31 ? 0x80000000u : 0xffffffffu)));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if ((in >> i & 1u) && !(high[i] < bound)) {
          const float d = below(v[i]);
          const float score = (direct ? v[i] / ts : -(d / ts)) - logf(r[i]);
          if (score > best) best = score, at = j + i;     // (a thread's indices rise: the lowest on ties)
        }
    }
  }
  unsigned long long choice =
      at < 0 ? 0 : ((unsigned long long)key_of(best + 0.f) << 32) | (0xffffffffu - (uint32_t)(i0 + at));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long v = __shfl_xor_sync(0xffffffffu, choice, o);
    if (v > choice) choice = v;
  }
  if (lane == 0 && choice) atomicMax(&s.best, choice);
  cl.sync();
  if (rank == 0 && tid == 0) {
    const unsigned long long c = over_cluster(
        cl, &s.best, [](unsigned long long u, unsigned long long v) { return u > v ? u : v; });
    if (c == 0) {
      a.tokens[row] = -1, a.logprobs[row] = -INFINITY;
    } else {
      const int i = (int)(0xffffffffu - (uint32_t)c);
      a.tokens[row] = i;
      a.logprobs[row] = scaled(value(to_f32(l[i])), top, ts) - lse;
    }
  }
  cl.sync();
}

constexpr int CHUNK_MAX = 176 * 1024;   // bytes of a row in a CTA (one an SM beyond 80 KB)

template <typename T>
int run(const SampleArgs& a, cudaStream_t st) {
  auto chunk_of = [&](int c) { return ((a.v + c - 1) / c + 7) / 8 * 8; };
  // CTAs per row: as few as two CTAs an SM hold it with, more (of 2048 values at least) while
  // the rows alone leave the device empty
  int c = 1;
  while (c < 16 && (size_t)chunk_of(c) * sizeof(T) > 80 * 1024) c *= 2;
  while (c < 8 && (long long)a.b * c * 2 <= 296 && chunk_of(2 * c) >= 2048) c *= 2;
  const size_t bytes = (size_t)chunk_of(c) * sizeof(T);
  if (bytes > CHUNK_MAX || (long long)a.b * c > 0x7fffffffLL) {
    sample_rows<T><<<a.b, NT, 0, st>>>(a);
    return check_launch("sample");
  }
  auto kern = sample_cluster<T>;
  static std::atomic<uint64_t> ready{0};      // devices whose limits are raised
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, CHUNK_MAX));
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.b * c));
  cfg.blockDim = dim3(CT);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VERACE_CUDA(cudaLaunchKernelEx(&cfg, kern, a, chunk_of(c)));
  return check_launch("sample");
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
  if (dtype == VERACE_F32) return run<float>(a, st);
  if (dtype == VERACE_BF16) return run<__nv_bfloat16>(a, st);
  return run<__half>(a, st);
}
