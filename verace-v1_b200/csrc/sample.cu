// Choice of a token per row of logits l (NaN counts as -inf).  z = (l - max l) / T, which no T
// sends above 0; kept are the tokens with l at least the k-th largest, then (over those) with
// less than p of the mass exp(z) above them, and with exp(z) >= min_p.  Equal values stand or fall together, so the kept
// set depends on no order.  token = argmax over the kept of z - log(noise), the lowest index
// on ties: with noise drawn from Exp(1) this is a draw from the softmax over the kept (the
// smallest of exponentials with rates w_i is i with probability w_i / sum w).  T = 0 takes
// the largest logit.  logprob = log softmax(z)[token] over the whole row (T = 0: of l).
//
// Two kernels.  sample_cluster: a cluster of CTAs per row, the row read once and kept in shared
// memory, where the passes after the first run, or (HELD false) read by each pass, from L2 mostly.  The cuts by count (k) and by mass (p) come from
// histograms in shared memory, joined over the cluster: first 512 bins linear in z (values
// near the top spread over many bins; bins of the float's bits would put most of a row into a
// handful), then within the bin of the cut 512 bins of the values' order-preserving keys, until
// a bin holds one value or one key: two or three levels for most rows, five at worst.
// sample_rows: one CTA per row that reads it again for every pass; for rows of more than 16 x 65536
// values.  Mass is summed in whole numbers (2^-40 of the largest weight; in sample_cluster's histograms
// 2^-20 of the bin's largest, and nothing for the last bin, below exp(-31)), so that the order of the
// atomics changes nothing.  A cut by p so moves only where it is within about 1e-6 of a value's edge.
//
// Bound: one read of the row, and of the noise where every value draws.  Measured on the device: one
// row of 32000 at T = 0 6.1 us (launch and cluster barriers); 64 fp32 rows of 163840 with k = 50,
// p = 0.9 and min_p 26 us for 42 MB (1.6 TB/s: two passes, the second from L2, then about eight steps
// between barriers of the cluster; one CTA a row that read it again for every step: 1924), with p alone
// 54 to 69; 256 bf16 rows of 32000 without cuts 25 us for 49 MB with the noise (2.0 TB/s: three passes with
// the cluster's barriers between, and the arithmetic per value, about 9 us of it).
#include "common.cuh"

#include <cooperative_groups.h>

#include <atomic>
#include <cstddef>

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
  const float ts = greedy ? 1.f : fminf(t, 3.4028235e38f);      // (an infinite T: as good as the largest)
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
  // the unit of mass: 2^40 to the largest weight, or so many that no sum over the row passes 64 bits
  const float unit = ldexpf(1.f, min(40, 32 + __clz(a.v)));

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
                      by_mass ? (unsigned long long)(expf(scaled(x, top, ts)) * unit + 0.5f) : 1ull);
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
constexpr int GATHER = 1024;           // listed values of a row that one CTA cuts and chooses from by itself
constexpr int LIST = 8192;             // values kept by the first level that a CTA lists (by 16-bit index)
struct Shared {
  Hist hist[2];                        // of alternate levels: a level clears the next one's
  float top, ties, rest;
  unsigned long long best;
  float red[32];
  unsigned long long red64[32];
  unsigned short list[LIST];
  uint32_t listed;
  int bin;
  uint32_t found;                      // the values in it
  unsigned long long left;             // of the target, before that bin
  unsigned long long target;           // the mass that the cut by p leaves, absolute
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
__device__ __forceinline__ float exp2_of(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float log2_of(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void add_to(Hist& h, int b, bool by_mass, float part) {
  atomicAdd(&h.count[b], 1u);
  if (by_mass) {
    const uint32_t lack = (uint32_t)fminf(fmaxf((1.f - part) * 1048576.f + 0.5f, 0.f), 65535.f);
    if (lack) atomicAdd(&h.lack[b], lack);
  }
}

// The mass that a cut by p leaves, of a total.
__device__ __forceinline__ unsigned long long target_of(float p, double total) {
  const double target = ceil((double)p * total);
  return target > 1. ? (unsigned long long)target : 1ull;
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
    left = target_of(p, (double)total);
    if (tid == 0) s.target = left;
  }
  if ((run >= left && run - mine < left) || (tid == BINS - 1 && run < left)) {
    s.bin = tid;
    s.found = count;
    s.left = left - (run - mine);
  }
  __syncthreads();
}

// HELD: the row is kept in shared memory; else every pass reads it from L2.
template <typename T, bool HELD>
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
  const float ts = greedy ? 1.f : fminf(t, 3.4028235e38f);      // (an infinite T: as good as the largest)
  const int k = a.k_rows ? a.k_rows[row] : a.k;
  const float p = a.p_rows ? a.p_rows[row] : a.p;
  const float minp = a.minp_rows ? a.minp_rows[row] : a.minp;
  const float log_minp = minp > 0.f ? logf(minp) : -INFINITY;

  // ---- this CTA's part of the row
  const int i0 = rank * chunk, n = max(0, min(chunk, a.v - i0));
  const bool cut_k = !greedy && k > 0 && k < a.v, cut_p = !greedy && p < 1.f, cuts = cut_k || cut_p;
  const float* noise = a.noise + row * a.noise_ld + i0;
  if (!greedy && !cuts && !(minp > 0.f)) {              // all of the noise is wanted: into L2 while the row is read
    for (int j = tid * 32; j < n; j += CT * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(noise + j));
  }
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
      if constexpr (HELD) *reinterpret_cast<uint4*>(xs + j) = u;
      if (HELD && nan) {
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
    if constexpr (HELD) xs[j] = f != f ? none : u;
    top = fmaxf(top, f);
  }
  top = top + 0.f;
  const float mine = top;              // the thread's largest
  const int n8 = (n + 7) / 8;
  if (HELD && tid < n8 * 8 - n) xs[n + tid] = none;
  auto values = [&](int j8, float (&v)[8]) {
    if constexpr (!HELD) {
      if (8 * j8 + 8 <= done) {
        const uint4* u = reinterpret_cast<const uint4*>(src + 8 * j8);
        const uint4 g = __ldg(u);
        if constexpr (sizeof(T) == 4) {
          const uint4 q = __ldg(u + 1);
          v[0] = __uint_as_float(g.x); v[1] = __uint_as_float(g.y);
          v[2] = __uint_as_float(g.z); v[3] = __uint_as_float(g.w);
          v[4] = __uint_as_float(q.x); v[5] = __uint_as_float(q.y);
          v[6] = __uint_as_float(q.z); v[7] = __uint_as_float(q.w);
        } else {
          unpack8<T>(g, v);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 8 * j8 + i < n ? to_f32(src[8 * j8 + i]) : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaxf(v[i], -INFINITY);          // (a NaN's place)
    } else if constexpr (sizeof(T) == 4) {
      const float4 u = reinterpret_cast<const float4*>(xs)[2 * j8], g = reinterpret_cast<const float4*>(xs)[2 * j8 + 1];
      v[0] = u.x; v[1] = u.y; v[2] = u.z; v[3] = u.w;
      v[4] = g.x; v[5] = g.y; v[6] = g.z; v[7] = g.w;
    } else {
      unpack8<T>(reinterpret_cast<const uint4*>(xs)[j8], v);
    }
  };
  // f(eight values, the first one's index in the CTA's part)
  auto each = [&](auto f) {
    for (int j = tid; j < n8; j += CT) {
      float v[8];
      values(j, v);
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
  const float inv = 1.f / ts, per = 16.f * inv;         // bins of 1/16 in z
  auto below = [&](float x) { return x == top ? 0.f : top - x; };
  // the first-level bin of a value, not yet cut to a whole number
  auto place = [&](float x) { return fminf(below(x) * per, (float)(BINS - 1)); };
  // a weight in units of its first-level bin's largest
  auto part_of = [&](float d, int b) { return __expf(0.0625f * b - d * inv); };
  // keys: order-preserving, without the bits that a 16-bit type leaves empty
  constexpr int EMPTY = sizeof(T) == 4 ? 0 : std::is_same<T, __half>::value ? 13 : 16;
  auto key = [&](float x) { return key_of(x + 0.f) >> EMPTY; };
  // For a k well below the number of threads, k of the threads' largest values bound the k-th
  // largest from below: what is under that bound goes into no histogram, and what is not is listed
  // in the pass that sums the weights.
  int h = 0, edge = BINS;
  uint32_t least = 0;
  bool listing = false;
  const bool bounded = cut_k && k <= (int)cl.num_blocks() * (CT / 2);
  const bool by_least = !greedy && !cuts && minp > 0.f;
  float list_from = INFINITY;
  if (bounded) {
    if (mine > -INFINITY) atomicAdd(&s.hist[0].count[(int)place(mine)], 1u);
    cl.sync();
    find_bin(cl, s, 0, false, true, p, (unsigned long long)k, 1.f);
    h = 1;
    for (int i = tid; i < BINS; i += CT) s.hist[1].count[i] = 0, s.hist[1].lack[i] = 0;
  }
  // a value that every value of bins up to `bin` reaches (place's roundings allowed for)
  auto floor_of = [&](int bin) {
    if (bin >= BINS - 1 || !(fabsf(top) <= 3.4028235e38f)) return -3.4028235e38f;
    const float wide = (bin + 1) * (0.0625f * ts);
    return fmaxf(top - wide - (fabsf(top) + wide) * 1e-6f, -3.4028235e38f);   // (-inf is no value: it fills)
  };
  // lists the values from `least` on
  auto list = [&](const float (&v)[8], int j, float least) {
    uint32_t in = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) in |= (v[i] >= least ? 1u : 0u) << i;
    if (in) {
      uint32_t at = atomicAdd(&s.listed, (uint32_t)__popc(in));
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (in >> i & 1u) {
          if (at < LIST) s.list[at] = (unsigned short)(j + i);
          ++at;
        }
    }
  };
  // f(value, index) for what is listed, or for every value where the list did not hold it
  auto visit = [&](auto f) {
    if (listing) {
      for (int i = tid; i < (int)s.listed; i += CT) f(to_f32(HELD ? xs[s.list[i]] : src[s.list[i]]), (int)s.list[i]);
    } else {
      each([&](const float (&v)[8], int j) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (v[i] > -INFINITY) f(v[i], j + i);
      });
    }
  };
  if (bounded) list_from = floor_of(s.bin);
  if (by_least) {
    const float deep = fmaxf(-log_minp * ts, 0.f);
    list_from = fabsf(top) <= 3.4028235e38f ? fmaxf(top - deep - (fabsf(top) + deep) * 1e-5f, -3.4028235e38f)
                                            : -3.4028235e38f;
  }
  float ties = 0.f, rest = 0.f;
  const bool mass = cut_p && !cut_k;
  const float rate = -1.44269504f * inv;         // weights as powers of two
  if (!cuts || bounded) {
    each([&](const float (&v)[8], int j) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = exp2_of(rate * (top - v[i]));
        if (v[i] == top) ties += 1.f;
        else rest += e;
      }
      if (list_from < INFINITY) list(v, j, list_from);
    });
  } else {
    each([&](const float (&v)[8], int j) {
      float d[8], e[8];
      int b[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        d[i] = below(v[i]);
        e[i] = exp2_of(rate * d[i]);
        b[i] = (int)place(v[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (d[i] == 0.f) ties += 1.f;
        else rest += e[i];
      }
      if (mass) {
#pragma unroll
        for (int i = 0; i < 8; ++i) e[i] = part_of(d[i], b[i]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] > -INFINITY) add_to(s.hist[0], b[i], mass, e[i]);
    });
  }
  {
    // both sums at once; they are joined over the cluster with the choice
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
  if (bounded || by_least) listing = s.listed <= LIST;
  if (cuts) cl.sync();

  // A short list, as it mostly is, goes to the first CTA, which sorts it: the cut by k is the value
  // at that place, the cut by p the one at which the running mass reaches the target.  (No more
  // levels and barriers over the cluster.  Comparing every value with every other instead took 60 k
  // clocks for a list of 1000.)
  const float shift = top * inv;
  // the score: l / T - log(noise) while that loses no more digits than z - log(noise), the latter beyond
  const bool direct = fabsf(top / ts) <= 64.f;
  auto score_of = [&](float x, float r) { return (direct ? x / ts : -(below(x) / ts)) - logf(r); };
  unsigned long long choice = 0;
  auto pack = [&](float score, int i) {
    return ((unsigned long long)key_of(score + 0.f) << 32) | (0xffffffffu - (uint32_t)i);
  };
  auto gather = [&] {
    const int ranks = cl.num_blocks();
    int total = 0;
    for (int q = 0; q < ranks; ++q) total += (int)min(*cl.map_shared_rank(&s.listed, q), (uint32_t)(GATHER + 1));
    if (total < 1 || total > GATHER) return false;
    if (rank > 0) return true;
    // (the histograms are read no more; the sorted keys go where this CTA's list was)
    float* gx = reinterpret_cast<float*>(s.hist);
    int* gi = reinterpret_cast<int*>(gx + GATHER);
    uint32_t* gk = reinterpret_cast<uint32_t*>(s.list);
    static_assert(sizeof(s.hist) >= GATHER * 8 && sizeof(s.list) >= GATHER * 4 && offsetof(Shared, list) % 4 == 0,
                  "gathered values fit");
    for (int e = tid; e < total; e += CT) {
      int q = 0, i = e;                          // which CTA's, and its place there
      for (int c = (int)*cl.map_shared_rank(&s.listed, 0); i >= c; c = (int)*cl.map_shared_rank(&s.listed, q)) i -= c, ++q;
      const int at = cl.map_shared_rank(&s, q)->list[i];
      gx[e] = to_f32(HELD ? cl.map_shared_rank(xs, q)[at] : l[q * chunk + at]);
      gi[e] = q * chunk + at;
    }
    __syncthreads();
    int size = 2;
    while (size < total) size *= 2;
    for (int e = tid; e < size; e += CT) gk[e] = e < total ? key_of(gx[e] + 0.f) : 0u;
    // bitonic, descending
    for (int run = 2; run <= size; run *= 2) {
      for (int apart = run / 2; apart > 0; apart /= 2) {
        __syncthreads();
        if (tid < size / 2) {
          const int i = 2 * tid - (tid & (apart - 1)), j = i + apart;
          const uint32_t u = gk[i], v = gk[j];
          if ((u < v) == ((i & run) == 0)) gk[i] = v, gk[j] = u;
        }
      }
    }
    __syncthreads();
    uint32_t cut = cut_k ? gk[min(k, total) - 1] : 1u;
    if (cut_p) {
      static_assert(GATHER == 2 * CT, "two places a thread");
      unsigned long long w[2], sum;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t q = 2 * tid + e < size ? gk[2 * tid + e] : 0u;
        const float x = __uint_as_float(q ^ (q >> 31 ? 0x80000000u : 0xffffffffu));
        w[e] = q && q >= cut ? (unsigned long long)(expf(-(below(x) / ts)) * 1099511627776.f + 0.5f) : 0ull;
      }
      sum = w[0] + w[1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long v = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += v;
      }
      if (lane == 31) s.red64[tid / 32] = sum;
      if (tid == 0) s.found = cut;
      __syncthreads();
      unsigned long long all = 0;
      for (int i = 0; i < CT / 32; ++i) {
        sum += i < tid / 32 ? s.red64[i] : 0;
        all += s.red64[i];
      }
      const unsigned long long target = cut_k ? target_of(p, (double)all) : s.target;
      // (at one place only)
      if (sum >= target && sum - w[1] < target) s.found = gk[2 * tid + 1];
      if (sum - w[1] >= target && sum - w[1] - w[0] < target) s.found = gk[2 * tid];
      __syncthreads();
      cut = s.found;
    }
    for (int e = tid; e < total; e += CT) {
      const float x = gx[e], d = below(x);
      if (key_of(x + 0.f) < cut || (minp > 0.f && d != 0.f && !(-d * inv >= log_minp))) continue;
      const float score = score_of(x, __ldg(noise + gi[e]));       // (the first CTA's noise is the row's)
      if (score > -INFINITY) choice = max(choice, pack(score, gi[e]));
    }
    return true;
  };
  bool chosen = false;
  if (bounded) {
    chosen = gather();
    if (!chosen) {
      visit([&](float x, int) { add_to(s.hist[1], (int)place(x), false, 0.f); });
      cl.sync();
    }
  }

  // ---- the cuts: what is kept is every value in a bin before `edge`, and in it the keys from
  // `least` on
  // (`listing` is each CTA's own: one CTA's list may overflow where another's holds, as for a row whose
  // ties or unmasked tokens all lie in one part.  So no barrier over the cluster and no gather may
  // depend on it; every other condition here is the same for all of a cluster's CTAs.)
  for (int by_mass = 0; by_mass < 2 && !chosen; ++by_mass) {
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
      __syncthreads();
      if (tid == 0) s.listed = 0;
      __syncthreads();
      const float from = floor_of(cut);
      each([&](const float (&v)[8], int j) { list(v, j, from); });
      __syncthreads();
      listing = s.listed <= LIST;
    }
    if (by_mass && !cut_k) {           // (nothing was listed before: every CTA has just done it)
      cl.sync();
      chosen = gather();
      if (chosen) break;
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
  float best = -INFINITY;
  int at = -1;
  if (chosen) {
  } else if (greedy) {
    each([&](const float (&v)[8], int j) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (v[i] > best) best = v[i], at = j + i;
    });
  } else if (cuts || by_least) {
    visit([&](float x, int j) {
      const float f = place(x), d = below(x);
      if (f >= (float)edge && (f >= (float)(edge + 1) || key(x) < least)) return;
      if (minp > 0.f && d != 0.f && !(-d * inv >= log_minp)) return;
      const float score = score_of(x, __ldg(noise + j));
      if (score > best || (score == best && score > -INFINITY && j < at)) best = score, at = j;
    });
  } else {
    // Every value's noise.  Fast arithmetic (off by less than `off`) passes over all that the best
    // of the warp so far rules out, which leaves a handful for the division and the logarithm.
    const bool wide = reinterpret_cast<size_t>(noise) % 16 == 0;
    const float off = direct ? 1e-3f + 1e-5f * fabsf(shift) : 1e-3f;
    float bound = -INFINITY;             // no score of the warp's that counts is below this
    for (int j0 = 0; j0 < n8; j0 += CT) {      // (whole warps)
      const int j = 8 * (j0 + tid);
      float v[8], r[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = -INFINITY, r[i] = 1.f;
      if (j < n) {
        if (wide && j + 8 <= n) {
          const float4 u = __ldg(reinterpret_cast<const float4*>(noise + j));
          const float4 q = __ldg(reinterpret_cast<const float4*>(noise + j + 4));
          r[0] = u.x; r[1] = u.y; r[2] = u.z; r[3] = u.w;
          r[4] = q.x; r[5] = q.y; r[6] = q.z; r[7] = q.w;
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (j + i < n) r[i] = __ldg(noise + j + i);
        }
        values(j / 8, v);
      }
      float high[8], log2_r[8], sure = -INFINITY, peak = -INFINITY, least_r = r[0];
#pragma unroll
      for (int i = 0; i < 8; ++i) log2_r[i] = log2_of(r[i]), least_r = fminf(least_r, r[i]);
      if (least_r < 1.17549435e-38f) {         // (log2_of takes subnormal noise for 0)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (r[i] < 1.17549435e-38f) log2_r[i] = log2_of(r[i] * 4294967296.f) - 32.f;
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float z = v[i] == top ? 0.f : (v[i] - top) * inv;
        const float near = fmaf(-0.693147181f, log2_r[i], direct ? z + shift : z), o = fmaf(-1e-6f, z, off);
        high[i] = near + o;
        peak = fmaxf(peak, high[i]);
        sure = fmaxf(sure, near - o);
      }
      const uint32_t most = __reduce_max_sync(0xffffffffu, key_of(sure + 0.f));
      bound = fmaxf(bound, __uint_as_float(most ^ (most >> 31 ? 0x80000000u : 0xffffffffu)));
      if (!(peak < bound)) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (v[i] > -INFINITY && !(high[i] < bound)) {
            const float score = score_of(v[i], r[i]);
            if (score > best) best = score, at = j + i;     // (a thread's indices rise: the lowest on ties)
          }
      }
    }
  }
  if (at >= 0) choice = pack(best, i0 + at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long v = __shfl_xor_sync(0xffffffffu, choice, o);
    if (v > choice) choice = v;
  }
  if (lane == 0 && choice) atomicMax(&s.best, choice);
  cl.sync();
  if (rank == 0 && tid < 32) {
    // a lane per CTA, joined in a fixed order
    unsigned long long c = 0;
    float all_ties = 0.f, all_rest = 0.f;
    if (lane < (int)cl.num_blocks()) {
      const Shared* r = cl.map_shared_rank(&s, lane);
      c = r->best;
      all_ties = r->ties;
      all_rest = r->rest;
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const unsigned long long u = __shfl_down_sync(0xffffffffu, c, o);
      if (u > c) c = u;
      all_ties += __shfl_down_sync(0xffffffffu, all_ties, o);
      all_rest += __shfl_down_sync(0xffffffffu, all_rest, o);
    }
    if (lane == 0) {
      const int i = (int)(0xffffffffu - (uint32_t)c);
      a.tokens[row] = c ? i : -1;
      a.logprobs[row] =
          c ? scaled(value(to_f32(l[i])), top, ts) - (logf(all_ties) + log1pf(all_rest / all_ties)) : -INFINITY;
    }
  }
  cl.sync();
}

constexpr int HELD_MAX = 80 * 1024;     // bytes of a row in a CTA: two CTAs share an SM

template <typename T, bool HELD>
int launch(const SampleArgs& a, int c, int chunk, cudaStream_t st) {
  auto kern = sample_cluster<T, HELD>;
  static std::atomic<uint64_t> ready{0};      // devices whose limits are raised
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, HELD ? HELD_MAX : 0));
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.b * c));
  cfg.blockDim = dim3(CT);
  cfg.dynamicSmemBytes = HELD ? (size_t)chunk * sizeof(T) : 0;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VERACE_CUDA(cudaLaunchKernelEx(&cfg, kern, a, chunk));
  return check_launch("sample");
}

template <typename T>
int run(const SampleArgs& a, cudaStream_t st) {
  auto chunk_of = [&](int c) { return ((a.v + c - 1) / c + 7) / 8 * 8; };
  // CTAs per row: as few as hold it, more (of 2048 values at least) while the rows alone leave
  // the device empty
  auto split = [&](int most) {
    int c = 1;
    while (c < 16 && chunk_of(c) > most) c *= 2;
    while (c < 8 && (long long)a.b * c * 2 <= 296 && chunk_of(2 * c) >= 2048) c *= 2;
    return c;
  };
  const int c = split(HELD_MAX / sizeof(T)), free = split(65536);
  if (chunk_of(free) > 65536 || (long long)a.b * c > 0x7fffffffLL) {
    sample_rows<T><<<a.b, NT, 0, st>>>(a);
    return check_launch("sample");
  }
  // Held rows take less time for a pass (64 bf16 rows of 163840, 4 CTAs a row either way: 19.9 us
  // with k and p against 20.9), but large ones more CTAs, which may be more waves (64 fp32 rows of
  // 163840: 41.7 against 26.0; 256 fp32 rows of 32000: 32.0 against 20.5).
  auto waves = [&](int c) { return ((long long)a.b * c + 295) / 296; };
  if (chunk_of(c) * (int)sizeof(T) > HELD_MAX || waves(free) < waves(c))
    return launch<T, false>(a, free, chunk_of(free), st);
  return launch<T, true>(a, c, chunk_of(c), st);
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
  // (indices run a stride past the end in 32 bits)
  VERACE_REQUIRE(v <= 1 << 30, VERACE_ERR_UNSUPPORTED, "sample: %d tokens (at most 2^30)", v);
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
