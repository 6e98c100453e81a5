// Products of one to a few tokens by dot products, the third engine behind linear.cu:
//     out(m, n) = epilogue(sum_k x(m, k) W(n, k))
// Bound: the weights' bytes; at small sizes the launch.  No tensor core: a weight is used for at most
// MT tokens, which the FMA pipes keep up with (a 16-byte vector of bf16 weights a lane costs 8 unpacking
// instructions and 8 FMAs a token; the memory rate leaves an SM 88 issue slots for it), and a kernel
// without TMEM, barriers and clusters starts and ends sooner: 1 x 1024 x 1024 bf16 2.5 us in a chain of calls, 1 x 8192 x
// 4096 13.8 us (4.9 TB/s); 8 x 4096 x 4096 fp32, whose operands are used as they are, 23 us.  (The rule between the
// engines, with both sides' times, is in linear.cu.)
//
// A warp takes RG rows of W (gated: RG of each weight) and MT tokens; its lanes walk K in 16-byte
// vectors, RG loads of W in flight beside each other for every step.  Few rows: the warps of a CTA share
// K and join their sums through shared memory in a fixed order.  fp32 rows that are not 16-byte aligned are
// read value by value, in the same order.  More tokens than MT: CTAs of the same rows run beside each other and share W in L2.
#include "linear_tc.cuh"

#include <cuda_fp8.h>

namespace verace {
namespace {

using namespace lin;

constexpr int WARPS = 8;

struct Args {
  const void *x, *w, *w_up;
  long long ldx, ldw;
  long long M, N, K;
  int share;            // warps that share a row's K: 1, 2, 4 or 8
  long long groups;     // of RG rows
  Epilogue e;
};

// a lane's vector as loaded, and its values
template <typename T, bool VEC>
struct Lot {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void load(const T* p, long long left) {   // (left: values up to the row's end)
    if constexpr (VEC) {
      raw = *reinterpret_cast<const uint4*>(p);
    } else {
      const uint32_t* f = reinterpret_cast<const uint32_t*>(p);
      raw = make_uint4(f[0], left > 1 ? f[1] : 0u, left > 2 ? f[2] : 0u, left > 3 ? f[3] : 0u);
    }
  }
  // values from `left` on are 0: what lies behind a row's end is not read as a number
  __device__ __forceinline__ void values(long long left, float (&v)[N]) const {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y);
      v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
    } else if constexpr (sizeof(T) == 2) {
      unpack8<T>(raw, v);
    } else {
      const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (16 * (i & 1))), __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
    if (left < N) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j >= left) v[j] = 0.f;
    }
  }
};

template <bool GATED>
__device__ __forceinline__ void finish(const Epilogue& e, long long m, long long n, float g, float u) {
  if (e.col_scale) {
    const float rs = e.row_scale[m];
    g = scaled_by(g, rs, e.col_scale[n]);
    if (GATED) u = scaled_by(u, rs, e.up_scale[n]);
  }
  if (!GATED && e.bias) g += load_as(e.bias, n, e.bias_type);
  if (e.pre) {
    e.pre[m * e.ld + n] = g;
    if (GATED) e.pre_up[m * e.ld + n] = u;
  }
  float v[1] = {g}, w[1] = {u};
  if (e.type == VERACE_F32) activate<GATED, false>(e, v, w);
  else activate<GATED, true>(e, v, w);
  g = v[0];
  if (!GATED && e.residual) g += load_as(e.residual, m * e.ld_res + n, e.type);
  store_as(e.out, m * e.ld + n, g, e.type);
}

template <typename T, int MT, int RG, bool GATED, bool VEC>
__global__ void __launch_bounds__(32 * WARPS) dot_product(const __grid_constant__ Args p) {
  constexpr int H = GATED ? 2 : 1, SUMS = MT * RG, STEP = 4 / RG > 1 ? 4 / RG : 1;   // STEP: vectors of a row in flight
  static_assert(SUMS <= 32, "a lane holds one output");
  using L = Lot<T, VEC>;
  __shared__ float join[H][WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = warp % p.share;
  const long long group = (long long)blockIdx.y * (WARPS / p.share) + warp / p.share;
  const long long m0 = (long long)blockIdx.x * MT, n0 = group * RG;
  float acc[H][MT][RG] = {};
  depend();
  if (group < p.groups) {
    const T* x[MT];
    const T* w[H][RG];
#pragma unroll
    for (int t = 0; t < MT; ++t) x[t] = static_cast<const T*>(p.x) + min(m0 + t, p.M - 1) * p.ldx;
#pragma unroll
    for (int r = 0; r < RG; ++r) {
      const long long row = min(n0 + r, p.N - 1) * p.ldw;
      w[0][r] = static_cast<const T*>(p.w) + row;
      if (GATED) w[H - 1][r] = static_cast<const T*>(p.w_up) + row;
    }
    const int stride = 32 * p.share * L::N;
    for (long long k = (32 * part + lane) * L::N; k < p.K; k += (long long)STEP * stride) {
      L lw[STEP][H][RG];
#pragma unroll
      for (int s = 0; s < STEP; ++s)
        if (s == 0 || k + s * stride < p.K)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int r = 0; r < RG; ++r) lw[s][h][r].load(w[h][r] + k + s * stride, p.K - k - s * stride);
#pragma unroll
      for (int s = 0; s < STEP; ++s) {
        const long long at = k + s * stride, left = p.K - at;
        if (s > 0 && left <= 0) break;
        float xv[MT][L::N];
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          L lx;
          lx.load(x[t] + at, left);
          lx.values(left, xv[t]);
        }
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int r = 0; r < RG; ++r) {
            float wv[L::N];
            lw[s][h][r].values(left, wv);
#pragma unroll
            for (int t = 0; t < MT; ++t)
#pragma unroll
              for (int j = 0; j < L::N; ++j) acc[h][t][r] = fmaf(xv[t][j], wv[j], acc[h][t][r]);
          }
      }
    }
  }
  // the lanes' sums; lane i keeps output i
  float mine[H] = {};
#pragma unroll
  for (int h = 0; h < H; ++h)
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int r = 0; r < RG; ++r) {
        float s = acc[h][t][r];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == t * RG + r) mine[h] = s;
      }
  if (p.share > 1) {
#pragma unroll
    for (int h = 0; h < H; ++h) join[h][warp][lane] = mine[h];
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int h = 0; h < H; ++h)
      for (int i = 1; i < p.share; ++i) mine[h] += join[h][warp + i][lane];
  }
  const long long m = m0 + lane / RG, n = n0 + lane % RG;
  if (lane < SUMS && group < p.groups && m < p.M && n < p.N) finish<GATED>(p.e, m, n, mine[0], mine[H - 1]);
}

template <typename T, int MT, int RG, bool GATED, bool VEC>
int launch(const Product& p, cudaStream_t st) {
  Args a{};
  a.x = p.a.p; a.w = p.b[0].p; a.w_up = p.b[1].p;
  a.ldx = p.a.ld; a.ldw = p.b[0].ld;
  a.M = p.M; a.N = p.N; a.K = p.K;
  a.e = p.e;
  a.groups = (p.N + RG - 1) / RG;
  const long long tokens = (p.M + MT - 1) / MT, vectors = p.K * sizeof(T) / 512;
  // warps share a row until 16 of them an SM have work, each at least four vectors of it a lane
  a.share = 1;
  while (a.share < WARPS && a.groups * tokens * a.share < 148 * 16 && vectors >= 4 * a.share) a.share *= 2;
  const long long blocks = (a.groups * a.share + WARPS - 1) / WARPS;
  VERACE_REQUIRE(tokens < 1LL << 31 && blocks <= 65535, VERACE_ERR_UNSUPPORTED, "linear: %lld x %lld outputs are too many", p.M,
                 p.N);
  return launch_after("dot_product", dot_product<T, MT, RG, GATED, VEC>, dim3((unsigned)tokens, (unsigned)blocks), 32 * WARPS, 0,
                      st, 1, a);
}

template <typename T, int MT, int RG, bool VEC = true>
int by_gate(const Product& p, cudaStream_t st) {
  if constexpr (RG >= 2) {
    if (p.gated) return launch<T, MT, RG / 2, true, VEC>(p, st);
  } else {
    if (p.gated) return launch<T, MT, 1, true, VEC>(p, st);
  }
  return launch<T, MT, RG, false, VEC>(p, st);
}

}  // namespace

namespace lin {

// x and W stored [M][K] and [N][K], one segment; p.type may be VERACE_F32 here.
int product_dot(const Product& p, cudaStream_t st) {
  if (p.type == VERACE_F32) {
    const bool vec = (((size_t)p.a.p | (size_t)p.b[0].p | (size_t)p.b[1].p) % 16 | (p.a.ld | p.b[0].ld) % 4) == 0;
    if (p.M == 1) return vec ? by_gate<float, 1, 2>(p, st) : by_gate<float, 1, 2, false>(p, st);
    if (p.M <= 4) return vec ? by_gate<float, 4, 4>(p, st) : by_gate<float, 4, 4, false>(p, st);
    return vec ? by_gate<float, 8, 4>(p, st) : by_gate<float, 8, 4, false>(p, st);
  }
  if (p.type == VERACE_E4M3)
    return p.M == 1 ? by_gate<__nv_fp8_e4m3, 1, 2>(p, st)
                    : p.M == 2 ? by_gate<__nv_fp8_e4m3, 2, 2>(p, st) : by_gate<__nv_fp8_e4m3, 4, 4>(p, st);
  if (p.type == VERACE_BF16)
    return p.M == 1 ? by_gate<__nv_bfloat16, 1, 2>(p, st)
                    : p.M == 2 ? by_gate<__nv_bfloat16, 2, 2>(p, st) : by_gate<__nv_bfloat16, 4, 4>(p, st);
  return p.M == 1 ? by_gate<__half, 1, 2>(p, st) : p.M == 2 ? by_gate<__half, 2, 2>(p, st) : by_gate<__half, 4, 4>(p, st);
}

}  // namespace lin
}  // namespace verace
