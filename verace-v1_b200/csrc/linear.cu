// Dense products of the feed-forward sub-layer with their epilogues, forward and backward:
//     linear:  out = act(x W^T + bias) + residual
//     gated:   out = act(x Wg^T) up(x Wu^T)
// fp32, bf16 or fp16, and e4m3 operands with a scale for each row.  Sums are fp32, outputs are
// rounded once.  Formulas of the activations: linear.cuh.
//
// Backward: p = d act'(pre) (gated: dg and du) in one pass over the saved sums, then
// dx = p W (dg Wg + du Wu), dW = p^T x, and the bias gradient as column sums in a fixed order.
#include "linear.cuh"

#include <cuda_fp8.h>

namespace verace {
namespace {

using namespace lin;

template <typename T>
__device__ __forceinline__ float val(T x) { return to_f32(x); }
template <>
__device__ __forceinline__ float val<__nv_fp8_e4m3>(__nv_fp8_e4m3 x) { return float(x); }

// ------------------------------------------------------------------ simple product
// out(m, n) = sum over `pairs` and k of a(m, k) b(n, k): 64 x 64 tiles, 4 x 4 a thread, through
// shared memory.  GATED: b[0] and b[1] give two sums of one row and column.
struct SimpleArgs {
  const void *a[2], *b[2];
  long long sam, sak, sbn, sbk;
  long long M, N, K;
  int pairs;
  Epilogue e;
};

__device__ __forceinline__ void finish_linear(const Epilogue& e, long long m, long long n, float v) {
  if (e.row_scale) v *= e.row_scale[m] * e.col_scale[n];
  if (e.bias) v += load_as(e.bias, n, e.bias_type);
  if (e.pre) store_as(e.pre, m * e.ld + n, v, e.type);
  by_act(e.act, e.type != VERACE_F32, [&](auto act, auto fast) { v = act_<decltype(act)::value, decltype(fast)::value>(v); });
  if (e.residual) v += load_as(e.residual, m * e.ld_res + n, e.type);
  store_as(e.out, m * e.ld + n, v, e.type);
}
__device__ __forceinline__ void finish_gated(const Epilogue& e, long long m, long long n, float g, float u) {
  if (e.row_scale) {
    g *= e.row_scale[m] * e.col_scale[n];
    u *= e.row_scale[m] * e.up_scale[n];
  }
  if (e.pre) {
    store_as(e.pre, m * e.ld + n, g, e.type);
    store_as(e.pre_up, m * e.ld + n, u, e.type);
  }
  float v = 0.f;
  by_act(e.act, e.type != VERACE_F32, [&](auto act, auto fast) {
    v = gate_<decltype(act)::value, decltype(fast)::value>(g, u, e.b1, e.b2, e.r1, e.r2);
  });
  store_as(e.out, m * e.ld + n, v, e.type);
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(256) simple_product(SimpleArgs p) {
  __shared__ float sa[16][65], sb[GATED ? 2 : 1][16][65];
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const long long n0 = (long long)blockIdx.x * 64, m0 = (long long)blockIdx.y * 64;
  float acc[GATED ? 2 : 1][4][4] = {};
  for (int pair = 0; pair < (GATED ? 1 : p.pairs); ++pair) {
    const T* a = static_cast<const T*>(p.a[pair]);
    for (long long k0 = 0; k0 < p.K; k0 += 16) {
      for (int i = tid; i < 1024; i += 256) {
        // neighbouring threads along the contiguous direction
        const int km = p.sak == 1 ? i & 15 : i >> 6, r = p.sak == 1 ? i >> 4 : i & 63;
        const bool in = m0 + r < p.M && k0 + km < p.K;
        sa[km][r] = in ? val(a[(m0 + r) * p.sam + (k0 + km) * p.sak]) : 0.f;
        const int kn = p.sbk == 1 ? i & 15 : i >> 6, c = p.sbk == 1 ? i >> 4 : i & 63;
        const bool inb = n0 + c < p.N && k0 + kn < p.K;
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h) {
          const T* b = static_cast<const T*>(p.b[GATED ? h : pair]);
          sb[h][kn][c] = inb ? val(b[(n0 + c) * p.sbn + (k0 + kn) * p.sbk]) : 0.f;
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int h = 0; h < (GATED ? 2 : 1); ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[h][i][j] = fmaf(sa[k][ty * 4 + i], sb[h][k][tx + 16 * j], acc[h][i][j]);
      __syncthreads();
    }
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const long long m = m0 + ty * 4 + i, n = n0 + tx + 16 * j;
      if (m >= p.M || n >= p.N) continue;
      if constexpr (GATED) finish_gated(p.e, m, n, acc[0][i][j], acc[1][i][j]);
      else finish_linear(p.e, m, n, acc[0][i][j]);
    }
}

template <bool GATED>
int run_simple(const SimpleArgs& p, int type, cudaStream_t st) {
  if (p.M == 0 || p.N == 0) return VERACE_OK;
  const dim3 grid((unsigned)((p.N + 63) / 64), (unsigned)((p.M + 63) / 64));
  switch (type) {
    case VERACE_F32: simple_product<float, GATED><<<grid, 256, 0, st>>>(p); break;
    case VERACE_BF16: simple_product<__nv_bfloat16, GATED><<<grid, 256, 0, st>>>(p); break;
    case VERACE_F16: simple_product<__half, GATED><<<grid, 256, 0, st>>>(p); break;
    default: simple_product<__nv_fp8_e4m3, GATED><<<grid, 256, 0, st>>>(p); break;
  }
  return check_launch("simple_product");
}

// ------------------------------------------------------------------ backward of the epilogues
// p = d act'(pre), in the products' type (rounded once: it is an operand of dx and dW).
template <typename T, typename O>
__global__ void __launch_bounds__(256) linear_slope(const O* __restrict__ d, const O* __restrict__ pre, T* __restrict__ p,
                                                    long long total, int act) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const float z = pre ? to_f32(pre[i]) : 0.f;
  float a, da = 1.f;
  by_act(act, sizeof(O) == 2, [&](auto c, auto fast) { act_slope_<decltype(c)::value, decltype(fast)::value>(z, a, da); });
  p[i] = from_f32<T>(to_f32(d[i]) * da);
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) gated_slope(const O* __restrict__ d, const O* __restrict__ gate,
                                                   const O* __restrict__ up, T* __restrict__ dg, T* __restrict__ du,
                                                   long long total, int act, float b1, float b2, float r1, float r2) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  float x = 0.f, y = 0.f;
  by_act(act, sizeof(O) == 2, [&](auto c, auto fast) {
    gate_slope_<decltype(c)::value, decltype(fast)::value>(to_f32(d[i]), to_f32(gate[i]), to_f32(up[i]), b1, b2, r1, r2, x, y);
  });
  dg[i] = from_f32<T>(x);
  du[i] = from_f32<T>(y);
}

// dbias = the column sums of d act'(pre), rows in order
template <typename T, typename O>
__global__ void __launch_bounds__(256) bias_sum(const O* __restrict__ d, const O* __restrict__ pre, T* __restrict__ out,
                                                long long m, long long n, int act) {
  const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
  if (c >= n) return;
  float s = 0.f;
  for (long long r = 0; r < m; ++r) {
    const float z = pre ? to_f32(pre[r * n + c]) : 0.f;
    float a, da = 1.f;
    by_act(act, sizeof(O) == 2, [&](auto k, auto fast) { act_slope_<decltype(k)::value, decltype(fast)::value>(z, a, da); });
    s += to_f32(d[r * n + c]) * da;
  }
  out[c] = from_f32<T>(s);
}

// ------------------------------------------------------------------ checks
constexpr long long MOST = 1 << 24;   // rows and columns of any operand

int check_sizes(const char* who, long long m, long long n, long long k) {
  VERACE_REQUIRE(m >= 0 && n >= 0 && k >= 0, VERACE_ERR_INVALID, "%s: negative size", who);
  VERACE_REQUIRE(m <= MOST && n <= MOST && k <= MOST, VERACE_ERR_UNSUPPORTED, "%s: m %lld, n %lld, k %lld too large", who, m,
                 n, k);
  return VERACE_OK;
}
int check_types(const char* who, int dtype, int out_dtype, bool eight) {
  VERACE_REQUIRE((dtype >= VERACE_F32 && dtype <= VERACE_F16) || (eight && dtype == VERACE_E4M3), VERACE_ERR_INVALID,
                 "%s: dtype %d", who, dtype);
  VERACE_REQUIRE(dtype == VERACE_E4M3 ? out_dtype >= VERACE_F32 && out_dtype <= VERACE_F16
                                      : out_dtype == dtype || out_dtype == VERACE_F32,
                 VERACE_ERR_INVALID, "%s: out_dtype %d for dtype %d", who, out_dtype, dtype);
  return VERACE_OK;
}
int check_rows(const char* who, const char* name, const void* p, long long ld, long long cols, int dtype) {
  VERACE_REQUIRE(p, VERACE_ERR_INVALID, "%s: NULL %s", who, name);
  VERACE_REQUIRE(ld >= cols, VERACE_ERR_INVALID, "%s: row stride %lld of %s < %lld", who, ld, name, cols);
  VERACE_REQUIRE(dtype == VERACE_F32 || ((size_t)p % 16 == 0 && ld * size_of(dtype) % 16 == 0), VERACE_ERR_INVALID,
                 "%s: the rows of %s must be 16-byte aligned", who, name);
  return VERACE_OK;
}

// Calls f(T(), O()) for the products' type and the outputs' of a differentiable call.
template <typename F>
int by_types(int dtype, int out_dtype, F f) {
  if (dtype == VERACE_F32) return f(float(), float());
  if (dtype == VERACE_BF16) return out_dtype == VERACE_F32 ? f(__nv_bfloat16(), float()) : f(__nv_bfloat16(), __nv_bfloat16());
  return out_dtype == VERACE_F32 ? f(__half(), float()) : f(__half(), __half());
}

Epilogue plain_out(void* out, long long ld, int type) {
  Epilogue e{};
  e.out = out; e.ld = ld; e.type = type; e.act = VERACE_ACT_NONE;
  return e;
}

}  // namespace
}  // namespace verace

using namespace verace;
using namespace verace::lin;

extern "C" size_t verace_linear_workspace(long long m, int n, int k, int dtype) { return 0; }

extern "C" int verace_linear(const void* x, long long ldx, const float* x_scale, const void* w, long long ldw,
                             const float* w_scale, const void* bias, const void* residual, long long ld_res, void* out,
                             void* pre, long long m, int n, int k, int act, int dtype, int out_dtype, void* workspace,
                             size_t workspace_bytes, void* stream) {
  constexpr const char* who = "verace_linear";
  int rc;
  if ((rc = check_sizes(who, m, n, k)) || (rc = check_types(who, dtype, out_dtype, true))) return rc;
  VERACE_REQUIRE(act >= VERACE_ACT_NONE && act <= VERACE_ACT_GELU_TANH, VERACE_ERR_INVALID, "%s: activation %d", who, act);
  if (m == 0 || n == 0) return VERACE_OK;
  if (k > 0 && ((rc = check_rows(who, "x", x, ldx, k, dtype)) || (rc = check_rows(who, "w", w, ldw, k, dtype)))) return rc;
  VERACE_REQUIRE(out && (dtype == VERACE_E4M3) == (x_scale != nullptr) && (dtype == VERACE_E4M3) == (w_scale != nullptr),
                 VERACE_ERR_INVALID, "%s: NULL out, or scales that do not go with the type", who);
  VERACE_REQUIRE(!residual || ld_res >= n, VERACE_ERR_INVALID, "%s: row stride %lld of the residual < %d", who, ld_res, n);
  SimpleArgs p{};
  p.a[0] = x; p.b[0] = w; p.sam = ldx; p.sak = 1; p.sbn = ldw; p.sbk = 1;
  p.M = m; p.N = n; p.K = k; p.pairs = 1;
  p.e = plain_out(out, n, out_dtype);
  p.e.row_scale = x_scale; p.e.col_scale = w_scale; p.e.bias = bias; p.e.residual = residual; p.e.ld_res = ld_res;
  p.e.pre = pre; p.e.act = act;
  p.e.bias_type = dtype == VERACE_E4M3 ? out_dtype : dtype;
  return run_simple<false>(p, dtype, (cudaStream_t)stream);
}

extern "C" size_t verace_linear_backward_workspace(long long m, int n, int k, int dtype) {
  if (m <= 0 || n <= 0) return 0;
  return align_up((size_t)m * n * size_of(dtype), 256) + 256;
}

extern "C" int verace_linear_backward(const void* dout, const void* x, long long ldx, const void* w, long long ldw,
                                      const void* pre, void* dx, void* dw, void* dbias, long long m, int n, int k, int act,
                                      int dtype, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  constexpr const char* who = "verace_linear_backward";
  int rc;
  if ((rc = check_sizes(who, m, n, k)) || (rc = check_types(who, dtype, out_dtype, false))) return rc;
  VERACE_REQUIRE(act >= VERACE_ACT_NONE && act <= VERACE_ACT_GELU_TANH, VERACE_ERR_INVALID, "%s: activation %d", who, act);
  VERACE_REQUIRE(m == 0 || n == 0 || (dout && (pre || act == VERACE_ACT_NONE)), VERACE_ERR_INVALID, "%s: NULL pointer", who);
  if (m > 0 && n > 0 && k > 0 && ((rc = check_rows(who, "x", x, ldx, k, dtype)) || (rc = check_rows(who, "w", w, ldw, k, dtype)))) return rc;
  const size_t need = verace_linear_backward_workspace(m, n, k, dtype);
  VERACE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VERACE_ERR_WORKSPACE,
                 "%s: workspace of %zu bytes required, %zu given", who, need, workspace ? workspace_bytes : (size_t)0);
  cudaStream_t st = (cudaStream_t)stream;
  return by_types(dtype, out_dtype, [&](auto t, auto o) -> int {
    using T = decltype(t);
    using O = decltype(o);
    T* p = reinterpret_cast<T*>(align_up((size_t)workspace, 256));
    const O* z = act == VERACE_ACT_NONE ? nullptr : (const O*)pre;
    int rc;
    if (m > 0 && n > 0) {
      linear_slope<T, O><<<(unsigned)((m * n + 255) / 256), 256, 0, st>>>((const O*)dout, z, p, m * n, act);
      if ((rc = check_launch("linear_slope"))) return rc;
    }
    if (dbias && n > 0) {
      bias_sum<T, O><<<(n + 255) / 256, 256, 0, st>>>((const O*)dout, z, (T*)dbias, m, n, act);
      if ((rc = check_launch("bias_sum"))) return rc;
    }
    SimpleArgs a{};
    a.pairs = 1;
    if (dx) {
      a.a[0] = p; a.sam = n; a.sak = 1; a.b[0] = w; a.sbn = 1; a.sbk = ldw;
      a.M = m; a.N = k; a.K = n; a.e = plain_out(dx, k, dtype);
      if ((rc = run_simple<false>(a, dtype, st))) return rc;
    }
    if (dw) {
      a.a[0] = p; a.sam = 1; a.sak = n; a.b[0] = x; a.sbn = 1; a.sbk = ldx;
      a.M = n; a.N = k; a.K = m; a.e = plain_out(dw, k, dtype);
      if ((rc = run_simple<false>(a, dtype, st))) return rc;
    }
    return VERACE_OK;
  });
}

extern "C" size_t verace_gated_linear_workspace(long long m, int f, int k, int dtype) { return 0; }

extern "C" int verace_gated_linear(const void* x, long long ldx, const float* x_scale, const void* w_gate, const void* w_up,
                                   long long ldw, const float* gate_scale, const float* up_scale, void* out, void* gate,
                                   void* up, long long m, int f, int k, int act, float beta1, float beta2, int dtype,
                                   int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  constexpr const char* who = "verace_gated_linear";
  int rc;
  if ((rc = check_sizes(who, m, f, k)) || (rc = check_types(who, dtype, out_dtype, true))) return rc;
  VERACE_REQUIRE(act >= VERACE_ACT_RELU && act <= VERACE_ACT_SITU, VERACE_ERR_INVALID, "%s: activation %d", who, act);
  VERACE_REQUIRE(act != VERACE_ACT_SITU || (beta1 != 0.f && beta2 != 0.f), VERACE_ERR_INVALID, "%s: beta of 0", who);
  if (m == 0 || f == 0) return VERACE_OK;
  if (k > 0 && ((rc = check_rows(who, "x", x, ldx, k, dtype)) || (rc = check_rows(who, "w_gate", w_gate, ldw, k, dtype)) ||
                (rc = check_rows(who, "w_up", w_up, ldw, k, dtype))))
    return rc;
  const bool eight = dtype == VERACE_E4M3;
  VERACE_REQUIRE(out && (gate != nullptr) == (up != nullptr) && eight == (x_scale != nullptr) &&
                     eight == (gate_scale != nullptr) && eight == (up_scale != nullptr),
                 VERACE_ERR_INVALID, "%s: NULL out, one of gate and up, or scales that do not go with the type", who);
  SimpleArgs p{};
  p.a[0] = x; p.b[0] = w_gate; p.b[1] = w_up; p.sam = ldx; p.sak = 1; p.sbn = ldw; p.sbk = 1;
  p.M = m; p.N = f; p.K = k; p.pairs = 1;
  p.e = plain_out(out, f, out_dtype);
  p.e.row_scale = x_scale; p.e.col_scale = gate_scale; p.e.up_scale = up_scale;
  p.e.pre = gate; p.e.pre_up = up; p.e.act = act;
  p.e.b1 = beta1; p.e.b2 = beta2; p.e.r1 = 1.f / beta1; p.e.r2 = 1.f / beta2;
  return run_simple<true>(p, dtype, (cudaStream_t)stream);
}

extern "C" size_t verace_gated_linear_backward_workspace(long long m, int f, int k, int dtype) {
  if (m <= 0 || f <= 0) return 0;
  return 2 * align_up((size_t)m * f * size_of(dtype), 256) + 256;
}

extern "C" int verace_gated_linear_backward(const void* dout, const void* x, long long ldx, const void* w_gate,
                                            const void* w_up, long long ldw, const void* gate, const void* up, void* dx,
                                            void* dw_gate, void* dw_up, long long m, int f, int k, int act, float beta1,
                                            float beta2, int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                                            void* stream) {
  constexpr const char* who = "verace_gated_linear_backward";
  int rc;
  if ((rc = check_sizes(who, m, f, k)) || (rc = check_types(who, dtype, out_dtype, false))) return rc;
  VERACE_REQUIRE(act >= VERACE_ACT_RELU && act <= VERACE_ACT_SITU, VERACE_ERR_INVALID, "%s: activation %d", who, act);
  VERACE_REQUIRE(act != VERACE_ACT_SITU || (beta1 != 0.f && beta2 != 0.f), VERACE_ERR_INVALID, "%s: beta of 0", who);
  VERACE_REQUIRE(m == 0 || f == 0 || (dout && gate && up), VERACE_ERR_INVALID, "%s: NULL pointer", who);
  if (m > 0 && f > 0 && k > 0 &&
      ((rc = check_rows(who, "x", x, ldx, k, dtype)) || (rc = check_rows(who, "w_gate", w_gate, ldw, k, dtype)) ||
       (rc = check_rows(who, "w_up", w_up, ldw, k, dtype))))
    return rc;
  const size_t need = verace_gated_linear_backward_workspace(m, f, k, dtype);
  VERACE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), VERACE_ERR_WORKSPACE,
                 "%s: workspace of %zu bytes required, %zu given", who, need, workspace ? workspace_bytes : (size_t)0);
  cudaStream_t st = (cudaStream_t)stream;
  return by_types(dtype, out_dtype, [&](auto t, auto o) -> int {
    using T = decltype(t);
    using O = decltype(o);
    T* dg = reinterpret_cast<T*>(align_up((size_t)workspace, 256));
    T* du = reinterpret_cast<T*>(align_up((size_t)(dg + m * f), 256));
    int rc;
    if (m > 0 && f > 0) {
      gated_slope<T, O><<<(unsigned)((m * f + 255) / 256), 256, 0, st>>>((const O*)dout, (const O*)gate, (const O*)up, dg, du,
                                                                      m * f, act, beta1, beta2, 1.f / beta1, 1.f / beta2);
      if ((rc = check_launch("gated_slope"))) return rc;
    }
    SimpleArgs a{};
    a.pairs = 2;
    if (dx) {
      a.a[0] = dg; a.a[1] = du; a.sam = f; a.sak = 1; a.b[0] = w_gate; a.b[1] = w_up; a.sbn = 1; a.sbk = ldw;
      a.M = m; a.N = k; a.K = f; a.e = plain_out(dx, k, dtype);
      if ((rc = run_simple<false>(a, dtype, st))) return rc;
    }
    a.pairs = 1;
    a.sam = 1; a.sak = f; a.b[0] = x; a.sbn = 1; a.sbk = ldx;
    a.M = f; a.N = k; a.K = m;
    for (int h = 0; h < 2; ++h) {
      void* out = h ? dw_up : dw_gate;
      if (!out) continue;
      a.a[0] = h ? du : dg;
      a.e = plain_out(out, k, dtype);
      if ((rc = run_simple<false>(a, dtype, st))) return rc;
    }
    return VERACE_OK;
  });
}
