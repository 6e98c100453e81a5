// What the dense products of the feed-forward sub-layer share: the activations with their
// derivatives, and what a product's epilogue does with a sum.
//
//   linear:  out = act(s_m t_n sum + bias_n) + residual            (s, t: scales of 8-bit operands)
//   gated:   out = act(g) up(u),  g and u two sums of the same row and column;
//            situ: act(g) = b1 tanh(g/b1) sigmoid(g), up(u) = b2 tanh(u/b2); the others: up(u) = u
#pragma once

#include "common.cuh"

namespace verace {
namespace lin {

// ------------------------------------------------------------------ activations
// FAST serves outputs of 16 bits: exponentials and reciprocals by the approximate instructions, against the output's half
// step of 2^-9 or 2^-12.  exp(x) is about (2 + |x|) 2^-23 off (x log2 e is rounded before the instruction takes it: 2^-17 at
// 80), tanh a few 2^-22; what would be below 2^-126 on the way is 0 (sigmoid below -87.3, and with it SiLU, which is less
// than 1.2e-36 there).  fp32 outputs take the CUDA functions.
__device__ __forceinline__ float ex2_(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float LOG2E = 1.4426950408889634f;
template <bool FAST>
__device__ __forceinline__ float exp_(float x) {
  return FAST ? ex2_(x * LOG2E) : expf(x);
}
template <bool FAST>
__device__ __forceinline__ float sigmoid_(float x) {
  return FAST ? rcp_(1.f + ex2_(x * -LOG2E)) : 1.f / (1.f + expf(-x));
}
// tanh x = 1 - 2 / (1 + e^2x), which cancels near 0; there its odd Taylor series up to x^7 (the first
// term left out is 62/2835 x^9: 6e-8 relative at 1/5).
template <bool FAST>
__device__ __forceinline__ float tanh_(float x) {
  if (!FAST) return tanhf(x);
  const float q = x * x;
  const float s = x * fmaf(q, fmaf(q, fmaf(q, -17.f / 315.f, 2.f / 15.f), -1.f / 3.f), 1.f);
  const float t = fmaf(-2.f, rcp_(1.f + ex2_(x * (2.f * LOG2E))), 1.f);
  return q < 0.04f ? s : t;
}

constexpr float SQRT_HALF = 0.70710678118654752f, INV_SQRT_2PI = 0.39894228040143268f;
constexpr float GT0 = 0.79788456080286536f, GT1 = 0.044715f;   // gelu_tanh: sqrt(2/pi) (z + 0.044715 z^3)

// act(z) of the one-input activations (NaN stays NaN)
template <int ACT, bool FAST>
__device__ __forceinline__ float act_(float z) {
  if (ACT == VERACE_ACT_RELU) return z < 0.f ? 0.f : z;
  if (ACT == VERACE_ACT_SILU) return z * sigmoid_<FAST>(z);
  if (ACT == VERACE_ACT_GELU) return 0.5f * z * (1.f + erff(z * SQRT_HALF));
  if (ACT == VERACE_ACT_GELU_TANH) return 0.5f * z * (1.f + tanh_<FAST>(GT0 * fmaf(GT1 * z * z, z, z)));
  return z;
}
// act(z) and act'(z), but for relu
template <int ACT, bool FAST>
__device__ __forceinline__ void act_slope_(float z, float& a, float& da) {
  if (ACT == VERACE_ACT_SILU) {
    const float p = sigmoid_<FAST>(z);
    a = z * p;
    da = p * (1.f + z * (1.f - p));
  } else if (ACT == VERACE_ACT_GELU) {
    const float half = 0.5f * (1.f + erff(z * SQRT_HALF));
    a = z * half;
    da = fmaf(z * INV_SQRT_2PI, exp_<FAST>(-0.5f * z * z), half);
  } else if (ACT == VERACE_ACT_GELU_TANH) {
    const float t = tanh_<FAST>(GT0 * fmaf(GT1 * z * z, z, z));
    a = 0.5f * z * (1.f + t);
    da = 0.5f * (1.f + t) + 0.5f * z * (1.f - t * t) * GT0 * fmaf(3.f * GT1 * z, z, 1.f);
  } else {
    a = z;
    da = 1.f;
  }
}
// the gradient of z from d, the gradient of act(z).  (relu selects, as torch does: 0 where z <= 0, even of an infinite d,
// and d where z is NaN)
template <int ACT, bool FAST>
__device__ __forceinline__ float back_(float d, float z) {
  if (ACT == VERACE_ACT_RELU) return z <= 0.f ? 0.f : d;
  float a, da;
  act_slope_<ACT, FAST>(z, a, da);
  return d * da;
}
// act(g) up(u)
template <int ACT, bool FAST>
__device__ __forceinline__ float gate_(float g, float u, float b1, float b2, float r1, float r2) {
  if (ACT == VERACE_ACT_SITU) return (b1 * tanh_<FAST>(g * r1) * sigmoid_<FAST>(g)) * (b2 * tanh_<FAST>(u * r2));
  return act_<ACT, FAST>(g) * u;
}
// the gradients of g and u from d, the gradient of act(g) up(u)
template <int ACT, bool FAST>
__device__ __forceinline__ void gate_slope_(float d, float g, float u, float b1, float b2, float r1, float r2, float& dg,
                                            float& du) {
  if (ACT == VERACE_ACT_SITU) {
    const float tg = tanh_<FAST>(g * r1), tu = tanh_<FAST>(u * r2), p = sigmoid_<FAST>(g);
    dg = d * (b2 * tu) * ((1.f - tg * tg) * p + b1 * tg * p * (1.f - p));
    du = d * (b1 * tg * p) * (1.f - tu * tu);
  } else if (ACT == VERACE_ACT_RELU) {
    dg = back_<ACT, FAST>(d * u, g);
    du = d * act_<ACT, FAST>(g);
  } else {
    float a, da;
    act_slope_<ACT, FAST>(g, a, da);
    dg = d * da * u;
    du = d * a;
  }
}

// Calls f(std::integral_constant<int, ACT>) for a runtime activation.
template <typename F>
__device__ __forceinline__ void by_act(int act, F&& f) {
  switch (act) {
    case VERACE_ACT_RELU: f(std::integral_constant<int, VERACE_ACT_RELU>()); break;
    case VERACE_ACT_SILU: f(std::integral_constant<int, VERACE_ACT_SILU>()); break;
    case VERACE_ACT_GELU: f(std::integral_constant<int, VERACE_ACT_GELU>()); break;
    case VERACE_ACT_GELU_TANH: f(std::integral_constant<int, VERACE_ACT_GELU_TANH>()); break;
    case VERACE_ACT_SITU: f(std::integral_constant<int, VERACE_ACT_SITU>()); break;
    default: f(std::integral_constant<int, VERACE_ACT_NONE>());
  }
}
// v <- act(v), or act(v) up(u): U values, FAST with the output's type
template <bool GATED, bool FAST, int U, typename E>
__device__ __forceinline__ void activate(const E& e, float (&v)[U], const float (&u)[U]) {
  if (!GATED && e.act == VERACE_ACT_NONE) return;
  by_act(e.act, [&](auto act) {
#pragma unroll
    for (int j = 0; j < U; ++j) {
      if constexpr (GATED) v[j] = gate_<decltype(act)::value, FAST>(v[j], u[j], e.b1, e.b2, e.r1, e.r2);
      else v[j] = act_<decltype(act)::value, FAST>(v[j]);
    }
  });
}

// a sum of 8-bit products times the scales of its row and column, the smaller one first: then nothing on the way leaves
// fp32's range that the result does not (their product may: 1e20 by 1e20 times a sum of 0, 1e-25 by 1e-20 times one of 1e9)
__device__ __forceinline__ float scaled_by(float v, float row, float col) {
  const bool first = fabsf(row) < fabsf(col);
  return v * (first ? row : col) * (first ? col : row);
}

// ------------------------------------------------------------------ values by a runtime type
__device__ __forceinline__ float load_as(const void* p, long long i, int type) {
  if (type == VERACE_F32) return static_cast<const float*>(p)[i];
  if (type == VERACE_BF16) return to_f32(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_f32(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_as(void* p, long long i, float v, int type) {
  if (type == VERACE_F32) static_cast<float*>(p)[i] = v;
  else if (type == VERACE_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
inline size_t size_of(int type) { return type == VERACE_F32 ? 4 : type == VERACE_E4M3 ? 1 : 2; }

// ------------------------------------------------------------------ epilogue
struct Epilogue {
  const float *row_scale, *col_scale, *up_scale;   // of 8-bit operands, or null
  const void *bias, *residual;                     // or null
  void* out;
  float *pre, *pre_up;                             // the sums before the activation in fp32, for a backward pass, or null
  long long ld, ld_res;                            // row strides of out and pre, and of the residual
  int bias_type, type, act;                        // type: of out and the residual
  float b1, b2, r1, r2;                            // r = 1 / b
};

}  // namespace lin
}  // namespace verace
