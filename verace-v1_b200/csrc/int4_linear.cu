// Product of a few tokens with 4-bit weights:
//     y[i][n] = sum_k x[i][k] W[n][k] (+ bias[n]),   W[n][k] = s[k/G][n] (q[n][k] - z[k/G][n])
// q in [0, 15], two to a byte along k (the even k in the low half); z in [0, 15], 8 when no
// zeros are given.
//
// Bound: the weights' bytes (half a byte for 2 m operations), if nothing else is slower.  A
// first version unpacked the codes to bf16 (11 instructions for 8 codes) for mma.sync and ran
// at a quarter of the memory rate, bound by instructions.  Here the tensor cores take a code as
// it is: the bit pattern of an e4m3 number in [0, 15] reads code * 2^-9 (subnormal below 8, the
// first binade from 8 on, with the same step), so a word of 8 codes becomes 8 operands with one
// shift and two masks.  x goes in as fp8 pieces that add up to it, exactly:
//   * few tokens: e4m3 pieces, each the rest of the one before times 2^5, in columns of their
//     own (a 128-row MMA takes 50 clocks for anything up to 64 columns): y = d0 + 2^-5 d1 + ...
//     bf16's 8 bits are 2 pieces, fp16's 11 are 3, fp32's 24 are 5;
//   * up to 64 tokens of 16-bit types: an e4m3 piece and one or two e5m2 pieces of the rest, one
//     MMA after the other into the same columns.
// Each token is scaled by a power of two, its largest input to [2^7, 2^8); inputs 2^-22 of that
// and smaller lose digits.  tcgen05.mma adds fp8 products in full fp32 (measured: 2^23 + 1 is
// exact).  The zeros are one more MMA per group: 32 inputs that hold X = sum of the group's
// scaled x in 6 e5m2 pieces, against -z.  So D = 2^-9 (sum q x - z X) per group, and a row's
// thread adds s D in fp32.  No weight and no input is rounded.
// What q x and z X lose by cancelling is 2^-24 of the group's largest input.  Where at most a
// sixteenth of a group is 2^12 above all the rest, that could show in the outputs whose q = z
// there, so those inputs (and infinities and NaN) are left out of the pieces and added one by
// one as (q - z) x s at the end (rare).
//
// One CTA per SM, 128 output rows at a time, 16 warps: one feeds the weights by TMA (128 rows x
// 256 codes a stage, 128-byte swizzle: a row's thread reads 16 bytes without bank conflicts),
// one the staged x, two issue the MMAs, eight unpack codes into TMEM (the MMA's A operand; two
// sets of four take a stage's halves), four hold the rows' sums.  Few row tiles: k is split over
// a cluster and the partial sums are joined through distributed shared memory in rank order.
#include "common.cuh"
#include "tc.cuh"
#include "tmap.cuh"

#include <cooperative_groups.h>
#include <cuda_fp8.h>

#include <atomic>
#include <mutex>

namespace verace {

__device__ int g_int4_status = 0;   // non-zero after a bounded wait gave up

namespace {

namespace cg = cooperative_groups;

constexpr uint32_t POLLS = 1u << 22;
constexpr int NT = 512;                  // threads: 16 warps
constexpr int ROWS = 128;                // output rows per tile
constexpr int KC = 128;                  // inputs per chunk
constexpr int SW = 5;                    // weight stages of two chunks
constexpr int W_STAGE = ROWS * KC;       // bytes: 128 rows x 256 codes
constexpr int NA = 4;                    // A operands (one chunk each) in TMEM
constexpr int D_COL = 256;               // first TMEM column of the accumulators
constexpr int MAX_SB = 64;
constexpr int B_SMEM = 136 * 1024;
constexpr float FINITE = 3.4028235e38f;
constexpr float APART = 1.f / 4096.f;

// How a token tile's x is laid out.  MP tokens per tile; COLS: the pieces in columns of their own.
template <typename T, int MP_>
struct Shape {
  static constexpr bool IS32 = std::is_same<T, float>::value;
  static constexpr int MP = MP_;
  static constexpr bool COLS = IS32 || MP <= (std::is_same<T, __half>::value ? 16 : 32);
  static constexpr int P = IS32 ? 5 : std::is_same<T, __half>::value ? 3 : 2;    // pieces
  static constexpr int N = COLS ? (P * MP + 15) / 16 * 16 : MP;                  // MMA columns
  static constexpr int PASSES = COLS ? 1 : P;
  static constexpr int ND = 128 / N < 2 ? 1 : 2;                                 // accumulators per MMA warp
  // bytes of a chunk's B operands: the passes' [128 / 16][N][16], then per group the zeros' [2][N][16]
  static constexpr int block(int gpc) { return PASSES * KC * N + gpc * 32 * N; }
};

struct Int4Args {
  const void* x;
  long long ldx;
  const uint8_t* q;
  const void* s;
  const uint8_t* z;
  const void* bias;
  void* y;
  long long m;
  int n, k, out_f32;
  int tiles, ytiles;   // row tiles and token tiles
  int ck, per;         // CTAs that share a tile, each with `per` chunks of k
  int staged;          // x comes from the workspace (else every CTA stages its own)
  int sb;              // chunks of x in shared memory
  int resident;        // all of the CTA's chunks, loaded once
  const uint8_t* ws;   // staged x: blocks [token tile][chunk], then scales, then left-out masks
  const float* ws_scale;
  const uint32_t* ws_mask;
};

// ------------------------------------------------------------------ staging x
// Eight consecutive inputs of one token; out-of-range ones are 0.
template <typename T>
__device__ __forceinline__ void load8(const T* p, bool valid, float (&v)[8]) {
  uint4 u[sizeof(T) / 2];
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
    u[i] = valid ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
  if constexpr (std::is_same<T, float>::value) {
    const uint32_t w[8] = {u[0].x, u[0].y, u[0].z, u[0].w, u[1].x, u[1].y, u[1].z, u[1].w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  } else {
    unpack8<T>(u[0], v);
  }
}

// Zeroes the inputs that are added one by one; `LANES` lanes in a row hold one group.  Returns the
// lane's largest remaining |input|.
template <int LANES>
__device__ __forceinline__ float leave_out(float (&v)[8], bool& out) {
  float mine = 0.f;
  out = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if (!(fabsf(v[i]) <= FINITE)) out = true, v[i] = 0.f;
    mine = fmaxf(mine, fabsf(v[i]));
  }
  float top = mine;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // a lane whose inputs are all far below the largest: perhaps that one stands alone
  if (__any_sync(0xffffffffu, mine > 0.f && mine < top * APART)) {
    int high = 0, low = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      high += fabsf(v[i]) >= top * APART;
      low |= fabsf(v[i]) < top * APART && v[i] != 0.f;
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
      high += __shfl_xor_sync(0xffffffffu, high, o);
      low |= __shfl_xor_sync(0xffffffffu, low, o);
    }
    if (low && high <= LANES * 8 / 16) {
      mine = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (fabsf(v[i]) >= top * APART) out = true, v[i] = 0.f;
        mine = fmaxf(mine, fabsf(v[i]));
      }
    }
  }
  return mine;
}

// The exponent that brings `top` to [2^7, 2^8), at most 100.
__device__ __forceinline__ int shift_of(float top) {
  return min(7 - ((int)(__float_as_uint(top) >> 23) - 127), 100);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// Writes the pieces of lane l16's eight inputs of a chunk (token row t of the tile) and, from a
// group's first lane, X.  A word's codes 0, 2, 4, 6 unpack before 1, 3, 5, 7, and so do x's bytes.
template <typename T, typename S, int GPC>
__device__ __forceinline__ void stage8(float (&v)[8], float scale, uint8_t* block, int t, int l16) {
  constexpr int LANES = 16 / GPC;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= scale, sum += v[i];
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  constexpr int at[4][2] = {{0, 2}, {4, 6}, {1, 3}, {5, 7}};
  uint8_t* d = block + ((l16 / 2) * S::N + t) * 16 + (l16 % 2) * 8;
  auto put = [&](int p, const uint32_t (&b)[4]) {
    uint8_t* to = d + (S::COLS ? p * S::MP * 16 : p * KC * S::N);
    *reinterpret_cast<uint2*>(to) = make_uint2(b[0] | (b[1] << 16), b[2] | (b[3] << 16));
  };
  if constexpr (S::IS32) {
#pragma unroll
    for (int p = 0; p < S::P; ++p) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        b[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[at[i][0]], v[at[i][1]]), __NV_SATFINITE, __NV_E4M3);
        const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)b[i], __NV_E4M3);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        v[at[i][0]] = (v[at[i][0]] - f.x) * 32.f;
        v[at[i][1]] = (v[at[i][1]] - f.y) * 32.f;
      }
      put(p, b);
    }
  } else {
    // 8 or 11 bits: fp16 holds them
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[at[i][0]], v[at[i][1]]);
#pragma unroll
    for (int p = 0; p < S::P; ++p) {
      uint32_t b[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const __half2_raw hr = *reinterpret_cast<const __half2_raw*>(&h[i]);
        __half2_raw r;
        if (S::COLS || p == 0) {
          b[i] = __nv_cvt_halfraw2_to_fp8x2(hr, __NV_SATFINITE, __NV_E4M3);
          r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)b[i], __NV_E4M3);
        } else {
          b[i] = __nv_cvt_halfraw2_to_fp8x2(hr, __NV_SATFINITE, __NV_E5M2);
          r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)b[i], __NV_E5M2);
        }
        h[i] = __hsub2(h[i], *reinterpret_cast<const __half2*>(&r));
        if (S::COLS) h[i] = __hmul2(h[i], __float2half2_rn(32.f));
      }
      put(p, b);
    }
  }
  if (l16 % LANES == 0) {
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int p = 0; p < 6; ++p) {
      const uint32_t b = __nv_cvt_float_to_fp8(sum, __NV_SATFINITE, __NV_E5M2);
      w[p / 4] |= b << (8 * (p % 4));
      const __half_raw r = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E5M2);
      sum -= __half2float(*reinterpret_cast<const __half*>(&r));
    }
    uint4* z = reinterpret_cast<uint4*>(block + S::PASSES * KC * S::N + (l16 / LANES) * 32 * S::N) + t;
    z[0] = make_uint4(w[0], w[1], 0, 0);
    z[S::N] = make_uint4(0, 0, 0, 0);
    if constexpr (S::COLS) {
#pragma unroll
      for (int p = 1; p < S::P; ++p) z[p * S::MP] = z[S::N + p * S::MP] = make_uint4(0, 0, 0, 0);
    }
  }
}

// The staging kernel: one CTA per token.
template <typename T, int MP, int GPC>
__global__ void __launch_bounds__(NT) int4_stage_x(const T* __restrict__ x, long long ldx, int k, int chunks,
                                                   uint8_t* __restrict__ ws, float* __restrict__ scales,
                                                   uint32_t* __restrict__ masks) {
  using S = Shape<T, MP>;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int s_top;
  __shared__ uint32_t s_mask;
  const int tid = threadIdx.x, l16 = tid % 16;
  const long long tok = blockIdx.x;
  const T* row = x + tok * ldx;
  const int span = (chunks * GPC + 31) / 32;
  if (tid == 0) s_top = 0, s_mask = 0;
  __syncthreads();
  for (int c0 = 0; c0 < chunks; c0 += NT / 16) {
    const int c = c0 + tid / 16, at = c * KC + l16 * 8;
    float v[8];
    load8(row + at, c < chunks && at < k, v);
    bool out;
    float mine = leave_out<16 / GPC>(v, out);
    if (out) atomicOr(&s_mask, 1u << ((c * GPC + l16 / (16 / GPC)) / span));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
    if (tid % 32 == 0) atomicMax(&s_top, __float_as_int(mine));
  }
  __syncthreads();
  const int sh = shift_of(__int_as_float(s_top));
  uint8_t* base = ws + (tok / MP) * (long long)chunks * S::block(GPC);
  for (int c0 = 0; c0 < chunks; c0 += NT / 16) {
    const int c = c0 + tid / 16, at = c * KC + l16 * 8;
    float v[8];
    load8(row + at, c < chunks && at < k, v);
    bool out;
    leave_out<16 / GPC>(v, out);
    // (whole warps: a warp's two chunks are both in range or its second is dropped after the shuffles)
    uint8_t* block = base + (long long)min(c, chunks - 1) * S::block(GPC);
    if (__all_sync(0xffffffffu, c < chunks)) {
      stage8<T, S, GPC>(v, pow2(sh), block, (int)(tok % MP), l16);
    } else if (__any_sync(0xffffffffu, c < chunks)) {
      // the last, odd chunk: its lanes' twins write the same bytes
      float u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) u[i] = __shfl_sync(0xffffffffu, v[i], l16);
      stage8<T, S, GPC>(u, pow2(sh), base + (long long)(chunks - 1) * S::block(GPC), (int)(tok % MP), l16);
    }
  }
  if (tid == 0) {
    scales[tok] = pow2(-sh);
    masks[tok] = s_mask;
  }
}

// The terms of one output that leave_out zeroed, over the group that starts at input k0.
template <typename T>
__device__ __noinline__ float left_out(const Int4Args& a, const T* x, long long row, int k0, int group) {
  const int k1 = min(k0 + group, a.k);
  float top = 0.f;
  for (int k = k0; k < k1; ++k) {
    const float m = fabsf(to_f32(x[k]));
    if (m <= FINITE) top = fmaxf(top, m);
  }
  int high = 0, low = 0;
  for (int k = k0; k < k1; ++k) {
    const float m = fabsf(to_f32(x[k]));
    if (m <= FINITE) {
      high += m >= top * APART;
      low |= m < top * APART && m != 0.f;
    }
  }
  const bool alone = low && high <= group / 16;
  const long long at = (long long)(k0 / group) * a.n + row;
  const float zero = a.z ? (float)a.z[at] : 8.f, scale = to_f32(static_cast<const T*>(a.s)[at]);
  float v = 0.f;
  for (int k = k0; k < k1; ++k) {
    const float xv = to_f32(x[k]);
    if (fabsf(xv) <= FINITE && !(alone && fabsf(xv) >= top * APART)) continue;
    const uint8_t by = a.q[row * (a.k / 2) + k / 2];
    v += xv * (((float)(k & 1 ? by >> 4 : by & 15) - zero) * scale);
  }
  return v;
}

// ------------------------------------------------------------------ TMEM and MMA
__device__ __forceinline__ void mma_f8(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__host__ __device__ constexpr uint32_t idesc_f8(int n, int b_e5m2) {
  return (1u << 4) | ((uint32_t)b_e5m2 << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(ROWS >> 4) << 24);
}
__device__ __forceinline__ void tmem_st8(uint32_t a, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(a), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_ld16_issue(uint32_t a, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(a));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// keeps the uses of loaded values behind the wait
__device__ __forceinline__ void pin16(float* v) {
  asm volatile("" : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
               "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]));
}

struct Bars {
  uint64_t wfull[SW], wempty[SW], afull[NA], aempty[NA], dfull[4], dempty[4], bfull[MAX_SB], bempty[MAX_SB], drain;
};

__device__ __forceinline__ bool ready(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(tc::smem_addr(bar)), "r"(parity)
               : "memory");
  return done;
}
// One lane of a converged warp.  (With `lane == 0` instead, the MMAs' and copies' operands are
// moved to uniform registers lane by lane: 114 clocks an MMA against 52.)
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p;
}

// Waits for completion number `it` (0, 1, ...) of a barrier.
struct Waiter {
  volatile int* fail;
  __device__ __forceinline__ bool operator()(uint64_t* bar, uint32_t it) const {
    if (ready(bar, it & 1) || (!*fail && tc::mbar_wait(bar, it & 1, POLLS))) return true;
    *fail = 1;
    atomicExch(&g_int4_status, 1);
    return false;
  }
  // the same answer for a whole warp
  __device__ __forceinline__ bool warp(uint64_t* bar, uint32_t it) const {
    return __all_sync(0xffffffffu, (*this)(bar, it));
  }
};

template <typename T, int MP, int GPC>
__global__ void __launch_bounds__(NT, 1) int4_linear_kernel(const __grid_constant__ CUtensorMap wmap, Int4Args a) {
  using S = Shape<T, MP>;
  constexpr int BLK = S::block(GPC), N = S::N, G = KC / GPC;
  constexpr int A_COLS = 32 + 8 * GPC;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bar;
  __shared__ uint32_t s_slot;
  __shared__ int s_fail;
  __shared__ int s_top[MP];
  __shared__ uint32_t s_mask[MP];
  __shared__ float s_scale[MP];
  uint8_t* wst = smem;
  uint8_t* bst = smem + SW * W_STAGE;
  const int tid = threadIdx.x, lane = tid % 32, w = __shfl_sync(0xffffffffu, tid / 32, 0);
  const int rank = a.ck > 1 ? blockIdx.x % a.ck : 0;
  const int chunks = (a.k + KC - 1) / KC;
  const int c0 = min(rank * a.per, chunks), c1 = min(c0 + a.per, chunks), nc = c1 - c0;
  const int stages = (nc + 1) / 2;
  const int unit0 = blockIdx.x / a.ck, units = a.tiles * a.ytiles, step = gridDim.x / a.ck;
  const int span = ((a.staged ? chunks : a.per) * GPC + 31) / 32;     // groups per bit of a left-out mask

  if (w == 1) tc::tmem_alloc(&s_slot, 512);
  if (tid == 0) {
    for (int i = 0; i < SW; ++i) tc::mbar_init(&bar.wfull[i], 1), tc::mbar_init(&bar.wempty[i], 8);
    for (int i = 0; i < NA; ++i) tc::mbar_init(&bar.afull[i], 4), tc::mbar_init(&bar.aempty[i], 1);
    for (int i = 0; i < 4; ++i) tc::mbar_init(&bar.dfull[i], 1), tc::mbar_init(&bar.dempty[i], 4);
    for (int i = 0; i < a.sb; ++i) tc::mbar_init(&bar.bfull[i], 1), tc::mbar_init(&bar.bempty[i], 1);
    tc::mbar_init(&bar.drain, 2);
    tc::fence_mbar_init();
    s_fail = 0;
    // the first weights, before anything else
    for (int i = 0; i < SW && i < stages; ++i) {
      tc::mbar_expect_tx(&bar.wfull[i], W_STAGE);
      tc::tma_load_2d(wst + i * W_STAGE, &wmap, (c0 + 2 * i) * (KC / 2), unit0 % a.tiles * ROWS, &bar.wfull[i]);
    }
  }
  if (tid < MP) s_top[tid] = 0, s_mask[tid] = 0, s_scale[tid] = 0.f;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_slot, 0);
  const Waiter wait{&s_fail};

  if (!a.staged && nc > 0) {
    // every thread stages the CTA's range of x: the tokens' largest inputs, then the pieces
    const T* x = static_cast<const T*>(a.x);
    const int toks = (int)a.m, total = toks * nc, l16 = tid % 16;
    for (int u0 = 0; u0 < total; u0 += NT / 16) {
      const int u = u0 + tid / 16, tok = u / nc, c = u - tok * nc, at = (c0 + c) * KC + l16 * 8;
      float v[8];
      load8(x + (long long)tok * a.ldx + at, u < total && at < a.k, v);
      bool out;
      float mine = leave_out<16 / GPC>(v, out);
      if (out) atomicOr(&s_mask[tok], 1u << ((c * GPC + l16 / (16 / GPC)) / span));
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) mine = fmaxf(mine, __shfl_xor_sync(0xffffffffu, mine, o));
      if (l16 == 0 && u < total) atomicMax(&s_top[tok], __float_as_int(mine));
    }
    __syncthreads();
    for (int u0 = 0; u0 < total; u0 += NT / 16) {
      const int u = u0 + tid / 16, tok = min(u / nc, toks - 1), c = u - u / nc * nc, at = (c0 + c) * KC + l16 * 8;
      float v[8];
      load8(x + (long long)tok * a.ldx + at, u < total && at < a.k, v);
      bool out;
      leave_out<16 / GPC>(v, out);
      const int sh = shift_of(__int_as_float(s_top[tok]));
      if (__all_sync(0xffffffffu, u < total)) {
        stage8<T, S, GPC>(v, pow2(sh), bst + c * BLK, tok, l16);
      } else if (__any_sync(0xffffffffu, u < total)) {     // the last, odd one: both halves of the warp write it
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = __shfl_sync(0xffffffffu, v[i], l16);
        stage8<T, S, GPC>(d, pow2(shift_of(__int_as_float(s_top[toks - 1]))), bst + (nc - 1) * BLK, toks - 1, l16);
      }
    }
    if (tid < toks) s_scale[tid] = pow2(-shift_of(__int_as_float(s_top[tid])));
    tc::fence_proxy_async();
    __syncthreads();
  }

  if (w == 0) {
    if (elect()) {   // ---- weights
      int it = 0;
      bool ok = true;
      for (int u = unit0; ok && u < units; u += step)
        for (int i = 0; i < stages; ++i, ++it) {
          if (it < SW && u == unit0) continue;             // loaded above
          const int sl = it % SW;
          if (it >= SW && !wait(&bar.wempty[sl], it / SW - 1)) { ok = false; break; }
          tc::mbar_expect_tx(&bar.wfull[sl], W_STAGE);
          tc::tma_load_2d(wst + sl * W_STAGE, &wmap, (c0 + 2 * i) * (KC / 2), u % a.tiles * ROWS, &bar.wfull[sl]);
        }
      // copies still in flight land before the CTA may exit
      for (int j = it - SW < 0 ? 0 : it - SW; j < it; ++j) tc::mbar_wait(&bar.wfull[j % SW], j / SW & 1, POLLS);
    }
  } else if (w == 1) {
    if (a.staged && elect()) {   // ---- staged x
      asm volatile("griddepcontrol.wait;" ::: "memory");
      int it = 0;
      bool ok = true;
      for (int u = unit0; ok && u < units && !(a.resident && u > unit0); u += step)
        for (int c = 0; c < nc; ++c, ++it) {
          const int sl = it % a.sb;
          if (it >= a.sb && !wait(&bar.bempty[sl], it / a.sb - 1)) { ok = false; break; }
          tc::mbar_expect_tx(&bar.bfull[sl], BLK);
          tc::bulk_load(bst + sl * BLK, a.ws + ((long long)(u / a.tiles) * chunks + c0 + c) * BLK, BLK, &bar.bfull[sl]);
        }
      for (int j = it - a.sb < 0 ? 0 : it - a.sb; j < it; ++j)
        tc::mbar_wait(&bar.bfull[j % a.sb], j / a.sb & 1, POLLS);
    }
  } else if (w < 4) {
    // ---- MMAs: two warps, every other chunk each.  A chunk takes a thread 50 clocks an MMA and
    // 100 a wait to issue, more than the chunk's share of time.
    if (elect()) {
      const int mine = w - 2;
      int ia = 0;
      bool ok = true;
      for (int u = unit0; ok && u < units; u += step)
        for (int c = 0; c < nc; ++c, ++ia) {
          if (ia % 2 != mine) continue;
          const int sl = a.resident ? c : ia % a.sb;
          if (!wait(&bar.afull[ia % NA], ia / NA) ||
              (a.staged && !wait(&bar.bfull[sl], a.resident ? 0 : ia / a.sb))) { ok = false; break; }
          const uint32_t A = tmem + ia % NA * A_COLS;
          const uint64_t B = tc::sdesc(tc::smem_addr(bst + sl * BLK), N * 16, 128);
#pragma unroll
          for (int gi = 0; gi < GPC; ++gi) {
            // each warp's accumulators are its own: it meets their every turn in order
            const int i = ia / 2 * GPC + gi, e = mine * S::ND + i % S::ND, turn = i / S::ND;
            if (turn > 0 && !wait(&bar.dempty[e], turn - 1)) { ok = false; break; }
            tc::fence_after_sync();
            const uint32_t D = tmem + D_COL + e * N;
#pragma unroll
            for (int p = 0; p < S::PASSES; ++p)
#pragma unroll
              for (int b = gi * (4 / GPC); b < (gi + 1) * (4 / GPC); ++b)
                mma_f8(D, A + 8 * b, B + (uint64_t)((p * KC * N + b * 32 * N) >> 4), idesc_f8(N, p > 0),
                       p > 0 || b > gi * (4 / GPC));
            mma_f8(D, A + 32 + 8 * gi, B + (uint64_t)((S::PASSES * KC * N + gi * 32 * N) >> 4), idesc_f8(N, 1), true);
            tc::commit(&bar.dfull[e]);
          }
          tc::commit(&bar.aempty[ia % NA]);
          if (a.staged && !a.resident) tc::commit(&bar.bempty[sl]);
        }
      tc::commit(&bar.drain);        // every MMA issued is done before the TMEM goes
      tc::mbar_wait(&bar.drain, 0, POLLS);
    }
  } else if (w >= 4 && w < 12) {
    // ---- unpacking: set `half` takes that half of each weight stage; a thread is a row
    const int half = (w - 4) / 4, r = w % 4 * 32 + lane;
    const uint32_t at = tmem + ((uint32_t)(w % 4 * 32) << 16);
    int it = 0, ia = 0;
    bool ok = true;
    uint32_t zc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) zc[i] = 0x88888888u;
    for (int u = unit0; ok && u < units; u += step, ia += nc) {
      const long long row = (long long)(u % a.tiles) * ROWS + r;
      const uint8_t* zp = a.z && row < a.n ? a.z + row : nullptr;
      const int groups = (a.k + G - 1) / G;
      uint8_t zn[GPC];
      auto load_zeros = [&](int c) {
#pragma unroll
        for (int gi = 0; gi < GPC; ++gi) {
          const int g = (c0 + c) * GPC + gi;
          zn[gi] = zp && c < nc && g < groups ? __ldg(zp + (long long)g * a.n) : 8;
        }
      };
      load_zeros(half);
      for (int i = 0; i < stages; ++i, ++it) {
        const int sl = it % SW, c = 2 * i + half, e = (ia + c) % NA, en = (ia + c) / NA;
        if (!wait.warp(&bar.wfull[sl], it / SW)) { ok = false; break; }
        if (c < nc) {
          uint4 raw[4];
          const uint8_t* src = wst + sl * W_STAGE + r * KC;
#pragma unroll
          for (int j = 0; j < 4; ++j) raw[j] = *reinterpret_cast<const uint4*>(src + (((half * 4 + j) ^ (r & 7)) * 16));
          if (en > 0 && !wait.warp(&bar.aempty[e], en - 1)) { ok = false; break; }
          tc::fence_after_sync();
          const uint32_t A = at + e * A_COLS;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t b[8] = {raw[j].x & 0x0f0f0f0fu, (raw[j].x >> 4) & 0x0f0f0f0fu,
                                   raw[j].y & 0x0f0f0f0fu, (raw[j].y >> 4) & 0x0f0f0f0fu,
                                   raw[j].z & 0x0f0f0f0fu, (raw[j].z >> 4) & 0x0f0f0f0fu,
                                   raw[j].w & 0x0f0f0f0fu, (raw[j].w >> 4) & 0x0f0f0f0fu};
            tmem_st8(A + 8 * j, b);
          }
          if (a.z || en == 0) {        // without zeros, -8 stays where the first round wrote it
#pragma unroll
            for (int gi = 0; gi < GPC; ++gi) {
              if (a.z) {
#pragma unroll
                for (int j = 0; j < 8; ++j) zc[j] = (0x80u | zn[gi]) * 0x01010101u;
              }
              tmem_st8(A + 32 + 8 * gi, zc);
            }
            if (a.z) load_zeros(c + 2);
          }
          asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
          tc::fence_before_sync();
        }
        __syncwarp();
        if (lane == 0) {
          tc::mbar_arrive(&bar.wempty[sl]);
          if (c < nc) tc::mbar_arrive(&bar.afull[e]);
        }
      }
    }
  } else if (w >= 12) {
    // ---- sums: a thread is an output row
    const int r = w % 4 * 32 + lane;
    const uint32_t at = tmem + D_COL + ((uint32_t)(w % 4 * 32) << 16);
    const T* sp = static_cast<const T*>(a.s);
    const int groups = (a.k + G - 1) / G, ng = nc * GPC;
    if (a.staged) asm volatile("griddepcontrol.wait;" ::: "memory");
    int ia = 0;
    bool ok = true;
    for (int u = unit0; ok && u < units; u += step, ia += nc) {
      const long long row = (long long)(u % a.tiles) * ROWS + r, m0 = (long long)(u / a.tiles) * MP;
      const int toks = (int)min((long long)MP, a.m - m0);
      float acc[MP];
#pragma unroll
      for (int t = 0; t < MP; ++t) acc[t] = 0.f;
      auto scale_of = [&](int g) {
        const int gg = c0 * GPC + g;
        return row < a.n && g < ng && gg < groups ? __ldg(sp + (long long)gg * a.n + row) : from_f32<T>(0.f);
      };
      T sq[4];                          // the scales of the next four groups, as loaded (a conversion would wait)
#pragma unroll
      for (int i = 0; i < 4; ++i) sq[i] = scale_of(i);
      for (int g0 = 0; ok && g0 < ng; g0 += 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (g0 + i >= ng) break;
          const int ca = ia + (g0 + i) / GPC, di = ca / 2 * GPC + (g0 + i) % GPC, e = ca % 2 * S::ND + di % S::ND;
          if (!wait.warp(&bar.dfull[e], di / S::ND)) { ok = false; break; }
          tc::fence_after_sync();
          const uint32_t D = at + e * N;
          const float s = to_f32(sq[i]);
          sq[i] = scale_of(g0 + i + 4);
          if constexpr (S::COLS) {
            float d[N];
#pragma unroll
            for (int j = 0; j < N; j += 16) tmem_ld16_issue(D + j, d + j);
            tmem_wait_ld();
#pragma unroll
            for (int j = 0; j < N; j += 16) pin16(d + j);
#pragma unroll
            for (int t = 0; t < MP; ++t) {
              float v = d[(S::P - 1) * MP + t];
#pragma unroll
              for (int p = S::P - 2; p >= 0; --p) v = fmaf(v, 1.f / 32.f, d[p * MP + t]);
              acc[t] = fmaf(s, v, acc[t]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < N; j += 32) {
              float d[32];
              tmem_ld16_issue(D + j, d);
              tmem_ld16_issue(D + j + 16, d + 16);
              tmem_wait_ld();
              pin16(d);
              pin16(d + 16);
#pragma unroll
              for (int t = 0; t < 32; ++t) acc[j + t] = fmaf(s, d[t], acc[j + t]);
            }
          }
          tc::fence_before_sync();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&bar.dempty[e]);
        }
      }
      // the tile's outputs (or this CTA's part of them)
      if (ok) {
        const T* x = static_cast<const T*>(a.x);
        const T* bias = static_cast<const T*>(a.bias);
        float* red = reinterpret_cast<float*>(wst);
#pragma unroll
        for (int t = 0; t < MP; ++t) {
          if (t < toks && (row < a.n || a.ck > 1)) {
            const uint32_t mask = a.staged ? a.ws_mask[m0 + t] : s_mask[t];
            float v = acc[t] * 512.f * (a.staged ? a.ws_scale[m0 + t] : s_scale[t]);
            if (mask && row < a.n)
              for (int g = 0; g < ng; ++g)
                if ((mask >> (((a.staged ? c0 * GPC : 0) + g) / span) & 1u) && (c0 * GPC + g) * G < a.k)
                  v += left_out<T>(a, x + (m0 + t) * a.ldx, row, (c0 * GPC + g) * G, G);
            if (a.ck > 1) {
              red[t * ROWS + r] = v;    // (all stages are consumed: every group's sum is in)
            } else {
              if (bias) v += to_f32(bias[row]);
              const long long o = (m0 + t) * a.n + row;
              if (a.out_f32) static_cast<float*>(a.y)[o] = v;
              else static_cast<T*>(a.y)[o] = from_f32<T>(v);
            }
          }
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (w == 1) tc::tmem_dealloc(tmem, 512);
  if (a.ck > 1) {
    cg::cluster_group cl = cg::this_cluster();
    cl.sync();
    const float* red = reinterpret_cast<const float*>(wst);
    const T* bias = static_cast<const T*>(a.bias);
    const long long row0 = (long long)(unit0 % a.tiles) * ROWS, m0 = (long long)(unit0 / a.tiles) * MP;
    const int total = (int)min((long long)MP, a.m - m0) * ROWS;
    for (int e = rank * NT + tid; e < total; e += a.ck * NT) {
      const long long row = row0 + e % ROWS;
      if (row >= a.n) continue;
      float v = 0.f;
      for (int i = 0; i < a.ck; ++i) v += cl.map_shared_rank(red, i)[e];
      if (bias) v += to_f32(bias[row]);
      const long long o = (m0 + e / ROWS) * a.n + row;
      if (a.out_f32) static_cast<float*>(a.y)[o] = v;
      else static_cast<T*>(a.y)[o] = from_f32<T>(v);
    }
    cl.sync();
  }
}

// ------------------------------------------------------------------ host
int sm_count() {
  static std::atomic<int> sms{0};
  int v = sms.load(std::memory_order_relaxed);
  if (v == 0) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
      v = 148;
    sms.store(v, std::memory_order_relaxed);
  }
  return v;
}

// Sizes of a call; the same for the workspace query and the launch.
struct Plan {
  int tiles, ytiles, ck, per, staged, sb, resident;
  size_t ws_blocks, ws_total;
};

template <typename T, int MP, int GPC>
Plan plan(long long m, int n, int k) {
  using S = Shape<T, MP>;
  constexpr int BLK = S::block(GPC);
  Plan p{};
  const int chunks = (k + KC - 1) / KC;
  p.tiles = (n + ROWS - 1) / ROWS;
  p.ytiles = (int)((m + MP - 1) / MP);
  const long long units = (long long)p.tiles * p.ytiles;
  p.ck = 1;
  while (p.ck < 8 && units * p.ck * 2 <= 148 && chunks >= p.ck * 4) p.ck *= 2;
  p.per = (chunks + p.ck - 1) / p.ck;
  if (p.ck > 1) p.per = (p.per + 1) / 2 * 2;
  const bool fits = (long long)p.per * BLK <= B_SMEM && p.per <= MAX_SB;
  // every CTA stages x itself while that is at most four rounds of its threads
  p.staged = !(fits && p.ytiles == 1 && m * p.per * 16 <= 4 * NT);
  p.resident = fits && p.ytiles == 1;
  p.sb = p.resident ? (p.per > 0 ? p.per : 1) : (B_SMEM / BLK < 8 ? B_SMEM / BLK / 2 * 2 : 8);   // (even: each MMA warp has its own)
  p.ws_blocks = align_up((size_t)p.ytiles * chunks * BLK, 256);
  p.ws_total = p.staged ? p.ws_blocks + align_up((size_t)p.ytiles * MP * 8, 256) + 256 : 0;
  return p;
}

int weight_map(CUtensorMap* map, const void* q, int n, int k) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tmap_encoder();
  VERACE_REQUIRE(enc, VERACE_ERR_CUDA, "int4_linear: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)k / 2, (cuuint64_t)n}, strides[1] = {(cuuint64_t)k / 2};
  const cuuint32_t box[2] = {KC, ROWS}, el[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(q), dims, strides, box, el,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VERACE_REQUIRE(r == CUDA_SUCCESS, VERACE_ERR_CUDA, "int4_linear: tensor map of n=%d k=%d refused (%d)", n, k, (int)r);
  return VERACE_OK;
}

template <typename T, int MP, int GPC>
int launch(Int4Args a, void* workspace, size_t ws_bytes, cudaStream_t st) {
  using S = Shape<T, MP>;
  constexpr int BLK = S::block(GPC);
  const Plan p = plan<T, MP, GPC>(a.m, a.n, a.k);
  VERACE_REQUIRE(!p.staged || (workspace && ws_bytes >= p.ws_total), VERACE_ERR_WORKSPACE,
                 "int4_linear: workspace of %zu bytes required, %zu given", p.ws_total, workspace ? ws_bytes : (size_t)0);
  a.tiles = p.tiles; a.ytiles = p.ytiles; a.ck = p.ck; a.per = p.per;
  a.staged = p.staged; a.sb = p.sb; a.resident = p.resident;
  const int chunks = (a.k + KC - 1) / KC;
  if (p.staged) {
    uint8_t* base = reinterpret_cast<uint8_t*>(align_up((size_t)workspace, 256));
    float* scales = reinterpret_cast<float*>(base + p.ws_blocks);
    a.ws = base;
    a.ws_scale = scales;
    a.ws_mask = reinterpret_cast<uint32_t*>(scales + (size_t)p.ytiles * MP);
    int4_stage_x<T, MP, GPC><<<(unsigned)a.m, NT, 0, st>>>(static_cast<const T*>(a.x), a.ldx, a.k, chunks, base, scales,
                                                         const_cast<uint32_t*>(a.ws_mask));
    const int rc = check_launch("int4_stage_x");
    if (rc) return rc;
  }
  CUtensorMap map;
  if (a.k > 0) {
    const int rc = weight_map(&map, a.q, a.n, a.k);
    if (rc) return rc;
  }
  auto kern = int4_linear_kernel<T, MP, GPC>;
  const int smem = SW * W_STAGE + p.sb * BLK;
  static std::atomic<uint64_t> ready{0};      // devices whose limit is raised
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SW * W_STAGE + B_SMEM));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  const int units = p.tiles * p.ytiles;
  cfg.gridDim = dim3((unsigned)(p.ck > 1 ? units * p.ck : units < sm_count() ? units : sm_count()));
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (p.ck > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = p.ck;
    attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
    ++na;
  }
  if (p.staged) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = na;
  VERACE_CUDA(cudaLaunchKernelEx(&cfg, kern, map, a));
  return check_launch("int4_linear");
}

// Calls f with the (type, tokens per tile, groups per chunk) of a problem.
template <typename F>
auto dispatch(long long m, int group, int dtype, F f) {
  auto by_group = [&](auto t, auto mp) {
    if (group == 128) return f(t, mp, std::integral_constant<int, 1>());
    if (group == 64) return f(t, mp, std::integral_constant<int, 2>());
    return f(t, mp, std::integral_constant<int, 4>());
  };
  auto by_tokens = [&](auto t) {
    if (m <= 8) return by_group(t, std::integral_constant<int, 8>());
    if (m <= 16) return by_group(t, std::integral_constant<int, 16>());
    if (m <= 32) return by_group(t, std::integral_constant<int, 32>());
    return by_group(t, std::integral_constant<int, 64>());
  };
  if (dtype == VERACE_F32) {
    if (m <= 3) return by_group(float(), std::integral_constant<int, 3>());
    if (m <= 8) return by_group(float(), std::integral_constant<int, 8>());
    return by_group(float(), std::integral_constant<int, 16>());
  }
  if (dtype == VERACE_BF16) return by_tokens(__nv_bfloat16());
  return by_tokens(__half());
}

}  // namespace

int int4_read_status(int* status) {
  int h = 0;
  VERACE_CUDA(cudaMemcpyFromSymbol(&h, g_int4_status, sizeof(int)));
  if (h) {
    const int zero = 0;
    VERACE_CUDA(cudaMemcpyToSymbol(g_int4_status, &zero, sizeof(int)));
  }
  *status = h;
  return VERACE_OK;
}

}  // namespace verace

using namespace verace;

extern "C" size_t verace_int4_linear_workspace(long long m, int n, int k, int group, int dtype) {
  if (m <= 0 || n <= 0 || k < 0 || k % 32 || (group != 32 && group != 64 && group != 128) || dtype < VERACE_F32 ||
      dtype > VERACE_F16)
    return 0;
  return dispatch(m, group, dtype, [&](auto t, auto mp, auto gpc) {
    return plan<decltype(t), decltype(mp)::value, decltype(gpc)::value>(m, n, k).ws_total;
  });
}

extern "C" int verace_int4_linear(const void* x, long long ldx, const void* qweight, const void* scales,
                                  const void* zeros, const void* bias, void* y, long long m, int n, int k,
                                  int group, int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
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
  VERACE_REQUIRE(m <= 1LL << 20 && n <= 1 << 28 && (m + 2) / 3 * ((n + ROWS - 1) / ROWS) < 1LL << 30,
                 VERACE_ERR_UNSUPPORTED, "int4_linear: m %lld, n %d too large", m, n);
  Int4Args a{};
  a.x = x; a.ldx = ldx; a.q = static_cast<const uint8_t*>(qweight); a.s = scales;
  a.z = static_cast<const uint8_t*>(zeros); a.bias = bias; a.y = y; a.m = m; a.n = n; a.k = k;
  a.out_f32 = out_dtype == VERACE_F32;
  return dispatch(m, group, dtype, [&](auto t, auto mp, auto gpc) {
    return launch<decltype(t), decltype(mp)::value, decltype(gpc)::value>(a, workspace, workspace_bytes,
                                                                          static_cast<cudaStream_t>(stream));
  });
}
