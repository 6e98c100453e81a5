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
// shift and two masks.  x goes in as fp8 pieces that add up to it:
//   * few tokens: e4m3 pieces, each the rest of the one before times 2^5, in columns of their
//     own (a 128-row MMA takes 50 clocks for anything up to 64 columns): y = d0 + 2^-5 d1 + ...
//     bf16's 8 bits are 2 pieces, fp16's 11 are 3, fp32's 24 are 5;
//   * up to 64 tokens of 16-bit types: an e4m3 piece and one or two e5m2 pieces of the rest, one
//     MMA after the other into the same columns.
// Each token (of a CTA's share of k, where CTAs stage x themselves) is scaled by a power of two, its
// largest input to [2^7, 2^8).  The pieces hold an input whole down to 2^-14 (bf16), 2^-16 (fp16, up to 16
// tokens) or 2^-13 (the others) of that largest; a smaller one is off by at most 2^-22 of the largest
// (bf16; 2^-21 beyond 32 tokens), 2^-26 (fp16; 2^-23 beyond 16 tokens) or 2^-37 (fp32).  The zeros run
// over the same pieces, so y is the product of these inputs but for fp32 sums.  (A scale for each group
// as well, one more factor in the sums, would keep more digits where a whole group is far above the rest
// and has no weight.  It cost 4 to 20 % of every call, 125 to 147 us against 119 for 16 x 65536 x 16384 in
// five forms: the summing warps have neither registers nor issue slots left.)
// tcgen05.mma adds fp8 products in full fp32 (measured: 2^23 + 1 is exact).  The zeros are one
// more MMA per group: 32 inputs that hold X = the sum of a column's pieces over the group, in 6 e5m2
// pieces, against -z.  So D = 2^-9 (sum q x - z X) per group, and a row's thread adds s D in fp32.  No
// weight is rounded.
// What q x and z X lose by cancelling is 2^-24 of the sums of q |x|.  Where at most a
// sixteenth of a group is 2^12 above all the rest, that could show in the outputs whose q = z
// there, so those inputs (and what is above 2^100, infinities and NaN) are left out of the pieces and
// added one by one as (q - z) x s at the end (rare).
//
// One CTA per SM, 128 output rows at a time, 20 warps.  One warp feeds the weights by TMA (128
// rows x 256 codes a stage, 128-byte swizzle: a row's thread reads 16 bytes without bank
// conflicts), one the staged x.  The rest are two lines that take every other chunk of 256 inputs,
// each with four warps that unpack codes into TMEM (the MMA's A operand), one that issues the
// MMAs, four that hold the rows' sums, and its own places in TMEM.  Every role is a chain of
// dependent steps of 30 to 100 clocks (a barrier, a shared-memory or TMEM round trip; an MMA takes
// a warp 33 clocks to issue), 600 to 1000 a chunk; a chunk's weights take 712 clocks of an SM's
// share of the memory rate, and two lines have twice that.  Few row tiles: k is split over a
// cluster and the partial sums are joined through distributed shared memory in rank order.
//
// Measured on the device (copies run at 6.55 TB/s): 1 x 163840 x 1024 bf16 22 to 23 us, 3.9 TB/s;
// 16 x 65536 x 16384 118 to 122 us, 4.6 TB/s (512 tiles over 148 CTAs: three rounds and half a one);
// 64 x 16384 x 4096 20.7 us, 415 TFLOP/s, 3 us of it the staging of x; 7 x 4096 x 8192 fp16 12.5 to 13.1 us
// and 1 x 3080 x 1024 6.7 us, of which set-up and joins are 5.
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

constexpr uint32_t POLLS = 1u << 16;     // of 64 polls each
constexpr int NT = 640;                  // threads: 20 warps
constexpr int ROWS = 128;                // output rows per tile
constexpr int KC = 256;                  // inputs per chunk
constexpr int W_STAGE = ROWS * KC / 2;   // bytes: 128 rows x 256 codes
constexpr int MAX_SB = 32;
constexpr int SMEM = 220 * 1024;
constexpr float KEPT = 1.2676506e30f;    // 2^100: inputs above it (infinities, NaN) are added one by one
constexpr float APART = 1.f / 4096.f;

// How a token tile's x is laid out.  MP tokens per tile; COLS: the pieces in columns of their own.
// GPC: groups per chunk.
template <typename T, int MP_, int GPC_>
struct Shape {
  static constexpr bool IS32 = std::is_same<T, float>::value;
  static constexpr int MP = MP_, GPC = GPC_;
  static constexpr bool COLS = IS32 || MP <= (std::is_same<T, __half>::value ? 16 : 32);
  static constexpr int P = IS32 ? 5 : std::is_same<T, __half>::value ? 3 : 2;    // pieces
  static constexpr int N = COLS ? (P * MP + 15) / 16 * 16 : MP;                  // MMA columns
  static constexpr int PASSES = COLS ? 1 : P;
  // sums: a line's warps hold all tokens of their chunks, and one line's sums are added to the
  // other's at the end; for 64 tokens, more than the registers hold, both lines' warps take half
  // of the tokens of every chunk
  static constexpr bool HALVES = MP > 32;
  static constexpr int TB = MP < 16 ? MP : 16;                                   // tokens summed at a time
  static constexpr int PART = HALVES ? 0 : 2 * MP * ROWS * 4;                    // bytes of sums handed over
  // TMEM: two accumulators (a pair of groups) per line, the rest for chunks of A, as many per line
  static constexpr int D_COL = 512 - 4 * N;
  static constexpr int A_COLS = KC / 4 + 8 * GPC;
  static constexpr int NA = D_COL / A_COLS >= 4 ? 4 : 2;
  static_assert(NA * A_COLS <= D_COL, "TMEM");
  // bytes of a chunk's B operands: the passes' [256 / 16][N][16], then per group the zeros' [2][N][16]
  static constexpr int BLK = PASSES * KC * N + GPC * 32 * N;
  // weight stages (even): fewer where x's blocks are large and want the room (64 fp32 tokens of 16384 x
  // 4096, blocks of 25.6 KB: 44.7 us with 6, 42.0 with 4; 5 of 32001 x 1056 in groups of 32, 24 KB:
  // 17.9 and 19.6)
  static constexpr int SW = BLK > 24 * 1024 ? 4 : 6;
  static constexpr int B_SMEM = SMEM - SW * W_STAGE - PART;                      // bytes for x
  static_assert(B_SMEM >= 2 * BLK, "x is at least double-buffered");
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
  int first, last;     // the launch's units (a row tile of a token tile)
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
    if (!(fabsf(v[i]) <= KEPT)) out = true, v[i] = 0.f;
    mine = fmaxf(mine, fabsf(v[i]));
  }
  float top = mine;
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // any input far below the largest: perhaps that one stands alone.  (left_out decides by the same rule,
  // for every group that shares a bit of the mask: what this leaves in it must not add again.)
  int low = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) low |= fabsf(v[i]) < top * APART && v[i] != 0.f;
  if (__any_sync(0xffffffffu, low)) {
    int high = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) high += fabsf(v[i]) >= top * APART;
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

// The exponent that brings `top` (at most KEPT) to [2^7, 2^8), or as far as 2^126 does: what is below
// 2^-119 has no digits that the last piece would miss.  The sums' factor, with the codes' 2^9, stays a
// normal number at both ends.
__device__ __forceinline__ int shift_of(float top) {
  return min(7 - ((int)(__float_as_uint(top) >> 23) - 127), 126);
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
__device__ __forceinline__ float factor_of(int shift) { return pow2(9 - shift); }

// Writes the pieces of a lane's eight inputs of a chunk (token row t of the tile; a warp holds the
// chunk) and, from a group's first lanes, X.  A word's codes 0, 2, 4, 6 unpack before 1, 3, 5, 7, and so do x's bytes.
template <typename T, typename S>
__device__ __forceinline__ void stage8(float (&v)[8], float scale, uint8_t* block, int t, int lane) {
  constexpr int LANES = 32 / S::GPC, NX = S::COLS ? S::P : 1;     // NX: the X of a group
  float sum[NX];
#pragma unroll
  for (int p = 0; p < NX; ++p) sum[p] = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] *= scale;
  constexpr int at[4][2] = {{0, 2}, {4, 6}, {1, 3}, {5, 7}};
  uint8_t* d = block + ((lane / 2) * S::N + t) * 16 + (lane % 2) * 8;
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
        sum[p] += f.x + f.y;
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
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&r));
        sum[S::COLS ? p : 0] += f.x + f.y;
        h[i] = __hsub2(h[i], *reinterpret_cast<const __half2*>(&r));
        if (S::COLS) h[i] = __hmul2(h[i], __float2half2_rn(32.f));
      }
      put(p, b);
    }
  }
#pragma unroll
  for (int p = 0; p < NX; ++p)
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) sum[p] += __shfl_xor_sync(0xffffffffu, sum[p], o);
  // X of each column in e5m2 pieces, 4 bits each: 24, which hold a column's sum whole (of multiples of
  // 2^-9 below 2^15), so that code = zero adds nothing
  uint4* z = reinterpret_cast<uint4*>(block + S::PASSES * KC * S::N + (lane / LANES) * 32 * S::N) + t;
#pragma unroll
  for (int p0 = 0; p0 < NX; p0 += LANES) {          // a lane per column
    float x = sum[p0];
#pragma unroll
    for (int p = p0 + 1; p < NX && p < p0 + LANES; ++p)
      if (lane % LANES == p - p0) x = sum[p];
    const int p = p0 + lane % LANES;
    if (p < NX) {
      uint32_t w[2] = {0, 0};
#pragma unroll
      for (int i = 0; i < 6; ++i) {
        const uint32_t b = __nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E5M2);
        w[i / 4] |= b << (8 * (i % 4));
        const __half_raw r = __nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)b, __NV_E5M2);
        x -= __half2float(*reinterpret_cast<const __half*>(&r));
      }
      z[p * S::MP] = make_uint4(w[0], w[1], 0, 0);
      z[S::N + p * S::MP] = make_uint4(0, 0, 0, 0);
    }
  }
}

// The staging kernel: one CTA per token, a warp per chunk.
constexpr int STAGE_NT = 512;
template <typename T, typename S>
__global__ void __launch_bounds__(STAGE_NT) int4_stage_x(const T* __restrict__ x, long long ldx, int k, int chunks,
                                                         uint8_t* __restrict__ ws, float* __restrict__ scales,
                                                         uint32_t* __restrict__ masks) {
  constexpr int LANES = 32 / S::GPC;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ int s_top;
  __shared__ uint32_t s_mask;
  const int tid = threadIdx.x, lane = tid % 32;
  const long long tok = blockIdx.x;
  const T* row = x + tok * ldx;
  const int span = (chunks * S::GPC + 31) / 32;
  if (tid == 0) s_top = 0, s_mask = 0;
  __syncthreads();
  float most = 0.f;
  for (int c = tid / 32; c < chunks; c += STAGE_NT / 32) {
    const int at = c * KC + lane * 8;
    float v[8];
    load8(row + at, at < k, v);
    bool out;
    most = fmaxf(most, leave_out<LANES>(v, out));
    if (out) atomicOr(&s_mask, 1u << ((c * S::GPC + lane / LANES) / span));
  }
  atomicMax(&s_top, __reduce_max_sync(0xffffffffu, __float_as_int(most)));
  __syncthreads();
  const int sh = shift_of(__int_as_float(s_top));
  uint8_t* block = ws + (tok / S::MP) * (long long)chunks * S::BLK;
  for (int c = tid / 32; c < chunks; c += STAGE_NT / 32) {
    const int at = c * KC + lane * 8;
    float v[8];
    load8(row + at, at < k, v);
    bool out;
    leave_out<LANES>(v, out);
    stage8<T, S>(v, pow2(sh), block + (long long)c * S::BLK, (int)(tok % S::MP), lane);
  }
  if (tid == 0) {
    scales[tok] = factor_of(sh);
    masks[tok] = s_mask;
  }
}

// The terms of one output that leave_out zeroed, over the group that starts at input k0.
template <typename T>
__device__ __noinline__ float left_out(const T* x, const uint8_t* q, const T* s, const uint8_t* z, int n, int k_all,
                                       long long row, int k0, int group) {
  const int k1 = min(k0 + group, k_all);
  float top = 0.f;
  for (int k = k0; k < k1; ++k) {
    const float m = fabsf(to_f32(x[k]));
    if (m <= KEPT) top = fmaxf(top, m);
  }
  int high = 0, low = 0;
  for (int k = k0; k < k1; ++k) {
    const float m = fabsf(to_f32(x[k]));
    if (m <= KEPT) {
      high += m >= top * APART;
      low |= m < top * APART && m != 0.f;
    }
  }
  const bool alone = low && high <= group / 16;
  const long long at = (long long)(k0 / group) * n + row;
  const float zero = z ? (float)z[at] : 8.f, scale = to_f32(s[at]);
  float v = 0.f;
  for (int k = k0; k < k1; ++k) {
    const float xv = to_f32(x[k]);
    if (fabsf(xv) <= KEPT && !(alone && fabsf(xv) >= top * APART)) continue;
    const uint8_t by = q[row * (k_all / 2) + k / 2];
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
__device__ __forceinline__ void tmem_st32(uint32_t a, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(a),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// Issues the load of n consecutive columns of this thread's lane; pin() keeps the uses behind the wait.
template <int n>
__device__ __forceinline__ void tmem_ld(uint32_t a, float* v) {
  static_assert(n == 2 || n == 4 || n == 8 || n == 16 || n == 32, "columns");
  if constexpr (n == 2) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x2.b32 {%0,%1}, [%2];" : "=f"(v[0]), "=f"(v[1]) : "r"(a));
  } else if constexpr (n == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]) : "r"(a));
  } else if constexpr (n == 8) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                 : "r"(a));
  } else {
#pragma unroll
    for (int i = 0; i < n; i += 16)
      asm volatile(
          "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
          : "=f"(v[i]), "=f"(v[i + 1]), "=f"(v[i + 2]), "=f"(v[i + 3]), "=f"(v[i + 4]), "=f"(v[i + 5]),
            "=f"(v[i + 6]), "=f"(v[i + 7]), "=f"(v[i + 8]), "=f"(v[i + 9]), "=f"(v[i + 10]), "=f"(v[i + 11]),
            "=f"(v[i + 12]), "=f"(v[i + 13]), "=f"(v[i + 14]), "=f"(v[i + 15])
          : "r"(a + i));
  }
}
template <int n>
__device__ __forceinline__ void pin(float* v) {
#pragma unroll
  for (int i = 0; i < n; i += 2) asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
struct Bars {
  uint64_t wfull[6], wempty[6], afull[4], aempty[4], dfull[2], dempty[2], bfull[MAX_SB], bempty[MAX_SB], xready, drain;
};

// A place in a ring of barriers, and the parity of the completion awaited there: `phase` for one
// that fills, phase ^ 1 for one that empties (which passes on the first turn).
struct Turn {
  int slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++slot == n) slot = 0, phase ^= 1;
  }
  // every other place of an even ring
  __device__ __forceinline__ void next2(int n) {
    slot += 2;
    if (slot >= n) slot -= n, phase ^= 1;
  }
};

__device__ __forceinline__ bool try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
               : "=r"(done)
               : "r"(tc::smem_addr(bar)), "r"(parity)
               : "memory");
  return done;
}
// One lane of a converged warp.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p;
}

// Waits for a completion, but not for ever: when one does not come, the status word is set and no
// wait of the CTA blocks any more.  The roles then run to their ends on whatever is there (every
// address stays in range), the copies and MMAs in flight are waited for with the same bound, and
// the TMEM is freed.
__device__ __noinline__ void wait_longer(uint64_t* bar, uint32_t parity, volatile int* fail) {
  for (uint32_t i = 0; i < POLLS; ++i) {
    if (tc::mbar_wait(bar, parity, 64)) return;
    if (*fail) return;
  }
  *fail = 1;
  atomicExch(&g_int4_status, 1);
}
struct Waiter {
  volatile int* fail;
  __device__ __forceinline__ void operator()(uint64_t* bar, uint32_t parity) const {
    if (!try_wait(bar, parity)) wait_longer(bar, parity, fail);
  }
};

template <typename T, typename S>
__global__ void __launch_bounds__(NT, 1) int4_linear_kernel(const __grid_constant__ CUtensorMap wmap, Int4Args a) {
  constexpr int BLK = S::BLK, N = S::N, MP = S::MP, GPC = S::GPC, G = KC / GPC, KB = 8 / GPC;   // KB: k blocks a group
  constexpr int SW = S::SW, PAIRS = GPC / 2;     // pairs of groups per chunk
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Bars bar;
  __shared__ uint32_t s_slot;
  __shared__ int s_fail;
  __shared__ int s_top[MP];
  __shared__ uint32_t s_mask[MP];
  __shared__ float s_factor[8][MP];            // of the token tile at hand, a copy for each summing warp
  __shared__ uint32_t s_marks[8][MP];
  uint8_t* wst = smem;
  uint8_t* bst = smem + SW * W_STAGE;
  float* part = reinterpret_cast<float*>(bst + (size_t)a.sb * BLK);   // [2][MP][ROWS]: one line's sums for the other
  const int tid = threadIdx.x, lane = tid % 32, w = __shfl_sync(0xffffffffu, tid / 32, 0);
  const int rank = a.ck > 1 ? blockIdx.x % a.ck : 0;
  const int chunks = (a.k + KC - 1) / KC;
  const int c0 = min(rank * a.per, chunks), nc = min(a.per, chunks - c0);
  const int unit0 = a.first + blockIdx.x / a.ck, units = a.last, step = gridDim.x / a.ck;
  const int span = ((a.staged ? chunks : a.per) * GPC + 31) / 32;     // groups per bit of a left-out mask

  if (w == 1) tc::tmem_alloc(&s_slot, 512);
  if (tid == 0) {
    for (int i = 0; i < SW; ++i) tc::mbar_init(&bar.wfull[i], 1), tc::mbar_init(&bar.wempty[i], 4);
    for (int i = 0; i < S::NA; ++i) tc::mbar_init(&bar.afull[i], 4), tc::mbar_init(&bar.aempty[i], 1);
    for (int i = 0; i < 2; ++i) tc::mbar_init(&bar.dfull[i], 1), tc::mbar_init(&bar.dempty[i], S::HALVES ? 8 : 4);
    for (int i = 0; i < a.sb; ++i) tc::mbar_init(&bar.bfull[i], 1), tc::mbar_init(&bar.bempty[i], 1);
    tc::mbar_init(&bar.xready, 8);
    tc::mbar_init(&bar.drain, 2);
    tc::fence_mbar_init();
    s_fail = 0;
    // the first weights, before anything else
    for (int i = 0; i < SW && i < nc; ++i) {
      tc::mbar_expect_tx(&bar.wfull[i], W_STAGE);
      tc::tma_load_2d(wst + i * W_STAGE, &wmap, (c0 + i) * (KC / 2), unit0 % a.tiles * ROWS, &bar.wfull[i]);
    }
  }
  if (tid < MP) s_top[tid] = 0, s_mask[tid] = 0;
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  // all 512 columns are this CTA's, so they start at column 0 (addresses without the base stay
  // in uniform registers)
  const Waiter wait{&s_fail};
  if (tid == 0 && s_slot != 0) {
    s_fail = 1;
    atomicExch(&g_int4_status, 1);
  }

  if (w == 0) {
    // ---- weights
    if (elect()) {
      Turn tw;
      int it = 0;
      for (int u = unit0; u < units; u += step) {
        const int y = u % a.tiles * ROWS;
        for (int c = 0; c < nc; ++c, ++it, tw.next(SW)) {
          if (it < SW && u == unit0) continue;             // loaded above
          wait(&bar.wempty[tw.slot], tw.phase ^ 1);
          tc::mbar_expect_tx(&bar.wfull[tw.slot], W_STAGE);
          tc::tma_load_2d(wst + tw.slot * W_STAGE, &wmap, (c0 + c) * (KC / 2), y, &bar.wfull[tw.slot]);
        }
      }
      // copies still in flight land before the CTA may exit
      for (int j = it - SW < 0 ? 0 : it - SW; j < it; ++j) wait(&bar.wfull[j % SW], j / SW & 1);
    }
  } else if (w == 1) {
    // ---- staged x
    if (a.staged && elect()) {
      asm volatile("griddepcontrol.wait;" ::: "memory");
      Turn tb;
      int it = 0;
      for (int u = unit0; u < units && !(a.resident && u > unit0); u += step) {
        const uint8_t* src = a.ws + ((long long)(u / a.tiles) * chunks + c0) * BLK;
        for (int c = 0; c < nc; ++c, ++it, tb.next(a.sb), src += BLK) {
          wait(&bar.bempty[tb.slot], tb.phase ^ 1);
          tc::mbar_expect_tx(&bar.bfull[tb.slot], BLK);
          tc::bulk_load(bst + tb.slot * BLK, src, BLK, &bar.bfull[tb.slot]);
        }
      }
      for (int j = it - a.sb < 0 ? 0 : it - a.sb; j < it; ++j) wait(&bar.bfull[j % a.sb], j / a.sb & 1);
    }
  } else if (w < 4) {
    // ---- MMAs.  The whole warp walks the loop, so that the operands sit in uniform registers (33
    // clocks an MMA; a single lane's loop took 114).
    const bool lead = elect();
    const int line = w - 2;
    Turn ta, tb;
    ta.slot = tb.slot = line;
    uint32_t dphase = 0;
    int first = line;
    if (!a.staged && nc > 0) wait(&bar.xready, 0);
    for (int u = unit0; u < units; u += step) {
      int c = first;
      for (; c < nc; c += 2) {
        const int slot = a.resident ? c : tb.slot;
        wait(&bar.afull[ta.slot], ta.phase);
        if (a.staged) wait(&bar.bfull[slot], a.resident ? 0 : tb.phase);
        const uint32_t A = ta.slot * S::A_COLS;
        const uint64_t B = tc::sdesc(tc::smem_addr(bst + slot * BLK), N * 16, 128);
#pragma unroll
        for (int gj = 0; gj < PAIRS; ++gj, dphase ^= 1) {
          wait(&bar.dempty[line], dphase ^ 1);
          tc::fence_after_sync();
          if (lead) {
            constexpr uint32_t main0 = idesc_f8(N, 0), rest = idesc_f8(N, 1);
#pragma unroll
            for (int gi = 2 * gj; gi < 2 * gj + 2; ++gi) {
              const uint32_t D = S::D_COL + (2 * line + gi % 2) * N, Ag = A + gi * (8 * KB);
              const uint64_t Bg = B + (uint64_t)(gi * (KB * 32 * N >> 4));
#pragma unroll
              for (int p = 0; p < S::PASSES; ++p)
#pragma unroll
                for (int b = 0; b < KB; ++b)
                  mma_f8(D, Ag + 8 * b, Bg + (uint64_t)((p * KC * N + b * 32 * N) >> 4), p > 0 ? rest : main0,
                         p + b > 0);
              mma_f8(D, A + KC / 4 + 8 * gi, B + (uint64_t)((S::PASSES * KC * N >> 4) + gi * (32 * N >> 4)), rest, true);
            }
            tc::commit(&bar.dfull[line]);
          }
        }
        if (lead) {
          tc::commit(&bar.aempty[ta.slot]);
          if (a.staged && !a.resident) tc::commit(&bar.bempty[slot]);
        }
        ta.next2(S::NA);
        if (!a.resident) tb.next2(a.sb);
      }
      first = c - nc;
    }
    if (lead) {
      tc::commit(&bar.drain);        // every MMA issued is done before the TMEM goes
      wait(&bar.drain, 0);
    }
  } else if (w < 12) {
    // ---- unpacking: a thread is a row
    const int line = (w - 4) / 4, r = w % 4 * 32 + lane;
    const uint32_t lanes = (uint32_t)(w % 4 * 32) << 16;
    Turn tw, ta;
    tw.slot = ta.slot = line;
    const int groups = (a.k + G - 1) / G - c0 * GPC;         // from this CTA's first
    // the zeros of the line's next chunk, a chunk ahead (across units)
    int zu = unit0, ztile = unit0 % a.tiles, zc = line;
    const uint8_t* zp = nullptr;
    bool zlive = false;
    uint8_t zn[GPC];
    auto zeros_at = [&] {
      const long long row = (long long)ztile * ROWS + r;
      zlive = zu < units && row < a.n;
      zp = a.z + (long long)(c0 + zc) * GPC * a.n + row;
    };
    auto load_zeros = [&] {
      if (zc >= nc) {
        while (zc >= nc && zu < units) {
          zc -= nc, zu += step, ztile += step;
          while (ztile >= a.tiles) ztile -= a.tiles;
        }
        zeros_at();
      }
#pragma unroll
      for (int gi = 0; gi < GPC; ++gi)
        zn[gi] = zlive && zc * GPC + gi < groups ? __ldg(zp + (long long)gi * a.n) : 8;
      zc += 2;
      zp += 2LL * GPC * a.n;
    };
    if (a.z && nc > 0) {
      zeros_at();
      load_zeros();
    }
    int first = line, fresh = S::NA / 2;
    for (int u = unit0; u < units; u += step) {
      int c = first;
      for (; c < nc; c += 2) {
        wait(&bar.wfull[tw.slot], tw.phase);
        const uint8_t* src = wst + tw.slot * W_STAGE + r * (KC / 2);
        uint4 raw[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) raw[j] = *reinterpret_cast<const uint4*>(src + ((j ^ (r & 7)) * 16));
        wait(&bar.aempty[ta.slot], ta.phase ^ 1);
        __syncwarp();
        tc::fence_after_sync();
        const uint32_t A = lanes + ta.slot * S::A_COLS;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t code[32];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 q = raw[4 * h + j];
            const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              code[8 * j + 2 * i] = word[i] & 0x0f0f0f0fu;
              code[8 * j + 2 * i + 1] = (word[i] >> 4) & 0x0f0f0f0fu;
            }
          }
          tmem_st32(A + 32 * h, code);
        }
        if (lane == 0) tc::mbar_arrive(&bar.wempty[tw.slot]);       // (the warp's loads are in registers)
        if (a.z || fresh > 0) {        // without zeros, -8 stays where the first rounds wrote it
#pragma unroll
          for (int gi = 0; gi < GPC; ++gi) {
            uint32_t zw[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) zw[j] = a.z ? (0x80u | zn[gi]) * 0x01010101u : 0x88888888u;
            tmem_st8(A + KC / 4 + 8 * gi, zw);
          }
          if (a.z) load_zeros();
          --fresh;
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        tc::fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&bar.afull[ta.slot]);
        tw.next2(SW);
        ta.next2(S::NA);
      }
      first = c - nc;
    }
  } else {
    // ---- sums: a thread is an output row
    const int line = (w - 12) / 4, r = w % 4 * 32 + lane;
    if (!a.staged && nc > 0) {
      // first these warps stage the CTA's range of x: the tokens' largest inputs, then the pieces
      constexpr int LANES = 32 / GPC;
      const T* x = static_cast<const T*>(a.x) + c0 * KC + lane * 8;
      const int toks = (int)a.m, total = toks * nc;
      for (int u = w - 12; u < total; u += 8) {
        const int tok = u / nc, c = u - tok * nc;
        float v[8];
        load8(x + (long long)tok * a.ldx + c * KC, (c0 + c) * KC + lane * 8 < a.k, v);
        bool out;
        const float most = leave_out<LANES>(v, out);
        if (out) atomicOr(&s_mask[tok], 1u << ((c * GPC + lane / LANES) / span));
        const int m = __reduce_max_sync(0xffffffffu, __float_as_int(most));
        if (lane == 0) atomicMax(&s_top[tok], m);
      }
      tc::named_sync(1, 256);
      for (int u = w - 12; u < total; u += 8) {
        const int tok = u / nc, c = u - tok * nc;
        float v[8];
        load8(x + (long long)tok * a.ldx + c * KC, (c0 + c) * KC + lane * 8 < a.k, v);
        bool out;
        leave_out<LANES>(v, out);
        stage8<T, S>(v, pow2(shift_of(__int_as_float(s_top[tok]))), bst + c * BLK, tok, lane);
      }
      tc::fence_proxy_async();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&bar.xready);
    }
    if (a.staged) asm volatile("griddepcontrol.wait;" ::: "memory");
    constexpr int TH = S::HALVES ? MP / 2 : MP, TB = S::TB;
    constexpr int STRIDE = S::HALVES ? 1 : 2;      // chunks of the warp
    const int t0 = S::HALVES ? line * TH : 0;
    const uint32_t at = S::D_COL + ((uint32_t)(w % 4 * 32) << 16) + t0;
    const int groups = (a.k + G - 1) / G - c0 * GPC;         // from this CTA's first
    // the scales of the warp's next two pairs (across units), as loaded: 16-bit ones in words of
    // their own, since a conversion or a packed pair would wait for the load
    using Raw = typename std::conditional<S::IS32, uint32_t, unsigned short>::type;
    int su = unit0, stile = unit0 % a.tiles, sc = S::HALVES ? 0 : line, sg = 0;     // sg: group in the chunk
    const Raw* sp = nullptr;
    bool slive = false;
    auto scales_at = [&] {
      const long long row = (long long)stile * ROWS + r;
      slive = su < units && row < a.n;
      sp = reinterpret_cast<const Raw*>(a.s) + (long long)(c0 + sc) * GPC * a.n + row;
    };
    auto load_scales = [&](uint32_t (&to)[2]) {
      if (sg == GPC) {
        sg = 0, sc += STRIDE, sp += (long long)(STRIDE - 1) * GPC * a.n;
        if (sc >= nc) {
          while (sc >= nc && su < units) {
            sc -= nc, su += step, stile += step;
            while (stile >= a.tiles) stile -= a.tiles;
          }
          scales_at();
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j, sp += a.n) {
        to[j] = 0;
        if (slive && sc * GPC + sg + j < groups) to[j] = __ldg(sp);
      }
      sg += 2;
    };
    uint32_t s0[2] = {0, 0}, s1[2] = {0, 0};
    if (nc > 0) {
      if (sc >= nc) sg = GPC, sc -= STRIDE;        // (the first unit has no chunk of this line)
      else scales_at();
      load_scales(s0);
      load_scales(s1);
    }
    int first = S::HALVES ? 0 : line, buf = 0, turn = 0;     // turn: the line of the next chunk (HALVES)
    uint32_t dphase[2] = {0, 0};
    long long tile_m = -1;
    uint32_t any = 0;                   // whether inputs of its tokens were left out
    for (int u = unit0; u < units; u += step, buf ^= 1) {
      const long long row = (long long)(u % a.tiles) * ROWS + r, m0 = (long long)(u / a.tiles) * MP;
      const int toks = (int)min((long long)MP, a.m - m0);
      float bv = 0.f;
      if (a.bias && row < a.n) bv = to_f32(static_cast<const T*>(a.bias)[row]);
      if (m0 != tile_m) {
        tile_m = m0;
        __syncwarp();
        for (int t = lane; t < toks; t += 32) {
          s_factor[w - 12][t] = a.staged ? a.ws_scale[m0 + t]
                                         : nc > 0 ? factor_of(shift_of(__int_as_float(s_top[t]))) : 0.f;
          s_marks[w - 12][t] = a.staged ? a.ws_mask[m0 + t] : s_mask[t];
        }
        __syncwarp();
        any = 0;
        for (int t = t0; t < min(t0 + TH, toks); ++t) any |= s_marks[w - 12][t];
      }
      float acc[TH];
#pragma unroll
      for (int t = 0; t < TH; ++t) acc[t] = 0.f;
      int c = first;
      for (; c < nc; c += STRIDE) {
        const int from = S::HALVES ? turn : line;
#pragma unroll
        for (int gj = 0; gj < PAIRS; ++gj) {
          wait(&bar.dfull[from], S::HALVES ? (from ? dphase[1] : dphase[0]) : dphase[0]);
          __syncwarp();
          tc::fence_after_sync();
          const uint32_t D = at + 2 * from * N;
          constexpr int NP = S::COLS ? S::P : 1;          // columns of a token
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float s;
            if constexpr (S::IS32) s = __uint_as_float(s0[j]);
            else if constexpr (std::is_same<T, __half>::value) s = __half2float(__ushort_as_half((unsigned short)s0[j]));
            else s = __uint_as_float(s0[j] << 16);
#pragma unroll
            for (int b = 0; b < TH; b += TB) {
              float d[NP][TB];
#pragma unroll
              for (int p = 0; p < NP; ++p) tmem_ld<TB>(D + j * N + p * MP + b, d[p]);
              tmem_wait_ld();
              if (j == 1 && b + TB == TH) {
                tc::fence_before_sync();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&bar.dempty[from]);
              }
#pragma unroll
              for (int p = 0; p < NP; ++p) pin<TB>(d[p]);
#pragma unroll
              for (int t = 0; t < TB; ++t) {
                float v = d[NP - 1][t];
#pragma unroll
                for (int p = NP - 2; p >= 0; --p) v = fmaf(v, 1.f / 32.f, d[p][t]);
                acc[b + t] = fmaf(s, v, acc[b + t]);
              }
            }
          }
          s0[0] = s1[0];
          s0[1] = s1[1];
          load_scales(s1);
          if (S::HALVES && from) dphase[1] ^= 1;
          else dphase[0] ^= 1;
        }
        turn ^= 1;
      }
      first = c - nc;
      if (!S::HALVES) {
        // one line's sums go to the other, which writes the tile out; they change places every tile.
        // (Two buffers: a line writes one again after it has seen the other line's next sums, which
        // that line has not handed over before reading these.)
        float* to = part + buf * MP * ROWS + r;
        if (line != buf) {
#pragma unroll
          for (int t = 0; t < TH; ++t) to[t * ROWS] = acc[t];
          __threadfence_block();
          asm volatile("bar.arrive %0, 256;" ::"r"(2 + buf) : "memory");
          continue;
        }
        tc::named_sync(2 + buf, 256);
#pragma unroll
        for (int t = 0; t < TH; ++t) acc[t] = line ? to[t * ROWS] + acc[t] : acc[t] + to[t * ROWS];
      }
      // the tile's outputs (or this CTA's part of them)
#pragma unroll
      for (int t = 0; t < TH; ++t) acc[t] *= s_factor[w - 12][t0 + t];      // (what is beyond toks is not stored)
      if (any && row < a.n) {
        const T* x = static_cast<const T*>(a.x);
#pragma unroll
        for (int t = 0; t < TH; ++t) {
          const uint32_t mask = t0 + t < toks ? s_marks[w - 12][t0 + t] : 0u;
          for (int g = 0; mask && g < nc * GPC; ++g)
            if ((mask >> (((a.staged ? c0 * GPC : 0) + g) / span) & 1u) && (c0 * GPC + g) * G < a.k)
              acc[t] += left_out<T>(x + (m0 + t0 + t) * a.ldx, a.q, static_cast<const T*>(a.s), a.z, a.n, a.k, row,
                                    (c0 * GPC + g) * G, G);
        }
      }
      if (a.ck > 1) {
        float* red = reinterpret_cast<float*>(wst) + t0 * ROWS + r;   // (all stages are consumed: every sum is in)
#pragma unroll
        for (int t = 0; t < TH; ++t)
          if (t0 + t < toks) red[t * ROWS] = acc[t];
      } else if (row < a.n) {
        const long long o = (m0 + t0) * a.n + row;
        if (a.out_f32) {
          float* y = static_cast<float*>(a.y) + o;
#pragma unroll
          for (int t = 0; t < TH; ++t, y += a.n)
            if (t0 + t < toks) *y = acc[t] + bv;
        } else {
          T* y = static_cast<T*>(a.y) + o;
#pragma unroll
          for (int t = 0; t < TH; ++t, y += a.n)
            if (t0 + t < toks) *y = from_f32<T>(acc[t] + bv);
        }
      }
    }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (w == 1) tc::tmem_dealloc(s_slot, 512);
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
  int rest, rest_ck;   // units of a last round, in a launch of their own
  size_t ws_blocks, ws_total;
};

template <typename T, typename S>
Plan plan(long long m, int n, int k) {
  Plan p{};
  const int chunks = (k + KC - 1) / KC;
  p.tiles = (n + ROWS - 1) / ROWS;
  p.ytiles = (int)((m + S::MP - 1) / S::MP);
  const long long units = (long long)p.tiles * p.ytiles;
  p.ck = 1;
  while (p.ck < 8 && units * p.ck * 2 <= 148 && chunks >= p.ck * 2) p.ck *= 2;
  p.per = (chunks + p.ck - 1) / p.ck;
  const bool fits = (long long)p.per * S::BLK <= S::B_SMEM && p.per <= MAX_SB;
  // Every CTA stages x itself while that is at most five chunks for each of the eight warps that do it.
  // (There a kernel of its own is 2 us less on the device, 10.6 against 12.5 for 2 x 16384 x 4096, but
  // its launch takes the host 3 to 4; at 56 chunks, 7 x 4096 x 8192, 11.3 against 16.0.)
  p.staged = !(fits && p.ytiles == 1 && m * p.per <= 40);
  p.resident = fits && p.ytiles == 1;
  p.sb = p.resident ? (p.per > 0 ? p.per : 1) : (S::B_SMEM / S::BLK < 8 ? S::B_SMEM / S::BLK / 2 * 2 : 8);   // (even)
  // A last round that leaves half of the CTAs idle shares its tiles' k instead, where that saves more
  // than the second launch costs (16 x 20480 x 16384 fp16, 160 tiles: 94 -> 67 us; 16 x 65536 x 16384, 512
  // tiles: 120 -> 116).
  p.rest = units > 148 ? (int)(units % 148) : 0;
  for (p.rest_ck = 1; p.rest > 0 && p.rest_ck < 8 && p.rest * p.rest_ck * 2 <= 148;) p.rest_ck *= 2;
  if (!p.staged || p.resident || chunks - chunks / p.rest_ck < 24) p.rest = 0;
  p.ws_blocks = align_up((size_t)p.ytiles * chunks * S::BLK, 256);
  p.ws_total = p.staged ? p.ws_blocks + align_up((size_t)p.ytiles * S::MP * 8, 256) + 256 : 0;
  return p;
}

int weight_map(CUtensorMap* map, const void* q, int n, int k) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tmap_encoder();
  VERACE_REQUIRE(enc, VERACE_ERR_CUDA, "int4_linear: the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[2] = {(cuuint64_t)k / 2, (cuuint64_t)n}, strides[1] = {(cuuint64_t)k / 2};
  const cuuint32_t box[2] = {KC / 2, ROWS}, el[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(q), dims, strides, box, el,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VERACE_REQUIRE(r == CUDA_SUCCESS, VERACE_ERR_CUDA, "int4_linear: tensor map of n=%d k=%d refused (%d)", n, k, (int)r);
  return VERACE_OK;
}

template <typename T, typename S>
int launch(Int4Args a, void* workspace, size_t ws_bytes, cudaStream_t st) {
  constexpr int BLK = S::BLK;
  const Plan p = plan<T, S>(a.m, a.n, a.k);
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
    a.ws_mask = reinterpret_cast<uint32_t*>(scales + (size_t)p.ytiles * S::MP);
    int4_stage_x<T, S><<<(unsigned)a.m, STAGE_NT, 0, st>>>(static_cast<const T*>(a.x), a.ldx, a.k, chunks, base, scales,
                                                         const_cast<uint32_t*>(a.ws_mask));
    const int rc = check_launch("int4_stage_x");
    if (rc) return rc;
  }
  CUtensorMap map;
  if (a.k > 0) {
    const int rc = weight_map(&map, a.q, a.n, a.k);
    if (rc) return rc;
  }
  auto kern = int4_linear_kernel<T, S>;
  const int smem = S::SW * W_STAGE + p.sb * BLK + S::PART;
  static std::atomic<uint64_t> ready{0};      // devices whose limit is raised
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int sms = sm_count();
  auto go = [&](int first, int last, int ck, bool dependent) -> int {
    const int units = last - first;
    a.first = first, a.last = last;
    a.ck = ck, a.per = (chunks + ck - 1) / ck;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(ck > 1 ? units * ck : units < sms ? units : sms));
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    int na = 0;
    if (ck > 1) {
      attr[na].id = cudaLaunchAttributeClusterDimension;
      attr[na].val.clusterDim.x = ck;
      attr[na].val.clusterDim.y = attr[na].val.clusterDim.z = 1;
      ++na;
    }
    if (dependent) {
      attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[na].val.programmaticStreamSerializationAllowed = 1;
      ++na;
    }
    cfg.attrs = attr;
    cfg.numAttrs = na;
    VERACE_CUDA(cudaLaunchKernelEx(&cfg, kern, map, a));
    return check_launch("int4_linear");
  };
  const int units = p.tiles * p.ytiles;
  if (p.rest == 0) return go(0, units, p.ck, p.staged);
  const int rc = go(0, units - p.rest, 1, p.staged);
  return rc ? rc : go(units - p.rest, units, p.rest_ck, false);
}

// Calls f with a problem's type and shape.
template <typename F>
auto dispatch(long long m, int group, int dtype, F f) {
  auto by_group = [&](auto t, auto mp) {
    using T = decltype(t);
    constexpr int MP = decltype(mp)::value;
    if (group == 128) return f(t, Shape<T, MP, 2>());
    if (group == 64) return f(t, Shape<T, MP, 4>());
    return f(t, Shape<T, MP, 8>());
  };
  auto by_tokens = [&](auto t) {
    if (m <= 8) return by_group(t, std::integral_constant<int, 8>());
    if (m <= 16) return by_group(t, std::integral_constant<int, 16>());
    if (m <= 32) return by_group(t, std::integral_constant<int, 32>());
    return by_group(t, std::integral_constant<int, 64>());
  };
  if (dtype == VERACE_F32) {
    if (m <= 4) return by_group(float(), std::integral_constant<int, 4>());
    // (16 tokens' accumulators and the zeros of 8 groups do not fit TMEM together)
    if (m <= 8) return by_group(float(), std::integral_constant<int, 8>());
    if (group == 32) return f(float(), Shape<float, 8, 8>());
    if (group == 64) return f(float(), Shape<float, 16, 4>());
    return f(float(), Shape<float, 16, 2>());
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
  if (m <= 0 || n <= 0 || k < 0 || k > 1 << 30 || k % 32 || (group != 32 && group != 64 && group != 128) || dtype < VERACE_F32 ||
      dtype > VERACE_F16)
    return 0;
  return dispatch(m, group, dtype, [&](auto t, auto s) {
    return plan<decltype(t), decltype(s)>(m, n, k).ws_total;
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
  VERACE_REQUIRE(m <= 1LL << 20 && n <= 1 << 28 && k <= 1 << 30 && (m + 3) / 4 * ((n + ROWS - 1) / ROWS) < 1LL << 30,
                 VERACE_ERR_UNSUPPORTED, "int4_linear: m %lld, n %d, k %d too large", m, n, k);
  Int4Args a{};
  a.x = x; a.ldx = ldx; a.q = static_cast<const uint8_t*>(qweight); a.s = scales;
  a.z = static_cast<const uint8_t*>(zeros); a.bias = bias; a.y = y; a.m = m; a.n = n; a.k = k;
  a.out_f32 = out_dtype == VERACE_F32;
  return dispatch(m, group, dtype, [&](auto t, auto s) {
    return launch<decltype(t), decltype(s)>(a, workspace, workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}
