// Product of a few tokens with 4-bit weights:
//     y[i][n] = sum_k x[i][k] W[n][k] (+ bias[n]),   W[n][k] = s[k/G][n] (q[n][k] - z[k/G][n])
// q in [0, 15], two to a byte along k (the even k in the low half); z in [0, 15], 8 when no
// zeros are given.  One group's terms are summed with the integers q - z, exact in bf16 and
// fp16, and scaled once: y = sum_g s_g (sum_{k in g} x_k (q_k - z_g)), all sums in fp32.  No
// weight is ever rounded.
//
// Bound: the weights' bytes (half a byte for 2 m operations), as long as the tensor cores keep
// up.  So the weights stream through shared memory once, each warp on its own: 32 output rows
// by a chunk of 128 inputs at a time, three chunks in flight by cp.async, no barrier between
// warps.  mma.sync with the weights as the 16-row operand fits few tokens better than a
// 128-row tile: eight tokens are one instruction's columns.  The order of k inside a chunk is
// free (both operands use the same one): lane t of a row's four takes one 32-bit word of
// every 16 bytes, whose nibbles i and i + 4 unpack as a pair with one logic operation, and x
// is staged in that order, so that a lane's operand is one 16-byte load.
// fp32 inputs are cut into three bf16 columns of 8 significant bits each (exact).
#include "common.cuh"
#include "tc.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace verace {
namespace {

namespace cg = cooperative_groups;

constexpr int NT = 256;           // threads per CTA: 8 warps
constexpr int WARPS = NT / 32;
constexpr int ROWS = 32;          // output rows per warp
constexpr int KC = 128;           // inputs per chunk (64 bytes of a weight row)
constexpr int STAGES = 3;         // chunks in flight per warp
// A row's 64 bytes at a pitch of 80: the word loads of a fragment (8 rows x 4 lanes) hit 32 banks.
constexpr int PITCH = 80;
constexpr int STAGE_BYTES = ROWS * PITCH;
constexpr int RPITCH = 36;        // row pitch (floats) of the partial tiles, conflict-free likewise
constexpr int XSTREAM = 16384;    // bytes of x in one of the two streamed buffers, before padding

// A group's unscaled sum reaches 128 * 15 times its largest input: bf16 and fp32 inputs are
// brought down by 2^12 (exact) and the result back up, so that sums of any finite inputs stay
// finite.  fp16 inputs are below 2^16 and need none.
template <typename T> constexpr float down() { return std::is_same<T, __half>::value ? 1.f : 1.f / 4096.f; }
template <typename T> constexpr float up() { return std::is_same<T, __half>::value ? 1.f : 4096.f; }

// operand type of the products, and columns of the product per token
template <typename T> struct Op { using type = T; static constexpr int cols = 1; };
template <> struct Op<float> { using type = __nv_bfloat16; static constexpr int cols = 3; };

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
  int wk;        // warps of a CTA that share a row tile, interleaved along k
  int ck;        // CTAs of a cluster that share a row tile, each with a range of k
  int per;       // chunks in a CTA's range of k
  int resident;  // the whole range's x staged once (else 16 KB at a time, double-buffered)
  int x_bytes;   // shared memory of x
};

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Nibbles i and i + 4 of w (already shifted down by 4 i) minus the zero, as a pair: the code in
// the low mantissa bits of 128 (bf16) or 1024 (fp16) is that number plus the code.
template <typename T>
__device__ __forceinline__ uint32_t unpack(uint32_t w, uint32_t zero2) {
  constexpr uint32_t magic = std::is_same<T, __half>::value ? 0x64006400u : 0x43004300u;
  const uint32_t c = (w & 0x000f000fu) | magic;
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&c), *reinterpret_cast<const __half2*>(&zero2));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __nv_bfloat162 r =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&c), *reinterpret_cast<const __nv_bfloat162*>(&zero2));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t zero_pair(uint32_t z) {
  return ((std::is_same<T, __half>::value ? 0x6400u : 0x4300u) | z) * 0x10001u;
}

// Eight consecutive inputs as loaded, and their staging: pairs (0,4) (1,5) (2,6) (3,7).
template <typename T> struct Raw { uint4 u[sizeof(T) / 2]; };

template <typename T>
__device__ __forceinline__ void load_raw(Raw<T>& r, const T* p, bool valid) {
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
    r.u[i] = valid ? __ldg(reinterpret_cast<const uint4*>(p) + i) : make_uint4(0, 0, 0, 0);
}

__device__ __forceinline__ uint4 pair_up(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  // words (0,1) (2,3) (4,5) (6,7) -> (0,4) (1,5) (2,6) (3,7)
  return make_uint4(__byte_perm(a, c, 0x5410), __byte_perm(a, c, 0x7632), __byte_perm(b, d, 0x5410),
                    __byte_perm(b, d, 0x7632));
}

__device__ __forceinline__ uint32_t bf16_down(uint32_t w) {
  const __nv_bfloat162 f = __float2bfloat162_rn(1.f / 4096.f);
  const __nv_bfloat162 r = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&w), f);
  return *reinterpret_cast<const uint32_t*>(&r);
}

template <typename T>
__device__ __forceinline__ void store_staged(uint8_t* dst, int pitch, const Raw<T>& r) {
  if constexpr (std::is_same<T, float>::value) {
    // x = h + m + l exactly: the top 8 significant bits, the next 8, the rest (truncated, so
    // that nothing rounds up past the range; an infinity or NaN stays whole in h)
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.u);
    uint32_t h[4], m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t p[2][3];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = __uint_as_float(w[i + 4 * e]) * down<float>();
        const bool fin = fabsf(x) <= 3.4e38f;
        // a NaN keeps a bit in its top half
        const uint32_t hb = fin ? __float_as_uint(x) & 0xffff0000u
                                : (x != x ? 0x7fc00000u : __float_as_uint(x));
        const float rest = fin ? x - __uint_as_float(hb) : 0.f;
        const uint32_t mb = __float_as_uint(rest) & 0xffff0000u;
        const float last = rest - __uint_as_float(mb);
        p[e][0] = hb; p[e][1] = mb; p[e][2] = __float_as_uint(last);
      }
      h[i] = __byte_perm(p[0][0], p[1][0], 0x7632);
      m[i] = __byte_perm(p[0][1], p[1][1], 0x7632);
      l[i] = __byte_perm(p[0][2], p[1][2], 0x7632);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4*>(dst + pitch) = make_uint4(m[0], m[1], m[2], m[3]);
    *reinterpret_cast<uint4*>(dst + 2 * pitch) = make_uint4(l[0], l[1], l[2], l[3]);
  } else {
    uint4 u = r.u[0];
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
      u = make_uint4(bf16_down(u.x), bf16_down(u.y), bf16_down(u.z), bf16_down(u.w));
    *reinterpret_cast<uint4*>(dst) = pair_up(u.x, u.y, u.z, u.w);
  }
}

// scale bits and zero of one output row and group, carried by the row's lane
template <typename T> struct Scale { uint32_t v; };            // scale | zero << 16
template <> struct Scale<float> { uint32_t v; uint32_t zero; };

// C8: columns in tiles of 8.  GPC: groups per chunk.
template <typename T, int C8, int GPC>
__global__ void __launch_bounds__(NT, C8 <= 2 ? 2 : 1) int4_linear_mma(Int4Args a) {
  using O = typename Op<T>::type;
  constexpr int PER_TOK = Op<T>::cols;
  constexpr int TOK = 8 * C8 / PER_TOK;          // tokens per CTA
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* xs = smem;
  uint8_t* ws = smem + a.x_bytes;
  const int tid = threadIdx.x, lane = tid % 32, w = tid / 32, g = lane / 4, t = lane % 4;
  const int wk = w % a.wk, wr = w / a.wk;
  const int rank = blockIdx.x % a.ck;
  const long long tile0 = (long long)(blockIdx.x / a.ck) * (WARPS / a.wk) * ROWS;   // the CTA's first row
  const long long row0 = tile0 + wr * ROWS;
  const long long m0 = (long long)blockIdx.y * TOK;
  const int toks = (int)(a.m - m0 < TOK ? a.m - m0 : TOK);
  const int cols = toks * PER_TOK;
  const int chunks = (a.k + KC - 1) / KC;
  const int c0 = rank * a.per, c1 = min(chunks, c0 + a.per);
  const int steps = (max(c1 - c0, 0) + a.wk - 1) / a.wk;
  const size_t qrow = a.k / 2;

  // ---- weights: this warp's ring
  uint8_t* ring = ws + w * STAGES * STAGE_BYTES;
  const bool rows_live = row0 < a.n;
  const uint8_t* qp = a.q + (rows_live ? row0 + g : 0) * qrow + t * 16;
  auto load_stage = [&](int j) {
    const int c = c0 + j * a.wk + wk;
    if (rows_live && c < c1) {
      uint8_t* d = ring + (j % STAGES) * STAGE_BYTES + g * PITCH + t * 16;
      const bool in_k = c * 64 + t * 16 < (int)qrow;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const bool v = in_k && row0 + g + 8 * i < a.n;
        tc::cp_async16(d + 8 * i * PITCH, v ? qp + 8 * i * qrow + (size_t)c * 64 : a.q, v);
      }
    }
    tc::cp_async_commit();
  };
  // ---- scales and zeros: lane l carries row l's
  const T* sp = static_cast<const T*>(a.s) + row0 + lane;
  const uint8_t* zp = a.z ? a.z + row0 + lane : nullptr;
  const int groups = (a.k + KC / GPC - 1) / (KC / GPC);
  Scale<T> next[GPC];
  auto load_scales = [&](int j) {
    const int c = c0 + j * a.wk + wk;
#pragma unroll
    for (int i = 0; i < GPC; ++i) {
      const long long gi = (long long)c * GPC + i;
      const bool v = c < c1 && gi < groups && row0 + lane < a.n;
      const uint32_t zero = v && zp ? __ldg(zp + gi * a.n) : 8u;
      if constexpr (std::is_same<T, float>::value) {
        next[i].v = v ? __float_as_uint(__ldg(sp + gi * a.n)) : 0u;
        next[i].zero = zero;
      } else {
        next[i].v = (v ? (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(sp) + gi * a.n) : 0u) | (zero << 16);
      }
    }
  };
#pragma unroll
  for (int j = 0; j < STAGES; ++j) load_stage(j);
  load_scales(0);

  // ---- x: staged whole, or streamed XSTREAM bytes at a time
  const int sx = a.resident ? max(steps, 1) : (8 / C8) / a.wk;      // steps per buffer
  const int xk = sx * a.wk * KC;                                    // inputs per buffer
  const int xpitch = xk * 2 + 64;
  const int xbuf = 8 * C8 * xpitch;
  const T* x = static_cast<const T*>(a.x) + m0 * a.ldx;
  const int units_k = xk / 8;
  constexpr int XR = (XSTREAM / 16 + NT - 1) / NT;                  // units per thread and buffer, at most
  Raw<T> xr[XR];
  auto fetch_x = [&](int b) {
    const int kb = (c0 * KC) + b * xk;
#pragma unroll
    for (int i = 0; i < XR; ++i) {
      const int u = tid + i * NT, tok = u / units_k, k = kb + (u - tok * units_k) * 8;
      if (tok < toks) load_raw(xr[i], x + (long long)min(tok, toks - 1) * a.ldx + k, k < a.k);
    }
  };
  auto store_x = [&](int b) {
#pragma unroll
    for (int i = 0; i < XR; ++i) {
      const int u = tid + i * NT, tok = u / units_k;
      if (tok < toks)
        store_staged<T>(xs + (b & 1) * xbuf + tok * PER_TOK * xpitch + (u - tok * units_k) * 16, xpitch, xr[i]);
    }
  };
  if (a.resident) {
    const int units = toks * units_k;
    for (int u0 = 0; u0 < units; u0 += 4 * NT) {
      Raw<T> r[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = u0 + tid + i * NT, tok = u / units_k, k = c0 * KC + (u - tok * units_k) * 8;
        if (u < units) load_raw(r[i], x + (long long)tok * a.ldx + k, k < a.k);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int u = u0 + tid + i * NT, tok = u / units_k;
        if (u < units) store_staged<T>(xs + tok * PER_TOK * xpitch + (u - tok * units_k) * 16, xpitch, r[i]);
      }
    }
  } else {
    fetch_x(0);
    store_x(0);
  }
  __syncthreads();

  float acc[2][C8][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < C8; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][c][e] = 0.f;

  // a lane's columns (clamped: what a column without a token computes is not stored)
  int xcol[C8];
#pragma unroll
  for (int c = 0; c < C8; ++c) xcol[c] = min(8 * c + g, cols - 1) * xpitch + t * 16;

  for (int j = 0; j < steps; ++j) {
    const int b = j / sx, jb = j - b * sx;
    if (!a.resident && jb == 0) {
      if (j > 0) {
        store_x(b);
        __syncthreads();
      }
      if ((b + 1) * sx < steps) fetch_x(b + 1);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
    __syncwarp();
    Scale<T> sc[GPC];
#pragma unroll
    for (int i = 0; i < GPC; ++i) sc[i] = next[i];
    if (j + 1 < steps) load_scales(j + 1);
    if (rows_live && c0 + j * a.wk + wk < c1) {
      const uint8_t* st = ring + (j % STAGES) * STAGE_BYTES + g * PITCH + t * 4;
      const uint8_t* xb = xs + (a.resident ? 0 : (b & 1) * xbuf) + (jb * a.wk + wk) * KC * 2;
#pragma unroll
      for (int gi = 0; gi < GPC; ++gi) {
        uint32_t zero[4];
        float scale[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const uint32_t v = __shfl_sync(0xffffffffu, sc[gi].v, 8 * r + g);
          if constexpr (std::is_same<T, float>::value) {
            scale[r] = __uint_as_float(v);
            zero[r] = zero_pair<O>(__shfl_sync(0xffffffffu, sc[gi].zero, 8 * r + g));
          } else {
            scale[r] = std::is_same<T, __half>::value
                           ? __half2float(__ushort_as_half((unsigned short)(v & 0xffffu)))
                           : __uint_as_float(v << 16);
            zero[r] = zero_pair<O>(v >> 16);
          }
        }
        float part[2][C8][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < C8; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[i][c][e] = 0.f;
#pragma unroll
        for (int kb = 0; kb < 4 / GPC; ++kb) {
          const int i = gi * (4 / GPC) + kb;     // 16-byte block of the chunk: 32 inputs
          uint4 xf[C8];
#pragma unroll
          for (int c = 0; c < C8; ++c) xf[c] = *reinterpret_cast<const uint4*>(xb + xcol[c] + i * 64);
#pragma unroll
          for (int mt = 0; mt < 2; ++mt) {
            const uint32_t w0 = *reinterpret_cast<const uint32_t*>(st + mt * 16 * PITCH + i * 16);
            const uint32_t w1 = *reinterpret_cast<const uint32_t*>(st + (mt * 16 + 8) * PITCH + i * 16);
            const uint32_t z0 = zero[2 * mt], z1 = zero[2 * mt + 1];
            const uint32_t a0[4] = {unpack<O>(w0, z0), unpack<O>(w1, z1), unpack<O>(w0 >> 4, z0),
                                    unpack<O>(w1 >> 4, z1)};
            const uint32_t a1[4] = {unpack<O>(w0 >> 8, z0), unpack<O>(w1 >> 8, z1), unpack<O>(w0 >> 12, z0),
                                    unpack<O>(w1 >> 12, z1)};
#pragma unroll
            for (int c = 0; c < C8; ++c) {
              mma<O>(part[mt][c], a0, xf[c].x, xf[c].y);
              mma<O>(part[mt][c], a1, xf[c].z, xf[c].w);
            }
          }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
          for (int c = 0; c < C8; ++c) {
            acc[mt][c][0] = fmaf(scale[2 * mt], part[mt][c][0], acc[mt][c][0]);
            acc[mt][c][1] = fmaf(scale[2 * mt], part[mt][c][1], acc[mt][c][1]);
            acc[mt][c][2] = fmaf(scale[2 * mt + 1], part[mt][c][2], acc[mt][c][2]);
            acc[mt][c][3] = fmaf(scale[2 * mt + 1], part[mt][c][3], acc[mt][c][3]);
          }
      }
    }
    __syncwarp();                  // every lane has read the slot
    load_stage(j + STAGES);
  }
  tc::cp_async_wait_all();
  __syncthreads();

  // ---- partial tiles [warp][column][row] over the rings, summed in a fixed order
  float* red = reinterpret_cast<float*>(ws);
  float* mine = red + w * 8 * C8 * RPITCH;
#pragma unroll
  for (int mt = 0; mt < 2; ++mt)
#pragma unroll
    for (int c = 0; c < C8; ++c) {
      float* d = mine + (8 * c + 2 * t) * RPITCH + 16 * mt + g;
      d[0] = acc[mt][c][0];
      d[RPITCH] = acc[mt][c][1];
      d[8] = acc[mt][c][2];
      d[RPITCH + 8] = acc[mt][c][3];
    }
  __syncthreads();
  const int nrows = WARPS / a.wk * ROWS;
  const int total = toks * nrows;
  const T* bias = static_cast<const T*>(a.bias);
  auto local = [&](const float* r, int tok, int row) {
    float v = 0.f;
    for (int i = 0; i < a.wk; ++i) {
      const float* p = r + ((row / ROWS) * a.wk + i) * 8 * C8 * RPITCH + tok * PER_TOK * RPITCH + row % ROWS;
#pragma unroll
      for (int e = 0; e < PER_TOK; ++e) v += p[e * RPITCH];
    }
    return v;
  };
  auto write = [&](int tok, int row, float v) {
    const long long r = tile0 + row;
    if (r < a.n) {
      v = v * up<T>() + (bias ? to_f32(bias[r]) : 0.f);
      const long long at = (m0 + tok) * a.n + r;
      if (a.out_f32) static_cast<float*>(a.y)[at] = v;
      else static_cast<T*>(a.y)[at] = from_f32<T>(v);
    }
  };
  if (a.ck == 1) {
    for (int e = tid; e < total; e += NT) write(e / nrows, e % nrows, local(red, e / nrows, e % nrows));
  } else {
    cg::cluster_group cl = cg::this_cluster();
    float* sum = reinterpret_cast<float*>(xs);      // the CTA's own tile [token][row]
    for (int e = tid; e < total; e += NT) sum[e] = local(red, e / nrows, e % nrows);
    cl.sync();
    for (int e = rank * NT + tid; e < total; e += a.ck * NT) {
      float v = 0.f;
      for (int i = 0; i < a.ck; ++i) v += cl.map_shared_rank(sum, i)[e];
      write(e / nrows, e % nrows, v);
    }
    cl.sync();
  }
}

constexpr int SMS = 148;
constexpr int SMEM_MAX = 112 * 1024;   // two CTAs an SM

template <typename T, int C8, int GPC>
int launch(Int4Args a, cudaStream_t st) {
  constexpr int PER_TOK = Op<T>::cols;
  constexpr int TOK = 8 * C8 / PER_TOK;
  auto kern = int4_linear_mma<T, C8, GPC>;
  const int chunks = (a.k + KC - 1) / KC;
  const int tiles = (a.n + ROWS - 1) / ROWS;
  const long long ytiles = (a.m + TOK - 1) / TOK;
  // split k over warps, then over CTAs, while the device has room for more warps (16 an SM)
  // and every warp keeps a chunk; a streamed buffer holds wk chunks of every column
  int wk = 1, ck = 1;
  while (wk * 2 * C8 <= 8 && wk * 2 <= chunks && (long long)tiles * ytiles * wk * 2 <= SMS * 16) wk *= 2;
  while (ck < 8 && wk * ck * 4 <= chunks && (long long)tiles * ytiles * wk * ck * 2 <= SMS * 16) ck *= 2;
  a.wk = wk;
  a.ck = ck;
  a.per = (chunks + ck - 1) / ck;
  a.per = (a.per + wk - 1) / wk * wk;
  const int nrows = WARPS / wk * ROWS;
  const long long whole = 8LL * C8 * (a.per * KC * 2 + 64);
  a.resident = whole <= 32768;
  const int streamed = 2 * 8 * C8 * ((8 / C8) * KC * 2 + 64);
  a.x_bytes = a.resident ? (int)whole : streamed;
  if (ck > 1 && a.x_bytes < TOK * nrows * 4) a.x_bytes = TOK * nrows * 4;
  a.x_bytes = (int)align_up(a.x_bytes, 128);
  const int smem = a.x_bytes + WARPS * STAGES * STAGE_BYTES;
  static_assert(WARPS * 8 * C8 * RPITCH * 4 <= WARPS * STAGES * STAGE_BYTES, "partial tiles fit the rings");
  static_assert(32768 + 8192 + WARPS * STAGES * STAGE_BYTES <= SMEM_MAX, "x and the rings fit");
  static std::atomic<uint64_t> ready{0};      // devices whose limit is raised
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MAX));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((tiles * wk + WARPS - 1) / WARPS * ck), (unsigned)ytiles);
  cfg.blockDim = dim3(NT);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ck;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = ck > 1 ? 1 : 0;
  VERACE_CUDA(cudaLaunchKernelEx(&cfg, kern, a));
  return check_launch("int4_linear");
}

template <typename T, int GPC>
int by_columns(const Int4Args& a, cudaStream_t st) {
  const long long cols = a.m * Op<T>::cols;
  if (cols <= 8 / Op<T>::cols * Op<T>::cols) return launch<T, 1, GPC>(a, st);
  if (cols <= 16 / Op<T>::cols * Op<T>::cols) return launch<T, 2, GPC>(a, st);
  return launch<T, 4, GPC>(a, st);
}

template <typename T>
int by_group(const Int4Args& a, int group, cudaStream_t st) {
  if (group == 128) return by_columns<T, 1>(a, st);
  if (group == 64) return by_columns<T, 2>(a, st);
  return by_columns<T, 4>(a, st);
}

}  // namespace
}  // namespace verace

using namespace verace;

extern "C" int verace_int4_linear(const void* x, long long ldx, const void* qweight, const void* scales,
                                  const void* zeros, const void* bias, void* y, long long m, int n, int k,
                                  int group, int dtype, int out_dtype, void* stream) {
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
  VERACE_REQUIRE(m <= 65535LL * 8, VERACE_ERR_UNSUPPORTED, "int4_linear: m %lld too large", m);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Int4Args a{};
  a.x = x; a.ldx = ldx; a.q = static_cast<const uint8_t*>(qweight); a.s = scales;
  a.z = static_cast<const uint8_t*>(zeros); a.bias = bias; a.y = y; a.m = m; a.n = n; a.k = k;
  a.out_f32 = out_dtype == VERACE_F32;
  if (dtype == VERACE_F32) return by_group<float>(a, group, st);
  if (dtype == VERACE_BF16) return by_group<__nv_bfloat16>(a, group, st);
  return by_group<__half>(a, group, st);
}
