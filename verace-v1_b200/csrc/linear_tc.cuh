// The tensor-core products behind linear.cu: what the host hands them.
#pragma once

#include "linear.cuh"
#include "tc.cuh"
#include "tmap.cuh"

namespace verace {
namespace lin {

// A matrix in memory: `pieces` times rows x cols, rows `ld` and pieces `piece` values apart.
struct Mat {
  const void* p;
  long long rows, cols, ld;
  int pieces;
  long long piece;
};

// out[z](m, n) = epilogue(sum over s < segments and k of A_s(m, k) B_s(n, k)).
// A_s is a's matrix a_first + s + z (the parts of an fp32 matrix `a_step` further each); B_s is b[s].
// A and B are stored [M][K] and [N][K], or [K][M] and [K][N] where a_mn, b_mn are set (16-bit types).
// gated: one segment, b[0] and b[1] give the two sums of a row and column (N: columns of each).
struct Product {
  int type;             // VERACE_BF16, VERACE_F16 or VERACE_E4M3
  bool parts;           // the operands are the parts of fp32 matrices
  long long M, N, K;
  Mat a, b[2];
  bool a_mn, b_mn, gated;
  int segments, a_first, a_step;
  int nz;               // outputs: 1 or 2
  void* out_z[2];       // where nz is 2
  Epilogue e;
  void* ws;             // split_bytes(...) bytes, for partial sums where K is split
};
// What product_large may take for partial sums (M x N outputs each, nz of them).
size_t split_bytes(long long M, long long N, long long K, int segments, int nz, bool gated, int type, bool parts);

// Tokens up to which weights may be streamed past them (linear_few.cu).
constexpr int FEW = 160;

// Values of K that a sum of 16- or 8-bit operands may run over in the tensor core, which cuts every product to the last place
// of the running sum (and two bits more) instead of rounding the sum.  Where all terms have one sign that takes 6.4e-9 of the
// sum a term (fp16; bf16 5e-9 to 6.2e-9, e4m3 up to 1.2e-9; 2048 x 2048 outputs, K = 2^12 ... 2^18): 2.1e-4 of it at 2^15 and
// 8e-4 at 2^17, less than half of fp16's and of bf16's half step.  Longer sums are split, and the splits' sums added with
// rounding.  (fp16, us, against sums unsplit: 4096 x 65536 x 4096 1495 to 1584 and 1530 to 1595, 4096 x 65536 x 1024 425 to 474 and
// 394 to 469, 16 x 65536 x 16384 335 to 341 and 347 to 359.)
inline long long run_of(int type) { return type == VERACE_F16 ? 1 << 15 : 1 << 17; }

// CTAs of a cluster that share K in linear_few.cu: while there is an SM for each, or a sum would be too long.
inline int few_splits(long long N, long long K, int segments, int type) {
  const int step = type == VERACE_E4M3 ? 128 : 64;
  const long long tiles = (N + 127) / 128, steps = (K + step - 1) / step * segments;
  int ck = 1;
  while (ck < 8 && ((tiles * ck * 2 <= 148 && steps >= ck * 4) || K * segments > run_of(type) * ck)) ck *= 2;
  return ck;
}

int product_large(const Product& p, cudaStream_t st);   // linear_large.cu
int product_few(const Product& p, cudaStream_t st);     // linear_few.cu: up to FEW rows of A
int product_dot(const Product& p, cudaStream_t st);     // linear_dot.cu: a few rows of A, fp32 operands as they are

// ------------------------------------------------------------------ launches
// Every kernel here is launched as a programmatic dependent of the one before it on the stream: it may be
// resident, and set itself up, while that one ends, waits for it (depend()) before its first access to global
// memory, and only then lets its own dependents in, so that whatever came before is complete for
// them too (chains of small products: 1.5 to 2 us a launch).
template <typename K, typename... A>
int launch_after(const char* what, K kernel, dim3 grid, int threads, size_t smem, cudaStream_t st, int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  VERACE_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
  return check_launch(what);
}
__device__ __forceinline__ void depend() {
  asm volatile("griddepcontrol.wait;\n\tgriddepcontrol.launch_dependents;" ::: "memory");
}

// The tensor map of an operand: boxes of 128 bytes x `rows`.
int operand_map(CUtensorMap* map, const Mat& m, int type, int rows);

// ------------------------------------------------------------------ device parts of both engines
__device__ __forceinline__ bool elect() {   // one lane of a converged warp
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
// two 16-bit values of a runtime type in a word, and back
__device__ __forceinline__ uint32_t pack_pair(float a, float b, int type) {   // (one packed conversion: the single ones share the
  uint32_t w;                                                                    // unit of the exponentials)
  if (type == VERACE_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(b), "f"(a));
  return w;
}
__device__ __forceinline__ float2 unpack_pair(uint32_t w, int type) {
  return type == VERACE_BF16 ? unpack2<__nv_bfloat16>(w) : unpack2<__half>(w);
}

// 16 columns of this thread's TMEM row, without waiting for them
__device__ __forceinline__ void tmem_ld_async(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
// waits for the loads; the registers pass through so that nothing reads them earlier
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}

// U values from column n0 on of a vector of N, the same ones for every lane (0 beyond the end)
template <int U>
__device__ __forceinline__ void column_values(const void* p, int type, long long n0, long long N, float (&v)[U]) {
  const char* at = static_cast<const char*>(p) + n0 * (type == VERACE_F32 ? 4 : 2);
  if (n0 + U <= N && ((size_t)at & 15) == 0) {
    if (type == VERACE_F32) {
#pragma unroll
      for (int j = 0; j < U / 4; ++j) {
        const float4 f = reinterpret_cast<const float4*>(at)[j];
        v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < U / 8; ++j) {
        const uint4 w = reinterpret_cast<const uint4*>(at)[j];
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = unpack_pair(x[i], type);
          v[8 * j + 2 * i] = f.x;
          v[8 * j + 2 * i + 1] = f.y;
        }
      }
    }
  } else if (type == VERACE_F32) {
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = n0 + j < N ? reinterpret_cast<const float*>(at)[j] : 0.f;
  } else {
    uint32_t w[U];
#pragma unroll
    for (int j = 0; j < U; ++j) w[j] = n0 + j < N ? reinterpret_cast<const unsigned short*>(at)[j] : 0u;
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = unpack_pair(w[j], type).x;
  }
}

// four neighbouring values of a row, `n` of them inside of it
__device__ __forceinline__ void load4(const void* p, long long i, int n, int type, float (&v)[4]) {
  const size_t at = (size_t)p + i * (type == VERACE_F32 ? 4 : 2);
  if (n == 4 && type != VERACE_F32 && (at & 7) == 0) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    const float2 a = unpack_pair(w.x, type), b = unpack_pair(w.y, type);
    v[0] = a.x; v[1] = a.y; v[2] = b.x; v[3] = b.y;
  } else if (n == 4 && type == VERACE_F32 && (at & 15) == 0) {
    const float4 f = *reinterpret_cast<const float4*>(at);
    v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = j < n ? load_as(p, i + j, type) : 0.f;
  }
}
__device__ __forceinline__ void store4(void* p, long long i, int n, int type, const float (&v)[4]) {
  const size_t at = (size_t)p + i * (type == VERACE_F32 ? 4 : 2);
  if (n == 4 && type != VERACE_F32 && (at & 7) == 0) {
    *reinterpret_cast<uint2*>(at) = make_uint2(pack_pair(v[0], v[1], type), pack_pair(v[2], v[3], type));
  } else if (n == 4 && type == VERACE_F32 && (at & 15) == 0) {
    *reinterpret_cast<float4*>(at) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) store_as(p, i + j, v[j], type);
  }
}

// four outputs (n of them inside of the row) of row m from their sums (u: the up projection's), the columns' scales, their
// bias (a gated product's: the up projection's scales), the row's scale and the residual, each read where e has it
template <bool GATED>
__device__ __forceinline__ void finish4(const Epilogue& e, long long m, long long c, int n, const float* col_scale,
                                        const float* col_add, float row_scale, const float (&res)[4], float (&g)[4],
                                        float (&u)[4]) {
  if (e.col_scale) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      g[j] = scaled_by(g[j], row_scale, col_scale[j]);
      if (GATED) u[j] = scaled_by(u[j], row_scale, col_add[j]);
    }
  }
  if (!GATED && e.bias) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] += col_add[j];
  }
  if (e.pre) {
    store4(e.pre, m * e.ld + c, n, VERACE_F32, g);
    if (GATED) store4(e.pre_up, m * e.ld + c, n, VERACE_F32, u);
  }
  if (e.type == VERACE_F32) activate<GATED, false>(e, g, u);
  else activate<GATED, true>(e, g, u);
  if (!GATED && e.residual) {
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] += res[j];
  }
  store4(e.out, m * e.ld + c, n, e.type, g);
}

}  // namespace lin
}  // namespace verace
