// Dense products of the feed-forward sub-layer with their epilogues, forward and backward:
//     linear:  out = act(x W^T + bias) + residual
//     gated:   out = act(x Wg^T) up(x Wu^T)
// fp32, bf16 or fp16, and e4m3 operands with a scale for each row.  Sums are fp32, outputs are
// rounded once.  Formulas of the activations: linear.cuh; the products: linear_large.cu.
//
// Backward: p = d act'(pre) (gated: dg and du) in one pass over the saved sums, which are kept in
// fp32 (rounded to bf16 they add as much error to the gradients as all the rest: 4096 x 4096 x 8192
// gated, 3.0e-3 of the gradients' norm against 2.3e-3; 4 bytes a sum instead of 2; p itself is rounded to the operands' 16
// bits, which the tensor core takes: in fp32 the gradients would be 1.7e-3 off, for twice the products), then
// dx = p W (dg Wg + du Wu) and dW = p^T x.  W, p and x are read there as they are stored; no
// operand is transposed in memory.  The bias gradient is summed in the pass, in fp32 and in a
// fixed order (32 rows at a time, then the partial sums).
//
// fp32 operands are split into three bf16 parts first (x = h + 2^-8 m + 2^-16 l, 24 bits; the powers of two keep the
// lower parts of small values inside of bf16's range), and the product takes the six pairs of parts down to 2^-24 of the
// largest (hh, hm, mh, hl, mm, lh).  Exact for every finite value: one that rounds to more than bf16's largest has that
// as its part, and the rest in the next ones.  An infinity's second part is NaN, and so is every output that it enters.
#include "linear_tc.cuh"

#include <algorithm>

namespace verace {
namespace {

using namespace lin;

// ------------------------------------------------------------------ operands in memory
template <typename T>
constexpr bool split_v = sizeof(T) == 4;      // fp32: three bf16 parts
template <typename T>
using Part = std::conditional_t<split_v<T>, __nv_bfloat16, T>;

// 8 values of a row from column c on (0 beyond the row's end)
template <typename T>
__device__ __forceinline__ void load8(const T* row, long long c, long long cols, bool vec, float (&v)[8]) {
  if (vec) {        // (cols is a multiple of 8)
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(row + c)[0], b = reinterpret_cast<const float4*>(row + c)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      unpack8<T>(*reinterpret_cast<const uint4*>(row + c), v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? to_f32(row[c + j]) : 0.f;
  }
}
constexpr float BF16_MOST = 0x1.fep127f;
// 8 values as an operand of the products: rounded to T, or split into three parts `piece` apart
template <typename T>
__device__ __forceinline__ void store_operand(Part<T>* o, long long piece, const float (&v)[8]) {
  if constexpr (split_v<T>) {
    float r[8], h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = v[j];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      // (an infinity stays one)
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = fabsf(r[j]) > BF16_MOST && fabsf(r[j]) < INFINITY ? copysignf(BF16_MOST, r[j]) : r[j];
      const uint4 w = pack8<__nv_bfloat16>(h);
      *reinterpret_cast<uint4*>(o + i * piece) = w;
      unpack8<__nv_bfloat16>(w, h);
#pragma unroll
      for (int j = 0; j < 8; ++j) r[j] = (r[j] - h[j]) * 256.f;
    }
  } else {
    *reinterpret_cast<uint4*>(o) = pack8<T>(v);
  }
}

// Matrices that the products cannot read as they lie, up to three in one launch (one after the other they took 2 to 3 us
// more each), 8 values or 16 bytes a thread.
struct Copy {
  const char* src;
  char* dst;
  long long ld_src, ld, rows, width;   // in values of fp32 parts, else in bytes
  unsigned blocks;
  bool vec;                            // (fp32) whole aligned words
};
struct Copies {
  Copy m[3];
};
// fp32 rows -> three bf16 parts [3][rows][ld], ld = width rounded up to 8
__device__ __forceinline__ void split_row(const Copy& a, long long row, long long c) {
  float v[8];
  load8<float>(reinterpret_cast<const float*>(a.src) + row * a.ld_src, c, a.width, a.vec, v);
  store_operand<float>(reinterpret_cast<__nv_bfloat16*>(a.dst) + row * a.ld + c, a.rows * a.ld, v);
}
// rows that start anywhere -> rows ld apart (a multiple of 16), zeros behind them; read as the aligned words around them
__device__ __forceinline__ void align_row(const Copy& a, long long row, long long c) {
  const char* s = a.src + row * a.ld_src + c;
  const int off = (int)((size_t)s & 3), left = (int)min(16LL, a.width - c);    // (left > 0: ld is width rounded up)
  const uint32_t* w = reinterpret_cast<const uint32_t*>(s - off);
  uint32_t x[5];
#pragma unroll
  for (int j = 0; j < 5; ++j) x[j] = 4 * j < off + left ? w[j] : 0u;
  uint32_t o[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    o[j] = __funnelshift_r(x[j], x[j + 1], 8 * off);
    const int valid = left - 4 * j;
    if (valid < 4) o[j] = valid <= 0 ? 0u : o[j] & ((1u << (8 * valid)) - 1u);
  }
  *reinterpret_cast<uint4*>(a.dst + row * a.ld + c) = make_uint4(o[0], o[1], o[2], o[3]);
}
template <bool SPLIT>
__global__ void __launch_bounds__(256) copy_rows(const __grid_constant__ Copies all) {
  constexpr int U = SPLIT ? 8 : 16;
  depend();
  unsigned block = blockIdx.x;
  int z = 0;
  while (z < 2 && block >= all.m[z].blocks) block -= all.m[z++].blocks;
  const Copy& a = all.m[z];
  const unsigned per_row = (unsigned)(a.ld / U);
  // (a division of 64 bits once in a matrix of 2^36 bytes alone)
  const unsigned long long first = (unsigned long long)block * 256;
  const unsigned long long row0 = first >> 32 ? first / per_row : (unsigned)first / per_row;
  const unsigned at = (unsigned)(first - row0 * per_row) + threadIdx.x;
  const long long row = (long long)row0 + at / per_row;
  if (row >= a.rows) return;
  if constexpr (SPLIT) split_row(a, row, (long long)(at % per_row) * U);
  else align_row(a, row, (long long)(at % per_row) * U);
}

long long padded(long long cols, int type = VERACE_BF16) {
  return type == VERACE_E4M3 ? (cols + 15) / 16 * 16 : (cols + 7) / 8 * 8;
}
// bytes of an operand that a pass writes
size_t operand_bytes(long long rows, long long cols, int type) {
  return align_up((size_t)rows * padded(cols, type) * (type == VERACE_F32 ? 6 : size_of(type)), 256);
}
// bytes of an operand made of a user's matrix: its parts, or its rows at 16-byte borders where their width is no
// multiple of 16 bytes
size_t copy_bytes(long long rows, long long cols, int type) {
  return type == VERACE_F32 || cols * size_of(type) % 16 ? operand_bytes(rows, cols, type) : 0;
}
Mat operand_at(void* p, long long rows, long long cols, int type) {
  const long long ld = padded(cols);
  return Mat{p, rows, cols, ld, type == VERACE_F32 ? 3 : 1, rows * ld};
}

// The workspace, taken from its start.
struct Taker {
  char* at;
  explicit Taker(void* ws) : at((char*)align_up((size_t)ws, 256)) {}
  void* take(size_t bytes) {
    void* p = at;
    at += align_up(bytes, 256);
    return p;
  }
};

bool aligned_rows(const void* p, long long ld, int type) { return (size_t)p % 16 == 0 && ld * size_of(type) % 16 == 0; }

// Operands of the products from a user's matrices: as they are, split into parts or copied in the workspace.
struct Operands {
  int type;
  Taker& ws;
  Copies all = {};
  int n = 0;
  long long blocks = 0;
  void add(Mat* out, const void* p, long long ld, long long rows, long long cols) {
    const bool split = type == VERACE_F32;
    if (!split && aligned_rows(p, ld, type)) {
      *out = Mat{p, rows, cols, ld, 1, 0};
      return;
    }
    const long long es = split ? 1 : size_of(type);
    void* dst = ws.take(operand_bytes(rows, cols, type));
    *out = split ? operand_at(dst, rows, cols, type) : Mat{dst, rows, cols, padded(cols, type), 1, 0};
    const long long mine = (rows * (out->ld * es / (split ? 8 : 16)) + 255) / 256;
    blocks += mine;
    all.m[n++] = Copy{(const char*)p, (char*)dst, ld * es, out->ld * es, rows, cols * es, (unsigned)mine,
                      cols % 8 == 0 && ld % 4 == 0 && (size_t)p % 16 == 0};
  }
  int make(cudaStream_t st) {
    if (n == 0) return VERACE_OK;
    VERACE_REQUIRE(blocks < 1LL << 31, VERACE_ERR_UNSUPPORTED, "linear: operands of %lld bytes are too large", blocks * 4096);
    return launch_after("copy_rows", type == VERACE_F32 ? copy_rows<true> : copy_rows<false>, dim3((unsigned)blocks), 256, 0, st,
                        1, all);
  }
};

// ------------------------------------------------------------------ sums over nothing (k = 0)
__global__ void __launch_bounds__(256) empty_sum(Epilogue e, long long m, long long n) {
  depend();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= m * n) return;
  const long long r = i / n, c = i % n;
  float v = e.bias ? load_as(e.bias, c, e.bias_type) : 0.f;
  if (e.pre) e.pre[r * e.ld + c] = v;
  if (e.pre_up) e.pre_up[r * e.ld + c] = 0.f;
  by_act(e.act, [&](auto act) { v = act_<decltype(act)::value, false>(v); });
  if (e.residual) v += load_as(e.residual, r * e.ld_res + c, e.type);
  store_as(e.out, r * e.ld + c, v, e.type);
}

// Whether a forward product goes to the engine of dot products.  In fp32 that saves splitting the weights
// (8 x 4096 x 4096: 23 us against 71, 24 tokens 63 against 72; gated 16 tokens 111 against 135, 24 tokens 162 against
// 135).  In 16 and 8 bits the tensor cores win where the weights' bytes count, the dot products where the launch does
// (us, dot products against the others, in chains of calls; bf16: 1 x 1024 x 1024 2.5 and 4.4, 1 x 4096 x 4096 8.4 and
// 9.6, 1 x 8192 x 4096 13.8 and 14.7; gated 1 x 1024 x 4096 5.7 and 6.3, 1 x 2048 x 4096 8.8 and 8.2; 4 x 1024 x 4096 4.9
// and 5.6, 4 x 2048 x 4096 8.6 and 6.8; e4m3: 1 x 2048 x 4096 5.9 and 6.1, 1 x 4096 x 4096 8.7 and 7.4).
bool by_dots(long long m, long long n, long long k, int type, int weights) {
  if (k == 0 || n > 65535LL * 8) return false;
  if (type == VERACE_F32) return m <= (weights == 1 ? 24 : 16);
  const long long most = m > 4 ? 0 : m > 1 ? 5 : weights == 1 && type != VERACE_E4M3 ? 32 : 10;   // millions of weights
  return n * k * weights <= most << 20;
}

// Whether a product of operands in memory goes to the engine that streams the weights past its rows (us, against tiles
// of 256 rows, in chains of calls; bf16: 32 x 4096 x 8192 15.6 and 19.0, 128 x 8192 x 4096 17.2 and 23.9, 160 x 4096 x 32000
// 52.7 and 59.8, 160 x 1024 x 4096 8.4 and 8.2, but 200 x 4096 x 32000 63.1 and 60.4; gated 128 x 4096 x 8192 30.9 and 33.8,
// 160 x 4096 x 32000 106 and 114, of small weights 112 x 1024 x 4096 10.5 and 10.5, 128 x 4096 x 1024 13.4 and 12.4; e4m3:
// 160 x 4096 x 8192 13.8 and 14.7, gated 19.7 and 23.1).
bool by_few(long long M, long long N, long long K, int segments, bool gated, int type, bool a_mn) {
  return !a_mn && type != VERACE_F32 && M <= (gated && N * K <= 4 << 20 ? 112 : FEW) &&
         K * segments <= run_of(type) * few_splits(N, K, segments, type);
}

// Workspace of a product's partial sums.
size_t partial_bytes(long long M, long long N, long long K, int sums, int nz, bool gated, int type, bool a_mn) {
  const bool parts = type == VERACE_F32;
  return by_few(M, N, K, sums, gated, type, a_mn) ? 0 : split_bytes(M, N, K, sums, nz, gated, parts ? VERACE_BF16 : type, parts);
}

int run_product(Product& p, cudaStream_t st) {
  if (p.M == 0 || p.N == 0) return VERACE_OK;
  if (p.K == 0) {
    for (int z = 0; z < (p.nz > 1 ? p.nz : 1); ++z) {
      Epilogue e = p.e;
      if (p.nz > 1) e.out = p.out_z[z];
      const long long blocks = (p.M * p.N + 255) / 256;
      VERACE_REQUIRE(blocks < 1LL << 31, VERACE_ERR_UNSUPPORTED, "linear: %lld x %lld outputs are too many", p.M, p.N);
      if (int rc = launch_after("empty_sum", empty_sum, dim3((unsigned)blocks), 256, 0, st, 1, e, p.M, p.N)) return rc;
    }
    return VERACE_OK;
  }
  const bool few = by_few(p.M, p.N, p.K, p.segments, p.gated, p.type, p.a_mn);
  p.parts = p.type == VERACE_F32;
  if (p.parts) p.type = VERACE_BF16;
  return few ? product_few(p, st) : product_large(p, st);
}

// ------------------------------------------------------------------ backward of the epilogues
// p = d act'(pre) as an operand of the products (rounded to the type of x, or in three parts), and its
// column sums: a CTA takes 32 rows (gated: 16) of 256 columns, a thread every eighth row of 8 columns.
// Bound: bytes (d and pre read, p written): gated 4096 x 8192 bf16 90 us for 470 MB, 5.2 TB/s.
constexpr int CHUNK = 32, GATED_CHUNK = 16;
struct SlopeArgs {
  const void* d;
  const float *pre, *up;
  void *out;            // p, or dg; null: the sums alone
  long long piece, second;   // between the parts, and from dg to du
  float* partial;       // [chunks][n], or null
  long long m, n, ld;   // ld: of out
  int act, vec, colblocks;
  float b1, b2, r1, r2;
};

template <typename T, typename O>
__global__ void __launch_bounds__(256) linear_slope(SlopeArgs a) {
  depend();
  __shared__ float part[8][256];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long chunk = blockIdx.x / a.colblocks, c = (blockIdx.x % a.colblocks) * 256LL + lane * 8;
  const long long end = min(a.m, (chunk + 1) * CHUNK);
  float sum[8] = {};
  if (c < a.ld)
    for (long long r = chunk * CHUNK + w; r < end; r += 8) {
      float d[8], z[8];
      load8<O>(static_cast<const O*>(a.d) + r * a.n, c, a.n, a.vec, d);
      if (a.pre) {
        load8<float>(a.pre + r * a.n, c, a.n, a.vec, z);
        by_act(a.act, [&](auto k) {
#pragma unroll
          for (int j = 0; j < 8; ++j) d[j] = back_<decltype(k)::value, sizeof(O) == 2>(d[j], z[j]);
        });
      }
      if (a.out) store_operand<T>(static_cast<Part<T>*>(a.out) + r * a.ld + c, a.piece, d);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[j] += d[j];
    }
  if (!a.partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) part[w][lane * 8 + j] = sum[j];
  __syncthreads();
  const long long n = (blockIdx.x % a.colblocks) * 256LL + threadIdx.x;
  if (n >= a.n) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
  a.partial[chunk * a.n + n] = s;
}

// the sums of the chunks, always in the same order: 32 columns a CTA, eight runs of chunks each.  (`partial` is still being
// written while this kernel is resident: no restricted pointer.)
template <typename T>
__global__ void __launch_bounds__(256) sum_chunks(const float* partial, long long chunks, long long n, T* out) {
  depend();
  __shared__ float part[8][32];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < n)
#pragma unroll 8
    for (long long i = w; i < chunks; i += 8) s += partial[i * n + c];
  part[w][lane] = s;
  __syncthreads();
  if (w > 0 || c >= n) return;
#pragma unroll
  for (int i = 1; i < 8; ++i) s += part[i][lane];
  out[c] = from_f32<T>(s);
}

template <typename T, typename O>
__global__ void __launch_bounds__(256) gated_slope(SlopeArgs a) {
  depend();
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const long long chunk = blockIdx.x / a.colblocks, c = (blockIdx.x % a.colblocks) * 256LL + lane * 8;
  const long long end = min(a.m, (chunk + 1) * GATED_CHUNK);
  if (c >= a.ld) return;
  for (long long r = chunk * GATED_CHUNK + w; r < end; r += 8) {
    float d[8], g[8], u[8];
    load8<O>(static_cast<const O*>(a.d) + r * a.n, c, a.n, a.vec, d);
    load8<float>(a.pre + r * a.n, c, a.n, a.vec, g);
    load8<float>(a.up + r * a.n, c, a.n, a.vec, u);
    by_act(a.act, [&](auto k) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float x, y;
        gate_slope_<decltype(k)::value, sizeof(O) == 2>(d[j], g[j], u[j], a.b1, a.b2, a.r1, a.r2, x, y);
        g[j] = x;
        u[j] = y;
      }
    });
    Part<T>* o = static_cast<Part<T>*>(a.out) + r * a.ld + c;
    store_operand<T>(o, a.piece, g);
    store_operand<T>(o + a.second, a.piece, u);
  }
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
  VERACE_REQUIRE(dtype == VERACE_F32 || cols * size_of(dtype) % 16 || aligned_rows(p, ld, dtype), VERACE_ERR_INVALID,
                 "%s: the rows of %s must be 16-byte aligned", who, name);
  return VERACE_OK;
}

int check_workspace(const char* who, size_t need, const void* ws, size_t given) {
  VERACE_REQUIRE(need == 0 || (ws && given >= need), VERACE_ERR_WORKSPACE, "%s: workspace of %zu bytes required, %zu given",
                 who, need, ws ? given : (size_t)0);
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

long long chunks_of(long long m) { return (m + CHUNK - 1) / CHUNK; }

int slope_grid(const SlopeArgs& a, int rows, unsigned* grid) {
  const long long blocks = (a.m + rows - 1) / rows * a.colblocks;
  VERACE_REQUIRE(blocks < 1LL << 31, VERACE_ERR_UNSUPPORTED, "linear: %lld x %lld outputs are too many", a.m, a.n);
  *grid = (unsigned)blocks;
  return VERACE_OK;
}

}  // namespace
}  // namespace verace

using namespace verace;
using namespace verace::lin;

extern "C" size_t verace_linear_workspace(long long m, int n, int k, int dtype) {
  if (m <= 0 || n <= 0 || k <= 0) return 0;
  const bool dots = by_dots(m, n, k, dtype, 1);
  if (dots && dtype == VERACE_F32) return 0;
  const size_t copies = copy_bytes(m, k, dtype) + copy_bytes(n, k, dtype);
  const size_t part = dots ? 0 : partial_bytes(m, n, k, 1, 1, false, dtype, false);
  return copies + part ? copies + part + 256 : 0;
}

extern "C" int verace_linear(const void* x, long long ldx, const float* x_scale, const void* w, long long ldw,
                             const float* w_scale, const void* bias, const void* residual, long long ld_res, void* out,
                             float* pre, long long m, int n, int k, int act, int dtype, int out_dtype, void* workspace,
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
  if ((rc = check_workspace(who, verace_linear_workspace(m, n, k, dtype), workspace, workspace_bytes))) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  Taker ws(workspace);
  Product p{};
  p.type = dtype; p.M = m; p.N = n; p.K = k; p.nz = 1;
  p.e = plain_out(out, n, out_dtype);
  p.e.row_scale = x_scale; p.e.col_scale = w_scale; p.e.bias = bias; p.e.residual = residual; p.e.ld_res = ld_res;
  p.e.pre = pre; p.e.act = act;
  p.e.bias_type = dtype == VERACE_E4M3 ? out_dtype : dtype;
  const bool dots = by_dots(m, n, k, dtype, 1);
  if (dots && dtype == VERACE_F32) {
    p.a = Mat{x, m, k, ldx, 1, 0};
    p.b[0] = Mat{w, n, k, ldw, 1, 0};
  } else if (k > 0) {
    Operands o{dtype, ws};
    o.add(&p.a, x, ldx, m, k);
    o.add(&p.b[0], w, ldw, n, k);
    if ((rc = o.make(st))) return rc;
  }
  if (dots) return product_dot(p, st);
  p.segments = p.a_step = 1;
  p.ws = ws.at;
  return run_product(p, st);
}

extern "C" size_t verace_linear_backward_workspace(long long m, int n, int k, int dtype) {
  if (m <= 0 || n <= 0) return 0;
  size_t s = operand_bytes(m, n, dtype) + align_up((size_t)chunks_of(m) * n * 4, 256) + 256;
  // (dx and dw follow each other: one place for the partial sums of either)
  s += std::max(partial_bytes(m, k, n, 1, 1, false, dtype, false), partial_bytes(n, k, m, 1, 1, false, dtype, true));
  if (k > 0) s += copy_bytes(m, k, dtype) + copy_bytes(n, k, dtype);
  return s;
}

extern "C" int verace_linear_backward(const void* dout, const void* x, long long ldx, const void* w, long long ldw,
                                      const float* pre, void* dx, void* dw, void* dbias, long long m, int n, int k, int act,
                                      int dtype, int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  constexpr const char* who = "verace_linear_backward";
  int rc;
  if ((rc = check_sizes(who, m, n, k)) || (rc = check_types(who, dtype, out_dtype, false))) return rc;
  VERACE_REQUIRE(act >= VERACE_ACT_NONE && act <= VERACE_ACT_GELU_TANH, VERACE_ERR_INVALID, "%s: activation %d", who, act);
  const bool any = m > 0 && n > 0;
  VERACE_REQUIRE(!any || (dout && (pre || act == VERACE_ACT_NONE)), VERACE_ERR_INVALID, "%s: NULL pointer", who);
  if (any && k > 0 &&
      ((dw && (rc = check_rows(who, "x", x, ldx, k, dtype))) || (dx && (rc = check_rows(who, "w", w, ldw, k, dtype)))))
    return rc;
  if ((rc = check_workspace(who, verace_linear_backward_workspace(m, n, k, dtype), workspace, workspace_bytes))) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  return by_types(dtype, out_dtype, [&](auto t, auto o) -> int {
    using T = decltype(t);
    using O = decltype(o);
    int rc;
    Taker ws(workspace);
    Mat p{nullptr, m, n, padded(n), 1, 0};
    SlopeArgs s{};
    s.d = dout; s.pre = act == VERACE_ACT_NONE ? nullptr : pre; s.act = act;
    s.m = m; s.n = n; s.ld = padded(n);
    s.vec = n % 8 == 0 && ((size_t)dout | (size_t)s.pre) % 16 == 0;
    s.colblocks = (int)((s.ld + 255) / 256);
    if (any) {
      if (!split_v<T> && std::is_same<T, O>::value && !s.pre && s.vec) {
        p = Mat{dout, m, n, n, 1, 0};                   // d is p, and an operand as it is
      } else if ((dx || dw) && k > 0) {
        s.out = ws.take(operand_bytes(m, n, dtype));
        p = operand_at(s.out, m, n, dtype);
        s.piece = p.piece;
      }
      if (dbias) s.partial = (float*)ws.take((size_t)chunks_of(m) * n * 4);
      if (s.out || s.partial) {
        unsigned grid;
        if ((rc = slope_grid(s, CHUNK, &grid))) return rc;
        if ((rc = launch_after("linear_slope", linear_slope<T, O>, dim3(grid), 256, 0, st, 1, s))) return rc;
      }
    }
    if (dbias && n > 0) {
      if ((rc = launch_after("sum_chunks", sum_chunks<T>, dim3((n + 31) / 32), 256, 0, st, 1, (const float*)s.partial,
                             any ? chunks_of(m) : 0LL, (long long)n, (T*)dbias)))
        return rc;
    }
    Mat xm{}, wm{};
    if (any && k > 0) {
      Operands made{dtype, ws};
      if (dx) made.add(&wm, w, ldw, n, k);
      if (dw) made.add(&xm, x, ldx, m, k);
      if ((rc = made.make(st))) return rc;
    }
    if (dx && k > 0) {
      Product d{};
      d.type = dtype; d.M = m; d.N = k; d.K = n; d.nz = 1; d.b_mn = true;
      d.e = plain_out(dx, k, dtype);
      d.a = p;
      d.b[0] = wm;
      d.segments = d.a_step = 1;
      d.ws = ws.at;
      if ((rc = run_product(d, st))) return rc;
    }
    if (dw && k > 0) {
      Product d{};
      d.type = dtype; d.M = n; d.N = k; d.K = m; d.nz = 1; d.a_mn = d.b_mn = true;
      d.e = plain_out(dw, k, dtype);
      d.a = p;
      d.b[0] = xm;
      d.segments = d.a_step = 1;
      d.ws = ws.at;
      if ((rc = run_product(d, st))) return rc;
    }
    return VERACE_OK;
  });
}

extern "C" size_t verace_gated_linear_workspace(long long m, int f, int k, int dtype) {
  if (m <= 0 || f <= 0 || k <= 0) return 0;
  const bool dots = by_dots(m, f, k, dtype, 2);
  if (dots && dtype == VERACE_F32) return 0;
  const size_t copies = copy_bytes(m, k, dtype) + 2 * copy_bytes(f, k, dtype);
  const size_t part = dots ? 0 : partial_bytes(m, f, k, 1, 1, true, dtype, false);
  return copies + part ? copies + part + 256 : 0;
}

extern "C" int verace_gated_linear(const void* x, long long ldx, const float* x_scale, const void* w_gate, const void* w_up,
                                   long long ldw, const float* gate_scale, const float* up_scale, void* out, float* gate,
                                   float* up, long long m, int f, int k, int act, float beta1, float beta2, int dtype,
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
  if ((rc = check_workspace(who, verace_gated_linear_workspace(m, f, k, dtype), workspace, workspace_bytes))) return rc;
  cudaStream_t st = (cudaStream_t)stream;
  Taker ws(workspace);
  Product p{};
  p.type = dtype; p.M = m; p.N = f; p.K = k; p.nz = 1; p.gated = true;
  p.e = plain_out(out, f, out_dtype);
  p.e.row_scale = x_scale; p.e.col_scale = gate_scale; p.e.up_scale = up_scale;
  p.e.pre = gate; p.e.pre_up = up; p.e.act = act;
  p.e.b1 = beta1; p.e.b2 = beta2; p.e.r1 = 1.f / beta1; p.e.r2 = 1.f / beta2;
  const bool dots = by_dots(m, f, k, dtype, 2);
  if (dots && dtype == VERACE_F32) {
    p.a = Mat{x, m, k, ldx, 1, 0};
    p.b[0] = Mat{w_gate, f, k, ldw, 1, 0};
    p.b[1] = Mat{w_up, f, k, ldw, 1, 0};
  } else if (k > 0) {
    Operands o{dtype, ws};
    o.add(&p.a, x, ldx, m, k);
    o.add(&p.b[0], w_gate, ldw, f, k);
    o.add(&p.b[1], w_up, ldw, f, k);
    if ((rc = o.make(st))) return rc;
  }
  if (dots) return product_dot(p, st);
  p.segments = p.a_step = 1;
  p.ws = ws.at;
  return run_product(p, st);
}

extern "C" size_t verace_gated_linear_backward_workspace(long long m, int f, int k, int dtype) {
  if (m <= 0 || f <= 0) return 0;
  size_t s = 2 * operand_bytes(m, f, dtype) + 256;
  // (dx and the weights' gradients follow each other: one place for the partial sums of either)
  s += std::max(partial_bytes(m, k, f, 2, 1, false, dtype, false),
                std::max(partial_bytes(f, k, m, 1, 1, false, dtype, true), partial_bytes(f, k, m, 1, 2, false, dtype, true)));
  if (k > 0) s += copy_bytes(m, k, dtype) + 2 * copy_bytes(f, k, dtype);
  return s;
}

extern "C" int verace_gated_linear_backward(const void* dout, const void* x, long long ldx, const void* w_gate,
                                            const void* w_up, long long ldw, const float* gate, const float* up, void* dx,
                                            void* dw_gate, void* dw_up, long long m, int f, int k, int act, float beta1,
                                            float beta2, int dtype, int out_dtype, void* workspace, size_t workspace_bytes,
                                            void* stream) {
  constexpr const char* who = "verace_gated_linear_backward";
  int rc;
  if ((rc = check_sizes(who, m, f, k)) || (rc = check_types(who, dtype, out_dtype, false))) return rc;
  VERACE_REQUIRE(act >= VERACE_ACT_RELU && act <= VERACE_ACT_SITU, VERACE_ERR_INVALID, "%s: activation %d", who, act);
  VERACE_REQUIRE(act != VERACE_ACT_SITU || (beta1 != 0.f && beta2 != 0.f), VERACE_ERR_INVALID, "%s: beta of 0", who);
  const bool any = m > 0 && f > 0;
  VERACE_REQUIRE(!any || (dout && gate && up), VERACE_ERR_INVALID, "%s: NULL pointer", who);
  if (any && k > 0 &&
      (((dw_gate || dw_up) && (rc = check_rows(who, "x", x, ldx, k, dtype))) ||
       (dx && ((rc = check_rows(who, "w_gate", w_gate, ldw, k, dtype)) || (rc = check_rows(who, "w_up", w_up, ldw, k, dtype))))))
    return rc;
  if ((rc = check_workspace(who, verace_gated_linear_backward_workspace(m, f, k, dtype), workspace, workspace_bytes))) return rc;
  if (k == 0) return VERACE_OK;   // (the gradients are empty)
  cudaStream_t st = (cudaStream_t)stream;
  return by_types(dtype, out_dtype, [&](auto t, auto o) -> int {
    using T = decltype(t);
    using O = decltype(o);
    int rc;
    Taker ws(workspace);
    // [part][gate, up][m][f]
    Mat p{nullptr, m, f, padded(f), 1, 0};
    if (any) {
      const long long one = m * padded(f), parts = split_v<T> ? 3 : 1;
      void* out = ws.take(2 * operand_bytes(m, f, dtype));
      p = Mat{out, m, f, padded(f), (int)(2 * parts), one};
      SlopeArgs s{};
      s.d = dout; s.pre = gate; s.up = up; s.out = out; s.piece = 2 * one; s.second = one;
      s.m = m; s.n = f; s.ld = padded(f); s.act = act;
      s.vec = f % 8 == 0 && ((size_t)dout | (size_t)gate | (size_t)up) % 16 == 0;
      s.colblocks = (int)((s.ld + 255) / 256);
      s.b1 = beta1; s.b2 = beta2; s.r1 = 1.f / beta1; s.r2 = 1.f / beta2;
      unsigned grid;
      if ((rc = slope_grid(s, GATED_CHUNK, &grid))) return rc;
      if ((rc = launch_after("gated_slope", gated_slope<T, O>, dim3(grid), 256, 0, st, 1, s))) return rc;
    }
    Mat xm{}, gm{}, um{};
    if (any) {
      Operands made{dtype, ws};
      if (dx) made.add(&gm, w_gate, ldw, f, k);
      if (dx) made.add(&um, w_up, ldw, f, k);
      if (dw_gate || dw_up) made.add(&xm, x, ldx, m, k);
      if ((rc = made.make(st))) return rc;
    }
    if (dx) {
      Product d{};
      d.type = dtype; d.M = m; d.N = k; d.K = f; d.nz = 1; d.b_mn = true;
      d.e = plain_out(dx, k, dtype);
      d.a = p;
      d.b[0] = gm;
      d.b[1] = um;
      d.segments = d.a_step = 2;
      d.ws = ws.at;
      if ((rc = run_product(d, st))) return rc;
    }
    if (dw_gate || dw_up) {
      Product d{};
      d.type = dtype; d.M = f; d.N = k; d.K = m; d.a_mn = d.b_mn = true;
      d.nz = dw_gate && dw_up ? 2 : 1;
      d.out_z[0] = dw_gate; d.out_z[1] = dw_up;
      d.e = plain_out(dw_gate ? dw_gate : dw_up, k, dtype);
      d.a = p;
      d.b[0] = xm;
      d.segments = 1;
      d.a_step = 2;
      d.a_first = dw_gate ? 0 : 1;
      d.ws = ws.at;
      if ((rc = run_product(d, st))) return rc;
    }
    return VERACE_OK;
  });
}
