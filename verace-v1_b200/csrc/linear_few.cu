// Products of few rows (tokens) on the tensor cores, the other engine behind linear.cu:
//     out(m, n) = epilogue(sum_k x(m, k) W(n, k)),  m up to 160
// Bound: the weights' bytes.  W's rows are the MMA's 128 rows and the tokens its 16 to 160 columns, so
// a weight crosses shared memory once and no row of the MMA is idle; a CTA streams its 128 rows (gated:
// 128 of each weight, two sums side by side in TMEM) by TMA in stages of 128 bytes of K.  Two
// CTAs share an SM where shared memory allows, so that one's set-up and epilogue run under the other's
// stream.  Few tiles: K is split over a cluster of up to 8 CTAs, whose partial sums are joined through
// distributed shared memory in rank order.
//
// Warps: 0 feeds the stages, 1 issues the MMAs; then all eight read the sums, two a quarter of TMEM: a thread holds a weight
// row, so neighbouring threads store neighbouring outputs of a token.  The input gradient of few tokens
// (a_mn: weights stored [K][N], read as MN-major) runs here too, for a gated block over both weights.
//
// Measured in chains of calls: 7 x 8192 x 4096 fp16 15.0 us (4.5 TB/s, 5 us of it set-up, first loads and the join),
// 16 x 1024 x 163840 bf16 63 us (5.3 TB/s), gated 64 x 4096 x 2 x 8192 e4m3 17.3 us (3.9 TB/s: the stream ends at 11.4,
// the sums are joined at 13, the gates and outputs take to 15.5, the next call begins 1.9 later).
#include "linear_tc.cuh"

#include <cooperative_groups.h>

#include <atomic>

namespace verace {

__device__ int g_linear_few_status = 0;   // non-zero after a bounded wait gave up

namespace {

namespace cg = cooperative_groups;
using namespace lin;

constexpr int NT = 256, ROWS = 128, MAX_STAGES = 8;
// shared memory for stages, or for the sums of up to FEW tokens, of a CTA that has an SM to itself, and of one that
// shares it (228 KB an SM, less 1 KB a CTA that the system takes, 2 KB of barriers and scales and 1 KB to align the stages)
constexpr int ROOM = 224 * 1024, HALF_ROOM = 110 * 1024;
constexpr uint32_t POLLS = 1u << 22, SUM_POLLS = 1u << 26;   // (a sum runs over up to run_of(type) values)

struct Maps {
  CUtensorMap w[2], x;
};

struct Args {
  long long M, N;       // tokens, outputs
  int mp;               // tokens, rounded up to 16
  int stages, stage;    // and a stage's bytes
  int kblocks, steps, per, ck, tiles_n;
  int cols;             // of TMEM
  int a_first;
  uint32_t idesc;
  Epilogue e;
};

template <bool F8>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (F8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate));
  else
    tc::mma_bf16(d, a, b, idesc, accumulate);   // (kind::f16; the descriptor names the type)
}

// one value of each of 16 rows `ld` apart (of `n` rows; 0 beyond), the loads in flight together
__device__ __forceinline__ void load_rows16(const void* p, long long i, long long ld, int n, int type, float (&v)[16]) {
  if (type == VERACE_F32) {
    const float* f = static_cast<const float*>(p) + i;
#pragma unroll
    for (int j = 0; j < 16; ++j, f += ld) v[j] = j < n ? *f : 0.f;
  } else {
    const unsigned short* f = static_cast<const unsigned short*>(p) + i;
    uint32_t w[16];
#pragma unroll
    for (int j = 0; j < 16; ++j, f += ld) w[j] = j < n ? *f : 0u;
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = unpack_pair(w[j], type).x;
  }
}
__device__ __forceinline__ void store_rows16(void* p, long long i, long long ld, int n, int type, const float (&v)[16]) {
  if (type == VERACE_F32) {
    float* f = static_cast<float*>(p) + i;
#pragma unroll
    for (int j = 0; j < 16; ++j, f += ld)
      if (j < n) *f = v[j];
  } else {
    unsigned short* f = static_cast<unsigned short*>(p) + i;
    uint32_t w[8];
    if (type == VERACE_BF16) {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = pack_pair(v[2 * j], v[2 * j + 1], VERACE_BF16);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = pack_pair(v[2 * j], v[2 * j + 1], VERACE_F16);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j, f += ld)
      if (j < n) *f = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
  }
}

template <bool F8, bool WMN, bool GATED>
__global__ void __launch_bounds__(NT, 2) few_product(const __grid_constant__ Maps maps, const __grid_constant__ Args p) {
  constexpr int KB = F8 ? 128 : 64, WB = GATED ? 2 * ROWS * 128 : ROWS * 128;
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(((size_t)raw + 1023) & ~(size_t)1023);
  __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], done;
  __shared__ uint32_t slot;
  __shared__ volatile int fail;
  __shared__ __align__(16) float row_scale[FEW], col_scale[ROWS], col_add[ROWS];   // (col_add: up_scale, or the bias)
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int tile_n = blockIdx.x / p.ck, rank = blockIdx.x - tile_n * p.ck, n0 = tile_n * ROWS;
  const int first = rank * p.per, last = min(p.steps, first + p.per);
  if (warp == 1) tc::tmem_alloc(&slot, p.cols);
  if (warp == 2 && lane < 3)
    asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 2 ? &maps.x : &maps.w[lane]) : "memory");
  if (tid == 0) {
    for (int i = 0; i < p.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&done, 1);
    fail = 0;
    tc::fence_mbar_init();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::fence_after_sync();
  depend();
  const uint32_t tmem = slot;

  if (warp == 0) {
    if (lane == 0) {   // ---- weights and tokens
      int i = 0, flying = 0, seg = first / p.kblocks, kb = first - seg * p.kblocks;
      uint32_t phase = 0;
      for (int s = first; s < last; ++s) {
        if (!tc::mbar_wait(&empty[i], phase ^ 1, POLLS)) {
          fail = 1;
          atomicExch(&g_linear_few_status, 1);
          break;
        }
        unsigned char* w = sm + i * p.stage;
        tc::mbar_expect_tx(&full[i], p.stage);
        if constexpr (WMN) {
          tc::tma_load_3d(w, &maps.w[seg], n0, kb * KB, 0, &full[i]);
          tc::tma_load_3d(w + 8192, &maps.w[seg], n0 + 64, kb * KB, 0, &full[i]);
        } else {
          tc::tma_load_3d(w, &maps.w[0], kb * KB, n0, 0, &full[i]);
          if (GATED) tc::tma_load_3d(w + ROWS * 128, &maps.w[1], kb * KB, n0, 0, &full[i]);
        }
        tc::tma_load_3d(w + WB, &maps.x, kb * KB, 0, p.a_first + seg, &full[i]);
        if (++kb == p.kblocks) kb = 0, ++seg;
        if (++i == p.stages) i = 0, phase ^= 1;
        flying = min(flying + 1, p.stages);
      }
      while (flying-- > 0) {   // copies in flight land before the CTA may end
        if (i == 0) i = p.stages, phase ^= 1;
        tc::mbar_wait(&full[--i], phase, POLLS);
      }
    }
  } else if (warp == 1) {   // ---- MMAs (the whole warp walks the loop: the operands sit in uniform registers)
    const bool lead = elect();
    int i = 0;
    uint32_t phase = 0;
    for (int s = first; s < last; ++s) {
      if (!tc::mbar_wait(&full[i], phase, POLLS)) {
        fail = 1;
        if (lane == 0) atomicExch(&g_linear_few_status, 1);
        break;
      }
      tc::fence_after_sync();
      const uint32_t w = tc::smem_addr(sm + i * p.stage), x = w + WB;
      if (lead) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint64_t dx = tc::sdesc_sw128(x + k * 32, 16, 1024);
          const uint64_t dw = WMN ? tc::sdesc_sw128(w + k * 2048, 8192, 1024) : tc::sdesc_sw128(w + k * 32, 16, 1024);
          const uint32_t more = s > first || k > 0;
          mma<F8>(tmem, dw, dx, p.idesc, more);
          if (GATED) mma<F8>(tmem + p.mp, tc::sdesc_sw128(w + ROWS * 128 + k * 32, 16, 1024), dx, p.idesc, more);
        }
        tc::commit(&empty[i]);
      }
      __syncwarp();
      if (++i == p.stages) i = 0, phase ^= 1;
    }
    if (lead) tc::commit(&done);
    __syncwarp();
  }
  __syncwarp();
  // ---- the sums.  What the epilogue reads beside them is fetched while the products run (read after them it took 2 us):
  // scales and bias go to shared memory, the residual to L2.
  const int tokens = (int)p.M;
  const bool joins = p.ck > 1;
  const Epilogue& e = p.e;
  if (warp >= 2) {
    for (int i = tid - 64; i < (FEW > ROWS ? FEW : ROWS); i += NT - 64) {
      if (e.row_scale && i < tokens) row_scale[i] = e.row_scale[i];
      if (i < ROWS && n0 + i < p.N) {
        if (e.col_scale) col_scale[i] = e.col_scale[n0 + i];
        if (GATED && e.col_scale) col_add[i] = e.up_scale[n0 + i];
        if (!GATED && e.bias) col_add[i] = load_as(e.bias, n0 + i, e.bias_type);
      }
    }
    if (!GATED && e.residual)
      for (int i = tid - 64; i < 4 * tokens; i += NT - 64) {
        const int c = n0 + 32 * (i & 3);
        const size_t at = (size_t)e.residual + ((i >> 2) * e.ld_res + c) * (e.type == VERACE_F32 ? 4 : 2);
        if (c < p.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
      }
  }
  const int quarter = warp & 3;
  const uint32_t mine = tmem + ((uint32_t)(32 * quarter) << 16);
  if (!joins) __syncthreads();   // (the scales; of a split K the barrier behind the sums)
  const bool ok = tc::mbar_wait(&done, 0, SUM_POLLS) && !fail;
  if (!ok && lane == 0) atomicExch(&g_linear_few_status, 1);
  tc::fence_after_sync();
  if (!joins) {
    if (ok) {
      const int c = 32 * quarter + lane, n = n0 + c;
      const bool in = n < p.N;
      const float cs = col_scale[c], ca = col_add[c];   // (read where they are set alone)
#pragma unroll 1
      for (int t = 16 * (warp >> 2); t < tokens; t += 32) {
        uint32_t r[16], s[16];
        tmem_ld_async(mine + t, r);
        if (GATED) tmem_ld_async(mine + p.mp + t, s);
        const int rows = in ? min(16, tokens - t) : 0;
        float res[16] = {};
        if (!GATED && e.residual) load_rows16(e.residual, (long long)t * e.ld_res + n, e.ld_res, rows, e.type, res);
        tmem_wait(r);
        if (GATED) tmem_wait(s);
        float g[16], u[16] = {};
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float rs = e.row_scale && t + j < tokens ? row_scale[t + j] : 1.f;
          g[j] = __uint_as_float(r[j]);
          if (e.col_scale) g[j] = scaled_by(g[j], rs, cs);
          if (!GATED && e.bias) g[j] += ca;
          if (GATED) {
            u[j] = __uint_as_float(s[j]);
            if (e.col_scale) u[j] = scaled_by(u[j], rs, ca);
          }
        }
        if (e.pre) {
          store_rows16(e.pre, (long long)t * e.ld + n, e.ld, rows, VERACE_F32, g);
          if (GATED) store_rows16(e.pre_up, (long long)t * e.ld + n, e.ld, rows, VERACE_F32, u);
        }
        if (e.type == VERACE_F32) activate<GATED, false>(e, g, u);
        else activate<GATED, true>(e, g, u);
#pragma unroll
        for (int j = 0; j < 16; ++j) g[j] += res[j];
        store_rows16(e.out, (long long)t * e.ld + n, e.ld, rows, e.type, g);
      }
    }
  } else {
    // every CTA's sums in its shared memory (the stages' place), [token][128].  TMEM is given back before the CTA
    // waits for the others of its cluster: one that held it there could wait for a CTA that waits for TMEM
    float* part = reinterpret_cast<float*>(sm);
    for (int t = 16 * (warp >> 2); t < tokens; t += 32)
#pragma unroll
      for (int h = 0; h < (GATED ? 2 : 1); ++h) {
        uint32_t r[16];
        tmem_ld_async(mine + h * p.mp + t, r);
        tmem_wait(r);
        float* o = part + (h * p.mp + t) * ROWS + 32 * quarter + lane;
#pragma unroll
        for (int j = 0; j < 16; ++j) o[j * ROWS] = ok && first < last ? __uint_as_float(r[j]) : 0.f;
      }
  }
  tc::fence_before_sync();
  __syncthreads();
  if (warp == 1) tc::tmem_dealloc(tmem, p.cols);
  if (joins) {
    cg::cluster_group cl = cg::this_cluster();
    const float* part = reinterpret_cast<const float*>(sm);
    auto met = cl.barrier_arrive();
    // a thread joins four columns of every 8 ck'th token
    const int col = 4 * lane, quad = (int)max(0LL, min(4LL, p.N - n0 - col)), joiner = rank * NT + tid,
              total = quad ? tokens * (ROWS / 4) : 0;
    const long long c0 = n0 + col;
    float res[4] = {};
    auto residual = [&](int i) {
      if (!GATED && e.residual && i < total) load4(e.residual, (long long)(i / (ROWS / 4)) * e.ld_res + c0, quad, e.type, res);
    };
    residual(joiner);
    cl.barrier_wait(std::move(met));
    // (the next vectors on their way while one is finished; one body for all of them: unrolled, it took 3.7 us for 64
    // gated tokens where it takes 2.2, most of it instructions on their way)
    auto join = [&](auto ck) {
      constexpr int CK = decltype(ck)::value, H = GATED ? 2 : 1;
      const float4* o[CK];
#pragma unroll
      for (int c = 0; c < CK; ++c) o[c] = reinterpret_cast<const float4*>(cl.map_shared_rank(part, c));
      float4 v[H][CK];
      auto load = [&](int i) {
        if (i < total)
#pragma unroll
          for (int h = 0; h < H; ++h)
#pragma unroll
            for (int c = 0; c < CK; ++c) v[h][c] = o[c][h * p.mp * (ROWS / 4) + i];
      };
      load(joiner);
#pragma unroll 1
      for (int i = joiner; i < total; i += CK * NT) {
        float s[2][4] = {}, r[4];
#pragma unroll
        for (int h = 0; h < H; ++h)
#pragma unroll
          for (int c = 0; c < CK; ++c) {
            s[h][0] += v[h][c].x; s[h][1] += v[h][c].y; s[h][2] += v[h][c].z; s[h][3] += v[h][c].w;
          }
#pragma unroll
        for (int j = 0; j < 4; ++j) r[j] = res[j];
        load(i + CK * NT);
        residual(i + CK * NT);
        const int t = i / (ROWS / 4);
        finish4<GATED>(e, t, c0, quad, col_scale + col, col_add + col, row_scale[t], r, s[0], s[1]);
      }
    };
    if (p.ck == 2) join(std::integral_constant<int, 2>());
    else if (p.ck == 4) join(std::integral_constant<int, 4>());
    else join(std::integral_constant<int, 8>());
    cl.sync();   // (the others may still read this CTA's sums)
  }
}

// ------------------------------------------------------------------ host
template <bool F8, bool WMN, bool GATED>
int launch(const Product& p, cudaStream_t st) {
  Maps maps;
  Args a{};
  int rc;
  a.M = p.M; a.N = p.N;
  static_assert(FEW % 16 == 0 && FEW * ROWS * 4 * 2 <= ROOM && 2 * FEW <= 512, "a CTA's sums fit in shared memory and TMEM");
  a.mp = (int)((p.M + 15) / 16 * 16);
  // A (x) in one box of all tokens, B (the weights) as the MMA's rows
  if ((rc = operand_map(&maps.x, p.a, p.type, a.mp))) return rc;
  for (int i = 0; i < 2; ++i)
    if ((rc = operand_map(&maps.w[i], p.b[p.b[i].p ? i : 0], p.type, WMN ? 64 : ROWS))) return rc;
  a.kblocks = (int)((p.K + (F8 ? 127 : 63)) / (F8 ? 128 : 64));
  a.a_first = p.a_first;
  a.steps = a.kblocks * p.segments;
  a.tiles_n = (int)((p.N + ROWS - 1) / ROWS);
  a.ck = few_splits(p.N, p.K, p.segments, p.type);
  a.per = (a.steps + a.ck - 1) / a.ck;
  a.stage = ROWS * 128 * (GATED ? 2 : 1) + a.mp * 128;
  // Two CTAs an SM while that leaves a CTA three stages (gated, 64 x 4096 x 32000: 89 us against 90, 48 of it for 8 bits
  // against 50); of a split K five, as there is a CTA for every SM at most (64 x 8192 x 4096: 17.4 us with four, 15.8 alone
  // on the SM with eight); clusters of eight always, which the SMs of a GPC hold only twice otherwise (32 x 16384 x 2048
  // 16.6 us against 26.1), unless their sums need more.
  const int sums = a.ck > 1 ? a.mp * ROWS * 4 * (GATED ? 2 : 1) : 0;
  int room = HALF_ROOM;
  if (sums > room || (a.ck < 8 && room / a.stage < (a.ck > 1 ? 5 : 3))) room = ROOM;
  a.stages = room / a.stage < MAX_STAGES ? room / a.stage : MAX_STAGES;
  if (a.stages > a.per) a.stages = a.per;
  const int want = a.mp * (GATED ? 2 : 1);
  a.cols = 32;
  while (a.cols < want) a.cols *= 2;
  int smem = a.stages * a.stage;
  if (smem < sums) smem = sums;
  smem += 1024;
  a.idesc = (1u << 4) | (uint32_t)(p.type == VERACE_BF16) << 7 | (uint32_t)(p.type == VERACE_BF16) << 10 |
            (uint32_t)WMN << 15 | (uint32_t)(a.mp >> 3) << 17 | (uint32_t)(ROWS >> 4) << 24;
  a.e = p.e;
  auto kern = few_product<F8, WMN, GATED>;
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  static std::atomic<uint64_t> ready{0};      // devices whose limit is raised
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, ROOM + 1024));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  return launch_after("few_product", kern, dim3(a.tiles_n * a.ck), NT, smem, st, a.ck, maps, a);
}

}  // namespace

namespace lin {

int product_few(const Product& p, cudaStream_t st) {
  if (p.type == VERACE_E4M3) return p.gated ? launch<true, false, true>(p, st) : launch<true, false, false>(p, st);
  if (p.gated) return launch<false, false, true>(p, st);
  return p.b_mn ? launch<false, true, false>(p, st) : launch<false, false, false>(p, st);
}

}  // namespace lin

int linear_few_read_status(int* status) {
  int h = 0;
  VERACE_CUDA(cudaMemcpyFromSymbol(&h, g_linear_few_status, sizeof(int)));
  if (h) {
    const int zero = 0;
    VERACE_CUDA(cudaMemcpyToSymbol(g_linear_few_status, &zero, sizeof(int)));
  }
  *status = h;
  return VERACE_OK;
}

}  // namespace verace
