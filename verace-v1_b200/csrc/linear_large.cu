// Products of many rows on the tensor cores (the engine behind linear.cu):
//     out(m, n) = epilogue(sum_k A(m, k) B(n, k))
// A pair of CTAs on neighbouring SMs computes a tile of 256 x BN: each holds 128 rows of A and
// half of B's rows in shared memory, and one tcgen05.mma.cta_group::2 a step of 32 bytes of K
// reads both, 128 rows x BN columns of fp32 sums landing in each CTA's TMEM.  (A single CTA's
// 128 x 256 tile would read 12 KB of shared memory for what the pair does with 8 KB a CTA.)
//
// Warps: 0 feeds stages of 128 bytes of K by TMA (128-byte swizzle; operands stored with K
// outermost come as boxes of 64 x 64 and go to the MMA as MN-major), 1 issues the MMAs (in the pair's
// first CTA), 4 to 11 are the epilogue.  Two sets of sums in TMEM: a tile's epilogue runs under
// the next one's products.  Persistent: a pair takes every 74th tile, eight rows of tiles
// beside each other so that the running tiles share their operands in L2.
//
// Gated products put 64 or 128 rows of each weight into one tile (the first CTA of the pair loads the
// gate's, the second the up projection's), so both sums of an output lie in one TMEM row and the product is formed in
// registers.  A sum of two products (the input gradient of a gated block) is two runs over K.
//
// fp32 operands come as three bf16 parts, three stages for 64 values of K (a stage holds one part of A and of B), and
// the MMAs take six pairs of them, the smallest first: the pairs of one order lie 2^8 above the next, by which the sums so
// far are brought down as the next order begins.  The tensor core cuts its sums to fp32 after every step instead
// of rounding them, which over a whole K adds up (K = 1001: 6e-6 of the result); so after every 64 values of K
// the epilogue's warps add them up in registers, rounding, while the next 64 run into the other set.  Sums of 16- and
// 8-bit operands stay there for up to run_of(type) values (linear_tc.cuh); K beyond that is split.
//
// Epilogue: a thread holds a row of the tile (as TMEM gives it), 64 columns at a time (32 of fp32),
// applies scales, bias and activation and puts the rounded values into the warp's block of shared memory, from where
// TMA stores them; rows that are not 16-byte aligned are stored word by word, the warp along a row.  Residuals come
// into the block that way too, fetched while the products run.
//
// Measured on the device: gated 8192 x 4096 x 2 x 8192 bf16 690 to 708 us (1.55 to 1.59 PFLOP/s, the tensor pipe 96 % active;
// a second of such calls runs into the power limit, 805 to 821 us), 8192 x 8192 x 4096 e4m3 188 to 194 us (2.8 to 2.9 PFLOP/s;
// bound by what the CTAs load, 32 KB each for 256 clocks of MMAs; in long runs 230), 8192 x 1024 x 4096 bf16 48 us (1.42),
// 4096^3 fp32 603 us (228 TFLOP/s).
#include "linear_tc.cuh"

#include <atomic>

namespace verace {

__device__ int g_linear_status = 0;   // non-zero after a bounded wait gave up

namespace {

using namespace lin;

constexpr int NT = 384, EPI_WARPS = 8;
constexpr uint32_t POLLS = 1u << 22, SUM_POLLS = 1u << 26;   // (a sum runs over up to run_of(type) values)
// 256 columns of parts: four warps give up registers for the epilogue's eight.  What the block was launched with has to cover
// both shares, or the increase would wait for ever; the host checks the kernels' count before it chooses them (wide_parts).
constexpr int SPLIT_REGISTERS = 168;
static_assert(128 * 72 + 256 * 216 <= NT * SPLIT_REGISTERS, "the shares' sum");
constexpr int TURN = 4096;             // a warp's block of the output: 32 rows of 128 bytes

template <int BN>
struct Shape {
  static constexpr int STAGE = 16384 + BN * 64;              // A: 128 rows x 128 bytes; B: BN / 2 rows
  static constexpr int STAGES = BN == 256 ? 6 : 8;
  static constexpr int TURNS = STAGE * STAGES, BARS = TURNS + EPI_WARPS * TURN, SMEM = BARS + 256 + 1024;
};

struct Maps {
  CUtensorMap a, b[2], out[2], pre[2];
};

struct Args {
  long long M, N;
  int kblocks, segments, a_first, a_step;
  int nz, tiles_m, tiles_n, tiles;
  int by_tma, pre_by_tma;   // whether the rows of the outputs and of the saved sums are 16-byte aligned
  int splits, per;      // of K: `per` stages (of every segment) each; the sums of split i go to the i-th partial outputs
  long long partial;    // values from one split's outputs to the next
  uint32_t idesc;
  void* out_z[2];
  Epilogue e;
};

__device__ __forceinline__ uint32_t in_cta0(const void* p) {   // the address of p's place in the pair's first CTA
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(tc::smem_addr(p)));
  return a;
}
__device__ __forceinline__ uint32_t cta_in_pair() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// a box into this CTA's shared memory, its bytes counted on the first CTA's barrier
__device__ __forceinline__ void load_box(void* smem, const CUtensorMap* map, int x, int y, int z, uint32_t bar0) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(tc::smem_addr(smem)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar0)
      : "memory");
}
// (SHIFT: the sums so far are multiplied by 2^-SHIFT)
template <bool F8, int SHIFT = 0>
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (F8)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate));
  else if constexpr (SHIFT == 0)
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate));
  else
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p, %5;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
                 "r"(accumulate), "n"(SHIFT));
}
// arrive on `bar` in both CTAs once the MMAs issued so far are done
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   tc::smem_addr(bar)),
               "h"((unsigned short)3)
               : "memory");
}
// (What it hands over is TMEM, ordered by the tcgen05 fences; a release over the cluster would wait for the
// warp's stores.)
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// tile t -> (split of K, output, row, column) of tiles: groups of eight rows, column by column
struct Place {
  int split, z, m, n;
};
__device__ __forceinline__ Place place(const Args& p, int t) {
  Place o;
  const int each = p.tiles_m * p.tiles_n;
  o.z = t / each;
  t -= o.z * each;
  o.split = o.z / p.nz;
  o.z -= o.split * p.nz;
  const int group = t / (8 * p.tiles_n), first = 8 * group, high = min(8, p.tiles_m - first);
  t -= group * 8 * p.tiles_n;
  o.n = t / high;
  o.m = first + t - o.n * high;
  return o;
}

// ------------------------------------------------------------------ the epilogue
// A warp's block: 32 rows of 128 bytes (32 columns of fp32, or 64 of 16-bit types) in shared memory, the 16-byte
// pieces of a row exchanged as TMA's 128-byte swizzle has them, which also keeps both a thread's walk along its own
// row and the warp's walk along one row free of bank conflicts.
struct Block {
  uint32_t turn;            // its address in shared memory
  long long m0, n0, M, N;   // first row and column; ends
};
// Where a block goes: by TMA through a map, or to rows in memory `ld` values apart.
struct Target {
  const CUtensorMap* map;
  int z;
  void* p;
  long long ld;
};

__device__ __forceinline__ uint32_t piece_at(const Block& b, int row, int piece) {   // the address of 16 bytes of a row
  return b.turn + row * 128 + ((piece ^ (row & 7)) << 4);
}
// (by their address: through pointers these would be generic accesses)
__device__ __forceinline__ uint32_t word(const Block& b, int row, int i) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(piece_at(b, row, i >> 2) + 4 * (i & 3)) : "memory");
  return v;
}
__device__ __forceinline__ void set_word(const Block& b, int row, int i, uint32_t v) {
  asm volatile("st.shared.b32 [%0], %1;" ::"r"(piece_at(b, row, i >> 2) + 4 * (i & 3)), "r"(v) : "memory");
}
__device__ __forceinline__ uint4 get_piece(const Block& b, int row, int piece) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(piece_at(b, row, piece))
               : "memory");
  return v;
}
__device__ __forceinline__ void set_piece(const Block& b, int row, int piece, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(piece_at(b, row, piece)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}
// the block's last copy to memory has left it
__device__ __forceinline__ void reclaim(int lane) {
  if (lane == 0) tc::bulk_wait_read<0>();
  __syncwarp();
}

// Where a warp reads or writes a block: row by row, a word (or its two halves) a lane.
struct Rows {
  char* at;           // the lane's word in the first row
  long long step;     // bytes of a row
  int rows;           // rows inside
  int part;           // 0: no column of the lane inside, 3: a whole word in every row, else 1: its first half alone, 2: both
};
template <bool WIDE>
__device__ __forceinline__ Rows rows_of(const Block& b, const void* p, long long ld, int lane) {
  constexpr int SIZE = WIDE ? 4 : 2, PER = WIDE ? 1 : 2;
  const long long n = b.n0 + PER * lane;
  Rows r;
  r.at = (char*)p + (b.m0 * ld + n) * SIZE;
  r.step = ld * SIZE;
  r.rows = (int)min(32LL, b.M - b.m0);
  if (WIDE) r.part = n < b.N ? 3 : 0;
  else r.part = n >= b.N ? 0 : n + 1 == b.N ? 1 : ((r.step | (size_t)r.at) & 3) == 0 ? 3 : 2;
  return r;
}
// the block to memory
template <bool WIDE>
__device__ __forceinline__ void write_block(const Block& b, const Target& to, int lane) {
  if (to.map) {
    tc::fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(to.map),
                   "r"((int)b.n0), "r"((int)b.m0), "r"(to.z), "r"(b.turn)
                   : "memory");
      tc::bulk_commit();
    }
    return;
  }
  __syncwarp();
  Rows r = rows_of<WIDE>(b, to.p, to.ld, lane);
  if (r.part == 3 && r.rows == 32) {
#pragma unroll
    for (int h = 0; h < 32; h += 16) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) w[i] = word(b, h + i, lane);
#pragma unroll
      for (int i = 0; i < 16; ++i, r.at += r.step) *reinterpret_cast<uint32_t*>(r.at) = w[i];
    }
  } else if (r.part == 3) {
    for (int i = 0; i < r.rows; ++i) *reinterpret_cast<uint32_t*>(r.at + i * r.step) = word(b, i, lane);
  } else if (!WIDE && r.part) {
    // rows off 4-byte borders (an odd row stride), or a last word cut in two: where the row's words lie between two
    // words of the block, a lane stores the column before its own and its first
    const int left = (int)min(64LL, b.N - b.n0) - 2 * lane;   // columns from the lane's on
#pragma unroll 8
    for (int i = 0; i < r.rows; ++i) {
      const uint32_t w = word(b, i, lane);
      unsigned short* o = reinterpret_cast<unsigned short*>(r.at + i * r.step);
      if (((size_t)o & 3) == 0) {
        if (left > 1) *reinterpret_cast<uint32_t*>(o) = w;
        else o[0] = (unsigned short)w;
      } else {
        if (lane == 0) o[0] = (unsigned short)w;
        else *reinterpret_cast<uint32_t*>(o - 1) = word(b, i, lane - 1) >> 16 | w << 16;
        if (left > 1 && (lane == 31 || left == 2)) o[1] = (unsigned short)(w >> 16);
      }
    }
  }
  __syncwarp();
}
// the words of a block of p, all loads in flight together
template <bool WIDE>
__device__ __forceinline__ void read_words(const Block& b, const void* p, long long ld, int lane, uint32_t (&w)[32]) {
  const Rows r = rows_of<WIDE>(b, p, ld, lane);
  if (r.part == 3) {
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i] = i < r.rows ? *reinterpret_cast<const uint32_t*>(r.at + i * r.step) : 0u;
  } else if (r.part) {
    const int second = r.part == 2 ? 1 : 0;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      w[i] = i < r.rows ? reinterpret_cast<const unsigned short*>(r.at + i * r.step)[0] : 0u;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (second && i < r.rows) w[i] |= (uint32_t)reinterpret_cast<const unsigned short*>(r.at + i * r.step)[1] << 16;
  }
}
// U values into the thread's own row of the block, from column c on
template <bool WIDE, int U>
__device__ __forceinline__ void put(const Block& b, int c, const float (&v)[U], int type, int lane) {
  if constexpr (WIDE) {
#pragma unroll
    for (int j = 0; j < U / 4; ++j)
      set_piece(b, lane, c / 4 + j, make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                                               __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3])));
  } else {
    uint32_t w[U / 2];
    if (type == VERACE_BF16) {
#pragma unroll
      for (int j = 0; j < U / 2; ++j) w[j] = pack_pair(v[2 * j], v[2 * j + 1], VERACE_BF16);
    } else {
#pragma unroll
      for (int j = 0; j < U / 2; ++j) w[j] = pack_pair(v[2 * j], v[2 * j + 1], VERACE_F16);
    }
#pragma unroll
    for (int j = 0; j < U / 8; ++j) set_piece(b, lane, c / 8 + j, make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]));
  }
}
template <bool WIDE, int U>
__device__ __forceinline__ void add(const Block& b, int c, float (&v)[U], int type, int lane) {
#pragma unroll
  for (int j = 0; j < U / (WIDE ? 4 : 8); ++j) {
    const uint4 w = get_piece(b, lane, c / (WIDE ? 4 : 8) + j);
    const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (WIDE) {
        v[4 * j + i] += __uint_as_float(x[i]);
      } else {
        const float2 f = unpack_pair(x[i], type);
        v[8 * j + 2 * i] += f.x;
        v[8 * j + 2 * i + 1] += f.y;
      }
    }
  }
}
// U sums of a row from column n0 on, with scales and bias
template <int U>
__device__ __forceinline__ void scaled(const Epilogue& e, const uint32_t (&r)[U], float (&v)[U], float rs,
                                       const float* col_scale, const void* bias, long long n0, long long N) {
#pragma unroll
  for (int j = 0; j < U; ++j) v[j] = __uint_as_float(r[j]);
  if (col_scale) {
    float s[U];
    column_values(col_scale, VERACE_F32, n0, N, s);
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] = scaled_by(v[j], rs, s[j]);
  }
  if (bias) {
    float s[U];
    column_values(bias, e.bias_type, n0, N, s);
#pragma unroll
    for (int j = 0; j < U; ++j) v[j] += s[j];
  }
}

// Where a block takes its sums from, 16 columns a lot: r, and of gated products the second sums s.
// TMEM: the next lot is on its way (ask) while one is worked on (have).
template <bool GATED>
struct TmemSums {
  uint32_t at, up;
  __device__ __forceinline__ void ask(int lot, uint32_t (&r)[16], uint32_t (&s)[16]) const {
    tmem_ld_async(at + 16 * lot, r);
    if constexpr (GATED) tmem_ld_async(up + 16 * lot, s);
  }
  __device__ __forceinline__ void have(uint32_t (&r)[16], uint32_t (&s)[16]) const {
    tmem_wait(r);
    if constexpr (GATED) tmem_wait(s);
  }
};
// local memory (parts): the warp's half of the tile's columns, of gated products half of each sum's; from lot `first` on
template <bool GATED, int N>
struct HeldSums {
  const float* sum;
  int first;
  __device__ __forceinline__ void ask(int lot, uint32_t (&r)[16], uint32_t (&s)[16]) const {
    const float4* f = reinterpret_cast<const float4*>(sum + 16 * (first + lot));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 a = f[j];
      r[4 * j] = __float_as_uint(a.x); r[4 * j + 1] = __float_as_uint(a.y);
      r[4 * j + 2] = __float_as_uint(a.z); r[4 * j + 3] = __float_as_uint(a.w);
      if constexpr (GATED) {
        const float4 b = f[N / 8 + j];
        s[4 * j] = __float_as_uint(b.x); s[4 * j + 1] = __float_as_uint(b.y);
        s[4 * j + 2] = __float_as_uint(b.z); s[4 * j + 3] = __float_as_uint(b.w);
      }
    }
  }
  __device__ __forceinline__ void have(uint32_t (&)[16], uint32_t (&)[16]) const {}
};

// The saved sums of `width` columns, in fp32: 32 columns at a time.  UP: the second sums.
template <bool UP, typename Sums>
__device__ __forceinline__ void save_sums(const Epilogue& e, Block b, const Sums& sums, int width, float rs,
                                          const float* col_scale, const void* bias, const Target& to, int lane) {
#pragma unroll 1
  for (int c = 0; c < width && b.n0 < b.N; c += 32, b.n0 += 32) {
    reclaim(lane);
#pragma unroll 1
    for (int h = 0; h < 32; h += 16) {
      uint32_t r[16], s[16];
      sums.ask((c + h) / 16, r, s);
      sums.have(r, s);
      float v[16];
      scaled(e, UP ? s : r, v, rs, col_scale, bias, b.n0 + h, b.N);
      put<true>(b, h, v, VERACE_F32, lane);
    }
    write_block<true>(b, to, lane);
  }
}

// One block, its residual in `res` (AHEAD) or read here.  `loaded` is called once the block's sums are in registers.
template <bool GATED, bool WIDE, bool AHEAD, typename Sums, typename F>
__device__ __forceinline__ void epilogue_block(const Epilogue& e, const Block& b, const Sums& sums,
                                               const uint32_t (&res)[AHEAD ? 32 : 1], const Target& out, const Target& pre,
                                               const Target& pre_up, int lane, F&& loaded) {
  constexpr int WIDTH = WIDE ? 32 : 64, U = 16, LOTS = WIDTH / U;
  const long long m = b.m0 + lane;
  const float rs = e.row_scale && m < b.M ? e.row_scale[m] : 0.f;
  if (e.pre) {
    save_sums<false>(e, b, sums, WIDTH, rs, e.col_scale, GATED ? nullptr : e.bias, pre, lane);
    if (GATED) save_sums<true>(e, b, sums, WIDTH, rs, e.up_scale, nullptr, pre_up, lane);
  }
  if (GATED && out.p == nullptr) {   // (partial sums: the two above are all)
    loaded();
    return;
  }
  uint32_t r[U], s[U];
  sums.ask(0, r, s);
  reclaim(lane);
  if (!GATED && e.residual) {
    if constexpr (AHEAD) {
#pragma unroll
      for (int i = 0; i < 32; ++i) set_word(b, i, lane, res[i]);
    } else {
      uint32_t w[32];
      read_words<WIDE>(b, e.residual, e.ld_res, lane, w);
#pragma unroll
      for (int i = 0; i < 32; ++i) set_word(b, i, lane, w[i]);
    }
    __syncwarp();
  }
#pragma unroll 1
  for (int l = 0; l < LOTS; ++l) {
    float v[U], u[U] = {};
    sums.have(r, s);
    scaled(e, r, v, rs, e.col_scale, GATED ? nullptr : e.bias, b.n0 + l * U, b.N);
    if constexpr (GATED) scaled(e, s, u, rs, e.up_scale, nullptr, b.n0 + l * U, b.N);
    if (l + 1 < LOTS) sums.ask(l + 1, r, s);
    else loaded();
    activate<GATED, !WIDE>(e, v, u);
    if (!GATED && e.residual) add<WIDE>(b, l * U, v, e.type, lane);
    put<WIDE>(b, l * U, v, e.type, lane);
  }
  write_block<WIDE>(b, out, lane);
}

// A warp's part of every tile of the pair: TMEM lanes 32 (warp % 4) ..., one half of the columns.
template <bool GATED, bool WIDE, int BN, bool PARTS, typename Wait, typename Free>
__device__ __forceinline__ void epilogue_tiles(const Args& p, const Maps& maps, uint32_t turn, uint32_t tmem, int pair, int pairs,
                                               int rank, int warp, int lane, Wait&& wait, Free&& release) {
  constexpr int HB = BN / 2, TN = GATED ? HB : BN, WIDTH = WIDE ? 32 : 64, PER = TN / 2 > WIDTH ? TN / 2 : WIDTH;
  const int half = (warp - 4) >> 2, first = half * PER, last = min(TN, first + PER);
  const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
  Block b;
  b.turn = turn;
  b.M = p.M;
  b.N = p.N;
  int n = 0;
  for (int t = pair; t < p.tiles; t += pairs, ++n) {
    const Place at = place(p, t);
    b.m0 = at.m * 256LL + rank * 128 + 32 * (warp & 3);
    b.n0 = (long long)at.n * TN + first;
    // the tile's outputs: of split i the i-th of the partial ones
    const long long first_of = p.splits > 1 ? (at.split * p.nz + at.z) * p.partial : 0;
    const int slot = p.splits > 1 ? 0 : at.z, z = p.splits > 1 ? at.split * p.nz + at.z : 0;
    Target out{p.by_tma ? &maps.out[slot] : nullptr, z, p.nz > 1 && p.splits == 1 ? p.out_z[at.z] : p.e.out, p.e.ld};
    Target pre{p.pre_by_tma ? &maps.pre[0] : nullptr, z, p.e.pre ? p.e.pre + first_of : nullptr, p.e.ld};
    Target pre_up{p.pre_by_tma ? &maps.pre[1] : nullptr, z, p.e.pre_up ? p.e.pre_up + first_of : nullptr, p.e.ld};
    if (!GATED && p.splits > 1) out.p = static_cast<float*>(p.e.out) + first_of;
    constexpr bool AHEAD = !PARTS;   // residuals on their way while the products run (parts' sums leave no registers for them)
    uint32_t res[AHEAD ? 32 : 1];
    if constexpr (AHEAD)
      if (!GATED && p.e.residual && b.m0 < b.M && b.n0 < b.N && first < last)
        read_words<WIDE>(b, p.e.residual, p.e.ld_res, lane, res);
    __align__(16) float held_sums[PARTS ? BN / 2 : 4];
    const int set = wait(n, held_sums);
    if (set < 0) break;
    const uint32_t sums = lanes + set;
    bool held = true;
    for (int c = first; c < last; c += WIDTH) {
      b.n0 = (long long)at.n * TN + c;
      if (b.m0 >= b.M || b.n0 >= b.N) break;
      Block after = b;
      after.n0 += WIDTH;
      const bool more = c + WIDTH < last && after.n0 < b.N;
      auto loaded = [&] {
        if (!more) {
          release(n);
          held = false;
        }
      };
      if constexpr (PARTS) {
        epilogue_block<GATED, WIDE, false>(p.e, b, HeldSums<GATED, BN / 2>{held_sums, (c - first) / 16}, res, out, pre, pre_up,
                                           lane, loaded);
      } else {
        uint32_t next[32];
        if (!GATED && p.e.residual && more) read_words<WIDE>(after, p.e.residual, p.e.ld_res, lane, next);
        epilogue_block<GATED, WIDE, true>(p.e, b, TmemSums<GATED>{sums + c, sums + HB + c}, res, out, pre, pre_up, lane, loaded);
        if (!GATED && p.e.residual)
#pragma unroll
          for (int i = 0; i < 32; ++i) res[i] = next[i];
      }
    }
    if (held) release(n);
  }
  if (lane == 0) tc::bulk_wait<0>();   // (the stores are done before the CTA ends)
}

template <bool F8, bool AMN, bool BMN, bool GATED, int BN, bool PARTS>
__global__ void __launch_bounds__(NT, 1)
large_product(const __grid_constant__ Maps maps, const __grid_constant__ Args p) {
  using S = Shape<BN>;
  constexpr int KB = F8 ? 128 : 64;            // values of K in a stage
  constexpr int HB = BN / 2;                   // rows of B in a CTA
  constexpr int COLS = 2 * BN;                 // of TMEM: two sets of sums
  extern __shared__ __align__(1024) unsigned char raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>(((size_t)raw + 1023) & ~(size_t)1023);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + S::BARS);
  uint64_t* empty = full + S::STAGES;
  uint64_t* acc_full = empty + S::STAGES;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* fail = reinterpret_cast<volatile int*>(slot + 1);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const uint32_t rank = cta_in_pair();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_addr(slot)), "r"(COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 2 && lane < 5)   // (the tensor maps on their way: a, b, b, out, out)
    asm volatile("prefetch.tensormap [%0];" ::"l"(&maps.a + lane) : "memory");
  if (tid == 0) {
    for (int i = 0; i < S::STAGES; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 2 * EPI_WARPS);
    }
    *fail = 0;
    tc::fence_mbar_init();
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc::fence_after_sync();
  depend();
  const uint32_t tmem = *slot;
  // sets of sums that make up a tile: one; of parts one for 64 values of K of a segment (as many for every split of K,
  // the last one's may be empty)
  const int sets = PARTS ? p.per * p.segments : 1;

  if (warp < 4) {
    if constexpr (PARTS && BN == 256) asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");   // (see SPLIT_REGISTERS)
    if (warp == 0) {
      if (lane == 0) {   // ---- operands
        int i = 0, flying = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int t = pair; t < p.tiles && ok; t += pairs) {
          const Place at = place(p, t);
          const int m0 = at.m * 256 + (int)rank * 128;
          const int n0 = GATED ? at.n * HB : at.n * BN + (int)rank * HB;
          const int k0 = at.split * p.per, k1 = min(k0 + p.per, p.kblocks);
          // (segment by segment; of parts 64 values of K of every segment, then the next)
          const int outer = PARTS ? k1 - k0 : p.segments, inner = PARTS ? 3 * p.segments : k1 - k0;
          for (int u = 0; u < outer && ok; ++u) {
            for (int v = 0; v < inner; ++v) {
              const int s = PARTS ? v / 3 : u, kb = k0 + (PARTS ? u : v), part = PARTS ? v % 3 : 0;
              const CUtensorMap* mb = &maps.b[GATED ? rank : s];
              const int az = part * p.a_step + p.a_first + s + at.z;
              if (!tc::mbar_wait(&empty[i], phase ^ 1, POLLS)) {   // (a fresh barrier lets the first round through)
                ok = false;
                break;
              }
              if (rank == 0) tc::mbar_expect_tx(&full[i], 2 * S::STAGE);
              const uint32_t bar = in_cta0(&full[i]);
              unsigned char* a = sm + i * S::STAGE;
              unsigned char* b = a + 16384;
              if constexpr (AMN) {
                load_box(a, &maps.a, m0, kb * KB, az, bar);
                load_box(a + 8192, &maps.a, m0 + 64, kb * KB, az, bar);
              } else {
                load_box(a, &maps.a, kb * KB, m0, az, bar);
              }
              if constexpr (BMN) {
#pragma unroll
                for (int h = 0; h < HB / 64; ++h) load_box(b + h * 8192, mb, n0 + 64 * h, kb * KB, part, bar);
              } else {
                load_box(b, mb, kb * KB, n0, part, bar);
              }
              if (++i == S::STAGES) i = 0, phase ^= 1;
              flying = min(flying + 1, S::STAGES);
            }
          }
        }
        if (!ok) {
          *fail = 1;
          atomicExch(&g_linear_status, 1);
        }
        // copies in flight land before the CTA may end (the first CTA's barriers count both CTAs'; the
        // second one stays for the first at the cluster's barrier below)
        if (rank == 0)
          while (flying-- > 0) {
            if (i == 0) i = S::STAGES, phase ^= 1;
            tc::mbar_wait(&full[--i], phase, POLLS);
          }
      }
    } else if (warp == 1) {
      if (rank == 0) {   // ---- MMAs of the pair.  The whole warp walks the loop, so that the operands sit in uniform registers:
        // by one thread's own loop a step of four MMAs took 657 clocks, the MMAs themselves take 512
        const bool lead = elect();
        constexpr std::integral_constant<int, 0> NONE;
        constexpr std::integral_constant<int, PARTS ? 8 : 0> PART;
        int i = 0, n = 0;
        uint32_t phase = 0;
        bool ok = true;
        const int mine = (p.tiles - pair + pairs - 1) / pairs * sets;   // sets to fill
        // four MMAs: 128 bytes of K of stage ia's A and stage ib's B
        auto step = [&](uint32_t d, int ia, int ib, bool more, auto shift) {
          const uint32_t a = tc::smem_addr(sm + ia * S::STAGE), bb = tc::smem_addr(sm + ib * S::STAGE) + 16384;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            // K-major: 32 bytes along the rows; MN-major: 16 rows of 128 bytes
            const uint64_t da = AMN ? tc::sdesc_sw128(a + k * 2048, 8192, 1024) : tc::sdesc_sw128(a + k * 32, 16, 1024);
            const uint64_t db = BMN ? tc::sdesc_sw128(bb + k * 2048, 8192, 1024) : tc::sdesc_sw128(bb + k * 32, 16, 1024);
            if (k == 0) mma_pair<F8, decltype(shift)::value>(d, da, db, p.idesc, more ? 1u : 0u);
            else mma_pair<F8>(d, da, db, p.idesc, 1u);
          }
        };
        for (; n < mine && ok; ++n) {
          const int b = n & 1, use = n >> 1;
          const int k0 = place(p, pair + n / sets * pairs).split * p.per;
          const int steps = PARTS ? k0 + n % sets / p.segments < p.kblocks : p.segments * (min(k0 + p.per, p.kblocks) - k0);
          if (!tc::mbar_wait(&acc_empty[b], (use & 1) ^ 1, POLLS)) {
            ok = false;
            break;
          }
          tc::fence_after_sync();
          const uint32_t d = tmem + b * BN;
          for (int s = 0; s < steps; ++s) {
            if constexpr (!PARTS) {
              if (!tc::mbar_wait(&full[i], phase, POLLS)) {
                ok = false;
                break;
              }
              tc::fence_after_sync();
              if (lead) {
                step(d, i, i, s > 0, NONE);
                commit_pair(&empty[i]);
              }
              __syncwarp();
              if (++i == S::STAGES) i = 0, phase ^= 1;
            } else {
              int at[3];
              for (int j = 0; j < 3 && ok; ++j) {
                at[j] = i;
                ok = tc::mbar_wait(&full[i], phase, POLLS);
                if (++i == S::STAGES) i = 0, phase ^= 1;
              }
              if (!ok) break;
              tc::fence_after_sync();
              if (lead) {   // parts: 0 the high one, 1 and 2 times 2^8 and 2^16
                step(d, at[2], at[0], false, NONE);
                step(d, at[1], at[1], true, NONE);
                step(d, at[0], at[2], true, NONE);
                commit_pair(&empty[at[2]]);
                step(d, at[1], at[0], true, PART);
                step(d, at[0], at[1], true, NONE);
                commit_pair(&empty[at[1]]);
                step(d, at[0], at[0], true, PART);
                commit_pair(&empty[at[0]]);
              }
              __syncwarp();
            }
          }
          if (lead) commit_pair(&acc_full[b]);   // (also after a failure: every MMA issued completes)
          __syncwarp();
          if (!ok) tc::mbar_wait(&acc_full[b], use & 1, POLLS);
        }
        if (!ok) {
          *fail = 1;
          if (lane == 0) atomicExch(&g_linear_status, 1);
        }
      }
    }
  } else {   // ---- epilogue
    if constexpr (PARTS && BN == 256) asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const uint32_t turn = tc::smem_addr(sm + S::TURNS + (warp - 4) * TURN);
    auto filled = [&](int n) {
      if (!tc::mbar_wait(&acc_full[n & 1], (n >> 1) & 1, SUM_POLLS)) {
        *fail = 1;
        if (lane == 0) atomicExch(&g_linear_status, 1);
        return false;
      }
      tc::fence_after_sync();
      return *fail == 0;
    };
    auto free = [&](int n) {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) arrive_at(in_cta0(&acc_empty[n & 1]));
    };
    // tile n's sums: the TMEM column of their set, or -1; of parts in `sum`, the warp's half of the columns (gated: of
    // both sums)
    auto wait = [&](int n, auto& sum) {
      if constexpr (!PARTS) {
        return filled(n) ? (n & 1) * BN : -1;
      } else {
        const uint32_t lanes = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        const int k0 = place(p, pair + n * pairs).split * p.per;
        auto col = [&](int h) {
          return GATED ? (h >= HB / 2 ? HB / 2 + h : h) + (warp >= 8 ? HB / 2 : 0) : h + (warp >= 8 ? HB : 0);
        };
        float acc[HB] = {};   // (in registers: no index but constants; `sum`, which the epilogue walks, is in local memory)
#pragma unroll 1
        for (int c = 0; c < sets; ++c) {
          const int set = n * sets + c;
          if (!filled(set)) return -1;
          if (k0 + c / p.segments < p.kblocks) {   // (a last split's missing stages)
#pragma unroll
            for (int h = 0; h < HB; h += 32) {
              uint32_t r[16], s[16];
              tmem_ld_async(lanes + (set & 1) * BN + col(h), r);
              tmem_ld_async(lanes + (set & 1) * BN + col(h + 16), s);
              tmem_wait(r);
              tmem_wait(s);
#pragma unroll
              for (int j = 0; j < 16; ++j) {
                acc[h + j] += __uint_as_float(r[j]);
                acc[h + 16 + j] += __uint_as_float(s[j]);
              }
            }
          }
          free(set);
        }
#pragma unroll
        for (int i = 0; i < HB; ++i) sum[i] = acc[i];
        return 0;
      }
    };
    auto release = [&](int n) {
      if (!PARTS) free(n);
    };
    if constexpr (PARTS) epilogue_tiles<GATED, true, BN, true>(p, maps, turn, tmem, pair, pairs, rank, warp, lane, wait, release);
    else if (p.e.type == VERACE_F32)
      epilogue_tiles<GATED, true, BN, false>(p, maps, turn, tmem, pair, pairs, rank, warp, lane, wait, release);
    else epilogue_tiles<GATED, false, BN, false>(p, maps, turn, tmem, pair, pairs, rank, warp, lane, wait, release);
  }
  tc::fence_before_sync();
  __syncthreads();
  cluster_sync();
  tc::fence_after_sync();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(COLS) : "memory");
}

// ------------------------------------------------------------------ host
template <bool F8, bool AMN, bool BMN, bool GATED, int BN, bool PARTS = false>
int launch(const Product& p, int splits, cudaStream_t st) {
  using S = Shape<BN>;
  constexpr int TN = GATED ? BN / 2 : BN;
  Maps maps;
  int rc;
  if ((rc = operand_map(&maps.a, p.a, p.type, AMN ? 64 : 128))) return rc;
  for (int i = 0; i < 2; ++i)
    if ((rc = operand_map(&maps.b[i], p.b[p.b[i].p ? i : 0], p.type, BMN ? 64 : BN / 2))) return rc;
  Args a{};
  a.M = p.M; a.N = p.N;
  a.e = p.e;
  a.partial = p.M * p.N;
  if (splits > 1) {
    Epilogue e{};
    e.ld = p.N; e.type = VERACE_F32; e.act = VERACE_ACT_NONE;
    if (GATED) {
      e.pre = static_cast<float*>(p.ws);
      e.pre_up = e.pre + splits * a.partial;
    } else {
      e.out = p.ws;
    }
    a.e = e;
  }
  // the outputs' maps (of splits: one, over all partial outputs)
  const int outs = splits > 1 ? 1 : p.nz, planes = splits > 1 ? splits * p.nz : 1;
  void* const out[2] = {outs > 1 ? p.out_z[0] : a.e.out, outs > 1 ? p.out_z[1] : nullptr};
  auto aligned = [&](const void* q, int type) { return q && (size_t)q % 16 == 0 && a.e.ld * size_of(type) % 16 == 0; };
  a.by_tma = aligned(out[0], a.e.type) && (outs == 1 || aligned(out[1], a.e.type));
  a.pre_by_tma = aligned(a.e.pre, VERACE_F32) && (!GATED || aligned(a.e.pre_up, VERACE_F32));
  for (int i = 0; i < outs && a.by_tma; ++i)
    if ((rc = operand_map(&maps.out[i], Mat{out[i], p.M, p.N, a.e.ld, planes, a.partial}, a.e.type, 32))) return rc;
  for (int i = 0; i < (GATED ? 2 : 1) && a.pre_by_tma; ++i)
    if ((rc = operand_map(&maps.pre[i], Mat{i ? a.e.pre_up : a.e.pre, p.M, p.N, a.e.ld, planes, a.partial}, VERACE_F32, 32)))
      return rc;
  a.kblocks = (int)((p.K + (F8 ? 127 : 63)) / (F8 ? 128 : 64));
  a.segments = p.segments; a.a_first = p.a_first; a.a_step = p.a_step;
  a.nz = p.nz;
  a.tiles_m = (int)((p.M + 255) / 256);
  a.tiles_n = (int)((p.N + TN - 1) / TN);
  a.splits = splits;
  a.per = (a.kblocks + splits - 1) / splits;
  const long long tiles = (long long)a.tiles_m * a.tiles_n * p.nz * splits;
  VERACE_REQUIRE(tiles < 1LL << 30, VERACE_ERR_UNSUPPORTED, "linear: %lld x %lld outputs are too many", p.M, p.N);
  a.tiles = (int)tiles;
  a.idesc = (1u << 4) | (uint32_t)(p.type == VERACE_BF16) << 7 | (uint32_t)(p.type == VERACE_BF16) << 10 |
            (uint32_t)AMN << 15 | (uint32_t)BMN << 16 | (uint32_t)(BN >> 3) << 17 | (uint32_t)(256 >> 4) << 24;
  a.out_z[0] = p.out_z[0]; a.out_z[1] = p.out_z[1];
  auto kern = large_product<F8, AMN, BMN, GATED, BN, PARTS>;
  int dev = 0;
  VERACE_CUDA(cudaGetDevice(&dev));
  static std::atomic<uint64_t> ready{0};      // devices whose limit is raised
  if (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1)) {
    if (PARTS && BN == 256) {     // (where wide_parts could not ask)
      cudaFuncAttributes fa;
      VERACE_CUDA(cudaFuncGetAttributes(&fa, kern));
      VERACE_REQUIRE(fa.numRegs == SPLIT_REGISTERS, VERACE_ERR_UNSUPPORTED, "linear: %d registers where %d are shared out",
                     fa.numRegs, SPLIT_REGISTERS);
    }
    VERACE_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM));
    if (dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int pairs = tiles < 74 ? (int)tiles : 74;
  return launch_after("large_product", kern, dim3(2 * pairs), NT, S::SMEM, st, 2, maps, a);
}

template <int BN>
int by_kind(const Product& p, int s, cudaStream_t st) {
  if (p.parts && p.gated) return launch<false, false, false, true, BN, true>(p, s, st);
  if (p.parts && p.a_mn) return launch<false, true, true, false, BN, true>(p, s, st);
  if (p.parts)
    return p.b_mn ? launch<false, false, true, false, BN, true>(p, s, st) : launch<false, false, false, false, BN, true>(p, s, st);
  if (p.type == VERACE_E4M3)
    return p.gated ? launch<true, false, false, true, BN>(p, s, st) : launch<true, false, false, false, BN>(p, s, st);
  if (p.gated) return launch<false, false, false, true, BN>(p, s, st);
  if (p.a_mn) return launch<false, true, true, false, BN>(p, s, st);
  return p.b_mn ? launch<false, false, true, false, BN>(p, s, st) : launch<false, false, false, false, BN>(p, s, st);
}

// ------------------------------------------------------------------ split K
// The outputs from the partial sums, added in order; four columns a thread.  (`part` is no restricted pointer: the kernel
// before this one still writes there while this one is resident, so these are no loads of constant memory.)
template <bool GATED>
__global__ void __launch_bounds__(256) join_splits(const float* part, int splits, long long partial, long long up,
                                                   Epilogue e, long long M, long long N, long long quads) {
  depend();
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long m = i / quads, c = i % quads * 4;
  if (m >= M) return;
  const int n = (int)min(4LL, N - c);
  float g[4] = {}, u[4] = {}, res[4] = {}, scale[4], add[4], row_scale = 1.f;   // (all on their way together)
  if (e.col_scale) {
    row_scale = e.row_scale[m];
    load4(e.col_scale, c, n, VERACE_F32, scale);
    if (GATED) load4(e.up_scale, c, n, VERACE_F32, add);
  }
  if (!GATED && e.bias) load4(e.bias, c, n, e.bias_type, add);
  if (!GATED && e.residual) load4(e.residual, m * e.ld_res + c, n, e.type, res);
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    float v[4];
    load4(part, s * partial + m * N + c, n, VERACE_F32, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) g[j] += v[j];
    if (GATED) {
      load4(part, up + s * partial + m * N + c, n, VERACE_F32, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] += v[j];
    }
  }
  finish4<GATED>(e, m, c, n, scale, add, row_scale, res, g, u);
}

// Whether the compiler gave the kernels of 256 columns of parts the registers that their warps share out among them; where
// it did not, products of parts run in tiles of 128 columns, which share none out.  (On a machine without a device, where
// nothing is launched, they are taken to be right.)
bool wide_parts() {
  static std::atomic<int> known{0};     // 0: not yet, 1: yes, 2: no
  int k = known.load(std::memory_order_relaxed);
  if (k == 0) {
    const void* kernels[] = {
        (const void*)large_product<false, false, false, true, 256, true>, (const void*)large_product<false, true, true, false, 256, true>,
        (const void*)large_product<false, false, true, false, 256, true>, (const void*)large_product<false, false, false, false, 256, true>};
    k = 1;
    for (const void* f : kernels) {
      cudaFuncAttributes a;
      if (cudaFuncGetAttributes(&a, f) != cudaSuccess) {
        cudaGetLastError();
        return true;
      }
      if (a.numRegs != SPLIT_REGISTERS) k = 2;
    }
    known.store(k, std::memory_order_relaxed);
  }
  return k == 1;
}

// How a product is cut: columns of a tile, and splits of K.  A pair's time in clocks: a step of four MMAs takes 512
// (BN 256) or 400 (BN 128, bound by shared memory: 8 KB for 64 clocks of an MMA), 64 values of parts 3200 or
// 2900, an epilogue about 40 a column (under the next tile's products but for the last), the first operands
// 6000; partial sums are written and read at about 2 KB a clock, and joining them takes another launch (5000).
struct Cut {
  int bn, splits;
};
Cut cut(long long M, long long N, long long K, int segments, int nz, bool gated, int type, bool parts) {
  const long long kblocks = (K + (type == VERACE_E4M3 ? 127 : 63)) / (type == VERACE_E4M3 ? 128 : 64);
  Cut best{256, 1};
  double least = 0;
  const int runs = parts ? 1 : (int)((K * segments + run_of(type) - 1) / run_of(type));   // (64 values of parts are a sum of their own)
  for (int bn = parts && !wide_parts() ? 128 : 256; bn >= 128; bn /= 2) {
    const int tn = gated ? bn / 2 : bn;
    const long long tiles = (M + 255) / 256 * ((N + tn - 1) / tn) * nz;
    for (int s = runs; s == runs || (s <= 16 && s * tiles <= 74 && kblocks >= 8 * s); ++s) {
      const long long stages = (kblocks + s - 1) / s;
      if ((s - 1) * stages >= kblocks) continue;      // (a split would be empty)
      const double per = (double)stages * segments * (parts ? bn == 256 ? 3200 : 2900 : bn == 256 ? 512 : 400), epi = 40. * bn;
      double t = (double)((tiles * s + 73) / 74) * (per > epi ? per : epi) + epi + 6000;
      if (s > 1) t += 5000 + (double)M * N * nz * (gated ? 8 : 4) * 2 * s / 2048;
      if (least == 0 || t < least) least = t, best = Cut{bn, s};
    }
  }
  return best;
}

}  // namespace

namespace lin {

int operand_map(CUtensorMap* map, const Mat& m, int type, int rows) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tmap_encoder();
  VERACE_REQUIRE(enc, VERACE_ERR_CUDA, "linear: the driver has no cuTensorMapEncodeTiled");
  const size_t es = size_of(type);
  const cuuint64_t dims[3] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows, (cuuint64_t)m.pieces};
  const cuuint64_t strides[2] = {m.ld * es, (m.pieces > 1 ? m.piece : m.ld) * es};
  const cuuint32_t box[3] = {(cuuint32_t)(128 / es), (cuuint32_t)rows, 1}, el[3] = {1, 1, 1};
  const CUtensorMapDataType dt = type == VERACE_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                 : type == VERACE_E4M3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                 : type == VERACE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const CUresult r = enc(map, dt, 3, const_cast<void*>(m.p), dims, strides, box, el, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  VERACE_REQUIRE(r == CUDA_SUCCESS, VERACE_ERR_CUDA, "linear: tensor map of %lld x %lld (stride %lld) refused (%d)", m.rows,
                 m.cols, m.ld, (int)r);
  return VERACE_OK;
}

size_t split_bytes(long long M, long long N, long long K, int segments, int nz, bool gated, int type, bool parts) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  const int s = cut(M, N, K, segments, nz, gated, type, parts).splits;
  return s > 1 ? align_up((size_t)M * N * nz * s * (gated ? 8 : 4), 256) : 0;
}

int product_large(const Product& p, cudaStream_t st) {
  const Cut c = cut(p.M, p.N, p.K, p.segments, p.nz, p.gated, p.type, p.parts);
  int rc = c.bn == 256 ? by_kind<256>(p, c.splits, st) : by_kind<128>(p, c.splits, st);
  if (rc || c.splits == 1) return rc;
  const long long quads = (p.N + 3) / 4, blocks = (p.M * quads + 255) / 256, one = p.M * p.N;
  for (int z = 0; z < p.nz; ++z) {
    Epilogue e = p.e;
    if (p.nz > 1) e.out = p.out_z[z];
    const float* part = static_cast<const float*>(p.ws) + z * one;
    rc = p.gated ? launch_after("join_splits", join_splits<true>, dim3((unsigned)blocks), 256, 0, st, 1, part, c.splits, one,
                                c.splits * one, e, (long long)p.M, (long long)p.N, quads)
                 : launch_after("join_splits", join_splits<false>, dim3((unsigned)blocks), 256, 0, st, 1, part, c.splits,
                                p.nz * one, 0LL, e, (long long)p.M, (long long)p.N, quads);
    if (rc) return rc;
  }
  return VERACE_OK;
}

}  // namespace lin

int linear_read_status(int* status) {
  int h = 0;
  VERACE_CUDA(cudaMemcpyFromSymbol(&h, g_linear_status, sizeof(int)));
  if (h) {
    const int zero = 0;
    VERACE_CUDA(cudaMemcpyToSymbol(g_linear_status, &zero, sizeof(int)));
  }
  *status = h;
  return VERACE_OK;
}

}  // namespace verace
