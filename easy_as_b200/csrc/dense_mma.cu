// dense_mma.cu — the dense layers' matrix products on tcgen05 (sm_100a).
//
// Operands are 16-bit matrices in either order: K-major (the contraction index is contiguous: x
// and W of the forward products) or MN-major (the output's index is: W in dx = dz W, both operands
// in dW = dz^T x).  TMA stages 64-deep k-blocks with 128-byte swizzle, the matrix instruction
// reads either order through its descriptors, and TMA fills what lies outside a matrix with
// zeros, so no size has to be a multiple of anything.
//
// A gated block is one product whose B tile is half gate rows and half up rows: the accumulator
// then holds g and u of the same outputs side by side in one row of TMEM, and the epilogue of one
// thread has both.  dx of a gated block is one product of two terms, whose k-blocks follow one
// another into the same accumulator.
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "dense_internal.h"
#include "dense_launch.h"
#include "dense_math.cuh"
#include "eas_internal.h"
#include "tcgen05_ptx.cuh"

namespace {

using namespace tc;
using namespace dense;

constexpr int kBK = 64;  // one 128-byte swizzle row

enum Mode { kForward = 0, kGatedForward = 1, kBackward = 2 };

// One product of a launch.
struct alignas(64) Job {
  CUtensorMap a[2], b[2], y[2];
  uint16_t* y_ptr[2];
  int64_t ldy[2];
  int M, N;
  int kb_term;         // k-blocks of one term
  int kb_total;        // of all terms
  int mt, nt, tiles;   // tiles along M and N, and in all
  int group;           // M tiles that are walked together
  int split;           // CTAs of a cluster that share a tile's k-blocks
  bool batch2, y_tma, a_mn;
};

struct alignas(64) Params {
  Job job[2];
  CUtensorMap pre, pre2;
  const uint16_t* bias;
  const uint16_t* residual;
  const float* unscale;
  uint16_t* pre_ptr;
  uint16_t* pre2_ptr;
  int64_t ldr, ldp, ldp2;
  int tiles;   // of all jobs
  int cluster; // CTAs per cluster: the largest split
  int ctas0;   // CTAs of job 0's tiles, and of all tiles (whole clusters each)
  int ctas;
  int ratio;   // tiles of job 1 that take as long as one of job 0
  int act;
  bool bf16, pre_tma, pre2_tma, bias_vec, res_vec;
  DenseColSum sums;
  int* status;
};

// The producer and MMA warps run their loops whole, one elected lane issuing: every address and
// descriptor is then uniform over the warp and stays in uniform registers, which these
// instructions want.  (Issued from a branch of one lane they came from vector registers, and a
// k-block took 566 cycles to issue whatever its tile: 300 ns per k-block, above the 270 ns that
// a 256 x 256 x 64 pair k-block computes.)
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int x,
                                                 int y) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
      "%4}], [%2];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y)
      : "memory");
}

__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar),
      "r"(bytes)
      : "memory");
}

// Arrive on `bar` when the MMAs issued so far are done; CG = 2: in both CTAs of the pair.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::
            "r"(bar),
        "h"((uint16_t)3)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
        : "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// Instruction descriptor, kind::f16: D = f32 (bits 4-5 = 1), A and B formats at bits 7-9 and 10-12
// (f16 0, bf16 1), A and B major at bits 15 and 16 (1 = MN), N >> 3 at bits 17-22, M >> 4 at 24-28.
__device__ __forceinline__ uint32_t instr_desc(int m, int n, bool a_mn, bool b_mn, bool bf16) {
  return (1u << 4) | (bf16 ? (1u << 7) | (1u << 10) : 0u) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Descriptor of a staged k-block.  K-major: rows of 128 bytes, 8 rows per swizzle atom; a step of
// 16 is 32 bytes along the row.  MN-major: 64 k-rows of 64 elements (128 bytes) per 64-wide piece,
// the next piece kBK * 128 bytes on; a step is 16 rows.  Descriptors count in 16-byte units.
template <bool MN>
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return MN ? smem_desc(addr, kBK * 128, 1024) : smem_desc(addr, 16, 1024);
}
template <bool MN>
constexpr int kStep = MN ? 2048 / 16 : 32 / 16;

// The four 16-deep MMAs of a k-block; the first overwrites D unless `accumulate`.
#define EAS_MMA_KBLOCK(GROUP)                                                                            \
  asm volatile(                                                                                          \
      "{\n\t.reg .pred e, p, t;\n\t.reg .b64 a, b;\n\t"                                                  \
      "elect.sync _|e, 0xffffffff;\n\t"                                                                  \
      "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 t, 0, 0;\n\t"                                                \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], %1, %2, %3, p;\n\t"                           \
      "add.s64 a, %1, %5;\n\tadd.s64 b, %2, %6;\n\t"                                                     \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], a, b, %3, t;\n\t"                             \
      "add.s64 a, a, %5;\n\tadd.s64 b, b, %6;\n\t"                                                       \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], a, b, %3, t;\n\t"                             \
      "add.s64 a, a, %5;\n\tadd.s64 b, b, %6;\n\t"                                                       \
      "@e tcgen05.mma.cta_group::" GROUP ".kind::f16 [%0], a, b, %3, t;\n\t}" ::"r"(d),                  \
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "l"(a_step), "n"(kStep<B_MN>)                   \
      : "memory")

template <int CG, bool B_MN>
__device__ __forceinline__ void mma_kblock(uint32_t d, uint64_t a_desc, uint64_t a_step, uint64_t b_desc,
                                           uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 2)
    EAS_MMA_KBLOCK("2");
  else
    EAS_MMA_KBLOCK("1");
}
#undef EAS_MMA_KBLOCK

// A whole warp's bounded wait (tc::mbar_wait is one thread's): the same answer in every lane, so
// that the warp leaves its loop together when a wait expires.
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  auto done = [&]() {
    return __all_sync(0xffffffffu, CLUSTER ? mbar_try_wait_cl(smem_u32(bar), parity) : mbar_try_wait(bar, parity));
  };
  if (done()) return true;
  const long long t0 = clock64();
  while (!done()) {
    const bool expired = clock64() - t0 > kWaitBudget;
    if (__any_sync(0xffffffffu, expired || *abort_flag)) {
      *abort_flag = 1;
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ bool going(volatile int* abort_flag) { return !__any_sync(0xffffffffu, *abort_flag); }

// After an expired wait: copies in flight land before the CTA's shared memory is given up.
__device__ __forceinline__ void settle() {
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000) {
  }
  __syncwarp();
}

// ---------------------------------------------------------------------------
// epilogue: 32 rows x 32 columns per warp at a time
// ---------------------------------------------------------------------------
//
// Each lane holds one row of 32 f32 columns from TMEM.  Results go through a 2 KB box of the warp
// (64-byte swizzle: 16-byte chunk j of row r lies at chunk j ^ (r / 2 & 3)) and leave by a TMA
// store, which clips at the matrix's edges; arrays whose base or pitch TMA cannot take are written
// from the box row by row, 32 neighbouring columns at a time.  Two boxes per warp take turns.

struct Boxes {
  uint8_t* base;
  int n;
};

constexpr int kBoxBytes = 32 * 64;

__device__ __forceinline__ uint8_t* box_chunk(uint8_t* box, int row, int chunk) {
  return box + row * 64 + ((chunk ^ ((row >> 1) & 3)) << 4);
}

// A lane's column of a box: its place in a row takes four values, by row.
struct ColumnInBox {
  uint8_t* base[4];
  __device__ __forceinline__ ColumnInBox(uint8_t* box, int lane) {
#pragma unroll
    for (int k = 0; k < 4; ++k) base[k] = box + (((lane >> 3) ^ k) << 4) + (lane & 7) * 2;
  }
  __device__ __forceinline__ uint16_t* at(int row) const {  // row known at compile time
    return reinterpret_cast<uint16_t*>(base[(row >> 1) & 3] + row * 64);
  }
};

__device__ __forceinline__ uint8_t* next_box(Boxes& bx, int lane) {
  uint8_t* box = bx.base + (bx.n & 1) * kBoxBytes;
  ++bx.n;
  if (lane == 0) bulk_wait_read1();  // the store that last used this box has read it
  __syncwarp();
  return box;
}

template <bool BF16>
__device__ __forceinline__ void put(Boxes& bx, int lane, const CUtensorMap* map, bool tma, uint16_t* ptr, int64_t ld,
                                    int M, int N, int m0, int n0, const float (&v)[32]) {
  uint8_t* box = next_box(bx, lane);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    *reinterpret_cast<uint4*>(box_chunk(box, lane, j)) =
        make_uint4(pack2<BF16>(v[8 * j], v[8 * j + 1]), pack2<BF16>(v[8 * j + 2], v[8 * j + 3]),
                   pack2<BF16>(v[8 * j + 4], v[8 * j + 5]), pack2<BF16>(v[8 * j + 6], v[8 * j + 7]));
  if (tma) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncwarp();
    if (lane == 0) tma_store_2d(map, box, n0, m0);
  } else {
    __syncwarp();
    const int rows = min(32, M - m0);
    if (n0 + lane < N) {
      uint16_t* dst = ptr + (int64_t)m0 * ld + n0 + lane;
      const ColumnInBox col(box, lane);
      if (rows == 32) {
#pragma unroll
        for (int r = 0; r < 32; ++r, dst += ld) *dst = *col.at(r);
      } else {
#pragma unroll
        for (int r = 0; r < 32; ++r, dst += ld)
          if (r < rows) *dst = *col.at(r);
      }
    }
  }
  if (lane == 0) bulk_commit();  // an empty group where nothing was stored: the boxes' turns count groups
}

// v += the residual's 32 x 32 piece
template <bool BF16>
__device__ __forceinline__ void add_residual(const Params& p, Boxes& bx, int lane, int m0, int n0, float (&v)[32]) {
  const int M = p.job[0].M, N = p.job[0].N;
  uint4 w[4];
  if (p.res_vec && n0 + 32 <= N) {
    const int m = min(m0 + lane, M - 1);  // rows past the last are not stored
    const uint4* src = reinterpret_cast<const uint4*>(p.residual + (int64_t)m * p.ldr + n0);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = src[j];
  } else {
    uint8_t* box = next_box(bx, lane);
    const int rows = n0 + lane < N ? min(32, M - m0) : 0;
    const uint16_t* src = p.residual + (int64_t)m0 * p.ldr + n0 + lane;
    const ColumnInBox col(box, lane);
#pragma unroll
    for (int r0 = 0; r0 < 32; r0 += 16) {  // 16 loads under way
      uint16_t h[16];
#pragma unroll
      for (int r = 0; r < 16; ++r, src += p.ldr) h[r] = r0 + r < rows ? *src : (uint16_t)0;
#pragma unroll
      for (int r = 0; r < 16; ++r) *col.at(r0 + r) = h[r];
    }
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const uint4*>(box_chunk(box, lane, j));
    if (lane == 0) bulk_commit();
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t q[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float lo, hi;
      unpack2<BF16>(q[i], lo, hi);
      v[8 * j + 2 * i] += lo;
      v[8 * j + 2 * i + 1] += hi;
    }
  }
}

template <bool BF16>
__device__ __forceinline__ void add_bias(const Params& p, int n0, float (&v)[32]) {
  const int N = p.job[0].N;
  if (p.bias_vec && n0 + 32 <= N) {
    const uint4* src = reinterpret_cast<const uint4*>(p.bias + n0);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint4 w = src[j];
      const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo, hi;
        unpack2<BF16>(q[i], lo, hi);
        v[8 * j + 2 * i] += lo;
        v[8 * j + 2 * i + 1] += hi;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (n0 + j < N) v[j] += to_f32<BF16>(p.bias[n0 + j]);
  }
}

// Finish 32 x 32 results of a job from their sums: v = z, or v = g and u.
template <int MODE, bool BF16>
__device__ __forceinline__ void finish_as(const Params& p, const Job& jb, Boxes& bx, int lane, int z, int m0, int n0,
                                          float (&v)[32], const float (&u)[MODE == kGatedForward ? 32 : 1]) {
  constexpr bool GATED = MODE == kGatedForward;
  if constexpr (MODE != kBackward) {
    if (!GATED && p.bias) add_bias<BF16>(p, n0, v);
    if (p.pre_ptr) put<BF16>(bx, lane, &p.pre, p.pre_tma, p.pre_ptr, p.ldp, jb.M, jb.N, m0, n0, v);
    if constexpr (GATED) {
      if (p.pre2_ptr) put<BF16>(bx, lane, &p.pre2, p.pre2_tma, p.pre2_ptr, p.ldp2, jb.M, jb.N, m0, n0, u);
    }
    with_act(p.act, [&](auto a) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        v[j] = act<decltype(a)::value>(v[j]);
        if constexpr (GATED) v[j] *= u[j];
      }
    });
    if (!GATED && p.residual) add_residual<BF16>(p, bx, lane, m0, n0, v);
  } else if (!BF16 && p.unscale) {
    const float s = *p.unscale;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= s;
  }
  put<BF16>(bx, lane, &jb.y[z], jb.y_tma, jb.y_ptr[z], jb.ldy[z], jb.M, jb.N, m0, n0, v);
}

template <int MODE>
__device__ __forceinline__ void finish(const Params& p, const Job& jb, Boxes& bx, int lane, int z, int m0, int n0,
                                       float (&v)[32], const float (&u)[MODE == kGatedForward ? 32 : 1]) {
  if (p.bf16)
    finish_as<MODE, true>(p, jb, bx, lane, z, m0, n0, v, u);
  else
    finish_as<MODE, false>(p, jb, bx, lane, z, m0, n0, v, u);
}

__device__ __forceinline__ void as_floats(const uint32_t (&r)[32], float (&v)[32]) {
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
}

struct Tile {
  int j, z, m, n;
};

// Tile t of all jobs' tiles.  Within a job they go in groups along M, so that the tiles in flight share
// operands in L2.
template <int MODE>
__device__ __forceinline__ Tile tile_at(const Params& p, int t) {
  Tile c;
  c.j = MODE == kBackward && t >= p.job[0].tiles ? 1 : 0;
  if (c.j) t -= p.job[0].tiles;
  const Job& jb = p.job[c.j];
  const int per_z = jb.mt * jb.nt;
  c.z = t / per_z;
  const int r = t - c.z * per_z;
  const int g = r / (jb.group * jb.nt);
  const int first = g * jb.group;
  const int size = min(jb.group, jb.mt - first);
  const int rr = r - g * jb.group * jb.nt;
  c.m = first + rr % size;
  c.n = rr / size;
  return c;
}

// The i-th tile of pair `cid` of `pairs` (past the last: -1).  One job: every pair in turn.  Two jobs: job 0
// is done in turn, and where its last round does not reach all pairs, the others take `ratio` tiles of
// job 1 meanwhile; then job 1 goes in turn.  (dx of 4096 x 8192 x 4096 has 256 tiles for 74 pairs: alone
// its fourth round leaves 40 of them idle.)
template <int MODE>
__device__ __forceinline__ int pair_tile(const Params& p, int i, int cid, int pairs) {
  if (MODE != kBackward || p.tiles == p.job[0].tiles) {
    const int64_t t = (int64_t)i * pairs + cid;
    return t < p.tiles ? (int)t : -1;
  }
  const int t0 = p.job[0].tiles, t1 = p.job[1].tiles;
  const int full = t0 / pairs, rest = t0 - full * pairs;
  const int mine = full + (cid < rest ? 1 : 0);
  if (i < mine) return i * pairs + cid;
  i -= mine;
  int64_t t;
  const int extra = rest ? p.ratio : 0;
  if (cid >= rest && i < extra) {
    t = (int64_t)i * (pairs - rest) + (cid - rest);
  } else {
    if (cid >= rest) i -= extra;
    t = (int64_t)extra * (pairs - rest) + (int64_t)i * pairs + cid;
  }
  return t < t1 ? t0 + (int)t : -1;
}

// ---------------------------------------------------------------------------
// CTA-pair kernel: 256 x 256 tiles, two accumulators
// ---------------------------------------------------------------------------
//
// A cluster of two CTAs, tcgen05.mma.cta_group::2 of M = 256, N = 256.  Each CTA stages its 128
// rows of A and 128 of the tile's 256 B rows (gated: CTA 0 the gate's, CTA 1 the up projection's);
// the leader issues the MMAs, and each CTA's TMEM receives its 128 rows of all 256 columns.  Two
// accumulators take turns, so the epilogue of one tile runs under the main loop of the next.
//   warp 0 TMA producer, warp 1 TMEM and (leader) MMA issue, warps 2-9 epilogue: two per TMEM
//   quarter, one for each half of the columns.
constexpr int kPairThreads = 320;
constexpr int kPairStages = 6;
constexpr int kPairStageBytes = 2 * 128 * kBK * 2;
constexpr int kPairBoxes = kPairStages * kPairStageBytes;
constexpr int kPairBars = kPairBoxes + 8 * 2 * kBoxBytes;
constexpr int kPairSmem = kPairBars + (2 * kPairStages + 4) * 8 + 16 + 1024;
static_assert(kPairSmem <= 232448, "shared memory over the 227 KB per-CTA limit");

template <int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    dense_pair_kernel(const __grid_constant__ Params p) {
  constexpr bool GATED = MODE == kGatedForward, B_MN = MODE == kBackward;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + kPairBars);
  uint64_t* empty = full + kPairStages;
  uint64_t* acc_full = empty + kPairStages;
  uint64_t* acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);  // uniform
  const int lane = threadIdx.x & 31;
  uint32_t rank;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));

  if (threadIdx.x == 0) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(&full[s], 1);  // armed by the leader with both CTAs' bytes (the leader's copy is used)
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 16);  // 8 epilogue warps x 2 CTAs (the leader's copy is used)
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    prefetch_map(&p.job[0].a[0]);
    prefetch_map(&p.job[0].b[0]);
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the peer's barriers are initialised before anyone signals them
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_order();

  const int cid = blockIdx.x >> 1, ncl = gridDim.x >> 1;
  const int kTileN = GATED ? 128 : 256;

  const uint32_t ring = smem_u32(smem), full0 = smem_u32(full), empty0 = smem_u32(empty);

  if (warp == 0) {
    const uint32_t leader_full = mapa_rank(full0, 0);
    int s = 0;
    uint32_t ph = 0;
    for (int i = 0; going(abort_flag); ++i) {
      const int t = pair_tile<MODE>(p, i, cid, ncl);
      if (t < 0) break;
      const Tile c = tile_at<MODE>(p, t);
      const Job& jb = p.job[c.j];
      const bool a_mn = MODE == kBackward && jb.a_mn;
      const int m0 = c.m * 256 + 128 * (int)rank;
      const int n0 = c.n * kTileN + (GATED ? 0 : 128 * (int)rank);
      int term = 0, k0 = 0;
      for (int kb = 0; kb < jb.kb_total; ++kb) {
        if (!warp_wait(&empty[s], ph ^ 1, abort_flag)) break;
        if (kb == jb.kb_term) term = 1, k0 = 0;
        const CUtensorMap* ma = &jb.a[jb.batch2 ? c.z : term];
        const CUtensorMap* mb = &jb.b[GATED ? (int)rank : term];
        const uint32_t fl = leader_full + s * 8;
        if (rank == 0) expect_tx(full0 + s * 8, 2 * kPairStageBytes);
        const uint32_t sa = ring + s * kPairStageBytes, sb = sa + 128 * kBK * 2;
        if (a_mn) {
          tma_load_2d_pair(sa, ma, fl, m0, k0);
          tma_load_2d_pair(sa + kBK * 128, ma, fl, m0 + 64, k0);
        } else {
          tma_load_2d_pair(sa, ma, fl, k0, m0);
        }
        if (B_MN) {
          tma_load_2d_pair(sb, mb, fl, n0, k0);
          tma_load_2d_pair(sb + kBK * 128, mb, fl, n0 + 64, k0);
        } else {
          tma_load_2d_pair(sb, mb, fl, k0, n0);
        }
        k0 += kBK;
        if (++s == kPairStages) {
          s = 0;
          ph ^= 1;
        }
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint64_t b0 = operand_desc<B_MN>(ring + 128 * kBK * 2);
      int s = 0;
      uint32_t ph = 0;
      for (int i = 0; going(abort_flag); ++i) {
        const int t = pair_tile<MODE>(p, i, cid, ncl);
        if (t < 0) break;
        const Job& jb = p.job[MODE == kBackward && t >= p.job[0].tiles ? 1 : 0];
        const bool a_mn = MODE == kBackward && jb.a_mn;
        const uint32_t idesc = instr_desc(256, 256, a_mn, B_MN, p.bf16);
        const uint64_t a0 = a_mn ? operand_desc<true>(ring) : operand_desc<false>(ring);
        const uint64_t a_step = a_mn ? kStep<true> : kStep<false>;
        const int buf = i & 1;
        if (!warp_wait<true>(&acc_empty[buf], ((i >> 1) & 1) ^ 1, abort_flag)) break;
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        bool ok = true;
        for (int kb = 0; kb < jb.kb_total; ++kb) {
          if (!warp_wait(&full[s], ph, abort_flag)) {
            ok = false;
            break;
          }
          const uint64_t at = (uint64_t)(s * (kPairStageBytes / 16));
          mma_kblock<2, B_MN>(d, a0 + at, a_step, b0 + at, idesc, kb);
          commit<2>(empty0 + s * 8);
          if (++s == kPairStages) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!ok) break;
        commit<2>(smem_u32(&acc_full[buf]));
      }
    }
  } else {
    const int q = warp & 3, half = (warp - 2) >> 2;
    Boxes bx = {smem + kPairBoxes + (warp - 2) * 2 * kBoxBytes, 0};
    const uint32_t leader[2] = {mapa_rank(smem_u32(&acc_empty[0]), 0), mapa_rank(smem_u32(&acc_empty[1]), 0)};
    for (int i = 0; going(abort_flag); ++i) {
      const int t = pair_tile<MODE>(p, i, cid, ncl);
      if (t < 0) break;
      const int buf = i & 1;
      if (!warp_wait(&acc_full[buf], (i >> 1) & 1, abort_flag)) break;
      tc_fence_after();
      const Tile c = tile_at<MODE>(p, t);
      const Job& jb = p.job[c.j];
      const int m0 = c.m * 256 + 128 * (int)rank + q * 32;
      const uint32_t acc = tmem + buf * 256 + ((uint32_t)(q * 32) << 16);
      constexpr int kCols = GATED ? 64 : 128;  // of this warp
      if (m0 < jb.M) {
#pragma unroll 1
        for (int cc = 0; cc < kCols; cc += 32) {
          const int col = half * kCols + cc, n0 = c.n * kTileN + col;
          if (n0 >= jb.N) break;
          uint32_t r[32];
          float v[32], u[GATED ? 32 : 1];
          tmem_ld32(acc + col, r);
          as_floats(r, v);
          if constexpr (GATED) {
            tmem_ld32(acc + 128 + col, r);
            as_floats(r, u);
          }
          finish<MODE>(p, jb, bx, lane, c.z, m0, n0, v, u);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader[buf]) : "memory");
    }
    if (lane == 0) bulk_wait_all0();  // the stores are done before the CTA's shared memory goes away
  }

  __syncwarp();
  if (*abort_flag) settle();
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the pair leaves together: no MMA still targets the peer's TMEM
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) *p.status = EAS_ERR_TIMEOUT;
}

// ---------------------------------------------------------------------------
// single-CTA kernel: 128 x BN tiles, K split over a cluster
// ---------------------------------------------------------------------------
//
// For outputs of too few 256 x 256 tiles.  One tile per cluster of S CTAs (S = 1, 2, 4, 8), each
// with its share of the k-blocks; two CTAs fit on an SM, so one's epilogue runs beside the
// other's main loop.  With S > 1 every CTA leaves its f32 sums in shared memory (column-major, over
// the ring, which is idle by then), and the cluster's warps share out the 32 x 32 pieces: a piece is
// summed over the CTAs in their order, through distributed shared memory, and finished.  No
// workspace, no atomics: the same bits on every run.
//   warp 0 TMA producer, warp 1 TMEM and MMA issue, warps 2-5 epilogue (one per TMEM quarter).
//
// Shapes: AR rows of A are staged (64 when the matrix has no more: the MMA then reads the rows
// behind them too, whatever they hold, into accumulator rows that nobody looks at).  DEEP rings
// take the whole SM, for launches of no more CTAs than SMs; else two CTAs share one.
constexpr int kTileThreads = 192;
template <int BN, int AR, bool DEEP>
struct TileShape {
  static constexpr int kABytes = AR * kBK * 2;
  static constexpr int kStageBytes = kABytes + BN * kBK * 2;
  static constexpr int kStages = (DEEP ? 196608 : 98304) / kStageBytes;
  static constexpr int kRing = kStages * kStageBytes;
  static constexpr int kOver = 128 * kBK * 2 > kStageBytes ? 128 * kBK * 2 - kStageBytes : 0;  // read past the ring
  static constexpr int kBoxes = 128 * BN * 4;  // after the partial sums, over the ring
  static constexpr int kBars = kRing + kOver;
  static constexpr int kSmem = kBars + (2 * kStages + 1) * 8 + 16 + 1024;
  static_assert(kBoxes + 4 * 2 * kBoxBytes <= kRing, "partial sums and boxes lie over the ring");
  static_assert(kSmem <= (DEEP ? 232448 : 115000), "shared memory");
};

// db of 32 columns from n0 on: each row of threads adds every 48th row, then the rows of threads
// are added in order.  `sums`: 48 x 33 floats.
template <bool BF16>
__device__ __forceinline__ void column_sums_of_matrix(const DenseColSum& c, int n0, float* sums) {
  constexpr int kRows = kTileThreads / 4;  // 4 threads of 8 columns per row
  const int tx = threadIdx.x & 3, ty = threadIdx.x >> 2, n = n0 + 8 * tx;
  float s[8] = {};
  if (n < c.N) {
    const uint16_t* end = c.matrix + (int64_t)(c.rows - 1) * c.ld + c.N;
#pragma unroll 4
    for (int r = ty; r < c.rows; r += kRows) {
      Gather8 from;
      from.fetch(c.matrix + (int64_t)r * c.ld + n, c.N - n, c.matrix, end);
      const uint4 w = from.get();
      float v[8];
      unpack2<BF16>(w.x, v[0], v[1]);
      unpack2<BF16>(w.y, v[2], v[3]);
      unpack2<BF16>(w.z, v[4], v[5]);
      unpack2<BF16>(w.w, v[6], v[7]);
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[ty * 33 + 8 * tx + j] = s[j];
  __syncthreads();
  const int col = threadIdx.x;
  if (col >= 32 || n0 + col >= c.N) return;
  float total = 0;
  for (int r = 0; r < kRows; ++r) total += sums[r * 33 + col];
  c.db[n0 + col] = to_16<BF16>(total);
}

__device__ __forceinline__ void column_sums(const DenseColSum& c, int n0, float* sums) {
  if (c.matrix) {
    if (c.bf16)
      column_sums_of_matrix<true>(c, n0, sums);
    else
      column_sums_of_matrix<false>(c, n0, sums);
    return;
  }
  constexpr int kRows = kTileThreads / 32;
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, n = n0 + tx;
  float s = 0;
  if (n < c.N) {
#pragma unroll 8
    for (int b = ty; b < c.rows; b += kRows) s += c.partial[(int64_t)b * c.N + n];
  }
  sums[ty * 32 + tx] = s;
  __syncthreads();
  if (ty || n >= c.N) return;
#pragma unroll
  for (int r = 1; r < kRows; ++r) s += sums[r * 32 + tx];
  c.db[n] = c.bf16 ? to_16<true>(s) : to_16<false>(s);
}

__global__ void __launch_bounds__(kTileThreads) column_sums_kernel(const __grid_constant__ DenseColSum c) {
  __shared__ float sums[48 * 33];
  grid_order();
  column_sums(c, blockIdx.x * 32, sums);
}

template <int BN, int AR, bool DEEP, int MODE>
__global__ void __launch_bounds__(kTileThreads, DEEP ? 1 : 2) dense_tile_kernel(const __grid_constant__ Params p) {
  constexpr bool GATED = MODE == kGatedForward, B_MN = MODE == kBackward;
  using L = TileShape<BN, AR, DEEP>;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + L::kStages;
  uint64_t* acc_full = empty + L::kStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);  // uniform
  const int lane = threadIdx.x & 31;
  if (MODE == kBackward && (int)blockIdx.x >= p.ctas) {  // CTAs behind the tiles': column sums
    grid_order();
    column_sums(p.sums, ((int)blockIdx.x - p.ctas) * 32, reinterpret_cast<float*>(smem));
    return;
  }
  const int second = MODE == kBackward && (int)blockIdx.x >= p.ctas0 ? 1 : 0;
  const int block = (int)blockIdx.x - second * p.ctas0;
  const int S = p.job[second].split;
  const int rank = block % S;  // consecutive blocks form a cluster, and share tiles by S
  if (MODE == kBackward && block / S >= p.job[second].tiles) {  // fills up the job's last cluster
    grid_order();
    if (S > 1) {  // the barriers of the CTAs that work
      cluster_sync_all();
      cluster_sync_all();
    }
    return;
  }

  constexpr int kTileN = GATED ? BN / 2 : BN;
  const Tile c = tile_at<MODE>(p, second * p.job[0].tiles + block / S);
  const Job& jb = p.job[c.j];
  const bool a_mn = MODE == kBackward && jb.a_mn;  // (only with AR = 128: it comes in 64-wide pieces of all rows)

  if (threadIdx.x == 32) {
    prefetch_map(&jb.a[jb.batch2 ? c.z : 0]);
    prefetch_map(&jb.b[0]);
    if (GATED) prefetch_map(&jb.b[1]);
  }
  if (threadIdx.x == 0) {
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(acc_full, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    __syncwarp();  // its first lane was elsewhere
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "n"(BN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  grid_order();

  const int m0 = c.m * 128, n0 = c.n * kTileN;
  const int kb_lo = (int)((int64_t)rank * jb.kb_total / S), kb_hi = (int)((int64_t)(rank + 1) * jb.kb_total / S);

  const uint32_t ring = smem_u32(smem), full0 = smem_u32(full), empty0 = smem_u32(empty);

  if (warp == 0) {
    int s = 0;
    uint32_t ph = 0;
    for (int kb = kb_lo; kb < kb_hi; ++kb) {
      if (!warp_wait(&empty[s], ph ^ 1, abort_flag)) break;
      const uint32_t fl = full0 + s * 8;
      expect_tx(fl, L::kStageBytes);
      const int term = kb >= jb.kb_term ? 1 : 0;
      const int k0 = (kb - term * jb.kb_term) * kBK;
      const CUtensorMap* ma = &jb.a[jb.batch2 ? c.z : term];
      const uint32_t sa = ring + s * L::kStageBytes, sb = sa + L::kABytes;
      if (a_mn) {
        tma_load_2d(sa, ma, fl, m0, k0);
        tma_load_2d(sa + kBK * 128, ma, fl, m0 + 64, k0);
      } else {
        tma_load_2d(sa, ma, fl, k0, m0);
      }
      if (GATED) {
        tma_load_2d(sb, &jb.b[0], fl, k0, n0);
        tma_load_2d(sb + kTileN * 128, &jb.b[1], fl, k0, n0);
      } else if (B_MN) {
#pragma unroll
        for (int j = 0; j < BN / 64; ++j) tma_load_2d(sb + j * kBK * 128, &jb.b[term], fl, n0 + 64 * j, k0);
      } else {
        tma_load_2d(sb, &jb.b[term], fl, k0, n0);
      }
      if (++s == L::kStages) {
        s = 0;
        ph ^= 1;
      }
    }
  } else if (warp == 1) {
    const uint32_t idesc = instr_desc(128, BN, a_mn, B_MN, p.bf16);
    const uint64_t a0 = a_mn ? operand_desc<true>(ring) : operand_desc<false>(ring);
    const uint64_t a_step = a_mn ? kStep<true> : kStep<false>;
    const uint64_t b0 = operand_desc<B_MN>(ring + L::kABytes);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb_lo; kb < kb_hi; ++kb) {
      if (!warp_wait(&full[s], ph, abort_flag)) {
        ok = false;
        break;
      }
      const uint64_t at = (uint64_t)(s * (L::kStageBytes / 16));
      mma_kblock<1, B_MN>(tmem, a0 + at, a_step, b0 + at, idesc, kb - kb_lo);
      commit<1>(empty0 + s * 8);
      if (++s == L::kStages) {
        s = 0;
        ph ^= 1;
      }
    }
    if (ok) commit<1>(smem_u32(acc_full));
  } else if (warp_wait(acc_full, 0, abort_flag)) {
    // every MMA has read its operands: the ring is free
    tc_fence_after();
    const int q = warp & 3;
    const uint32_t acc = tmem + ((uint32_t)(q * 32) << 16);
    if (S == 1) {
      Boxes bx = {smem + L::kBoxes + q * 2 * kBoxBytes, 0};
      if (m0 + q * 32 < jb.M) {
#pragma unroll 1
        for (int cc = 0; cc < kTileN && n0 + cc < jb.N; cc += 32) {
          uint32_t r[32];
          float v[32], u[GATED ? 32 : 1];
          tmem_ld32(acc + cc, r);
          as_floats(r, v);
          if constexpr (GATED) {
            tmem_ld32(acc + kTileN + cc, r);
            as_floats(r, u);
          }
          finish<MODE>(p, jb, bx, lane, c.z, m0 + q * 32, n0 + cc, v, u);
        }
      }
      if (lane == 0) bulk_wait_all0();
    } else if (m0 + q * 32 < jb.M) {
      float* part = reinterpret_cast<float*>(smem) + q * 32 + lane;
#pragma unroll 1
      for (int cc = 0; cc < BN; cc += 32) {
        uint32_t r[32];
        tmem_ld32(acc + cc, r);
#pragma unroll
        for (int j = 0; j < 32; ++j) part[(cc + j) * 128] = __uint_as_float(r[j]);
      }
    }
  }

  __syncwarp();
  if (*abort_flag) settle();
  if (S > 1) {
    cluster_sync_all();  // every CTA's sums are in its shared memory
    if (warp >= 2) {
      const int e = warp - 2;
      Boxes bx = {smem + L::kBoxes + e * 2 * kBoxBytes, 0};
      // the S CTAs of this tile are neighbours in the cluster, which may hold several tiles
      uint32_t first;
      asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(first));
      first -= (uint32_t)rank;
      const int quarters = min(4, (jb.M - m0 + 31) / 32);
      const int pieces = min(kTileN, jb.N - n0 + 31) / 32 * quarters;
      for (int i = rank + e * S; i < pieces; i += 4 * S) {
        const int q = i % quarters, cc = i / quarters * 32;
        const uint32_t at = smem_u32(smem) + (uint32_t)(cc * 128 + q * 32 + lane) * 4;
        float v[32], u[GATED ? 32 : 1];
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = 0;
        if constexpr (GATED) {
#pragma unroll
          for (int j = 0; j < 32; ++j) u[j] = 0;
        }
        for (int s = 0; s < S; ++s) {
          const uint32_t from = mapa_rank(at, first + (uint32_t)s);
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] += ld_cluster_f32(from + j * 512);
          if constexpr (GATED) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] += ld_cluster_f32(from + (kTileN + j) * 512);
          }
        }
        finish<MODE>(p, jb, bx, lane, c.z, m0 + q * 32, n0 + cc, v, u);
      }
      if (lane == 0) bulk_wait_all0();
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are being read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(BN) : "memory");
  }
  if (threadIdx.x == 0 && *abort_flag) *p.status = EAS_ERR_TIMEOUT;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// A row-major matrix [rows][cols] of 16-bit values for TMA boxes of box_rows x box_cols.
int encode(CUtensorMap* map, const void* base, uint64_t rows, uint64_t cols, uint64_t ld, uint32_t box_rows,
           uint32_t box_cols, CUtensorMapSwizzle swizzle, const char* who) {
  const cuuint64_t dims[2] = {cols, rows};
  const cuuint64_t strides[1] = {ld * 2};
  const cuuint32_t box[2] = {box_cols, box_rows};
  const cuuint32_t estr[2] = {1, 1};
  // 16-bit words are copied as they are, whichever of the two types they hold; zeros fill the outside
  return eas_drv_check(
      g_drv.tensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base), dims, strides, box,
                                 estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE),
      who, EAS_ERR_VALUE);
}

bool aligned16(const void* p, uint64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0; }

// One job: operand maps (a_rows, b_rows: rows of a K-major operand per box), results, tiles of tile_m x tile_n.
int fill_job(Job& q, const DenseProduct& p, int a_rows, int b_rows, int tile_m, int tile_n, const char* who) {
  int rc = EAS_OK;
  const int na = p.terms > 1 || p.batch > 1 ? 2 : 1;
  const int nb = p.terms > 1 || p.gated ? 2 : 1;
  for (int t = 0; t < na && !rc; ++t)
    rc = p.a_mn ? encode(&q.a[t], p.a[t], p.K, p.M, p.lda[t], kBK, 64, CU_TENSOR_MAP_SWIZZLE_128B, who)
                : encode(&q.a[t], p.a[t], p.M, p.K, p.lda[t], a_rows, kBK, CU_TENSOR_MAP_SWIZZLE_128B, who);
  for (int t = 0; t < nb && !rc; ++t)
    rc = p.b_mn ? encode(&q.b[t], p.b[t], p.K, p.N, p.ldb[t], kBK, 64, CU_TENSOR_MAP_SWIZZLE_128B, who)
                : encode(&q.b[t], p.b[t], p.N, p.K, p.ldb[t], b_rows, kBK, CU_TENSOR_MAP_SWIZZLE_128B, who);
  q.y_tma = aligned16(p.y[0], p.ldy[0]) && (p.batch < 2 || aligned16(p.y[1], p.ldy[1]));
  for (int z = 0; z < p.batch && q.y_tma && !rc; ++z)
    rc = encode(&q.y[z], p.y[z], p.M, p.N, p.ldy[z], 32, 32, CU_TENSOR_MAP_SWIZZLE_64B, who);
  if (rc) return rc;
  for (int z = 0; z < 2; ++z) q.y_ptr[z] = p.y[z], q.ldy[z] = (int64_t)p.ldy[z];
  q.M = p.M, q.N = p.N;
  q.kb_term = (p.K + kBK - 1) / kBK;
  q.kb_total = q.kb_term * p.terms;
  const int64_t mt = ((int64_t)p.M + tile_m - 1) / tile_m, nt = ((int64_t)p.N + tile_n - 1) / tile_n;
  if (mt * nt * p.batch > 0x1fffffff) return eas_fail(EAS_ERR_VALUE, "%s: too many output tiles", who);
  q.mt = (int)mt, q.nt = (int)nt, q.tiles = (int)(mt * nt * p.batch);
  // As many M tiles as keep their rows of A in half of L2 from one column of tiles to the next: 16 of
  // 256 rows up to K of 4882, else 8 (8192^3: 838 us by 8, 855 by 16; 8192 x 2 8192 x 4096: 773, 761).
  q.group = (int64_t)16 * tile_m * p.K * 2 <= 40000000 ? 16 : 8;
  q.batch2 = p.batch > 1;
  q.a_mn = p.a_mn;
  return EAS_OK;
}

// What the epilogue of a forward product takes.
int fill_epilogue(Params& q, const DenseProduct& p, const char* who) {
  int rc = EAS_OK;
  if (p.pre && (q.pre_tma = aligned16(p.pre, p.ldp)))
    rc = encode(&q.pre, p.pre, p.M, p.N, p.ldp, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B, who);
  if (!rc && p.pre2 && (q.pre2_tma = aligned16(p.pre2, p.ldp2)))
    rc = encode(&q.pre2, p.pre2, p.M, p.N, p.ldp2, 32, 32, CU_TENSOR_MAP_SWIZZLE_64B, who);
  if (rc) return rc;
  q.bias = p.bias, q.residual = p.residual;
  q.bias_vec = (reinterpret_cast<uintptr_t>(p.bias) & 15) == 0;
  q.res_vec = aligned16(p.residual, p.ldr);
  q.pre_ptr = p.pre, q.pre2_ptr = p.pre2;
  q.ldr = (int64_t)p.ldr, q.ldp = (int64_t)p.ldp, q.ldp2 = (int64_t)p.ldp2;
  q.act = p.act;
  return EAS_OK;
}

// Shared-memory opt-in and co-resident clusters of a kernel, once per device.
struct KernelState {
  int pairs[64] = {0};
};

template <int MODE>
int launch_pair(Params& q, int dev, cudaStream_t s, const char* who) {
  static KernelState st;
  const void* kernel = reinterpret_cast<const void*>(&dense_pair_kernel<MODE>);
  const int slot = dev >= 0 && dev < 64 ? dev : 0;
  if (!st.pairs[slot]) {
    int rc = eas_cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kPairSmem), who,
                            EAS_ERR_LAUNCH);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * (dense_sms(dev) / 2)), 1, 1);
    cfg.blockDim = dim3(kPairThreads, 1, 1);
    cfg.dynamicSmemBytes = kPairSmem;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      n = dense_sms(dev) / 2;
    }
    st.pairs[slot] = n;
  }
  const int pairs = q.tiles < st.pairs[slot] ? q.tiles : st.pairs[slot];
  return dense_launch(kernel, dim3(2 * pairs), 0, kPairThreads, kPairSmem, s, &q, who);
}

template <int BN, int AR, bool DEEP, int MODE>
int launch_tile(Params& q, int dev, cudaStream_t s, const char* who) {
  auto whole = [&](int ctas) { return (ctas + q.cluster - 1) / q.cluster * q.cluster; };
  q.ctas0 = whole(q.job[0].tiles * q.job[0].split);
  q.ctas = q.ctas0 + whole(q.job[1].tiles * q.job[1].split);
  const int sums = q.sums.db ? whole((q.sums.N + 31) / 32) : 0;
  static bool ready[64] = {false};
  using L = TileShape<BN, AR, DEEP>;
  const void* kernel = reinterpret_cast<const void*>(&dense_tile_kernel<BN, AR, DEEP, MODE>);
  const int slot = dev >= 0 && dev < 64 ? dev : 0;
  if (!ready[slot]) {
    int rc = eas_cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmem), who,
                            EAS_ERR_LAUNCH);
    if (rc) return rc;
    ready[slot] = true;
  }
  return dense_launch(kernel, dim3((unsigned)(q.ctas + sums)), q.cluster > 1 ? q.cluster : 0, kTileThreads, L::kSmem, s, &q,
                      who);
}

using Choice = DenseShape;

// The shape of least estimated time, in microseconds on one B200 at 1.9 GHz (operands from HBM).  A step is
// one 64-deep k-block of one CTA or pair.  The numbers are fitted to 650 random calls of all four operators, and
// tried on 2000 more, each timed with every shape: the choice takes 1.4 % longer than the best one (two
// products: 2.1) on geometric average.
//   pair, 256 x 256        7 + rounds x k-blocks x 0.28   (512 x 4096 x 4096: 25.3)
//   one CTA per SM         5.4 + k-blocks x step, step 0.125 (BN 64) or 0.215 (128), 0.11 or 0.19 with
//                          64 rows of A   (64 x 4096 x 4096: 12.3 BN 64, 15.0 BN 128)
//   two CTAs per SM        4.6 + CTAs per SM x (k-blocks x step + 0.7), step 0.2 or 0.3 (2048^3: 25.1
//                          BN 64, 17.5 BN 128), one product's in whole rounds (gated 736 x 3456 x 4608,
//                          324 CTAs for 296 places: 82; as pairs 52)
//   a split over 2 or 4    1.35 or 2.1 more for the exchange, and only while all CTAs are resident at
//                          once (16 x 4096 x 4096, BN 64: 11.9 whole, 10.2 split in 2, 17.9 in 8;
//                          184 x 560 x 1504: 6.9 whole, 5.9 split in 4)
//   two products           a few long sums beside many short ones are split over up to 8 CTAs (dx beside dW
//                          of 7 x 6215 x 795: 98 k-blocks beside 637 tiles of one; whole, they took 46),
//                          where each CTA also holds its place for 1.8 while it waits for the others
//   column sums            3 more with the pair kernel, which leaves them to a launch of their own
Choice choose(const DenseProduct* p, int count, bool sums, int sms) {
  const int pairs = sms / 2 > 0 ? sms / 2 : 1;
  int64_t kb[2] = {0, 0}, least_kb = INT64_MAX;
  int most_rows = 0;
  bool a_mn = false;
  for (int i = 0; i < count; ++i) {
    kb[i] = (int64_t)((p[i].K + kBK - 1) / kBK) * p[i].terms;
    least_kb = kb[i] < least_kb ? kb[i] : least_kb;
    most_rows = p[i].M > most_rows ? p[i].M : most_rows;
    a_mn |= p[i].a_mn;
  }
  auto tiles_of = [&](int i, int m, int width) {
    const int n = p[i].gated ? width / 2 : width;
    return (int64_t)((p[i].M + (int64_t)m - 1) / m) * ((p[i].N + (int64_t)n - 1) / n) * p[i].batch;
  };
  Choice best = {0, {1, 1}, 128, false};
  double best_us;
  if (count == 1) {
    best_us = 7 + (double)((tiles_of(0, 256, 256) + pairs - 1) / pairs) * kb[0] * 0.28;
  } else {  // the jobs (the longer tiles first) fill one another's last rounds
    double steps = 0;
    int64_t tiles = 0;
    for (int i = 0; i < count; ++i) {
      tiles += tiles_of(i, 256, 256);
      steps += (double)tiles_of(i, 256, 256) * kb[i];
    }
    steps = tiles <= pairs ? kb[0] : steps / pairs + 0.5 * least_kb;
    best_us = 7 + (steps > kb[0] ? steps : kb[0]) * 0.28;
  }
  if (sums) best_us += 3;
  const int64_t most_split = (int64_t)sms * 7 / 8;
  for (int bn = 64; bn <= 128; bn += 64) {
    int64_t tiles[2] = {0, 0};
    double work = 0;  // steps of all tiles, with what a tile costs beside its steps
    const double shared = bn == 64 ? 0.2 : 0.3, tile_us = 0.7;
    for (int i = 0; i < count; ++i) {
      tiles[i] = tiles_of(i, 128, bn);
      work += (double)tiles[i] * (kb[i] * shared + tile_us);
    }
    const bool few = most_rows <= 64 && !a_mn;
    const double step = bn == 64 ? (few ? 0.11 : 0.125) : (few ? 0.19 : 0.215);
    auto exchange = [](int split) { return split == 1 ? 0 : split == 2 ? 1.35 : 2.1; };
    for (int s0 = 1; s0 <= 8; s0 *= 2) {
      for (int s1 = 1; s1 <= (count > 1 ? s0 : 1); s1 *= 2) {
        const int64_t ctas = tiles[0] * s0 + tiles[1] * s1;
        if (s0 > 1 && (kb[0] < 2 * s0 || (s1 > 1 && kb[1] < 2 * s1))) continue;
        Choice c = {bn, {s0, s1}, 128, ctas <= sms};
        double us;
        if (c.deep) {
          if (s0 > 4 || (s0 > 1 && ctas > most_split)) continue;
          if (few) c.ar = 64;
          const double t0 = (double)((kb[0] + s0 - 1) / s0) * step + exchange(s0);
          const double t1 = (double)((kb[1] + s1 - 1) / s1) * step + exchange(s1);
          us = 5.4 + (t0 > t1 ? t0 : t1);
        } else {
          if (s1 > 1 || (s0 > 1 && count == 1)) continue;
          // the longer tiles beside another, and all work spread over the SMs
          const double meet = s0 == 1 ? 0 : s0 == 2 ? 2.2 : s0 == 4 ? 3.0 : 3.3;
          const double t0 = (double)((kb[0] + s0 - 1) / s0) * 1.1 * shared + 1.1 * tile_us + meet;
          double all = (work + (double)tiles[0] * (s0 * meet + (s0 - 1) * 1.8)) / sms;
          if (count == 1) {  // like tiles start and end together: whole rounds, two per SM
            const int64_t rounds = (ctas + 2 * sms - 1) / (2 * sms);
            if (rounds > 1) all = (double)rounds * 2 * work / ctas;
          }
          us = 4.6 + (all > t0 ? all : t0);
        }
        if (us < best_us) best = c, best_us = us;
      }
    }
  }
  return best;
}

template <int MODE>
int launch_choice(const Choice& c, Params& q, int dev, cudaStream_t s, const char* who) {
  if (c.bn == 0) {
    if (q.sums.db) {
      int rc = dense_column_sums(q.sums, s, who);
      if (rc) return rc;
    }
    return launch_pair<MODE>(q, dev, s, who);
  }
  if (c.ar == 64)
    return c.bn == 64 ? launch_tile<64, 64, true, MODE>(q, dev, s, who) : launch_tile<128, 64, true, MODE>(q, dev, s, who);
  if (c.bn == 64)
    return c.deep ? launch_tile<64, 128, true, MODE>(q, dev, s, who) : launch_tile<64, 128, false, MODE>(q, dev, s, who);
  return c.deep ? launch_tile<128, 128, true, MODE>(q, dev, s, who) : launch_tile<128, 128, false, MODE>(q, dev, s, who);
}

// The epilogue waits for a whole sum (0.3 us per k-block), with the budget of all waits, about 2 s.
constexpr int64_t kMostSteps = 1 << 22;

int64_t steps_of(const DenseProduct& p) { return (int64_t)((p.K + kBK - 1) / kBK) * p.terms; }

void longer_first(const DenseProduct* p, int count, DenseProduct (&order)[2]) {
  const bool swap = count > 1 && steps_of(p[0]) < steps_of(p[1]);
  order[0] = p[swap ? 1 : 0];
  order[1] = p[count > 1 && !swap ? 1 : 0];
}

}  // namespace

DenseShape dense_shape(const DenseProduct* p, int count, bool sums, int sms) {
  DenseProduct order[2];
  longer_first(p, count, order);
  return choose(order, count, sums, sms);
}

int dense_column_sums(const DenseColSum& sums, cudaStream_t stream, const char* who) {
  DenseColSum c = sums;
  return dense_launch(reinterpret_cast<const void*>(&column_sums_kernel), dim3((unsigned)((c.N + 31) / 32)), 0,
                      kTileThreads, 0, stream, &c, who);
}

int dense_mma(const DenseProduct* p, int count, const DenseColSum& sums, cudaStream_t stream, const char* who) {
  int dev = 0;
  int rc = eas_cuda_check(cudaGetDevice(&dev), who, EAS_ERR_UNAVAILABLE);
  if (rc) return rc;
  DenseProduct order[2];
  longer_first(p, count, order);
  for (int i = 0; i < count; ++i)
    if (steps_of(order[i]) > kMostSteps)
      return eas_fail(EAS_ERR_VALUE, "%s: sums of more than %lld products are not taken", who, (long long)kMostSteps * kBK);
  const Choice c = choose(order, count, sums.db != nullptr, dense_sms(dev));
  const bool gated = p[0].gated;
  const int width = c.bn ? c.bn : 256;  // of the accumulator: a gated tile has half as many outputs
  const int b_rows = !c.bn ? 128 : (gated ? c.bn / 2 : c.bn);
  Params q = {};
  for (int i = 0; i < count; ++i) {
    rc = fill_job(q.job[i], order[i], c.ar, b_rows, c.bn ? 128 : 256, gated ? width / 2 : width, who);
    if (rc) return rc;
    q.job[i].split = c.split[i];
    q.tiles += q.job[i].tiles;
  }
  if (count > 1) q.ratio = (q.job[0].kb_total + q.job[1].kb_total / 2) / q.job[1].kb_total;
  q.cluster = c.split[0] > c.split[1] ? c.split[0] : c.split[1];
  if (count == 1) q.job[1].split = 1;
  q.bf16 = p[0].bf16;
  q.unscale = p[0].unscale;
  q.sums = sums;
  q.status = eas_native_status_dev(dev);
  if (!q.status) return eas_fail(EAS_ERR_MEMORY, "%s: no status word, in which an expired wait would be reported", who);
  if (p[0].b_mn) return launch_choice<kBackward>(c, q, dev, stream, who);
  rc = fill_epilogue(q, p[0], who);
  if (rc) return rc;
  return gated ? launch_choice<kGatedForward>(c, q, dev, stream, who) : launch_choice<kForward>(c, q, dev, stream, who);
}
