// dense.cu — the dense layers of a model as operators: a linear layer with bias, activation and
// residual, a gated feed-forward block, and their backward passes (f16 or bf16, f32 sums).
//
//   linear            z = x W^T + b;  y = act(z) + r                      x [M,K], W [N,K], y [M,N]
//   linear_backward   dz = dy act'(z);  dx = dz W;  dW = dz^T x;  db = sum_m dz
//   gated             g = x Wg^T, u = x Wu^T;  h = act(g) u
//   gated_backward    dg = dh u act'(g), du = dh act(g);  dx = dg Wg + du Wu;  dWg = dg^T x;  dWu = du^T x
//
// A backward pass is one pass over dy (act_grad_kernel: dz, and the column sums of db) and the two
// products.  dz, dg and du are rounded to the operands' type there: they are operands of matrix
// products, as x and W are, and a matrix instruction takes 16-bit ones at this rate (a second term
// for the remainder would double the products).  Half a step more of each operand: the error of dx and
// dW against 64 bits grows from 1.66e-3 to 2.35e-3 in bf16.  In f16 their range would lose more than
// that; see "the range of f16" below.
#include <cuda_runtime.h>
#include <stdint.h>

#include <initializer_list>

#include "dense_internal.h"
#include "dense_launch.h"
#include "dense_math.cuh"
#include "eas_internal.h"

namespace {

using namespace dense;

// ---------------------------------------------------------------------------
// copies of operands whose rows TMA cannot read in place
// ---------------------------------------------------------------------------
//
// Up to three matrices, in rows of a multiple of 8 elements (zeros past the end), 8 elements per thread,
// beside the elementwise half of a backward pass or in a launch of their own.  Bound by HBM: 97 MB of
// 3648 x 6675 weights take 39 us, 5 TB/s.  (Loading aligned words and shifting them, as the other
// kernels do, took as long there and 2 us more on small matrices.)

struct Repitch {
  struct Matrix {
    const uint16_t* src;
    uint16_t* dst;
    int64_t ld, end;   // groups of this matrix and of those before it
    int cols, groups;  // groups of 8 per padded row
  } m[3];
  int count;
};

__device__ __forceinline__ void repitch(const Repitch& p, int64_t block, int64_t blocks) {
  const int64_t total = p.m[p.count - 1].end;
  const bool small = total < (1ll << 31);  // a division of 32 bits
  for (int64_t i = block * 256 + threadIdx.x; i < total; i += blocks * 256) {
    const int k = i < p.m[0].end ? 0 : i < p.m[1].end ? 1 : 2;
    const Repitch::Matrix& m = p.m[k];
    const int64_t g = i - (k ? p.m[k - 1].end : 0);
    const int64_t r = small ? (uint32_t)g / (uint32_t)m.groups : g / m.groups;
    const int c = (int)(g - r * m.groups) * 8;
    const uint16_t* src = m.src + r * m.ld + c;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t lo = c + 2 * j < m.cols ? src[2 * j] : 0;
      const uint32_t hi = c + 2 * j + 1 < m.cols ? src[2 * j + 1] : 0;
      w[j] = lo | (hi << 16);
    }
    *reinterpret_cast<uint4*>(m.dst + g * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

int repitch_blocks(const Repitch& p) {
  if (!p.count) return 0;
  const int64_t blocks = (p.m[p.count - 1].end + 255) / 256;
  return (int)(blocks < 24 * 148 ? blocks : 24 * 148);
}

__global__ void __launch_bounds__(256) repitch_kernel(const __grid_constant__ Repitch p) {
  grid_order();
  repitch(p, blockIdx.x, gridDim.x);
}

// ---------------------------------------------------------------------------
// the elementwise half of the backward pass
// ---------------------------------------------------------------------------
//
// linear: dz = dy act'(z);  gated: dg = dh u act'(g), du = dh act(g).  One pass, 8 columns (16
// bytes) per thread; a block covers 256 columns of rows_per_block() rows with 8 thread rows.  With
// db, each thread keeps the f32 sums of its columns, the block adds its 8 thread rows in shared
// memory and writes one row of partial sums, which the products' launch adds in a fixed order: no
// atomics, the same bits on every run.

bool vec_ok(const void* p, uint64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0; }

// Past the last value of a matrix.
const uint16_t* past_end(const uint16_t* p, int64_t ld, int64_t rows, int64_t cols) { return p + (rows - 1) * ld + cols; }

// What a block of act_grad_kernel saw of the values that it rounded to f16 (see "the range of f16").
struct Range {
  float largest;  // finite |value|
  float low;      // > 0: many groups of values have no full precision
};

struct ActGrad {
  const uint16_t* dy;
  const uint16_t* g;
  const uint16_t* u;
  const uint16_t *dy_end, *g_end, *u_end;  // past their last values
  uint16_t* dg;     // dz, or dg; null when dz is dy itself (act none) and only db is wanted
  uint16_t* du;
  float* partial;   // [row blocks][N] sums of dz, or null
  Range* range;     // [blocks], where f16 may need a scale, else null
  float* unscale;   // what the products have to be multiplied by, then
  int64_t lddy, ldg, ldu, ldo;
  int M, N, rows_per_block;
  int row_blocks;   // the blocks behind those make copies
  Repitch copies;
  int act;
  bool bf16;
};

template <bool BF16>
__device__ __forceinline__ void widen8(const uint4& w, float (&v)[8]) {
  unpack2<BF16>(w.x, v[0], v[1]);
  unpack2<BF16>(w.y, v[2], v[3]);
  unpack2<BF16>(w.z, v[4], v[5]);
  unpack2<BF16>(w.w, v[6], v[7]);
}

template <bool BF16>
__device__ __forceinline__ void store8(uint16_t* p, int n, const float (&v)[8]) {
  if (n >= 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2<BF16>(v[0], v[1]), pack2<BF16>(v[2], v[3]),
                                              pack2<BF16>(v[4], v[5]), pack2<BF16>(v[6], v[7]));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) p[j] = to_16<BF16>(v[j]);
  }
}

// ---- the range of f16 ----
//
// dz, dg and du can leave f16's range where dx and dW do not (dh = up = 300: dg would be infinite), or its
// full precision (gradients of 1e-5 are its subnormals).  They are linear in dy, so a power of two taken
// out of all of them and put back in the products' epilogue costs no rounding.  act_grad_kernel stores them
// unscaled and each of its blocks notes what it saw; act_again_kernel behind it looks at all notes
// and, where a scale is needed, makes the pass again with it.  Only sums over all blocks can choose it:
//   the largest finite |value| is past 65504: it is brought below 2^15;
//   of the groups of 8 neighbours that are not all zeros, more than one in 64 is below 2^-11
//   throughout: the largest value is brought up to 2^14 (or stays).
// Otherwise at most one group in 64 has typical values among f16's subnormals (below 2^-14), where the
// rounding error no longer falls with the value: it stays at 2^-25, that of 2^-14.
// act none and relu leave dy or 0, which f16 holds, and bf16 has the range of f32: neither needs this.
// The look costs a launch: linear 777 x 1000 x 2088 takes 23.2 us with it (20.6 without), gated 613 x 1376
// x 512 17.0 (14.1), 2048 x 4096 x 1024 70 (68), 4096 x 8192 x 4096 the same within 1 %.  Made again, with one
// block per SM, the pass takes 5 to 100 us more (those sizes: 27, 22, 97, 890).  More blocks make it
// faster and the look slower: with two per SM 2048 x 4096 x 1024 takes 72 and 87 us, for 70 and 97.

constexpr float kLow = 0x1p-11f;

// The values of one thread.
struct RangeNotes {
  float largest = 0;
  int low = 0;  // 63 for each low group, -1 for each other one (2^31 rows: 2 x 63 x 2^31 / 1184 / 8 < 2^25)

  __device__ __forceinline__ void add(const float (&v)[8]) {
    float g = fabsf(v[0]);
#pragma unroll
    for (int j = 1; j < 8; ++j) g = fmaxf(g, fabsf(v[j]));  // passes NaN by
    if (g == INFINITY) {
      g = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) g = fabsf(v[j]) < INFINITY ? fmaxf(g, fabsf(v[j])) : g;
    }
    largest = fmaxf(largest, g);
    low += g > 0 ? (g < kLow ? 63 : -1) : 0;
  }
};

// Of a block's 256 threads: the largest `largest` and the sum of all `low`.
__device__ __forceinline__ Range block_range(Range r) {
  __shared__ Range warps[8];
  // (the bits of values that are not negative are in their order)
  r.largest = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(r.largest)));
#pragma unroll
  for (int d = 16; d; d >>= 1) r.low += __shfl_xor_sync(0xffffffffu, r.low, d);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = r;
  __syncthreads();
  r = warps[0];
#pragma unroll
  for (int w = 1; w < 8; ++w) r.largest = fmaxf(r.largest, warps[w].largest), r.low += warps[w].low;
  return r;
}

// e of the scale 2^e: -18 (the largest values are below 65504^2 x 1.13 < 2^33) .. 100 (what is
// smaller yet is 0 in every result).
__device__ __forceinline__ int range_exponent(const Range& r) {
  const int e = 14 - ((int)(__float_as_uint(r.largest) >> 23) - 127);
  if (r.largest > 65504.0f) return e;
  return r.low > 0 && e > 0 ? min(e, 100) : 0;
}

// One block's part: 256 columns of rows_per_block rows.  VEC: every array takes 16-byte accesses, so that
// only the last columns need other ones.  (Others are gathered from aligned words.)  AGAIN: values times
// `scale`; else notes and column sums of them unscaled.
template <bool GATED, bool BF16, bool VEC, bool AGAIN>
__device__ __forceinline__ void act_grad_part(const ActGrad& p, int bx, int by, float scale, float (&sum)[8],
                                              RangeNotes& notes) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int n0 = (bx * 32 + tx) * 8;
  const int cols = p.N - n0;
  if (cols <= 0) return;
  const int64_t r0 = (int64_t)by * p.rows_per_block;
  const int64_t r1 = min((int64_t)p.M, r0 + p.rows_per_block);
  with_act(p.act, [&](auto a) {
    constexpr int ACT = decltype(a)::value;
    constexpr bool kG = GATED || ACT != kNone;
    constexpr bool kNotes = !BF16 && !AGAIN && (GATED || (ACT != kNone && ACT != kRelu));
    auto put = [&](uint16_t* to, float (&v)[8]) {
      if constexpr (kNotes) notes.add(v);
      if constexpr (AGAIN) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] *= scale;
      }
      store8<BF16>(to, cols, v);
    };
    auto row = [&](int64_t m, const float (&dy)[8], const float (&g)[8], const float (&u)[8]) {
      float o[8];
      if constexpr (GATED) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v, d;
          act_and_slope<ACT>(g[j], v, d);
          w[j] = dy[j] * u[j] * d;
          o[j] = dy[j] * v;
        }
        put(p.dg + m * p.ldo + n0, w);
        put(p.du + m * p.ldo + n0, o);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          float v, d = 1.0f;
          if (ACT != kNone) act_and_slope<ACT>(g[j], v, d);
          o[j] = dy[j] * d;
          if (!AGAIN) sum[j] += o[j];
        }
        if (p.dg) put(p.dg + m * p.ldo + n0, o);
      }
    };
    float dy[8], g[8], u[8];
    int64_t m = r0 + ty;
    if (VEC && cols >= 8) {
      // the next row's words are under way while this one is worked on
      const int64_t sd = 8 * p.lddy, sg = 8 * p.ldg, su = 8 * p.ldu;
      const uint16_t *pd = p.dy + m * p.lddy + n0, *pg = kG ? p.g + m * p.ldg + n0 : nullptr,
                     *pu = GATED ? p.u + m * p.ldu + n0 : nullptr;
      uint4 wd, wg, wu;
      auto fetch = [&]() {
        wd = *reinterpret_cast<const uint4*>(pd);
        if (kG) wg = *reinterpret_cast<const uint4*>(pg);
        if (GATED) wu = *reinterpret_cast<const uint4*>(pu);
        pd += sd, pg += sg, pu += su;
      };
      if (m < r1) fetch();
      for (; m < r1; m += 8) {
        widen8<BF16>(wd, dy);
        if (kG) widen8<BF16>(wg, g);
        if (GATED) widen8<BF16>(wu, u);
        if (m + 8 < r1) fetch();
        row(m, dy, g, u);
      }
    }
    for (; m < r1; m += 8) {
      const uint16_t *pd = p.dy + m * p.lddy + n0, *pg = kG ? p.g + m * p.ldg + n0 : nullptr,
                     *pu = GATED ? p.u + m * p.ldu + n0 : nullptr;
      if constexpr (VEC) {  // the last, partial words
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          dy[j] = j < cols ? to_f32<BF16>(pd[j]) : 0.0f;
          if (kG) g[j] = j < cols ? to_f32<BF16>(pg[j]) : 0.0f;
          if (GATED) u[j] = j < cols ? to_f32<BF16>(pu[j]) : 0.0f;
        }
      } else {
        Gather8 wd, wg, wu;
        wd.fetch(pd, cols, p.dy, p.dy_end);
        if (kG) wg.fetch(pg, cols, p.g, p.g_end);
        if (GATED) wu.fetch(pu, cols, p.u, p.u_end);
        widen8<BF16>(wd.get(), dy);
        if (kG) widen8<BF16>(wg.get(), g);
        if (GATED) widen8<BF16>(wu.get(), u);
      }
      row(m, dy, g, u);
    }
  });
}

// Four blocks per SM: the bytes under way are what the pass lives on (a gated backward call of 4096 x 8192
// with dWg of 64 columns alone: 73 us with three blocks, 65 with four).  Three where the notes of gathered
// gated values would spill at 64 registers (613 x 1375 x 512: 18.9 us, 19.4 with four).
template <bool GATED, bool BF16, bool VEC>
__global__ void __launch_bounds__(256, GATED && !BF16 && !VEC ? 3 : 4) act_grad_kernel(const __grid_constant__ ActGrad p) {
  __shared__ float sums[8][32][9];
  grid_order();
  if ((int)blockIdx.y >= p.row_blocks) {
    repitch(p.copies, (int64_t)(blockIdx.y - p.row_blocks) * gridDim.x + blockIdx.x,
            (int64_t)(gridDim.y - p.row_blocks) * gridDim.x);
    return;
  }
  float sum[8] = {};
  RangeNotes notes;
  act_grad_part<GATED, BF16, VEC, false>(p, blockIdx.x, blockIdx.y, 1.0f, sum, notes);
  if (!BF16 && p.range) {
    const Range r = block_range({notes.largest, (float)notes.low});
    if (threadIdx.x == 0) p.range[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = r;
  }
  if (GATED || !p.partial) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sums[threadIdx.x >> 5][threadIdx.x & 31][j] = sum[j];
  __syncthreads();
  const int c = threadIdx.x, n = blockIdx.x * 256 + c;  // one column per thread
  float s = 0;
#pragma unroll
  for (int r = 0; r < 8; ++r) s += sums[r][c >> 3][c & 7];
  if (n < p.N) p.partial[(int64_t)blockIdx.y * p.N + n] = s;
}

// The pass again (f16), with the scale that the blocks' notes ask for; mostly they ask for none.
template <bool GATED, bool VEC>
__global__ void __launch_bounds__(256, 2) act_again_kernel(const __grid_constant__ ActGrad p) {
  grid_order();
  const int width = (p.N + 255) / 256;
  const int64_t blocks = (int64_t)width * p.row_blocks;
  Range all = {0, 0};
  for (int64_t i = threadIdx.x; i < blocks; i += 256) {
    const Range r = p.range[i];
    all.largest = fmaxf(all.largest, r.largest);
    all.low += r.low;
  }
  const int e = range_exponent(block_range(all));
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.unscale = __uint_as_float((uint32_t)(127 - e) << 23);
  if (e == 0) return;
  float sum[8];
  RangeNotes notes;
  for (int64_t b = blockIdx.x; b < blocks; b += gridDim.x)
    act_grad_part<GATED, false, VEC, true>(p, (int)(b % width), (int)(b / width), __uint_as_float((uint32_t)(127 + e) << 23),
                                           sum, notes);
}

template <bool GATED>
int launch_act_grad(ActGrad& g, int blocks, cudaStream_t s, const char* who) {
  const bool kG = GATED || g.act != kNone;
  const bool vec = vec_ok(g.dy, g.lddy) && (!kG || vec_ok(g.g, g.ldg)) && (!GATED || vec_ok(g.u, g.ldu));
  g.dy_end = past_end(g.dy, g.lddy, g.M, g.N);
  if (kG) g.g_end = past_end(g.g, g.ldg, g.M, g.N);
  if (GATED) g.u_end = past_end(g.u, g.ldu, g.M, g.N);
  const void* kernel = g.bf16 ? (vec ? reinterpret_cast<const void*>(&act_grad_kernel<GATED, true, true>)
                                     : reinterpret_cast<const void*>(&act_grad_kernel<GATED, true, false>))
                              : (vec ? reinterpret_cast<const void*>(&act_grad_kernel<GATED, false, true>)
                                     : reinterpret_cast<const void*>(&act_grad_kernel<GATED, false, false>));
  const int width = (g.N + 255) / 256;
  g.row_blocks = blocks;
  const int64_t parts = (int64_t)width * blocks;
  blocks += (repitch_blocks(g.copies) + width - 1) / width;
  int rc = dense_launch(kernel, dim3((unsigned)width, (unsigned)blocks), 0, 256, 0, s, &g, who);
  if (rc || !g.range) return rc;
  kernel = vec ? reinterpret_cast<const void*>(&act_again_kernel<GATED, true>)
               : reinterpret_cast<const void*>(&act_again_kernel<GATED, false>);
  return dense_launch(kernel, dim3((unsigned)(parts < 148 ? parts : 148)), 0, 256, 0, s, &g, who);
}

// Rows per block: enough blocks for 8 per SM, at least 8 rows (one per thread row); with sums at most
// 128 row blocks (whose partial sums are added one after another).
int rows_per_block(int M, int N, bool sums) {
  const int64_t col_blocks = ((int64_t)N + 255) / 256;
  int64_t want = (8 * 148 + col_blocks - 1) / col_blocks;
  if (sums && want > 128) want = 128;
  int64_t rows = ((int64_t)M + want - 1) / want;
  rows = (rows + 7) / 8 * 8;
  return (int)(rows < 8 ? 8 : rows);
}

// Up to so many rows the products' launch sums the columns of dy itself where dz is dy (32 columns per
// CTA, beside the tiles); beyond, act_grad_kernel makes partial sums first.
constexpr uint32_t kDirectRows = 2048;

// Makes `dev` current for the scope of a call.
struct DeviceScope {
  int before = -1;
  int rc = EAS_OK;
  explicit DeviceScope(int dev) {
    rc = eas_driver_init();
    if (rc) return;
    int cur = -1;
    rc = eas_cuda_check(cudaGetDevice(&cur), "cudaGetDevice", EAS_ERR_UNAVAILABLE);
    if (rc || cur == dev) return;
    rc = eas_cuda_check(cudaSetDevice(dev), "cudaSetDevice", EAS_ERR_VALUE);
    if (!rc) before = cur;
  }
  ~DeviceScope() {
    if (before >= 0) cudaSetDevice(before);
  }
};

int check_sizes(const char* who, uint32_t M, uint32_t N, uint32_t K, int dtype, int act) {
  if (dtype < 0 || dtype >= kTypes) return eas_fail(EAS_ERR_VALUE, "%s: dtype must be 0 (f16) or 1 (bf16)", who);
  if (act < 0 || act >= kActs) return eas_fail(EAS_ERR_VALUE, "%s: unknown activation %d", who, act);
  if (M > 0x7fffff00u || N > 0x7fffff00u || K > 0x7fffff00u)
    return eas_fail(EAS_ERR_VALUE, "%s: a dimension exceeds 2^31 - 256", who);
  if (N == 0 || K == 0) return eas_fail(EAS_ERR_VALUE, "%s: N and K must be positive", who);
  return EAS_OK;
}

// A matrix of 16-bit values as it was passed; null ones are absent.
struct Given {
  const void* p;
  uint64_t ld;
  uint32_t rows, cols;
};

int check_matrices(const char* who, std::initializer_list<Given> all) {
  for (const Given& g : all) {
    if (!g.p) continue;
    if (reinterpret_cast<uintptr_t>(g.p) & 1) return eas_fail(EAS_ERR_VALUE, "%s: an address is odd", who);
    if (g.rows > 1 && g.ld < g.cols)
      return eas_fail(EAS_ERR_VALUE, "%s: a row pitch is smaller than the row", who);
  }
  return EAS_OK;
}

int zero_rows(void* p, uint64_t ld, uint32_t rows, uint32_t cols, cudaStream_t s, const char* who) {
  return eas_cuda_check(cudaMemset2DAsync(p, ld * 2, 0, (size_t)cols * 2, rows, s), who, EAS_ERR_LAUNCH);
}

uint64_t round256(uint64_t b) { return (b + 255) / 256 * 256; }

const uint16_t* u16(const void* p) { return static_cast<const uint16_t*>(p); }
uint16_t* u16(void* p) { return static_cast<uint16_t*>(p); }

// Which outputs a backward pass computes, and which operands TMA cannot read in place.
enum { kDx = 1, kDw = 2, kDb = 4 };
enum { kXOff = 1, kWOff = 2, kUpOff = 4, kDyOff = 8 };

// Layout of a call's scratch: operands that TMA cannot read in place, copied into rows padded to 8
// elements; of a backward pass also dz (or dg, du) in such rows, what was seen of their range, and the
// partial sums of db.
struct Scratch {
  uint64_t x = 0, w = 0, up = 0, dz = 0, dz2 = 0, partial = 0, range = 0, unscale = 0, total = 0;
  uint64_t ldk = 0, ldn = 0;  // padded pitches of rows of K and of N elements
  int rows = 0, blocks = 0;
  bool need_dz = false;
  bool ranged = false;  // in f16: dz, dg and du may need a scale
  bool direct = false;  // db straight from dy

  Scratch(uint32_t N, uint32_t K) : ldk(((uint64_t)K + 7) / 8 * 8), ldn(((uint64_t)N + 7) / 8 * 8) {}
  uint64_t take(uint64_t bytes) {
    const uint64_t at = total;
    total += round256(bytes);
    return at;
  }
};

Scratch forward_scratch(bool gated, uint32_t M, uint32_t N, uint32_t K, int off) {
  Scratch s(N, K);
  if (dense_rows_fit((int)M, (int)K)) return s;
  if (off & kXOff) s.x = s.take(2 * (uint64_t)M * s.ldk);
  if (off & kWOff) s.w = s.take(2 * (uint64_t)N * s.ldk);
  if (gated && (off & kUpOff)) s.up = s.take(2 * (uint64_t)N * s.ldk);
  return s;
}

Scratch backward_scratch(bool gated, uint32_t M, uint32_t N, uint32_t K, int act, int outputs, int off) {
  Scratch s(N, K);
  if ((outputs & kDw) && (off & kXOff)) s.x = s.take(2 * (uint64_t)M * s.ldk);
  if ((outputs & kDx) && (off & kWOff)) s.w = s.take(2 * (uint64_t)N * s.ldk);
  if (gated && (outputs & kDx) && (off & kUpOff)) s.up = s.take(2 * (uint64_t)N * s.ldk);
  s.rows = rows_per_block((int)M, (int)N, outputs & kDb);
  s.blocks = (int)(((uint64_t)M + s.rows - 1) / s.rows);
  s.need_dz = (outputs & (kDx | kDw)) && (gated || act != kNone || (off & kDyOff));
  if (s.need_dz) s.dz = s.take(2 * (uint64_t)M * s.ldn);
  if (s.need_dz && gated) s.dz2 = s.take(2 * (uint64_t)M * s.ldn);
  s.ranged = s.need_dz && (gated || (act != kNone && act != kRelu));
  if (s.ranged) {
    s.range = s.take((((uint64_t)N + 255) / 256) * s.blocks * sizeof(Range));
    s.unscale = s.take(sizeof(float));
  }
  s.direct = (outputs & kDb) && act == kNone && !s.need_dz && M <= kDirectRows;
  if ((outputs & kDb) && !s.direct) s.partial = s.take((uint64_t)s.blocks * N * 4);
  return s;
}

int check_scratch(const char* who, const Scratch& s, const void* p, uint64_t bytes) {
  if (s.total && (!p || bytes < s.total || (reinterpret_cast<uintptr_t>(p) & 255)))
    return eas_fail(EAS_ERR_VALUE, "%s: needs %llu bytes of 256-byte aligned scratch (eas_dense_scratch)", who,
                    (unsigned long long)s.total);
  return EAS_OK;
}

int off_mask(const void* p, uint64_t ld, int bit) { return vec_ok(p, ld) ? 0 : bit; }

// A matrix as a product's operand: itself, or its copy in scratch rows TMA can read.
struct Operand {
  const uint16_t* p;
  uint64_t ld;
};

struct Copies {
  Repitch r = {};

  Operand add(const void* src, uint64_t ld, uint32_t rows, uint32_t cols, bool off, void* scratch, uint64_t at,
              uint64_t ld_pad) {
    if (!off) return {u16(src), ld};
    uint16_t* dst = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(scratch) + at);
    const int groups = (int)(ld_pad / 8);
    const int64_t before = r.count ? r.m[r.count - 1].end : 0;
    r.m[r.count++] = {u16(src), dst, (int64_t)ld, before + (int64_t)rows * groups, (int)cols, groups};
    return {dst, ld_pad};
  }
  int launch(cudaStream_t s, const char* who) {
    if (!r.count) return EAS_OK;
    return dense_launch(reinterpret_cast<const void*>(&repitch_kernel), dim3((unsigned)repitch_blocks(r)), 0, 256, 0, s,
                        &r, who);
  }
};

// dx = sum_t dz_t W_t and dW_t = dz_t^T x, and db: independent of one another, so one launch.
int backward_products(const char* who, int terms, const Operand (&dz)[2], const Operand (&w)[2], const Operand& x,
                      void* dx, uint64_t lddx, void* const (&dw)[2], const uint64_t (&lddw)[2], const DenseColSum& sums,
                      const float* unscale, uint32_t M, uint32_t N, uint32_t K, int dtype, cudaStream_t s) {
  DenseProduct p[2];
  int count = 0;
  if (dx) {
    DenseProduct& d = p[count++];
    for (int t = 0; t < terms; ++t) d.a[t] = dz[t].p, d.lda[t] = dz[t].ld, d.b[t] = w[t].p, d.ldb[t] = w[t].ld;
    d.M = (int)M, d.N = (int)K, d.K = (int)N, d.terms = terms;
    d.y[0] = u16(dx), d.ldy[0] = lddx;
  }
  if (dw[0] || dw[1]) {
    DenseProduct& d = p[count++];
    d.batch = 0;
    for (int t = 0; t < terms; ++t) {
      if (!dw[t]) continue;
      const int z = d.batch++;
      d.a[z] = dz[t].p, d.lda[z] = dz[t].ld, d.y[z] = u16(dw[t]), d.ldy[z] = lddw[t];
    }
    d.b[0] = x.p, d.ldb[0] = x.ld;
    d.a_mn = true;
    d.M = (int)N, d.N = (int)K, d.K = (int)M;
  }
  for (int i = 0; i < count; ++i) p[i].b_mn = true, p[i].bf16 = dtype == kBF16, p[i].unscale = unscale;
  return dense_mma(p, count, sums, s, who);
}

}  // namespace

extern "C" int eas_dense_scratch(int op, uint32_t M, uint32_t N, uint32_t K, int act, int outputs, int unaligned,
                                 uint64_t* bytes) {
  if (!bytes) return eas_fail(EAS_ERR_VALUE, "eas_dense_scratch: null pointer");
  if (op < 0 || op > 3) return eas_fail(EAS_ERR_VALUE, "eas_dense_scratch: op must be 0..3");
  *bytes = 0;
  int rc = check_sizes("eas_dense_scratch", M, N, K, kF16, act);
  if (rc || M == 0) return rc;
  const bool gated = op & 1;
  *bytes = (op < 2 ? forward_scratch(gated, M, N, K, unaligned)
                   : backward_scratch(gated, M, N, K, act, outputs, unaligned)).total;
  return EAS_OK;
}

extern "C" int eas_dense_plan(int op, uint32_t M, uint32_t N, uint32_t K, int outputs, int num_sms, int* kernel,
                              int* width, int* split0, int* split1, int* a_rows, int* ctas_per_sm) {
  if (!kernel || !width || !split0 || !split1 || !a_rows || !ctas_per_sm)
    return eas_fail(EAS_ERR_VALUE, "eas_dense_plan: null pointer");
  if (op < 0 || op > 3) return eas_fail(EAS_ERR_VALUE, "eas_dense_plan: op must be 0..3");
  int rc = check_sizes("eas_dense_plan", M, N, K, kF16, kNone);
  if (rc) return rc;
  if (M == 0 || num_sms <= 0 || (op >= 2 && !(outputs & (kDx | kDw))))
    return eas_fail(EAS_ERR_VALUE, "eas_dense_plan: no product");
  const bool gated = op & 1;
  DenseProduct p[2];
  int count = 1;
  if (op < 2) {
    p[0].gated = gated;
    p[0].M = (int)M, p[0].N = (int)N, p[0].K = (int)K;
    if (dense_rows_fit((int)M, (int)K)) {
      const DenseRowsShape c = dense_rows_shape(p[0], true, num_sms);
      *kernel = 0, *width = gated ? 8 : 16, *split0 = c.split, *split1 = 1;
      *a_rows = kDenseRows, *ctas_per_sm = 0;  // (eas_dense_rows_plan)
      return EAS_OK;
    }
  } else {
    count = 0;
    if (outputs & kDx) {
      DenseProduct& d = p[count++];
      d.M = (int)M, d.N = (int)K, d.K = (int)N, d.terms = gated ? 2 : 1, d.b_mn = true;
    }
    if (outputs & kDw) {
      DenseProduct& d = p[count++];
      d.M = (int)N, d.N = (int)K, d.K = (int)M, d.batch = gated ? 2 : 1, d.a_mn = d.b_mn = true;
    }
  }
  const DenseShape s = dense_shape(p, count, outputs & kDb, num_sms);
  *kernel = s.bn ? 1 : 2, *width = s.bn ? s.bn : 256, *split0 = s.split[0], *split1 = s.split[1];
  *a_rows = s.ar, *ctas_per_sm = s.bn && !s.deep ? 2 : 1;
  return EAS_OK;
}

extern "C" int eas_dense_rows_plan(int op, uint32_t M, uint32_t N, uint32_t K, int unaligned, int num_sms, int* way,
                                   int* warps, int* split) {
  if (!way || !warps || !split) return eas_fail(EAS_ERR_VALUE, "eas_dense_rows_plan: null pointer");
  if (op != 0 && op != 1) return eas_fail(EAS_ERR_VALUE, "eas_dense_rows_plan: op must be 0 or 1");
  int rc = check_sizes("eas_dense_rows_plan", M, N, K, kF16, kNone);
  if (rc) return rc;
  if (M == 0 || num_sms <= 0 || !dense_rows_fit((int)M, (int)K))
    return eas_fail(EAS_ERR_VALUE, "eas_dense_rows_plan: no product of few rows");
  DenseProduct p;
  p.gated = op;
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  const DenseRowsShape c = dense_rows_shape(p, !(unaligned & (kXOff | kWOff | (op ? kUpOff : 0))), num_sms);
  *way = c.way, *warps = c.warps, *split = c.split;
  return EAS_OK;
}

extern "C" int eas_linear(const eas_linear_args* args, void* stream) {
  const char* who = "eas_linear";
  if (!args) return eas_fail(EAS_ERR_VALUE, "%s: null arguments", who);
  const void *const x = args->x, *const w = args->w, *const bias = args->bias, *const residual = args->residual;
  void *const y = args->y, *const pre = args->pre;
  const uint64_t ldx = args->ldx, ldw = args->ldw, ldr = args->ldr, ldy = args->ldy, ldp = args->ldp;
  const uint32_t M = args->M, N = args->N, K = args->K;
  const int dev = args->dev, dtype = args->dtype, act = args->act;
  void* const scratch = args->scratch;
  const uint64_t scratch_bytes = args->scratch_bytes;
  int rc = check_sizes(who, M, N, K, dtype, act);
  if (rc || M == 0) return rc;
  if (!x || !w || !y) return eas_fail(EAS_ERR_VALUE, "%s: null operand", who);
  rc = check_matrices(who, {{x, ldx, M, K}, {w, ldw, N, K}, {bias, N, 1, N}, {y, ldy, M, N}, {pre, ldp, M, N},
                            {residual, N, 1, N}});  // (the residual's rows may be one and the same)
  if (rc) return rc;
  const bool few = dense_rows_fit((int)M, (int)K);
  const int off = few ? 0 : off_mask(x, ldx, kXOff) | off_mask(w, ldw, kWOff);
  const Scratch sc = forward_scratch(false, M, N, K, off);
  if ((rc = check_scratch(who, sc, scratch, scratch_bytes))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceScope scope(dev);
  if (scope.rc) return scope.rc;
  Copies copies;
  const Operand X = copies.add(x, ldx, M, K, off & kXOff, scratch, sc.x, sc.ldk);
  const Operand W = copies.add(w, ldw, N, K, off & kWOff, scratch, sc.w, sc.ldk);
  if ((rc = copies.launch(s, who))) return rc;
  DenseProduct p;
  p.a[0] = X.p, p.lda[0] = X.ld, p.b[0] = W.p, p.ldb[0] = W.ld;
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  p.bias = u16(bias), p.residual = u16(residual), p.y[0] = u16(y), p.pre = u16(pre);
  p.ldr = ldr, p.ldy[0] = ldy, p.ldp = ldp;
  p.act = act, p.bf16 = dtype == kBF16;
  return few ? dense_rows(p, s, who) : dense_mma(&p, 1, DenseColSum(), s, who);
}

extern "C" int eas_gated(const eas_gated_args* args, void* stream) {
  const char* who = "eas_gated";
  if (!args) return eas_fail(EAS_ERR_VALUE, "%s: null arguments", who);
  const void *const x = args->x, *const w_gate = args->w_gate, *const w_up = args->w_up;
  void *const h = args->h, *const gate = args->gate, *const up = args->up;
  const uint64_t ldx = args->ldx, ldwg = args->ldwg, ldwu = args->ldwu, ldh = args->ldh, ldg = args->ldg, ldu = args->ldu;
  const uint32_t M = args->M, N = args->N, K = args->K;
  const int dev = args->dev, dtype = args->dtype, act = args->act;
  void* const scratch = args->scratch;
  const uint64_t scratch_bytes = args->scratch_bytes;
  int rc = check_sizes(who, M, N, K, dtype, act);
  if (rc || M == 0) return rc;
  if (!x || !w_gate || !w_up || !h) return eas_fail(EAS_ERR_VALUE, "%s: null operand", who);
  rc = check_matrices(who, {{x, ldx, M, K}, {w_gate, ldwg, N, K}, {w_up, ldwu, N, K}, {h, ldh, M, N}, {gate, ldg, M, N},
                            {up, ldu, M, N}});
  if (rc) return rc;
  if (!gate != !up) return eas_fail(EAS_ERR_VALUE, "%s: gate and up go together", who);
  const bool few = dense_rows_fit((int)M, (int)K);
  const int off = few ? 0 : off_mask(x, ldx, kXOff) | off_mask(w_gate, ldwg, kWOff) | off_mask(w_up, ldwu, kUpOff);
  const Scratch sc = forward_scratch(true, M, N, K, off);
  if ((rc = check_scratch(who, sc, scratch, scratch_bytes))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceScope scope(dev);
  if (scope.rc) return scope.rc;
  Copies copies;
  const Operand X = copies.add(x, ldx, M, K, off & kXOff, scratch, sc.x, sc.ldk);
  const Operand G = copies.add(w_gate, ldwg, N, K, off & kWOff, scratch, sc.w, sc.ldk);
  const Operand U = copies.add(w_up, ldwu, N, K, off & kUpOff, scratch, sc.up, sc.ldk);
  if ((rc = copies.launch(s, who))) return rc;
  DenseProduct p;
  p.gated = true;
  p.a[0] = X.p, p.lda[0] = X.ld, p.b[0] = G.p, p.ldb[0] = G.ld, p.b[1] = U.p, p.ldb[1] = U.ld;
  p.M = (int)M, p.N = (int)N, p.K = (int)K;
  p.y[0] = u16(h), p.pre = u16(gate), p.pre2 = u16(up);
  p.ldy[0] = ldh, p.ldp = ldg, p.ldp2 = ldu;
  p.act = act, p.bf16 = dtype == kBF16;
  return few ? dense_rows(p, s, who) : dense_mma(&p, 1, DenseColSum(), s, who);
}

extern "C" int eas_linear_backward(const eas_linear_backward_args* args, void* stream) {
  const char* who = "eas_linear_backward";
  if (!args) return eas_fail(EAS_ERR_VALUE, "%s: null arguments", who);
  const void *const dy = args->dy, *const pre = args->pre, *const x = args->x, *const w = args->w;
  void *const dx = args->dx, *const dw = args->dw, *const db = args->db;
  const uint64_t lddy = args->lddy, ldp = args->ldp, ldx = args->ldx, ldw = args->ldw, lddx = args->lddx, lddw = args->lddw;
  const uint32_t M = args->M, N = args->N, K = args->K;
  const int dev = args->dev, dtype = args->dtype, act = args->act;
  void* const scratch = args->scratch;
  const uint64_t scratch_bytes = args->scratch_bytes;
  int rc = check_sizes(who, M, N, K, dtype, act);
  if (rc) return rc;
  if ((M && !dy) || (M && act != kNone && !pre) || (dx && !w) || (M && dw && !x))
    return eas_fail(EAS_ERR_VALUE, "%s: null operand", who);
  rc = check_matrices(who, {{dy, lddy, M, N}, {pre, ldp, M, N}, {x, ldx, M, K}, {w, ldw, N, K}, {dx, lddx, M, K},
                            {dw, lddw, N, K}, {db, N, 1, N}});
  if (rc) return rc;
  const int outputs = (dx ? kDx : 0) | (dw ? kDw : 0) | (db ? kDb : 0);
  if (!outputs) return EAS_OK;
  const int off = off_mask(x, ldx, kXOff) | off_mask(w, ldw, kWOff) | off_mask(dy, lddy, kDyOff);
  const Scratch sc = backward_scratch(false, M, N, K, act, outputs, off);
  if (M && (rc = check_scratch(who, sc, scratch, scratch_bytes))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceScope scope(dev);
  if (scope.rc) return scope.rc;
  if (M == 0) {  // no rows: the sums over them are zero
    if (dw && (rc = zero_rows(dw, lddw, N, K, s, who))) return rc;
    if (db && (rc = zero_rows(db, N, 1, N, s, who))) return rc;
    return EAS_OK;
  }
  Copies copies;
  const Operand X = dw ? copies.add(x, ldx, M, K, off & kXOff, scratch, sc.x, sc.ldk) : Operand{};
  const Operand W = dx ? copies.add(w, ldw, N, K, off & kWOff, scratch, sc.w, sc.ldk) : Operand{};
  uint8_t* base = static_cast<uint8_t*>(scratch);
  uint16_t* dz = sc.need_dz ? reinterpret_cast<uint16_t*>(base + sc.dz) : nullptr;
  float* partial = db && !sc.direct ? reinterpret_cast<float*>(base + sc.partial) : nullptr;
  float* unscale = sc.ranged && dtype == kF16 ? reinterpret_cast<float*>(base + sc.unscale) : nullptr;
  if (dz || partial) {
    ActGrad g = {};
    g.dy = u16(dy), g.g = u16(pre), g.dg = dz, g.partial = partial;
    g.lddy = lddy, g.ldg = ldp, g.ldo = sc.ldn;
    g.M = M, g.N = N, g.rows_per_block = sc.rows, g.act = act, g.bf16 = dtype == kBF16;
    g.copies = copies.r;
    if (unscale) g.range = reinterpret_cast<Range*>(base + sc.range), g.unscale = unscale;
    rc = launch_act_grad<false>(g, sc.blocks, s, who);
  } else {
    rc = copies.launch(s, who);
  }
  if (rc) return rc;
  const Operand DZ = dz ? Operand{dz, sc.ldn} : Operand{u16(dy), lddy};
  DenseColSum sums;
  if (db) {
    sums.db = u16(db), sums.N = (int)N, sums.bf16 = dtype == kBF16;
    if (sc.direct)
      sums.matrix = u16(dy), sums.ld = (int64_t)lddy, sums.rows = (int)M;
    else
      sums.partial = partial, sums.rows = sc.blocks;
  }
  if (!dx && !dw) return dense_column_sums(sums, s, who);
  return backward_products(who, 1, {DZ, {}}, {W, {}}, X, dx, lddx, {dw, nullptr}, {lddw, 0}, sums, unscale, M, N, K, dtype,
                           s);
}

extern "C" int eas_gated_backward(const eas_gated_backward_args* args, void* stream) {
  const char* who = "eas_gated_backward";
  if (!args) return eas_fail(EAS_ERR_VALUE, "%s: null arguments", who);
  const void *const dh = args->dh, *const gate = args->gate, *const up = args->up, *const x = args->x, *const w_gate = args->w_gate, *const w_up = args->w_up;
  void *const dx = args->dx, *const dw_gate = args->dw_gate, *const dw_up = args->dw_up;
  const uint64_t lddh = args->lddh, ldg = args->ldg, ldu = args->ldu, ldx = args->ldx, ldwg = args->ldwg, ldwu = args->ldwu, lddx = args->lddx, lddwg = args->lddwg, lddwu = args->lddwu;
  const uint32_t M = args->M, N = args->N, K = args->K;
  const int dev = args->dev, dtype = args->dtype, act = args->act;
  void* const scratch = args->scratch;
  const uint64_t scratch_bytes = args->scratch_bytes;
  int rc = check_sizes(who, M, N, K, dtype, act);
  if (rc) return rc;
  if ((M && (!dh || !gate || !up)) || (dx && (!w_gate || !w_up)) || (M && (dw_gate || dw_up) && !x))
    return eas_fail(EAS_ERR_VALUE, "%s: null operand", who);
  rc = check_matrices(who, {{dh, lddh, M, N}, {gate, ldg, M, N}, {up, ldu, M, N}, {x, ldx, M, K}, {w_gate, ldwg, N, K},
                            {w_up, ldwu, N, K}, {dx, lddx, M, K}, {dw_gate, lddwg, N, K}, {dw_up, lddwu, N, K}});
  if (rc) return rc;
  const int outputs = (dx ? kDx : 0) | (dw_gate || dw_up ? kDw : 0);
  if (!outputs) return EAS_OK;
  const int off = off_mask(x, ldx, kXOff) | off_mask(w_gate, ldwg, kWOff) | off_mask(w_up, ldwu, kUpOff) |
                  off_mask(dh, lddh, kDyOff);
  const Scratch sc = backward_scratch(true, M, N, K, act, outputs, off);
  if (M && (rc = check_scratch(who, sc, scratch, scratch_bytes))) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  DeviceScope scope(dev);
  if (scope.rc) return scope.rc;
  if (M == 0) {
    if (dw_gate && (rc = zero_rows(dw_gate, lddwg, N, K, s, who))) return rc;
    if (dw_up && (rc = zero_rows(dw_up, lddwu, N, K, s, who))) return rc;
    return EAS_OK;
  }
  uint8_t* base = static_cast<uint8_t*>(scratch);
  const bool dw = outputs & kDw;
  Copies copies;
  const Operand X = dw ? copies.add(x, ldx, M, K, off & kXOff, scratch, sc.x, sc.ldk) : Operand{};
  const Operand G = dx ? copies.add(w_gate, ldwg, N, K, off & kWOff, scratch, sc.w, sc.ldk) : Operand{};
  const Operand U = dx ? copies.add(w_up, ldwu, N, K, off & kUpOff, scratch, sc.up, sc.ldk) : Operand{};
  uint16_t* dg = reinterpret_cast<uint16_t*>(base + sc.dz);  // need_dz: some output is asked for
  uint16_t* du = reinterpret_cast<uint16_t*>(base + sc.dz2);
  ActGrad g = {};
  g.dy = u16(dh), g.g = u16(gate), g.u = u16(up), g.dg = dg, g.du = du;
  g.lddy = lddh, g.ldg = ldg, g.ldu = ldu, g.ldo = sc.ldn;
  g.M = M, g.N = N, g.rows_per_block = sc.rows, g.act = act, g.bf16 = dtype == kBF16;
  g.copies = copies.r;
  float* unscale = dtype == kF16 ? reinterpret_cast<float*>(base + sc.unscale) : nullptr;
  if (unscale) g.range = reinterpret_cast<Range*>(base + sc.range), g.unscale = unscale;
  rc = launch_act_grad<true>(g, sc.blocks, s, who);
  if (rc) return rc;
  return backward_products(who, 2, {{dg, sc.ldn}, {du, sc.ldn}}, {G, U}, X, dx, lddx, {dw_gate, dw_up},
                           {lddwg, lddwu}, DenseColSum(), unscale, M, N, K, dtype, s);
}
