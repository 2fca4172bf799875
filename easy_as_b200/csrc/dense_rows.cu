// dense_rows.cu — the dense layers' forward products for a few rows (decoding steps).
//
//   plain   z[m][n] = sum_k x[m][k] W[n][k];  y = act(z + bias) + residual
//   gated   g = x Wg^T, u = x Wu^T;  y = act(g) u
//
// With so few rows the product reads W once and does almost nothing with it: the bound is HBM, and
// what counts is to keep bytes under way with few instructions.  Each warp copies 16 rows x 64 values
// at a time into a queue of its own in shared memory (cp.async), several pieces ahead, and hands them
// to mma.sync from there.  A warp reads only what it copied itself, so the queue needs no barrier
// between warps.  x lies in shared memory whole.  Rows of W are the instruction's 16 rows (gated: 8 of
// the gate, 8 of the up projection), rows of x its 8 columns.  Its k order is a convention between the
// two operands: lane t of a quad takes k = 8t .. 8t+7 of 32, as it lies in memory, and hands words 0-1
// to one m16n8k16 and words 2-3 to the next, on both operands alike.
//
// Rows that do not start on 16 bytes are copied as the aligned words that hold them, one more per row
// and piece, and shifted into place on their way from the queue to the instruction (4096 x 4096, one
// row: 7.8 us; K = 4095: 11.0, and 15.2 with 8 rows; loaded value by value they take 24).  Of less than
// 4 MB of weights they are loaded value by value straight into registers: that starts 2 us sooner (576 x
// 123 gated: 2.8 us, against 4.5; 3912 x 1000: 6.7, against 7.1; gated 3272 x 1408: 16.1, against 14.1).
//
// Two blocks of 8 warps stay on each SM (or one of 16, where x needs the room), each with an equal
// share of W's rows (N / 296 of them, give or take one, so that no SM has more to read than another),
// in tiles of at most 16 (gated: 8 of each weight).  The warps take every 8th (16th) 64-wide piece of K,
// and the queue runs on over the tiles' ends.  Where a share would be too few rows for a tile, the CTAs
// of a cluster share the rows of several and split K.  The sums of the warps, then of the cluster's
// CTAs, are added in a fixed order through (distributed) shared memory, so results are the same bits
// on every run.
#include <cuda_runtime.h>
#include <stdint.h>

#include "dense_internal.h"
#include "dense_launch.h"
#include "dense_math.cuh"
#include "eas_internal.h"
#include "tcgen05_ptx.cuh"

namespace {

using namespace dense;

struct RowsParams {
  const uint16_t* x;
  const uint16_t* w[2];
  const uint16_t *x_end, *w_end[2];  // past their last values
  const uint16_t* bias;
  const uint16_t* residual;
  uint16_t* y;
  uint16_t* pre;
  uint16_t* pre2;
  int64_t ldx, ldw[2], ldr, ldy, ldp, ldp2;
  int M, N, K, split, act;
};

template <bool BF16>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// 8 values of a row, of which `n` are left: zeros past them.
__device__ __forceinline__ uint4 load8(const uint16_t* p, int n) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t lo = 2 * j < n ? p[2 * j] : 0, hi = 2 * j + 1 < n ? p[2 * j + 1] : 0;
    w[j] = lo | (hi << 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

__device__ __forceinline__ void copy16(uint32_t dst, const uint16_t* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Copy 16 bytes past L1, of which the row has `n` values left: zeros past them.
__device__ __forceinline__ void copy8(uint32_t dst, const uint16_t* src, int n) {
  const int bytes = n >= 8 ? 16 : n > 0 ? 2 * n : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}

constexpr int kPiece = 64;       // values of K per row and piece

// How W comes: by words of its rows, which start on 16 bytes; by words that are shifted; value by value.
enum Way { kWords, kShifted, kValues };

// W warps per block, and of x in shared memory: two blocks of 8 warps per SM, or one of 16 with twice
// the room for x.  A slot holds a piece of 16 rows of W: 8 words
// each, and behind them (shifted) the 16 rows' ninth ones.
template <int W, Way WAY>
struct Shape {
  static constexpr int kSlot = 16 * 128 + (WAY == kShifted ? 16 * 16 : 0);
  static constexpr int kPieces = WAY == kWords ? 4 : 3;      // per warp
  static constexpr int kDepth = kPieces - 1;       // under way while one is consumed
  static constexpr int kQueue = WAY == kValues ? 0 : W * kPieces * kSlot;  // 64 or 54 KB, or twice that
};

template <int W>
constexpr int kMostX = W == 8 ? 40960 : 81920;

// x in shared memory: rows of whole pieces, 64 bytes apart modulo 128, so that the quads of a
// quarter warp read different banks.
__host__ __device__ constexpr int64_t x_pitch(int64_t K) { return (K + kPiece - 1) / kPiece * (2 * kPiece) + 64; }

template <int kWarps, bool GATED, Way WAY, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, 16 / kWarps)
    dense_rows_kernel(const __grid_constant__ RowsParams p) {
  constexpr int kTile = GATED ? 8 : 16;  // outputs; always 16 rows of W
  constexpr int kRows = kDenseRows, kCols = 16;
  constexpr bool VEC = WAY == kWords;
  using Q = Shape<kWarps, WAY>;
  constexpr int kSlot = Q::kSlot, kDepth = Q::kDepth;
  extern __shared__ __align__(128) uint8_t queue[];
  __shared__ float part[2][kWarps][kRows][kCols + 1];  // tiles take turns
  __shared__ float sums[kRows][kCols + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int S = p.split;
  const int rank = (int)blockIdx.x % S;
  const int64_t group = blockIdx.x / S, groups = gridDim.x / S;
  const int lo = (int)(group * p.N / groups), hi = (int)((group + 1) * p.N / groups);
  const int tiles = (hi - lo + kTile - 1) / kTile;
  auto tile_row = [&](int j) { return lo + (int)((int64_t)j * (hi - lo) / max(tiles, 1)); };  // equal tiles
  const int stride = kPiece * kWarps * S;
  const int first = kPiece * (rank * kWarps + warp);

  // Copies go 4 rows of W at a time, 8 lanes and so a whole 128-byte line per row (64 bytes of each
  // row at a time, the way the lanes read them, every line crossed from L2 twice: 273 MB for 134).
  // Chunk c of a row lies at place c ^ 4 (row & 1), so that two rows' quads read different banks.
  // Rows past the tile are not copied: whatever their place in the queue holds reaches only sums
  // that nobody looks at.
  // (Shifted: 9 words of each row, in the order of the lanes.)
  constexpr int kCopies = VEC ? 4 : 5;
  auto copy_row = [&](int i) { return VEC ? (lane >> 3) + 4 * i : (lane + 32 * i) / 9; };
  auto copy_word = [&](int i) { return VEC ? lane & 7 : (lane + 32 * i) % 9; };
  auto word_at = [](int r, int c) { return c == 8 ? 2048 + 16 * r : r * 128 + ((c ^ (4 * (r & 1))) << 4); };
  auto lag = [](const uint16_t* at) { return VEC ? 0 : (int)(reinterpret_cast<uintptr_t>(at) >> 1) & 7; };
  auto w_row = [&](int r, int n0, int n1) {  // row r of a tile's 16
    const int n = n0 + (GATED ? r & 7 : r), h = GATED && r >= 8;
    return p.w[h] + (int64_t)(n < n1 ? n : n0) * p.ldw[h];
  };
  const uint16_t* w[kCopies];
  int have = 0;
  int left_of[kCopies];  // (shifted) values of K behind the word's first
  auto aim = [&](int n0, int n1) {
    if (WAY == kValues) return;
    have = 0;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int r = min(copy_row(i), 15), c = copy_word(i);
      const uint16_t* at = w_row(r, n0, n1);
      const int s = lag(at);
      const bool use = copy_row(i) < 16 && n0 + (GATED ? r & 7 : r) < n1 && (c < 8 || s);
      have |= (use ? 1 : 0) << i;
      w[i] = at - s + 8 * c;
      left_of[i] = p.K - 8 * c + s;
    }
  };
  const int xrow = min(g, p.M - 1);

  grid_order();

  const uint32_t mine = tc::smem_u32(queue) + warp * (Q::kPieces * kSlot);
  const uint32_t take = mine + word_at(g, t);  // v = 1: ^ 64; row g + 8: + 1024
  // (shifted) the words behind those, of rows g and g + 8
  const uint32_t next0 = mine + word_at(g, t + 1), next1[2] = {mine + word_at(g, t + 5), mine + word_at(g + 8, t + 5)};
  const int64_t pitch = x_pitch(p.K);
  const uint32_t xs = tc::smem_u32(queue) + Q::kQueue;
  const uint32_t xmine = xs + (uint32_t)(xrow * pitch) + 16 * t;
  int in_tile = 0, in_k = first, in_slot = 0, out_slot = 0;
  if (tiles > 0) aim(tile_row(0), tile_row(1));
  auto issue = [&]() {  // always one group, empty past the end: the waits count groups
    if (WAY != kValues && in_tile < tiles && in_k < p.K) {
      const uint32_t at = mine + in_slot * kSlot;
      if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const uint32_t dst = at + word_at(copy_row(i), copy_word(i));
          const int h = GATED && copy_row(i) >= 8;
          const uint16_t* src = w[i] + in_k;
          if (!(have >> i & 1) || in_k >= left_of[i]) continue;
          if (src >= p.w[h] && src + 8 <= p.w_end[h]) {
            copy16(dst, src);
          } else {  // reaches out of the matrix's memory
            for (int j = 0; j < 8; ++j)
              if (src + j >= p.w[h] && src + j < p.w_end[h])
                asm volatile("st.shared.u16 [%0], %1;" ::"r"(dst + 2 * j), "h"(src[j]) : "memory");
          }
        }
      } else if (in_k + kPiece <= p.K) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
          if (have >> i & 1) copy16(at + word_at(copy_row(i), copy_word(i)), w[i] + in_k);
      } else {  // zeros past the end of K
        const int left = p.K - in_k - 8 * copy_word(0);
#pragma unroll
        for (int i = 0; i < kCopies; ++i)
          copy8(at + word_at(copy_row(i), copy_word(i)), w[i] + (left > 0 ? in_k : 0), left);
      }
      in_slot = in_slot == kDepth ? 0 : in_slot + 1;
      in_k += stride;
      if (in_k >= p.K) {
        in_k = first;
        if (++in_tile < tiles) aim(tile_row(in_tile), tile_row(in_tile + 1));
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  if constexpr (WAY != kValues) {
    // x once per block: from every warp's piece it would be read by all SMs at the same time, and
    // its few lines of L2 were what the kernel waited for (4 rows: 44 us where one took 34)
    const int words = (int)((pitch - 64) / 16);
    for (int e = threadIdx.x; e < p.M * words; e += kWarps * 32) {
      const int r = e / words, c = e % words;
      const int left = p.K - 8 * c;
      const uint16_t* src = p.x + (int64_t)r * p.ldx + (left > 0 ? 8 * c : 0);
      const uint32_t dst = xs + (uint32_t)(r * pitch) + 16 * c;
      if constexpr (VEC) {
        copy8(dst, src, left);
      } else {
        Gather8 from;
        from.fetch(src, left, p.x, p.x_end);
        const uint4 v = from.get();
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                     : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
    for (int i = 0; i < kDepth; ++i) issue();
    asm volatile("cp.async.wait_group %0;" ::"n"(kDepth) : "memory");
    __syncthreads();
  }

  for (int j = 0; j < tiles; ++j) {
    const int n0 = tile_row(j), width = tile_row(j + 1) - n0;
    int shift[2];  // of rows g and g + 8
#pragma unroll
    for (int i = 0; i < 2; ++i) shift[i] = lag(w_row(g + 8 * i, n0, n0 + width));
    const uint16_t* row[2] = {w_row(g, n0, n0 + width) + 8 * t, w_row(g + 8, n0, n0 + width) + 8 * t};
    float acc[4] = {};
    for (int k = first; k < p.K; k += stride) {
      uint32_t slot = 0;
      if constexpr (WAY != kValues) {
        asm volatile("cp.async.wait_group %0;" ::"n"(kDepth - 1) : "memory");
        __syncwarp();  // the piece is here, and everyone has read the one before it
        issue();
        slot = out_slot * kSlot;
        out_slot = out_slot == kDepth ? 0 : out_slot + 1;
      }
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint4 a[2];
        uint4 b;
        const int left = p.K - k - 32 * v - 8 * t;
        if constexpr (WAY == kValues) {
#pragma unroll
          for (int i = 0; i < 2; ++i) a[i] = load8(row[i] + k + 32 * v, left);
          b = load8(p.x + (int64_t)xrow * p.ldx + 8 * t + k + 32 * v, left);
        } else {
          b = lds128(xmine + 2 * k + v * 64);
          a[0] = lds128((take + slot) ^ (v * 64));
          a[1] = lds128(((take + slot) ^ (v * 64)) + 1024);
        }
        if constexpr (WAY == kShifted) {
          const uint4 c0 = lds128((v ? next1[0] : next0) + slot), c1 = lds128((v ? next1[1] : next0 + 1024) + slot);
          a[0] = shift8(a[0], c0, shift[0]);
          a[1] = shift8(a[1], c1, shift[1]);
          if (k + kPiece > p.K) {  // what lies behind the row's end
            a[0] = first8(a[0], left);
            a[1] = first8(a[1], left);
          }
        }
        const uint32_t a0[4] = {a[0].x, a[1].x, a[0].y, a[1].y};
        const uint32_t a1[4] = {a[0].z, a[1].z, a[0].w, a[1].w};
        __syncwarp();  // the copies and loads above may have split the warp, and the instruction is .aligned
        mma_16816<BF16>(acc, a0, b.x, b.y);
        mma_16816<BF16>(acc, a1, b.z, b.w);
      }
    }
    auto& mine_part = part[j & 1];
#pragma unroll
    for (int c = 0; c < 4; ++c) mine_part[warp][2 * t + (c & 1)][8 * (c >> 1) + g] = acc[c];
    __syncthreads();
    const int rows = p.M;
    if (S > 1) {
      for (int e = threadIdx.x; e < rows * kCols; e += kWarps * 32) {
        float s = 0;
#pragma unroll
        for (int v = 0; v < kWarps; ++v) s += mine_part[v][e / kCols][e % kCols];
        sums[e / kCols][e % kCols] = s;
      }
      tc::cluster_sync_all();
    }
    // this CTA's share of the tile's outputs
    const int e = threadIdx.x * S + rank;
    const int r = e / kTile, c = e % kTile, n = n0 + c;
    if (r < rows && c < width) {
      float z = 0, u = 0;
      if (S == 1) {
#pragma unroll
        for (int v = 0; v < kWarps; ++v) {
          z += mine_part[v][r][c];
          if (GATED) u += mine_part[v][r][c + 8];
        }
      } else {
        const uint32_t at = tc::smem_u32(&sums[r][c]);
        for (int s = 0; s < S; ++s) {
          const uint32_t from = tc::mapa_rank(at, (uint32_t)s);
          z += tc::ld_cluster_f32(from);
          if (GATED) u += tc::ld_cluster_f32(from + 4 * 8);
        }
      }
      if (!GATED && p.bias) z += to_f32<BF16>(p.bias[n]);
      if (p.pre) p.pre[r * p.ldp + n] = to_16<BF16>(z);
      float v = 0;
      with_act(p.act, [&](auto a) { v = act<decltype(a)::value>(z); });
      if (GATED) {
        if (p.pre2) p.pre2[r * p.ldp2 + n] = to_16<BF16>(u);
        v *= u;
      } else if (p.residual) {
        v += to_f32<BF16>(p.residual[r * p.ldr + n]);
      }
      p.y[r * p.ldy + n] = to_16<BF16>(v);
    }
    if (S > 1) tc::cluster_sync_all();  // nobody overwrites its sums, or leaves, while they are being read
  }
}

// Weights that are shifted rather than loaded value by value, where their rows do not start on 16 bytes.
constexpr int64_t kShiftFrom = 2 << 20;

bool aligned16(const void* p, uint64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld & 7) == 0; }

// CTAs that split K: two where each block's share of the rows would fill less than half a tile and
// K is long (1024 x 8192, one row: 7.9 us whole, 6.9 in two, 10.2 in four; 512 x 4096: 5.1, 5.1, 7.6).
int choose_split(const DenseProduct& p, int blocks, int warps) {
  const int tile = p.gated ? 8 : 16;
  return (int64_t)p.N < (int64_t)blocks * tile / 2 && p.K >= 8 * kPiece * warps ? 2 : 1;
}

// How a product's launch is made up; `aligned`: every row of x and W starts on 16 bytes.
DenseRowsShape choose_rows(const DenseProduct& p, bool aligned, int sms) {
  DenseRowsShape c;
  c.way = aligned ? kWords : (int64_t)p.N * p.K * (p.gated ? 2 : 1) < kShiftFrom ? kValues : kShifted;
  c.warps = c.way == kValues || p.M * x_pitch(p.K) <= kMostX<8> ? 8 : 16;
  c.split = choose_split(p, 16 / c.warps * sms, c.warps);
  return c;
}

template <int W, bool GATED, Way WAY, bool BF16>
int launch_rows(const DenseProduct& p, RowsParams& q, int split, int dev, cudaStream_t s, const char* who) {
  static bool ready[64] = {false};
  const void* kernel = reinterpret_cast<const void*>(&dense_rows_kernel<W, GATED, WAY, BF16>);
  constexpr int kQueue = Shape<W, WAY>::kQueue;
  if (WAY != kValues && !ready[dev & 63]) {
    int rc = eas_cuda_check(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kQueue + kMostX<W>),
                            who, EAS_ERR_LAUNCH);
    if (rc) return rc;
    ready[dev & 63] = true;
  }
  const int resident = 16 / W * dense_sms(dev);
  q.split = split;
  // no block without rows; four rows a block or more, where there are few
  int groups = resident / q.split;
  if (groups > (p.N + 3) / 4) groups = (p.N + 3) / 4;
  return dense_launch(kernel, dim3(groups * q.split), q.split > 1 ? q.split : 0, W * 32,
                      WAY == kValues ? 0 : kQueue + q.M * (int)x_pitch(q.K), s, &q, who);
}

template <int W, Way WAY>
int launch_rows(const DenseProduct& p, RowsParams& q, int split, int dev, cudaStream_t s, const char* who) {
  if (p.bf16)
    return p.gated ? launch_rows<W, true, WAY, true>(p, q, split, dev, s, who)
                   : launch_rows<W, false, WAY, true>(p, q, split, dev, s, who);
  return p.gated ? launch_rows<W, true, WAY, false>(p, q, split, dev, s, who)
                 : launch_rows<W, false, WAY, false>(p, q, split, dev, s, who);
}

}  // namespace

DenseRowsShape dense_rows_shape(const DenseProduct& p, bool aligned, int sms) { return choose_rows(p, aligned, sms); }

bool dense_rows_fit(int M, int K) { return M <= kDenseRows && M * x_pitch(K) <= kMostX<16>; }

int dense_rows(const DenseProduct& p, cudaStream_t stream, const char* who) {
  int dev = 0;
  int rc = eas_cuda_check(cudaGetDevice(&dev), who, EAS_ERR_UNAVAILABLE);
  if (rc) return rc;
  RowsParams q = {};
  q.x = p.a[0], q.w[0] = p.b[0], q.w[1] = p.b[1];
  q.bias = p.bias, q.residual = p.residual, q.y = p.y[0], q.pre = p.pre, q.pre2 = p.pre2;
  q.ldx = (int64_t)p.lda[0], q.ldw[0] = (int64_t)p.ldb[0], q.ldw[1] = (int64_t)p.ldb[1];
  q.ldr = (int64_t)p.ldr, q.ldy = (int64_t)p.ldy[0], q.ldp = (int64_t)p.ldp, q.ldp2 = (int64_t)p.ldp2;
  q.M = p.M, q.N = p.N, q.K = p.K, q.act = p.act;
  q.x_end = q.x + (q.M - 1) * q.ldx + q.K;
  for (int i = 0; i < (p.gated ? 2 : 1); ++i) q.w_end[i] = q.w[i] + (q.N - 1) * q.ldw[i] + q.K;
  const bool aligned = aligned16(p.a[0], p.M > 1 ? p.lda[0] : 0) && aligned16(p.b[0], p.N > 1 ? p.ldb[0] : 0) &&
                       (!p.gated || aligned16(p.b[1], p.N > 1 ? p.ldb[1] : 0));
  const DenseRowsShape c = choose_rows(p, aligned, dense_sms(dev));
  if (c.way == kValues) return launch_rows<8, kValues>(p, q, c.split, dev, stream, who);
  if (c.way == kWords)
    return c.warps == 8 ? launch_rows<8, kWords>(p, q, c.split, dev, stream, who)
                        : launch_rows<16, kWords>(p, q, c.split, dev, stream, who);
  return c.warps == 8 ? launch_rows<8, kShifted>(p, q, c.split, dev, stream, who)
                      : launch_rows<16, kShifted>(p, q, c.split, dev, stream, who);
}
