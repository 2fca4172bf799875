// dense_internal.h — the matrix products behind the dense-layer operators.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

// C = sum_t A_t B_t^T with an epilogue, on 16-bit matrices with f32 sums.
//   plain   z[m][n] = sum_{t < terms} sum_k A_t[m][k] B_t[n][k];  y = act(z + bias) + residual
//   gated   g = A_0 B_0^T, u = A_0 B_1^T;  y = act(g) u           (terms = 1)
//   batch 2 two products with one B: y_z = A_z B_0^T, z = 0, 1    (plain, terms = 1)
// A_t[m][k] is at a[t] + m lda[t] + k, or at a[t] + k lda[t] + m when a_mn; B_t likewise by n.
// Operand bases and pitches are multiples of 16 bytes; those of the other arrays are arbitrary.
// Forward products have K-major operands (neither a_mn nor b_mn) and one term; backward ones have b_mn
// and no epilogue but a factor, a power of two that was taken out of their first operands.
struct DenseProduct {
  const uint16_t* a[2] = {nullptr, nullptr};
  const uint16_t* b[2] = {nullptr, nullptr};
  uint64_t lda[2] = {0, 0}, ldb[2] = {0, 0};
  bool a_mn = false, b_mn = false, gated = false;
  int M = 0, N = 0, K = 0;
  int terms = 1, batch = 1;
  const uint16_t* bias = nullptr;
  const uint16_t* residual = nullptr;
  uint16_t* y[2] = {nullptr, nullptr};
  uint16_t* pre = nullptr;   // z, or g
  uint16_t* pre2 = nullptr;  // u
  uint64_t ldr = 0, ldy[2] = {0, 0}, ldp = 0, ldp2 = 0;
  const float* unscale = nullptr;  // of a backward launch: all sums are multiplied by it (null: by 1)
  int act = 0;
  bool bf16 = false;
};

// db[n] = the column sums of `rows` rows of N values, rounded to the type (db null: none wanted): of
// f32 partial sums, or of a matrix of the type itself.
struct DenseColSum {
  const float* partial = nullptr;
  const uint16_t* matrix = nullptr;
  int64_t ld = 0;  // of the matrix
  uint16_t* db = nullptr;
  int rows = 0, N = 0;
  bool bf16 = false;
};

int dense_column_sums(const DenseColSum& sums, cudaStream_t stream, const char* who);

// One forward product, or one or two backward ones (with column sums) that do not depend on one another.
int dense_mma(const DenseProduct* p, int count, const DenseColSum& sums, cudaStream_t stream, const char* who);

// The shape of kernel that dense_mma runs such products on.
struct DenseShape {
  int bn;        // 0: the pair kernel, else the single-CTA kernel's tile width
  int split[2];  // CTAs that share a tile's k-blocks, by product (the one of the longer sums first)
  int ar;        // rows of A staged
  bool deep;     // one CTA per SM
};
DenseShape dense_shape(const DenseProduct* p, int count, bool sums, int sms);

// The same for the forward products (K-major operands, one term, one product) of at most kDenseRows
// rows that fit in shared memory; operands of any alignment.
constexpr int kDenseRows = 8;
bool dense_rows_fit(int M, int K);
struct DenseRowsShape {
  int way;    // of reading W: 0 words of its rows, 1 words that are shifted, 2 values
  int warps;  // per block: 8 (two blocks per SM) or 16
  int split;  // CTAs of a cluster that share K
};
DenseRowsShape dense_rows_shape(const DenseProduct& p, bool aligned, int sms);
int dense_rows(const DenseProduct& p, cudaStream_t stream, const char* who);
