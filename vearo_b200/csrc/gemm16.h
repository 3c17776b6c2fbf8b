// Products of f32 matrices held as half-precision pairs (split16.cuh), and the forms of the vocabulary product that the
// projection-with-loss needs (gemm16.cu).
#pragma once
#include <cuda.h>
#include "common.h"

namespace vb {

// [rows, cols] as two half planes (hi, then lo `plane` halves later), rows `ld` halves apart; inv: 2^-e of each 128 x 128 block, [row
// block][column block], or of 128 columns of each row, [column block][row], or of 128 rows of each column, [row block][column].  By row (by column), a
// row keeps its bits beside one that is many times as large: for the M side of a product over its columns (rows), where a row's scale costs nothing.
enum class Scale16 { Block, Row, Column };
struct Split16 { void* planes; float* inv; i64 rows, cols, ld, plane, inv_ld; Scale16 scale; };
inline size_t split16_bytes(i64 rows, i64 cols, Scale16 scale = Scale16::Block) {
  const i64 ld = (cols + 7) / 8 * 8, rb = (rows + 127) / 128, cb = (cols + 127) / 128;
  return (size_t)(2 * rows * ld) * 2 + 16 + (size_t)(scale == Scale16::Row ? rows * cb : scale == Scale16::Column ? rb * ld : rb * cb) * sizeof(float);
}
Split16 split16_at(void* mem, i64 rows, i64 cols, Scale16 scale = Scale16::Block);                // lays the pair out in memory of that size
constexpr int kNoTarget = -(1 << 30);
struct SplitJob { const float* x; Split16 to; const int* keep = nullptr; };                       // x: [rows, cols] contiguous; keep[row] == kNoTarget: read as 0
// Target columns given as floats, one a row of the first job: as integers to `out`.  `zero`: ints that the launch sets to 0.
struct TargetRows { const float* targets; i64 ignore, vocab; int* out; int* zero; int n_zero; };
int launch_split16(const SplitJob* jobs, int n, const TargetRows* rows = nullptr);                // n <= 3, one launch

// What a product does with its tiles.
enum class Tile16 {
  Store,      // out (+)= alpha * product
  RowStats,   // per row and 128 columns the (max, sum of exp) of the product, and the product at the row's target column
  LossGrad    // exp(product - lse) - [column is the target] as half planes (rows without a target: 0): times 2^14, and with a scale for 128 rows of a column
};
// out[m, n] = sum_k A[m, k] B[n, k].  An operand is K-major ([mn, k] in memory) or, mn true, [k, mn] in memory; its extents and
// scales are those of the Split16 (inv null: all 1).
struct Op16 { Split16 s; bool mn; };
struct Product16 {
  Op16 a, b;
  i64 M, N, K;
  // Store
  float* out; i64 ldo; bool add;
  const float* alpha; float alpha_host;          // alpha (device, null: 1) times alpha_host
  // RowStats / LossGrad
  const int* target;                             // [M] column of the row's target, kNoTarget: none (LossGrad: the row is left out)
  i64 col0;                                      // what the target columns call column 0 of this product
  float2* stats;                                 // [ceil(N / 128), M]
  float* target_value;                           // [M], written where the target lies in this product
  const float* lse;                              // [M]
  Split16 grad, grad_by_column;                  // [M, N]; planes null: not wanted.  grad holds 2^14 times the values and has no scales
};
// n <= 2 (Store), independent of one another, one launch (and one for each whose long sums are formed in parts); counter: an int on the device that is 0 when the launch begins.  The RowStats
// kernel is launched by launch_early and waits for the kernel ahead of it by itself.
int launch_gemm16(Tile16 what, const Product16* products, int n, int* counter);

}  // namespace vb
