// Dense products of 16-bit matrices with a fused end, on tcgen05 (dense_dev.cuh): what their callers hand over.
#pragma once
#include <cuda.h>
#include "common.cuh"

namespace xkb {
namespace dense {

// What a product's accumulators become.
constexpr int kStore = 0;     // D, rounded to 16 bits; or kept / added to in fp32
constexpr int kSwiglu = 1;    // gate and up of the same column side by side: silu(gate) * up, and both if they are kept
constexpr int kDswiglu = 2;   // D is the gradient of silu(gate) * up: the gradients of both, and the product itself
constexpr int kCeStats = 3;   // D are logits: maximum and sum of exponentials of a row's piece, the label's logit
constexpr int kCeGrad = 4;    // D are logits: their gradient, rounded to 16 bits
// The launcher's choices: kStore of sums so long that they are added up in parts; the two gradients with second terms (End::second).
constexpr int kStoreLong = 5, kDswigluTwo = 6, kCeGradTwo = 7;

constexpr int kMaxProblems = 3;

// One product D[M, N] = A[M, K] B[N, K]^T.  Either operand lies in memory as its own rows (K contiguous) or as K rows
// (its own index contiguous).
struct Operand {
  const void* base;
  int64_t pitch;      // elements from one row in memory to the next, a multiple of 8; the base is 16-byte aligned
  bool k_rows;        // rows in memory are K
  int64_t row0;       // first row in memory (B of a piece of the vocabulary)
  int64_t rows, cols; // extents in memory; what lies outside reads as 0
  int64_t rest;       // elements to a second term of the same form (left operand of kStore, up to 64 rows; 0: none)
};

struct End {
  void* out;            // 16-bit
  int64_t ld;
  const int32_t* row_map;   // row of `out` for every row of D, nullptr: the same
  const float* scale;       // factor of D on the device, nullptr: 1
  float* acc;               // fp32 [k_parts, M, acc_ld]
  int64_t acc_ld, acc_part; // acc_part: elements from one part to the next
  int acc_in, acc_out;      // add what acc holds; write there and not to out
  // kSwiglu, kDswiglu
  void* h;
  int64_t ld_h;
  void* h_rest;             // kSwiglu: what the rounding left of h, rounded itself (nullptr: not wanted)
  void* gate_up;            // [M, 2 * half]
  int64_t ld_gu;
  int half;                 // columns of gate, which are in front of those of up
  float limit;
  // kCeStats, kCeGrad: arrays over the rows of D
  const int32_t* labels;
  const int64_t* labels64;  // kCeStats: in place of labels
  float2* part;             // [M, parts]
  int64_t part_ld;
  float* given;
  const float4* coef;       // m, l, factor of p, what is taken off at the label
  int col0;                 // first column of the piece in the vocabulary
  // kDswiglu, kCeGrad: what the rounding of row r left, itself rounded, is written to row second + r.  kStore: row second + r of D
  // is added to row r.  (0: one term.  16 at most, and no more rows.)
  int second;
  // which vector accesses their rows allow (bytes: 16 or 2), set by the launcher
  int vec_out, vec_h, vec_gu;
  int tma_out;          // rows of `out` leave by copies of 64 columns, set by the launcher
};

struct Product {
  Operand a, b;
  int64_t M, N, K;
  int k_parts;          // kStore with acc_out: K is taken in so many parts, a tile each (0: one)
  const int32_t* live;  // on the device: how many of M's rows (of K's, if a.k_rows) there are, nullptr: all
  End end;
};

// Launches `count` products with the same end and the same orientation of B as one kernel.  `chained`: may start while
// its predecessor on the stream runs (common.cuh); `early_b`: B is no output of a kernel of the same call.
int launch(const Product* products, int count, int end, int dtype, bool chained, bool early_b, cudaStream_t stream);
// In how many parts to take K of the first of two products [M0, N0, K0] (few long tiles) and [M1, N1, K1] (many short ones,
// or none) that one launch deals out, so that the long ones do not outlast the rest.
int k_parts_of(int64_t M0, int64_t N0, int64_t K0, int64_t M1, int64_t N1, int64_t K1);
// How many pieces a row's statistics come in (kCeStats), and no more than how many.
int ce_parts(int64_t M, int64_t N, int64_t K, int* parts);
int64_t ce_most_parts(int64_t M, int64_t N);
// xkb_lay_out_rows; exponent_host, if not null: bits of a type's exponent, for copies in which infinities and NaN become 0 (0: they stay).
int lay_out(const void* const* from_host, const int64_t* ld_host, const int64_t* rows_host, const int64_t* cols_host, void* const* to_host,
            const int* exponent_host, int count, cudaStream_t stream);

}  // namespace dense
}  // namespace xkb
