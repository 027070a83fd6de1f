// Products with one 16-bit or 4-bit weight: what linear_kernel.h's parts (linear_dense.hip, linear_q4.hip, linear_turned.hip)
// and their callers (linear.hip) share.
#pragma once

#include "moe_gemm.h"

namespace usaf {

// out[m, n] = dt( sum_k A[m, k] W[n, k] ), or with kept or gated set the gate and up product below.
struct LinArgs {
  const uint8_t* A;    // 16-bit rows, lda bytes apart (16-byte aligned, lda too)
  int64_t lda;
  int64_t M, K;        // K % 64 == 0 (4-bit: % 128)
  const uint8_t* W;    // 16-bit rows or packed codes, ldw bytes apart (16-byte aligned, ldw too)
  int64_t ldw;
  const uint32_t* sz;  // 4-bit: scale | zero << 16 of every group of 128, [K / 128, rows]
  int64_t N;           // columns of out; gated: W has 2 N rows, the gate's and then up's
  uint16_t* out;       // [M, ldo], act where gated
  int64_t ldo;
  // gated: what a backward reads (linear.hip), or nullptr
  void* kept;          // [M, 2, hs]: 16-bit values, hs = N in whole 8, or codes, hs = N in whole 128
  uint8_t* kept_s;     // scale bytes [M, 2, hs / 128] of codes; nullptr: 16-bit values
  int64_t hs;
  int n_nt;            // set at the launch
  // not gated: the contraction in parts, each part's fp32 sums [parts, M, ldp] to part instead of out
  int parts = 1;
  float* part = nullptr;
  int64_t ldp = 0;     // N in whole 4
};

// The tile for a product of these sizes, how many parts its contraction is taken in, and about how long it takes.
struct LinPlan {
  int (*launch)(const LinArgs&, int dt, bool gated, hipStream_t) = nullptr;
  int parts = 1;
  double us = 0;
  int rows = 0, w_rows = 0;  // of the tile: of A, of W
};
LinPlan plan_linear_dense(const LinArgs& g, bool gated);
LinPlan plan_linear_q4(const LinArgs& g, bool gated);
// C = A W of W [K, N] (both: C = A^T W of A [K, M] too), lda and ldw the distances of these rows; K % 64 == 0, N (M) % 8 == 0.
LinPlan plan_linear_turned(const LinArgs& g, bool both);
// A few rows of a 4-bit weight's product, out [M, N] (ldo = N), nothing kept: whether it takes them, and its launch (q4_small.hip).
bool q4_small_ok(int64_t M, int64_t N, int64_t K);
int q4_small(const LinArgs& g, int dt, bool gated, hipStream_t st);
void prepare_q4_small();
void prepare_linear_dense();
void prepare_linear_q4();
void prepare_linear_turned();
// Raises the products' dynamic-LDS limits, once per process (usaf_hip_init, or their first use).
void prepare_linear_kernels();

}  // namespace usaf
