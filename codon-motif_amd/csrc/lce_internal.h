// Softmax cross entropy straight from hidden states X [N, d] and the vocabulary's rows W [V, d]
// (linear_ce.hip: the entries and the row kernels; lce_general.hip: the products of fp32 inputs;
// lce_bf16.hip: those of bf16).
//
// With z_iv = x_i . w_v, s_i the gradient of row i's loss and t_i its label:
//   loss_i = log sum_v e^{z_iv} - z_{i t_i}
//   P_iv   = s_i (e^{z_iv} / sum_u e^{z_iu} - [v = t_i]),  dX = P W,  dW = P^T X
// Where all s_i are one number (sum, mean), it multiplies dX and dW instead: P rounded to bf16 with a
// factor 1 / 15565 in it was off by the same quarter of a percent in every row.
// The forward keeps one number per row (the base-2 log-sum-exp); the backward forms P again in
// pieces of the vocabulary and multiplies each piece on both sides.  Rows without a label are
// taken out first: every product runs over the `count` rows that have one, in their order.
#pragma once

#include "capi_internal.h"
#include "common.h"

namespace motif {

struct LceArgs {
  const void *x;       // [count, ldx]: the labelled rows
  const void *w;       // [V, d], row stride ldw
  int64_t ldx, ldw;
  int N, d, V, dk;     // dk: columns of x and w that the bf16 kernels read (d, or with zeros up to a multiple of 8)
  const int *row;      // [N] original row of labelled row i
  const int *label;    // [N] its label (-1: outside the vocabulary; loss and gradient are NaN)
  const int *pos;      // [N] labelled position of original row r, or -1
  const int *count;    // labelled rows
  float *part_m, *part_s;  // [nparts, N] maxima (times log2 e) and sums of a vocabulary part
  float *at_label;     // [N] z at the label
  float *lse;          // [N] base-2 log-sum-exp of z log2 e
  const float *dloss;  // gradient of the loss(es)
  int64_t dl_st;       // 0: one for all rows
  int reduction;       // 0: a gradient per row, 1: sum, 2: mean over count
  void *p;             // P of a vocabulary piece (layout: the kernels' own)
  int v0, vc, vn;      // the piece: first vocabulary row, rows laid out, rows of the vocabulary in it
  float *dx_part;      // partial dX, fp32: see lce_dx_shares
  int64_t n_pad;
  int dx_splits, dx_tiles, first;  // first: the first piece (nothing to add to)
  void *dw;            // [V, d]
};

// A launch has less than 2^32 threads along x: workgroups beyond kGridX go along y, in the same order.
constexpr int64_t kGridX = 1 << 21;
inline dim3 lce_grid(int64_t n) {
  const int64_t x = n < kGridX ? n : kGridX;
  return dim3(static_cast<unsigned>(x), static_cast<unsigned>((n + x - 1) / x));
}
__device__ __forceinline__ int64_t lce_block() { return int64_t(blockIdx.y) * gridDim.x + blockIdx.x; }

// A wave's accumulators of 32 x 32 products with the vocabulary (or P's rows) on the left: register
// i of lane l is row 8 (i / 4) + 4 (l / 32) + i % 4, column l % 32.
__device__ __forceinline__ int acc_row(int i, int h) { return 8 * (i >> 2) + 4 * h + (i & 3); }

// log-sum-exp pairs (m, s) = (max, sum 2^{z - m}); an empty pair is (-inf, 0)
__device__ __forceinline__ void lse_merge(float &m, float &s, float m2, float s2) {
  const float top = fmaxf(m, m2);
  const float ref = top == -INFINITY ? 0.f : top;
  s = s * fast_exp2(m - ref) + s2 * fast_exp2(m2 - ref);
  m = top;
}

// bf16: P is rounded to bf16 for its products.  Over many rows those roundings add up to less than the results' own (dx and dw
// are 1.15 to 1.35 times as far from 64 bits as without them); with a row or two they do not (up to 1.7 times).  Up to kFewRows
// labelled rows, what the rounding left over takes the places kRestAt further on, as rows of its own, for which the tiles have
// room (16 x 768 x 32000: 90 us with and without, 30 x 1024 x 40000: 115 and 108; up to 128 rows it would be 107 where 98 do
// for 128 x 768 x 32000).
constexpr int kFewRows = 32, kRestAt = 128;

// dX in shares of a piece's vocabulary rows: `dx_splits` of [n_pad, d] partial sums, or (dx_tiles: the tiles of 256
// that n_pad makes) as many of the labelled rows' as fit the same place.
constexpr int kMaxShares = 32;
struct DxShares { int n; int64_t rows; };
__device__ __forceinline__ DxShares lce_dx_shares(const LceArgs &a, int count) {
  if (!a.dx_tiles) return {a.dx_splits, a.n_pad};
  const int live = max(1, (count + 255) / 256);
  return {min(kMaxShares, a.dx_splits * a.dx_tiles / live), int64_t(live) * 256};
}

// Forward: the pair of a wave's MB x 32 vocabulary rows from v0 for each of its NB x 32 tokens from t0,
// into part `part`, and z at the labels among them.
template <int MB, int NB>
__device__ __forceinline__ void lce_row_stats(const LceArgs &a, f32x16 (&acc)[MB][NB], int v0, int t0, int count, int part) {
  const int l = threadIdx.x & 63, h = l >> 5;
  if (v0 + 32 * MB > a.V) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (v0 + 32 * mb + acc_row(i, h) >= a.V)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) acc[mb][nb][i] = -INFINITY;
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int t = t0 + 32 * nb + (l & 31);
    const bool live = t < count;
    const int rel = live ? a.label[t] - v0 : -1;
    if (live && rel >= 0 && rel < 32 * MB && ((rel >> 2) & 1) == h && a.label[t] >= 0) {
      float z = 0.f;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (rel == 32 * mb + acc_row(i, h)) z = acc[mb][nb][i];
      a.at_label[t] = z;
    }
    float m = -INFINITY;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, acc[mb][nb][i]);
    m *= kLog2e;
    const float ref = m == -INFINITY ? 0.f : m;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i & 3] += fast_exp2(fmaf(acc[mb][nb][i], kLog2e, -ref));
    float sum = (s[0] + s[1]) + (s[2] + s[3]);
    lse_merge(m, sum, __shfl_xor(m, 32, 64), __shfl_xor(sum, 32, 64));
    if (live && h == 0) {
      a.part_m[int64_t(part) * a.N + t] = m;
      a.part_s[int64_t(part) * a.N + t] = sum;
    }
  }
}

// What multiplies the products with P
__device__ __forceinline__ float lce_factor(const LceArgs &a, int count) {
  if (!a.reduction) return 1.f;
  return a.reduction == 1 ? *a.dloss : count ? *a.dloss / static_cast<float>(count) : 0.f;
}

// Backward: P over the same accumulators, in place; 0 behind the vocabulary.  What it holds for tokens behind the
// last labelled one (`live`: this lane's are not) is the caller's to leave out: a row of infinities in W times no
// row is no number.
template <int MB, int NB>
__device__ __forceinline__ void lce_row_grads(const LceArgs &a, f32x16 (&acc)[MB][NB], int v0, int t0, int count,
                                              bool (&live)[NB]) {
  const int l = threadIdx.x & 63, h = l >> 5;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int t = t0 + 32 * nb + (l & 31);
    live[nb] = t < count;
    const int label = live[nb] ? a.label[t] : 0, rel = live[nb] ? label - v0 : -1;
    float lse = live[nb] ? a.lse[t] : 0.f;
    if (live[nb] && label < 0) lse = __builtin_nanf("");  // (a label outside the vocabulary)
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mb][nb][i] = fast_exp2(fmaf(acc[mb][nb][i], kLog2e, -lse));
    if (rel >= 0 && rel < 32 * MB && ((rel >> 2) & 1) == h) {
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (rel == 32 * mb + acc_row(i, h)) acc[mb][nb][i] -= 1.f;
    }
    if (a.reduction == 0) {  // (a factor of each row; a common one multiplies the products)
      const float s = live[nb] ? a.dloss[int64_t(a.row[t]) * a.dl_st] : 0.f;
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[mb][nb][i] *= s;
    }
  }
  if (v0 + 32 * MB > a.V) {
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (v0 + 32 * mb + acc_row(i, h) >= a.V)
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) acc[mb][nb][i] = 0.f;
  }
}

// lce_general.hip: fp32 products, any alignment (P is fp32 [N, vc])
int lce_general_parts(int V);
int launch_lce_general_stats(const LceArgs &a, hipStream_t s);
int launch_lce_general_grads(const LceArgs &a, hipStream_t s);  // P of the piece
int lce_general_dx_splits(int64_t N, int d, int V, int vc);
int launch_lce_general_products(const LceArgs &a, bool dx, bool dw, hipStream_t s);

// lce_bf16.hip: bf16 (P is bf16 in blocks).  Vocabulary rows that do not start on 16-byte boundaries are
// copied to some that do first (`direct`: no need).
bool lce_bf16_direct(const void *w, int64_t ldw, int d);
int lce_bf16_parts(int V);
int lce_bf16_dx_splits(int64_t N, int d, int V, int vc);
int launch_lce_bf16_stats(const LceArgs &a, hipStream_t s);
int launch_lce_bf16_grads(const LceArgs &a, hipStream_t s);
int launch_lce_bf16_products(const LceArgs &a, bool dx, bool dw, hipStream_t s);

}  // namespace motif
