// Softmax cross entropy straight from hidden states: the C entries and the row kernels around the
// products of lce_bf16.hip and lce_general.hip.
//
// Forward: lce_plan (which rows have a label), lce_gather (those rows beside each other, the padding
// columns zero), one product with the row statistics in its epilogue, lce_combine (a row's parts),
// lce_loss (sum or mean).  Backward, per vocabulary piece: P, then dX += P W and dW = P^T X;
// lce_dx_rows sums the partial dX, rounds once and puts the rows back.
// No atomics: every sum has a fixed order, so results repeat bit for bit.
#include "lce_internal.h"

#include <algorithm>

namespace motif {

namespace {

// ------------------------------------------------------------ which rows have a label
// One workgroup, 16384 labels at a time: 16 a thread, all loaded before the first is looked at.
__global__ void __launch_bounds__(1024) lce_plan_kernel(const int64_t *labels, int64_t st, int64_t ignore, int N, int V,
                                                        int *row, int *label, int *pos, int *count, float *loss_rows) {
  constexpr int PER = 16;
  __shared__ int sums[PER * 16];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int base = 0;
  for (int64_t r0 = 0; r0 < N; r0 += 1024 * PER) {
    int64_t t[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t r = r0 + i * 1024 + tid;
      t[i] = r < N ? labels[r * st] : ignore;
    }
    uint64_t has[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      has[i] = __ballot(t[i] != ignore);
      if (lane == 0) sums[i * 16 + wave] = __popcll(has[i]);
    }
    __syncthreads();
    if (wave == 0) {  // exclusive sums of the 256 groups of 64 labels, in their order
      int v[4], n = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] = sums[4 * lane + j], n += v[j];
      int incl = n;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const int up = __shfl_up(incl, off, 64);
        if (lane >= off) incl += up;
      }
      int at = base + incl - n;
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[4 * lane + j] = at, at += v[j];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int64_t r = r0 + i * 1024 + tid;
      if (r >= N) continue;
      if (t[i] != ignore) {
        const int at = sums[i * 16 + wave] + __popcll(has[i] & ((uint64_t(1) << lane) - 1));
        row[at] = static_cast<int>(r);
        label[at] = t[i] >= 0 && t[i] < V ? static_cast<int>(t[i]) : -1;
        pos[r] = at;
      } else {
        pos[r] = -1;
        if (loss_rows) loss_rows[r] = 0.f;
      }
    }
    // (the last group's start and size: labels behind N count as ignored)
    base = sums[PER * 16 - 1];
    __shared__ int last;
    if (tid == 1023) last = __popcll(has[PER - 1]);
    __syncthreads();
    base += last;
    __syncthreads();
  }
  if (tid == 0) *count = base;
}

// One wave per labelled row: d elements, then zeros up to ldo (the products read whole 64-element steps).
// VEC: rows on 16-byte boundaries and d a multiple of 16 bytes' elements.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) lce_gather_kernel(const T *x, int64_t rs, const int *row, const int *count, T *out,
                                                         int d, int ldo) {
  constexpr int E = VEC ? 16 / sizeof(T) : 1;
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), l = threadIdx.x & 63;
  if (i >= *count) return;
  const T *src = x + int64_t(row[i]) * rs;
  T *dst = out + int64_t(i) * ldo;
  for (int c = l * E; c < ldo; c += 64 * E) {
    if (VEC)
      *reinterpret_cast<uint4 *>(dst + c) = c < d ? *reinterpret_cast<const uint4 *>(src + c) : uint4{0, 0, 0, 0};
    else
      dst[c] = c < d ? src[c] : T(0);
  }
}

// A row's parts joined: 32 rows a workgroup, 32 threads to each (250 parts of 4096 rows: 23 us with 64 rows and
// four threads to each, whose loads followed each other).
__global__ void __launch_bounds__(1024) lce_combine_kernel(LceArgs a, int nparts, float *nll, float *loss_rows) {
  __shared__ float sm[32][33], ss[32][33];
  const int l = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int count = *a.count, t = blockIdx.x * 32 + l;
  if (blockIdx.x * 32 >= count) return;
  float m = -INFINITY, s = 0.f;
  if (t < count)
    for (int p = w; p < nparts; p += 32) lse_merge(m, s, a.part_m[int64_t(p) * a.N + t], a.part_s[int64_t(p) * a.N + t]);
  sm[w][l] = m;
  ss[w][l] = s;
  __syncthreads();
  // (a wave holds two rows: row w of 32 pairs, one a lane)
  m = sm[l][w];
  s = ss[l][w];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) lse_merge(m, s, __shfl_xor(m, off, 64), __shfl_xor(s, off, 64));
  const int r = blockIdx.x * 32 + w;
  if (l != 0 || r >= count) return;
  const float lse = m + log2f(s);
  a.lse[r] = lse;
  const float z = a.label[r] < 0 ? __builtin_nanf("") : a.at_label[r];
  const float loss = (lse - z * kLog2e) * 0.6931471805599453f;
  if (loss_rows) loss_rows[a.row[r]] = loss;
  else nll[r] = loss;
}

// The sum (or mean) of the rows' losses, in 64 bits.
__global__ void __launch_bounds__(1024) lce_loss_kernel(const float *nll, const int *count, int mean, float *loss) {
  __shared__ double sums[16];
  const int n = *count;
  double s = 0;
  for (int i = threadIdx.x; i < n; i += 1024) s += nll[i];
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  s = 0;
  for (int i = 0; i < 16; ++i) s += sums[i];
  *loss = static_cast<float>(mean ? s / n : s);  // (no label at all: 0 / 0)
}

// dX rows: the partial sums of a labelled row times the common factor, rounded once; zeros for the others.  One wave
// a row; E = 4 where d is a multiple of 4.
template <typename T, int E>
__global__ void __launch_bounds__(256) lce_dx_rows_kernel(LceArgs a, T *dx) {
  const int64_t r = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= a.N) return;
  const int i = a.pos[r];
  const int count = *a.count;
  const float f = lce_factor(a, count);
  const DxShares sh = lce_dx_shares(a, count);
  const float *p = a.dx_part + int64_t(i < 0 ? 0 : i) * a.d;
  const int64_t plane = sh.rows * a.d;
  for (int c = (threadIdx.x & 63) * E; c < a.d; c += 64 * E) {
    float s[E] = {};
    if (i >= 0) {
#pragma unroll 4
      for (int k = 0; k < sh.n; ++k) {
        float v[E];
        if (E == 4) {
          const float4 u = *reinterpret_cast<const float4 *>(p + k * plane + c);
          v[0] = u.x, v[1 % E] = u.y, v[2 % E] = u.z, v[3 % E] = u.w;
        } else {
          v[0] = p[k * plane + c];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) s[e] += v[e];
      }
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] *= f;
    }
    T o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) st(o + e, s[e]);
    __builtin_memcpy(dx + r * a.d + c, o, sizeof(o));
  }
}

constexpr size_t kAlign = 256;
size_t up(size_t n, size_t m) { return (n + m - 1) / m * m; }

int esize(int dtype) { return dtype == MOTIF_F32 ? 4 : 2; }

// The forward's workspace: statistics of the vocabulary's parts, z at the labels, the rows' losses.
struct FwdSpace {
  size_t m, s, z, nll, bytes;
  FwdSpace(int N, int V) {
    const size_t parts = lce_general_parts(V, N), col = up(4 * size_t(N), kAlign);
    m = 0;
    s = up(parts * 4 * N, kAlign);
    z = 2 * s;
    nll = z + col;
    bytes = nll + col;
  }
};

// The backward's: P of a vocabulary piece and fp32 partial dX.  A piece holds P in 256 MB (so that it
// stays in the memory-side cache between its three products), but no fewer than 4096 vocabulary rows:
// every piece reads and writes the partial dX once.
struct BwdSpace {
  int vc, splits;
  int64_t n_pad;
  size_t p, dx, bytes;
  BwdSpace(int64_t N, int d, int V, bool general) {
    const size_t e = general ? 4 : 2;
    n_pad = static_cast<int64_t>(up(N, 256));
    const size_t rows = (size_t(1) << 28) / (n_pad * e) / 256 * 256;
    vc = static_cast<int>(std::min(std::max<size_t>(rows, 4096), up(V, 256)));
    splits = general ? lce_general_dx_splits(N, d, V, vc) : lce_bf16_dx_splits(N, d, V, vc);
    p = 0;
    dx = up(size_t(n_pad) * vc * e, kAlign);
    bytes = dx + size_t(splits) * n_pad * d * 4;
  }
};

bool sizes_ok(int N, int d, int V) { return N > 0 && d > 0 && V > 0 && V <= (1 << 30) && d <= (1 << 20); }

// kept: 4 N + 1 words: row, label, pos, lse, count
void bind_kept(LceArgs &a, int *kept) {
  const int64_t N = a.N;
  a.row = kept;
  a.label = kept + N;
  a.pos = kept + 2 * N;
  a.lse = reinterpret_cast<float *>(kept + 3 * N);
  a.count = kept + 4 * N;
}

template <typename T> int gather(const void *x, int64_t rs, const LceArgs &a, void *out, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && rs % E == 0 && a.d % E == 0;
  const dim3 g((a.N + 3) / 4);
  const T *src = static_cast<const T *>(x);
  if (vec) lce_gather_kernel<T, true><<<g, 256, 0, s>>>(src, rs, a.row, a.count, static_cast<T *>(out), a.d, static_cast<int>(a.ldx));
  else lce_gather_kernel<T, false><<<g, 256, 0, s>>>(src, rs, a.row, a.count, static_cast<T *>(out), a.d, static_cast<int>(a.ldx));
  return check_launch("lce_gather_kernel");
}

}  // namespace

}  // namespace motif

using namespace motif;

extern "C" size_t motif_linear_ce_rows_bytes(int N, int d, int dtype) {
  if (!sizes_ok(N, d, 1)) return 0;
  return size_t(N) * up(d, 64) * esize(dtype);
}

extern "C" size_t motif_linear_ce_workspace_bytes(int N, int d, int V, int dtype, int backward) {
  if (!sizes_ok(N, d, V)) return 0;
  if (!backward) return FwdSpace(N, V).bytes;
  const size_t g = BwdSpace(N, d, V, true).bytes;
  return dtype == MOTIF_BF16 ? std::max(g, BwdSpace(N, d, V, false).bytes) : g;
}

extern "C" int motif_linear_ce_fwd(const void *x, int64_t x_rs, const void *w, int64_t w_rs, const int64_t *labels,
                                   int64_t labels_st, int64_t ignore_index, int N, int d, int V, int reduction,
                                   void *rows, int *kept, float *loss, void *workspace, size_t workspace_bytes, int dtype,
                                   void *stream) {
  if (dtype != MOTIF_F32 && dtype != MOTIF_BF16) return set_error(MOTIF_ERR_UNSUPPORTED, "linear_ce_fwd: fp32 or bf16");
  if (!sizes_ok(N, d, V)) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: N, d, V out of range");
  if (reduction < 0 || reduction > 2) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: reduction is 0, 1 or 2");
  if (!x || !w || !labels || !rows || !kept || !loss || !workspace)
    return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: null pointer");
  if (x_rs < 0 || (V > 1 && w_rs < d)) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: rows overlap");
  const FwdSpace f(N, V);
  if (workspace_bytes < f.bytes) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  LceArgs a{};
  a.N = N, a.d = d, a.V = V;
  a.x = rows, a.ldx = static_cast<int64_t>(up(d, 64));
  a.w = w, a.ldw = w_rs;
  bind_kept(a, kept);
  char *ws = static_cast<char *>(workspace);
  a.part_m = reinterpret_cast<float *>(ws + f.m);
  a.part_s = reinterpret_cast<float *>(ws + f.s);
  a.at_label = reinterpret_cast<float *>(ws + f.z);
  float *nll = reinterpret_cast<float *>(ws + f.nll), *loss_rows = reduction == 0 ? loss : nullptr;
  lce_plan_kernel<<<1, 1024, 0, s>>>(labels, labels_st, ignore_index, N, V, kept, kept + N, kept + 2 * int64_t(N),
                                     kept + 4 * int64_t(N), loss_rows);
  int rc = check_launch("lce_plan_kernel");
  if (rc == MOTIF_OK) rc = dtype == MOTIF_F32 ? gather<float>(x, x_rs, a, rows, s) : gather<bf16_t>(x, x_rs, a, rows, s);
  if (rc != MOTIF_OK) return rc;
  const bool fast = lce_bf16_serves(w, w_rs, d, dtype);
  const int nparts = fast ? lce_bf16_parts(V) : lce_general_parts(V, N);
  rc = fast ? launch_lce_bf16_stats(a, s) : launch_lce_general_stats(a, dtype, s);
  if (rc != MOTIF_OK) return rc;
  lce_combine_kernel<<<(N + 31) / 32, 1024, 0, s>>>(a, nparts, nll, loss_rows);
  rc = check_launch("lce_combine_kernel");
  if (rc != MOTIF_OK || reduction == 0) return rc;
  lce_loss_kernel<<<1, 1024, 0, s>>>(nll, a.count, reduction == 2, loss);
  return check_launch("lce_loss_kernel");
}

extern "C" int motif_linear_ce_bwd(const void *rows, const void *w, int64_t w_rs, const int *kept, const float *dloss,
                                   int64_t dloss_st, int N, int d, int V, int reduction, void *dx, void *dw,
                                   void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  if (dtype != MOTIF_F32 && dtype != MOTIF_BF16) return set_error(MOTIF_ERR_UNSUPPORTED, "linear_ce_bwd: fp32 or bf16");
  if (!sizes_ok(N, d, V)) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: N, d, V out of range");
  if (reduction < 0 || reduction > 2) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: reduction is 0, 1 or 2");
  if (!rows || !w || !kept || !dloss || !workspace) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: null pointer");
  if (V > 1 && w_rs < d) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: rows overlap");
  if (!dx && !dw) return MOTIF_OK;
  const bool fast = lce_bf16_serves(w, w_rs, d, dtype);
  const BwdSpace b(N, d, V, !fast);
  if (workspace_bytes < b.bytes) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  LceArgs a{};
  a.N = N, a.d = d, a.V = V;
  a.x = rows, a.ldx = static_cast<int64_t>(up(d, 64));
  a.w = w, a.ldw = w_rs;
  bind_kept(a, const_cast<int *>(kept));
  a.dloss = dloss, a.dl_st = dloss_st, a.reduction = reduction;
  char *ws = static_cast<char *>(workspace);
  a.p = ws + b.p;
  a.dx_part = reinterpret_cast<float *>(ws + b.dx);
  a.n_pad = b.n_pad, a.dx_splits = b.splits, a.dx_tiles = fast ? static_cast<int>(b.n_pad / 256) : 0, a.vc = b.vc, a.dw = dw;
  int rc = MOTIF_OK;
  for (int v0 = 0; v0 < V && rc == MOTIF_OK; v0 += b.vc) {
    a.v0 = v0, a.vn = std::min(b.vc, V - v0), a.first = v0 == 0;
    rc = fast ? launch_lce_bf16_grads(a, s) : launch_lce_general_grads(a, dtype, s);
    if (rc != MOTIF_OK) break;
    if (fast) {
      rc = launch_lce_bf16_products(a, dx, dw, s);
    } else {
      if (dx) rc = launch_lce_general_dx(a, dtype, s);
      if (rc == MOTIF_OK && dw) rc = launch_lce_general_dw(a, dtype, s);
    }
  }
  if (rc != MOTIF_OK || !dx) return rc;
  const unsigned g = (N + 3) / 4;
  const bool f32 = dtype == MOTIF_F32;
  if (d % 4 == 0 && reinterpret_cast<uintptr_t>(dx) % 16 == 0) {
    if (f32) lce_dx_rows_kernel<float, 4><<<g, 256, 0, s>>>(a, static_cast<float *>(dx));
    else lce_dx_rows_kernel<bf16_t, 4><<<g, 256, 0, s>>>(a, static_cast<bf16_t *>(dx));
  } else {
    if (f32) lce_dx_rows_kernel<float, 1><<<g, 256, 0, s>>>(a, static_cast<float *>(dx));
    else lce_dx_rows_kernel<bf16_t, 1><<<g, 256, 0, s>>>(a, static_cast<bf16_t *>(dx));
  }
  return check_launch("lce_dx_rows_kernel");
}
