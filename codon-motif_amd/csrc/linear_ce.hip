// Softmax cross entropy straight from hidden states: the C entries and the row kernels around the
// products of lce_bf16.hip and lce_general.hip.
//
// Forward: lce_plan (which rows have a label) and lce_gather (those rows beside each other, the padding
// columns zero), in one launch for few rows; one product with the row statistics in its epilogue, lce_combine (a row's parts),
// lce_loss (sum or mean).  Backward, per vocabulary piece: P, then dX += P W and dW = P^T X;
// lce_dx_rows sums the partial dX, rounds once and puts the rows back.
// No atomics: every sum has a fixed order, so results repeat bit for bit.
#include "lce_internal.h"

#include <algorithm>

namespace motif {

namespace {

// ------------------------------------------------------------ which rows have a label
// One workgroup, 16384 labels at a time: 16 a thread, all loaded before the first is looked at (16384 labels 9.8 us; 45
// with a run of labels to each thread).
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

// Both in one launch for few rows: 16 rows a workgroup, which counts the labels before its own by itself (4096 rows: 11 us
// and a launch less, where the two take 6.7 and 6.0; 517: 6.5 against 8.3; every label is read up to N / 16 times, so only
// up to kOneLaunch rows).
constexpr int kOneLaunch = 8192;
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) lce_plan_gather_kernel(const int64_t *labels, int64_t st, int64_t ignore, int N, int V,
                                                              int *row, int *label, int *pos, int *count, float *loss_rows,
                                                              const T *x, int64_t rs, T *out, int d, int ldo) {
  __shared__ int sums[4], at_of[16];
  const int tid = threadIdx.x, l = tid & 63, w = tid >> 6, r0 = blockIdx.x * 16;
  int n = 0;
#pragma unroll 4
  for (int r = tid; r < r0; r += 256) n += labels[r * st] != ignore;
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) n += __shfl_xor(n, off, 64);
  if (l == 0) sums[w] = n;
  __syncthreads();
  const int before = sums[0] + sums[1] + sums[2] + sums[3];
  if (w == 0) {
    const int r = r0 + l;
    const bool in = l < 16 && r < N;
    const int64_t t = in ? labels[r * st] : ignore;
    const uint64_t has = __ballot(t != ignore);
    const int at = t != ignore ? before + __popcll(has & ((uint64_t(1) << l) - 1)) : -1;
    if (l < 16) at_of[l] = at;
    if (at >= 0) {
      row[at] = r;
      label[at] = t >= 0 && t < V ? static_cast<int>(t) : -1;
    }
    if (in) {
      pos[r] = at;
      if (at < 0 && loss_rows) loss_rows[r] = 0.f;
    }
    if (l == 0 && r0 + 16 >= N) *count = before + __popcll(has);
  }
  __syncthreads();
  constexpr int E = VEC ? 16 / sizeof(T) : 1;
  for (int i = w; i < 16; i += 4) {
    if (at_of[i] < 0) continue;
    const T *src = x + int64_t(r0 + i) * rs;
    T *dst = out + int64_t(at_of[i]) * ldo;
    for (int c = l * E; c < ldo; c += 64 * E) {
      if (VEC)
        *reinterpret_cast<uint4 *>(dst + c) = c < d ? *reinterpret_cast<const uint4 *>(src + c) : uint4{0, 0, 0, 0};
      else
        dst[c] = c < d ? src[c] : T(0);
    }
  }
}

// The vocabulary's rows on 16-byte boundaries with zeros up to ldo, one wave a row.
__global__ void __launch_bounds__(256) lce_copy_kernel(const bf16_t *w, int64_t rs, bf16_t *out, int V, int d, int ldo) {
  const int v = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (v >= V) return;
  for (int c = threadIdx.x & 63; c < ldo; c += 64) out[int64_t(v) * ldo + c] = c < d ? w[v * rs + c] : bf16_t(0);
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

// dX rows: the partial sums of a labelled row times the common factor, rounded once; zeros for the others.  A wave takes
// 64 E columns of a row (`per` of them make a row); E = 4 where d is a multiple of 4.
template <typename T, int E>
__global__ void __launch_bounds__(256) lce_dx_rows_kernel(LceArgs a, T *dx, int per) {
  const int64_t id = lce_block() * 4 + (threadIdx.x >> 6);
  const int64_t r = id / per;
  const int c = (static_cast<int>(id - r * per) * 64 + (threadIdx.x & 63)) * E;
  if (r >= a.N || c >= a.d) return;
  const int i = a.pos[r], count = *a.count;
  float s[E] = {};
  if (i >= 0) {
    const float f = lce_factor(a, count);
    const DxShares sh = lce_dx_shares(a, count);
    const float *p = a.dx_part + int64_t(i) * a.d + c;
    const int64_t plane = sh.rows * a.d;
    auto add = [&](const float *p) {
      float v[E];
      if (E == 4) {
        const float4 u = *reinterpret_cast<const float4 *>(p);
        v[0] = u.x, v[1 % E] = u.y, v[2 % E] = u.z, v[3 % E] = u.w;
      } else {
        v[0] = *p;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) s[e] += v[e];
    };
#pragma unroll 8
    for (int k = 0; k < sh.n; ++k) add(p + k * plane);
    if (a.dx_tiles && count <= kFewRows)  // (the rows of P's remainders)
#pragma unroll 8
      for (int k = 0; k < sh.n; ++k) add(p + k * plane + int64_t(kRestAt) * a.d);
#pragma unroll
    for (int e = 0; e < E; ++e) s[e] *= f;
  }
  T o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) st(o + e, s[e]);
  __builtin_memcpy(dx + r * a.d + c, o, sizeof(o));
}

constexpr size_t kAlign = 256;
size_t up(size_t n, size_t m) { return (n + m - 1) / m * m; }

int esize(int dtype) { return dtype == MOTIF_F32 ? 4 : 2; }

// Copies of vocabulary rows (bf16 off 16-byte boundaries); 0: none
size_t copy_bytes(const void *w, int64_t w_rs, int d, int V, int dtype) {
  return dtype != MOTIF_BF16 || lce_bf16_direct(w, w_rs, d) ? 0 : up(size_t(V) * up(d, 64) * 2, kAlign);
}

// The forward's workspace: copied vocabulary rows, statistics of the vocabulary's parts, z at the labels, the rows' losses.
struct FwdSpace {
  int parts;
  size_t m, s, z, nll, bytes;
  FwdSpace(int N, int V, int dtype, size_t copy) {
    parts = dtype == MOTIF_BF16 ? lce_bf16_parts(V) : lce_general_parts(V);
    const size_t col = up(4 * size_t(N), kAlign), part = up(size_t(parts) * 4 * N, kAlign);
    m = copy;
    s = m + part;
    z = s + part;
    nll = z + col;
    bytes = nll + col;
  }
};

// The backward's: copied vocabulary rows, P of a vocabulary piece and fp32 partial dX.  A piece holds P in 256 MB (so that
// it stays in the memory-side cache between its three products: 16384 x 768 x 40960 in five of them 3.3 ms, in four 3.6), but
// no fewer than 4096 vocabulary rows, since every piece reads and writes the partial dX once.  In bf16 a tile of dW sums
// N / 32 steps, and the launch has N vc tn / 32768 of them for each of 512 places (tn column tiles); where that is half as
// many or fewer, the piece grows, up to 1 GB, until they are as many (32768 x 768 x 32000: eight pieces 7.0 ms, three
// 5.2).  The pieces of a vocabulary are made alike.
struct BwdSpace {
  int vc, splits;
  int64_t n_pad;
  size_t p, dx, bytes;
  BwdSpace(int64_t N, int d, int V, int dtype, size_t copy) {
    const size_t e = esize(dtype);
    n_pad = static_cast<int64_t>(up(N, 256));
    const size_t near = std::max<size_t>((size_t(1) << 28) / (n_pad * e), 4096), tn = (d + 127) / 128;
    size_t rows = near;
    if (dtype == MOTIF_BF16 && 65536 >= 2 * near * tn) rows = std::max(near, std::min(65536 / tn, (size_t(1) << 30) / (n_pad * e)));
    rows = std::max<size_t>(rows / 256 * 256, 256);
    const size_t pieces = (V + rows - 1) / rows;
    vc = static_cast<int>(up((V + pieces - 1) / pieces, 256));
    splits = dtype == MOTIF_BF16 ? lce_bf16_dx_splits(N, d, V, vc) : lce_general_dx_splits(N, d, V, vc);
    p = copy;
    dx = p + up(size_t(n_pad) * vc * e, kAlign);
    bytes = dx + size_t(splits) * n_pad * d * 4;
  }
};

// Each size by itself, and the tiles of dX and dW together, which are one launch of 256 threads each (2^24 tiles: x and w of 1 TB
// in bf16, 275 GB in fp32; a small dX has up to 512 more in its shares).
bool sizes_ok(int N, int d, int V, int dtype) {
  if (N < 1 || N > (1 << 23) || d < 1 || d > (1 << 16) || V < 1 || V > (1 << 22) - 64) return false;
  const int64_t tm = dtype == MOTIF_BF16 ? 256 : 64, tn = dtype == MOTIF_BF16 ? 128 : 64;
  return ((N + tm - 1) / tm + (V + tm - 1) / tm) * ((d + tn - 1) / tn) <= (1 << 24) - 1024;
}

// kept: 4 N + 1 words: row, label, pos, lse, count
void bind_kept(LceArgs &a, int *kept) {
  const int64_t N = a.N;
  a.row = kept;
  a.label = kept + N;
  a.pos = kept + 2 * N;
  a.lse = reinterpret_cast<float *>(kept + 3 * N);
  a.count = kept + 4 * N;
}

// w, or its copy at `ws`
int bind_weight(LceArgs &a, const void *w, int64_t w_rs, size_t copy, void *ws, hipStream_t s) {
  a.w = w, a.ldw = w_rs, a.dk = static_cast<int>(up(a.d, 8));
  if (!copy) return MOTIF_OK;
  a.w = ws, a.ldw = static_cast<int64_t>(up(a.d, 64));
  lce_copy_kernel<<<(a.V + 3) / 4, 256, 0, s>>>(static_cast<const bf16_t *>(w), w_rs, static_cast<bf16_t *>(ws), a.V, a.d,
                                                 static_cast<int>(a.ldw));
  return check_launch("lce_copy_kernel");
}

struct Labels { const int64_t *p; int64_t st, ignore; float *loss_rows; };

// The plan in `kept` and the labelled rows in `out`
template <typename T> int gather(const void *x, int64_t rs, const LceArgs &a, const Labels &lb, int *kept, void *out, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const bool vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && rs % E == 0 && a.d % E == 0;
  const int64_t N = a.N;
  int *row = kept, *label = kept + N, *pos = kept + 2 * N, *count = kept + 4 * N;
  const T *src = static_cast<const T *>(x);
  T *dst = static_cast<T *>(out);
  const int ldo = static_cast<int>(a.ldx);
  if (N <= kOneLaunch) {
    const dim3 g((a.N + 15) / 16);
    if (vec) lce_plan_gather_kernel<T, true><<<g, 256, 0, s>>>(lb.p, lb.st, lb.ignore, a.N, a.V, row, label, pos, count, lb.loss_rows, src, rs, dst, a.d, ldo);
    else lce_plan_gather_kernel<T, false><<<g, 256, 0, s>>>(lb.p, lb.st, lb.ignore, a.N, a.V, row, label, pos, count, lb.loss_rows, src, rs, dst, a.d, ldo);
    return check_launch("lce_plan_gather_kernel");
  }
  lce_plan_kernel<<<1, 1024, 0, s>>>(lb.p, lb.st, lb.ignore, a.N, a.V, row, label, pos, count, lb.loss_rows);
  const int rc = check_launch("lce_plan_kernel");
  if (rc != MOTIF_OK) return rc;
  const dim3 g((a.N + 3) / 4);
  if (vec) lce_gather_kernel<T, true><<<g, 256, 0, s>>>(src, rs, row, count, dst, a.d, ldo);
  else lce_gather_kernel<T, false><<<g, 256, 0, s>>>(src, rs, row, count, dst, a.d, ldo);
  return check_launch("lce_gather_kernel");
}

}  // namespace

}  // namespace motif

using namespace motif;

extern "C" size_t motif_linear_ce_rows_bytes(int N, int d, int dtype) {
  if (!sizes_ok(N, d, 1, dtype)) return 0;
  return size_t(N) * up(d, 64) * esize(dtype);
}

extern "C" size_t motif_linear_ce_workspace_bytes(int N, int d, const void *w, int64_t w_rs, int V, int dtype, int backward) {
  if (!sizes_ok(N, d, V, dtype)) return 0;
  const size_t copy = copy_bytes(w, w_rs, d, V, dtype);
  return backward ? BwdSpace(N, d, V, dtype, copy).bytes : FwdSpace(N, V, dtype, copy).bytes;
}

extern "C" int motif_linear_ce_fwd(const void *x, int64_t x_rs, const void *w, int64_t w_rs, const int64_t *labels,
                                   int64_t labels_st, int64_t ignore_index, int N, int d, int V, int reduction,
                                   void *rows, int *kept, float *loss, void *workspace, size_t workspace_bytes, int dtype,
                                   void *stream) {
  if (dtype != MOTIF_F32 && dtype != MOTIF_BF16) return set_error(MOTIF_ERR_UNSUPPORTED, "linear_ce_fwd: fp32 or bf16");
  if (!sizes_ok(N, d, V, dtype)) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: N, d, V out of range");
  if (reduction < 0 || reduction > 2) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: reduction is 0, 1 or 2");
  if (!x || !w || !labels || !rows || !kept || !loss || !workspace)
    return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: null pointer");
  if (x_rs < 0 || (V > 1 && w_rs < d)) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: rows overlap");
  const size_t copy = copy_bytes(w, w_rs, d, V, dtype);
  const FwdSpace f(N, V, dtype, copy);
  if (workspace_bytes < f.bytes) return set_error(MOTIF_ERR_INVALID, "linear_ce_fwd: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  LceArgs a{};
  a.N = N, a.d = d, a.V = V;
  a.x = rows, a.ldx = static_cast<int64_t>(up(d, 64));
  bind_kept(a, kept);
  char *ws = static_cast<char *>(workspace);
  a.part_m = reinterpret_cast<float *>(ws + f.m);
  a.part_s = reinterpret_cast<float *>(ws + f.s);
  a.at_label = reinterpret_cast<float *>(ws + f.z);
  float *nll = reinterpret_cast<float *>(ws + f.nll), *loss_rows = reduction == 0 ? loss : nullptr;
  const Labels lb{labels, labels_st, ignore_index, loss_rows};
  int rc = dtype == MOTIF_F32 ? gather<float>(x, x_rs, a, lb, kept, rows, s) : gather<bf16_t>(x, x_rs, a, lb, kept, rows, s);
  if (rc == MOTIF_OK) rc = bind_weight(a, w, w_rs, copy, ws, s);
  if (rc != MOTIF_OK) return rc;
  rc = dtype == MOTIF_BF16 ? launch_lce_bf16_stats(a, s) : launch_lce_general_stats(a, s);
  if (rc != MOTIF_OK) return rc;
  lce_combine_kernel<<<(N + 31) / 32, 1024, 0, s>>>(a, f.parts, nll, loss_rows);
  rc = check_launch("lce_combine_kernel");
  if (rc != MOTIF_OK || reduction == 0) return rc;
  lce_loss_kernel<<<1, 1024, 0, s>>>(nll, a.count, reduction == 2, loss);
  return check_launch("lce_loss_kernel");
}

extern "C" int motif_linear_ce_bwd(const void *rows, const void *w, int64_t w_rs, const int *kept, const float *dloss,
                                   int64_t dloss_st, int N, int d, int V, int reduction, void *dx, void *dw,
                                   void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  if (dtype != MOTIF_F32 && dtype != MOTIF_BF16) return set_error(MOTIF_ERR_UNSUPPORTED, "linear_ce_bwd: fp32 or bf16");
  if (!sizes_ok(N, d, V, dtype)) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: N, d, V out of range");
  if (reduction < 0 || reduction > 2) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: reduction is 0, 1 or 2");
  if (!rows || !w || !kept || !dloss || !workspace) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: null pointer");
  if (V > 1 && w_rs < d) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: rows overlap");
  if (!dx && !dw) return MOTIF_OK;
  const bool bf16 = dtype == MOTIF_BF16;
  const size_t copy = copy_bytes(w, w_rs, d, V, dtype);
  const BwdSpace b(N, d, V, dtype, copy);
  if (workspace_bytes < b.bytes) return set_error(MOTIF_ERR_INVALID, "linear_ce_bwd: workspace too small");
  hipStream_t s = static_cast<hipStream_t>(stream);
  LceArgs a{};
  a.N = N, a.d = d, a.V = V;
  a.x = rows, a.ldx = static_cast<int64_t>(up(d, 64));
  bind_kept(a, const_cast<int *>(kept));
  a.dloss = dloss, a.dl_st = dloss_st, a.reduction = reduction;
  char *ws = static_cast<char *>(workspace);
  a.p = ws + b.p;
  a.dx_part = reinterpret_cast<float *>(ws + b.dx);
  a.n_pad = b.n_pad, a.dx_splits = b.splits, a.dx_tiles = bf16 ? static_cast<int>(b.n_pad / 256) : 0, a.vc = b.vc, a.dw = dw;
  int rc = bind_weight(a, w, w_rs, copy, ws, s);
  for (int v0 = 0; v0 < V && rc == MOTIF_OK; v0 += b.vc) {
    a.v0 = v0, a.vn = std::min(b.vc, V - v0), a.first = v0 == 0;
    rc = bf16 ? launch_lce_bf16_grads(a, s) : launch_lce_general_grads(a, s);
    if (rc != MOTIF_OK) break;
    rc = bf16 ? launch_lce_bf16_products(a, dx, dw, s) : launch_lce_general_products(a, dx, dw, s);
  }
  if (rc != MOTIF_OK || !dx) return rc;
  const bool four = d % 4 == 0 && reinterpret_cast<uintptr_t>(dx) % 16 == 0;
  const int per = (d + (four ? 256 : 64) - 1) / (four ? 256 : 64);
  const dim3 g = lce_grid((int64_t(N) * per + 3) / 4);
  if (four) {
    if (bf16) lce_dx_rows_kernel<bf16_t, 4><<<g, 256, 0, s>>>(a, static_cast<bf16_t *>(dx), per);
    else lce_dx_rows_kernel<float, 4><<<g, 256, 0, s>>>(a, static_cast<float *>(dx), per);
  } else {
    if (bf16) lce_dx_rows_kernel<bf16_t, 1><<<g, 256, 0, s>>>(a, static_cast<bf16_t *>(dx), per);
    else lce_dx_rows_kernel<float, 1><<<g, 256, 0, s>>>(a, static_cast<float *>(dx), per);
  }
  return check_launch("lce_dx_rows_kernel");
}
