// RMSNorm and LayerNorm of rows, forward and backward:
//   h = (x - m) r,  r = 1 / sqrt(mean((x - m)^2) + eps),  y = h w + b     (RMSNorm: m = 0, b = 0)
//   g = dy w,  dx = r (g - mean(g h) h - mean(g)),  dw = sum_rows dy h,  db = sum_rows dy
// (RMSNorm: no mean(g), no db).  All in fp32, y and dx rounded once; the forward keeps r (and m) of
// each row in fp32.
//
// Both passes are bound by memory: a row is read once into registers, by a group of 4 to 1024 lanes
// that holds it whole (NV accesses of E elements a lane, E elements being 16 bytes where every row
// starts on a 16-byte boundary, else one).  Variance is taken around the mean, from the registers.
// The backward walks its rows in a grid of at most kMaxGroups workgroups; each keeps its share of
// dw and db in registers, adds the row groups through LDS and leaves one partial row; a second
// kernel adds the partial rows in a fixed order (no atomics: results repeat bit for bit).
#include "capi_internal.h"
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace motif {

namespace {

constexpr int kMaxGroups = 512;
constexpr int kMaxD = 16384;  // features of a row

struct NormArgs {
  const void *x; int64_t x_rs;
  const void *w, *b;             // [D] or NULL
  const void *dy; int64_t dy_rs;
  void *y; int64_t y_rs;         // y, or dx
  float *rstd, *mean;            // [rows]
  float *part;                   // [2, groups, D] partial dw, db
  void *dw, *db;
  float eps;
  int rows, D, groups;
};

// One access: E elements as they lie in memory, and as floats.
template <typename T, int E> struct Raw {
  T e[E];
  __device__ __forceinline__ void load(const T *p) { e[0] = *p; }
};
template <typename T> struct __align__(16) Raw<T, 8> {
  T e[8];
  __device__ __forceinline__ void load(const T *p) { *this = *reinterpret_cast<const Raw *>(p); }
};
template <> struct __align__(16) Raw<float, 4> {
  float e[4];
  __device__ __forceinline__ void load(const float *p) { *this = *reinterpret_cast<const Raw *>(p); }
};
template <typename T, int E> __device__ __forceinline__ void load_row(const T *p, float *v) {
  Raw<T, E> r;
  r.load(p);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = ld(&r.e[e]);
}
template <typename T, int E> __device__ __forceinline__ void store_row(T *p, const float *v) {
  Raw<T, E> r;
#pragma unroll
  for (int e = 0; e < E; ++e) st(&r.e[e], v[e]);
  *reinterpret_cast<Raw<T, E> *>(p) = r;
}

// The sums of N values over a row's LPR lanes (more than a wave: through LDS, every lane of the workgroup with them).
template <int LPR, int N>
__device__ __forceinline__ void group_sum(float (&v)[N], float *lds) {
#pragma unroll
  for (int off = LPR < 64 ? LPR / 2 : 32; off > 0; off >>= 1)
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] += __shfl_xor(v[n], off, 64);
  if (LPR > 64) {
    constexpr int W = LPR / 64;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int n = 0; n < N; ++n) lds[N * (threadIdx.x >> 6) + n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) {
      v[n] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[n] += lds[N * (threadIdx.x / LPR * W + i) + n];
    }
    __syncthreads();
  }
}

template <int LPR> constexpr int block_size() { return LPR > 256 ? LPR : 256; }

template <typename T, int E, int LPR, int NV, bool LAYER>
__global__ void __launch_bounds__(block_size<LPR>()) row_norm_fwd_kernel(NormArgs a) {
  constexpr int BS = block_size<LPR>();
  __shared__ float lds[16];
  const int sub = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const int64_t row = int64_t(blockIdx.x) * (BS / LPR) + grp;
  const bool live = row < a.rows;
  const T *x = static_cast<const T *>(a.x) + (live ? row : 0) * a.x_rs;
  float v[NV][E];
  float sum[1] = {0.f};
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (sub + j * LPR) * E;
    if (c < a.D) load_row<T, E>(x + c, v[j]);
    else
#pragma unroll
      for (int e = 0; e < E; ++e) v[j][e] = 0.f;
  }
  const float inv = 1.f / static_cast<float>(a.D);
  float m = 0.f;
  if (LAYER) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) sum[0] += v[j][e];
    group_sum<LPR, 1>(sum, lds);
    m = sum[0] * inv;
    sum[0] = 0.f;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if ((sub + j * LPR) * E < a.D)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (LAYER) v[j][e] -= m;
        sum[0] = fmaf(v[j][e], v[j][e], sum[0]);
      }
  group_sum<LPR, 1>(sum, lds);
  const float r = 1.f / sqrtf(fmaf(sum[0], inv, a.eps));
  if (!live) return;
  if (sub == 0 && a.rstd) {
    a.rstd[row] = r;
    if (LAYER) a.mean[row] = m;
  }
  T *y = static_cast<T *>(a.y) + row * a.y_rs;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (sub + j * LPR) * E;
    if (c >= a.D) continue;
    float w[E], b[E], o[E];
    if (a.w) load_row<T, E>(static_cast<const T *>(a.w) + c, w);
    if (LAYER && a.b) load_row<T, E>(static_cast<const T *>(a.b) + c, b);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      o[e] = v[j][e] * r;
      if (a.w) o[e] *= w[e];
      if (LAYER && a.b) o[e] += b[e];
    }
    store_row<T, E>(y + c, o);
  }
}

// PARAMS: dw (and db) are wanted.
template <typename T, int E, int LPR, int NV, bool LAYER, bool PARAMS>
__global__ void __launch_bounds__(block_size<LPR>()) row_norm_bwd_kernel(NormArgs a) {
  constexpr int BS = block_size<LPR>(), RPB = BS / LPR;
  constexpr int NS = LAYER ? 2 : 1;
  __shared__ float lds[32];
  const int sub = threadIdx.x % LPR, grp = threadIdx.x / LPR;
  const float inv = 1.f / static_cast<float>(a.D);
  float dw[NV][E], db[NV][E];
  Raw<T, E> w[NV], xr[NV], gr[NV];  // w, and the next row's x and dy, in flight while this one is worked on
  float next_r = 0.f, next_m = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (sub + j * LPR) * E;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      dw[j][e] = db[j][e] = 0.f;
      st(&w[j].e[e], 1.f);
    }
    if (a.w && c < a.D) w[j].load(static_cast<const T *>(a.w) + c);
  }
  auto fetch = [&](int64_t row) {
    if (row >= a.rows) return;
    const T *x = static_cast<const T *>(a.x) + row * a.x_rs, *dy = static_cast<const T *>(a.dy) + row * a.dy_rs;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (sub + j * LPR) * E;
      if (c < a.D) xr[j].load(x + c), gr[j].load(dy + c);
    }
    next_r = a.rstd[row];
    if (LAYER) next_m = a.mean[row];
  };
  // A row of 1024 lanes leaves each of them 128 registers: it is read twice (the second time from the cache) instead of held.
  constexpr bool kTwice = LPR == 1024;
  if (!kTwice) fetch(int64_t(blockIdx.x) * RPB + grp);
  // (every lane of a workgroup takes every step: the sums below meet at barriers)
  for (int64_t row0 = int64_t(blockIdx.x) * RPB; row0 < a.rows; row0 += int64_t(gridDim.x) * RPB) {
    const int64_t row = row0 + grp;
    const bool live = row < a.rows;
    if (kTwice) {
      const int64_t rr = live ? row : 0;
      const T *x = static_cast<const T *>(a.x) + rr * a.x_rs, *dy = static_cast<const T *>(a.dy) + rr * a.dy_rs;
      const float r = a.rstd[rr], m = LAYER ? a.mean[rr] : 0.f;
      float s[NS] = {};
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (sub + j * LPR) * E;
        if (!live || c >= a.D) continue;
        float h[E], g[E];
        load_row<T, E>(x + c, h);
        load_row<T, E>(dy + c, g);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          h[e] = (h[e] - m) * r;
          if (PARAMS) {
            dw[j][e] = fmaf(g[e], h[e], dw[j][e]);
            if (LAYER) db[j][e] += g[e];
          }
          g[e] *= ld(&w[j].e[e]);
          s[0] = fmaf(g[e], h[e], s[0]);
          if (LAYER) s[NS - 1] += g[e];
        }
      }
      group_sum<LPR, NS>(s, lds);
      if (!live || !a.y) continue;
      const float c1 = s[0] * inv, c0 = LAYER ? s[NS - 1] * inv : 0.f;
      T *dx = static_cast<T *>(a.y) + row * a.y_rs;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (sub + j * LPR) * E;
        if (c >= a.D) continue;
        float h[E], g[E];
        load_row<T, E>(x + c, h);
        load_row<T, E>(dy + c, g);
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = r * (fmaf(-c1, (h[e] - m) * r, g[e] * ld(&w[j].e[e])) - c0);
        store_row<T, E>(dx + c, h);
      }
      continue;
    }
    const float r = next_r, m = next_m;
    float h[NV][E], g[NV][E], s[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) s[n] = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const bool in = live && (sub + j * LPR) * E < a.D;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        h[j][e] = in ? (ld(&xr[j].e[e]) - m) * r : 0.f;
        g[j][e] = in ? ld(&gr[j].e[e]) : 0.f;
      }
    }
    fetch(row + int64_t(gridDim.x) * RPB);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        if (PARAMS) {
          dw[j][e] = fmaf(g[j][e], h[j][e], dw[j][e]);
          if (LAYER) db[j][e] += g[j][e];
        }
        g[j][e] *= ld(&w[j].e[e]);
        s[0] = fmaf(g[j][e], h[j][e], s[0]);
        if (LAYER) s[NS - 1] += g[j][e];
      }
    group_sum<LPR, NS>(s, lds);
    if (!live || !a.y) continue;
    const float c1 = s[0] * inv, c0 = LAYER ? s[NS - 1] * inv : 0.f;
    T *dx = static_cast<T *>(a.y) + row * a.y_rs;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (sub + j * LPR) * E;
      if (c >= a.D) continue;
      float o[E];
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] = r * (fmaf(-c1, h[j][e], g[j][e]) - c0);
      store_row<T, E>(dx + c, o);
    }
  }
  if (!PARAMS) return;
  // the row groups of the workgroup: within a wave by shuffles, over its waves through LDS
  constexpr int CW = LPR > 64 ? LPR : 64, L = LPR < 64 ? LPR : CW, NC = BS / CW;  // NC groups of waves hold the same columns
  __shared__ float acc[NC > 1 ? (NC - 1) * L * E : 1];
  const int copy = threadIdx.x / CW, lane = threadIdx.x % CW;
#pragma unroll
  for (int k = 0; k < (LAYER ? 2 : 1); ++k) {
    float *out = a.part + (int64_t(k) * a.groups + blockIdx.x) * a.D;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float v[E];
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = k ? db[j][e] : dw[j][e];
        if (LPR < 64)
#pragma unroll
          for (int off = 32; off >= LPR; off >>= 1) v[e] += __shfl_xor(v[e], off, 64);
      }
      if (NC > 1) {
        __syncthreads();
        if (copy > 0 && lane < L)
#pragma unroll
          for (int e = 0; e < E; ++e) acc[((copy - 1) * E + e) * L + lane] = v[e];
        __syncthreads();
        if (copy == 0 && lane < L)
#pragma unroll
          for (int i = 0; i < NC - 1; ++i)
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] += acc[(i * E + e) * L + lane];
      }
      const int c = (sub + j * LPR) * E;
      if (grp == 0 && c < a.D)
#pragma unroll
        for (int e = 0; e < E; ++e) out[c + e] = v[e];
    }
  }
}

// dw (blockIdx.y 0) and db (1): the partial rows of 32 columns, 32 workgroups' shares beside each other
template <typename T>
__global__ void __launch_bounds__(1024) row_norm_params_kernel(NormArgs a) {
  __shared__ float lds[32][33];
  const int cl = threadIdx.x & 31, sl = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + cl;
  T *out = static_cast<T *>(blockIdx.y ? a.db : a.dw);
  if (!out) return;
  const float *p = a.part + int64_t(blockIdx.y) * a.groups * a.D;
  float v = 0.f;
  if (c < a.D)
#pragma unroll 8
    for (int g = sl; g < a.groups; g += 32) v += p[int64_t(g) * a.D + c];
  lds[sl][cl] = v;
  __syncthreads();
  if (sl != 0 || c >= a.D) return;
#pragma unroll
  for (int i = 1; i < 32; ++i) v += lds[i][cl];
  st(out + c, v);
}

// The lanes and accesses of a row: the fewest lanes that hold it in one to three accesses of 16 bytes (four of 2048
// features a wave: LayerNorm's backward outgrew the registers, 29.8 against 20.4 us for 8192 rows), or sixteen of one
// element (a row within one wave needs no barrier).
template <int E, typename F> bool with_shape(int D, F &&f) {
  const int n = (D + E - 1) / E;  // accesses
#define MOTIF_ROW(LPR, NV) \
  if (n <= (LPR) * (NV)) { f(std::integral_constant<int, LPR>{}, std::integral_constant<int, NV>{}); return true; }
  MOTIF_ROW(8, 1)
  MOTIF_ROW(16, 1)
  if constexpr (E > 1) {
    MOTIF_ROW(32, 1)
    MOTIF_ROW(32, 3)
    MOTIF_ROW(64, 2)
    MOTIF_ROW(128, 2)
    MOTIF_ROW(256, 2)
    MOTIF_ROW(512, 2)
    MOTIF_ROW(1024, 2)
    if constexpr (E == 4) MOTIF_ROW(1024, 4)
  } else {
    MOTIF_ROW(64, 1)
    MOTIF_ROW(64, 4)
    MOTIF_ROW(64, 16)
    MOTIF_ROW(256, 16)
    MOTIF_ROW(1024, 16)
  }
#undef MOTIF_ROW
  return false;
}

template <int LPR> int rows_per_block() { return (LPR > 256 ? LPR : 256) / LPR; }

// Workgroups of the backward: one for each set of rows that a workgroup takes at a time, at most kMaxGroups, which then go
// through the sets in turn
int bwd_groups(int rows, int rpb) {
  const int64_t blocks = (int64_t(rows) + rpb - 1) / rpb;
  return static_cast<int>(std::min<int64_t>(blocks, kMaxGroups));
}

template <typename T, int E> int launch_fwd(const NormArgs &a, bool layer, hipStream_t s) {
  const bool ok = with_shape<E>(a.D, [&](auto lpr, auto nv) {
    constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value;
    const int rpb = rows_per_block<LPR>();
    // (a launch has less than 2^32 threads: 2^29 rows of 8 lanes, 2^24 of 256)
    const int64_t most = int64_t(UINT32_MAX / block_size<LPR>()) * rpb;
    for (int64_t r0 = 0; r0 < a.rows; r0 += most) {
      NormArgs c = a;
      c.rows = static_cast<int>(std::min<int64_t>(most, a.rows - r0));
      c.x = static_cast<const T *>(a.x) + r0 * a.x_rs, c.y = static_cast<T *>(a.y) + r0 * a.y_rs;
      c.rstd = a.rstd ? a.rstd + r0 : nullptr, c.mean = a.mean ? a.mean + r0 : nullptr;
      const dim3 g(static_cast<unsigned>((int64_t(c.rows) + rpb - 1) / rpb)), b(block_size<LPR>());
      if (layer) row_norm_fwd_kernel<T, E, LPR, NV, true><<<g, b, 0, s>>>(c);
      else row_norm_fwd_kernel<T, E, LPR, NV, false><<<g, b, 0, s>>>(c);
    }
  });
  if (!ok) return set_error(MOTIF_ERR_UNSUPPORTED, "row_norm: rows longer than the kernels hold");
  return check_launch("row_norm_fwd_kernel");
}

template <typename T, int E> int launch_bwd(NormArgs a, bool layer, bool params, hipStream_t s) {
  const bool ok = with_shape<E>(a.D, [&](auto lpr, auto nv) {
    constexpr int LPR = decltype(lpr)::value, NV = decltype(nv)::value;
    a.groups = bwd_groups(a.rows, rows_per_block<LPR>());
    const dim3 g(a.groups), b(block_size<LPR>());
    if (layer) {
      if (params) row_norm_bwd_kernel<T, E, LPR, NV, true, true><<<g, b, 0, s>>>(a);
      else row_norm_bwd_kernel<T, E, LPR, NV, true, false><<<g, b, 0, s>>>(a);
    } else {
      if (params) row_norm_bwd_kernel<T, E, LPR, NV, false, true><<<g, b, 0, s>>>(a);
      else row_norm_bwd_kernel<T, E, LPR, NV, false, false><<<g, b, 0, s>>>(a);
    }
  });
  if (!ok) return set_error(MOTIF_ERR_UNSUPPORTED, "row_norm: rows longer than the kernels hold");
  int rc = check_launch("row_norm_bwd_kernel");
  if (rc != MOTIF_OK || !params) return rc;
  row_norm_params_kernel<T><<<dim3((a.D + 31) / 32, layer ? 2 : 1), 1024, 0, s>>>(a);
  return check_launch("row_norm_params_kernel");
}

// 16 bytes an access where every row of every tensor starts on a 16-byte boundary
bool wide(const NormArgs &a, int esize) {
  const int e = 16 / esize;
  const auto al = [](const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  return a.D % e == 0 && al(a.x) && al(a.w) && al(a.b) && al(a.dy) && al(a.y) && a.x_rs % e == 0 && a.dy_rs % e == 0 &&
         a.y_rs % e == 0;
}

int check_args(const NormArgs &a, const char *what) {
  if (a.rows < 1 || a.D < 1) return set_error(MOTIF_ERR_INVALID, std::string(what) + ": rows and features start at 1");
  if (a.D > kMaxD) return set_error(MOTIF_ERR_UNSUPPORTED, std::string(what) + ": at most 16384 features");
  if (!a.x) return set_error(MOTIF_ERR_INVALID, std::string(what) + ": null pointer");
  return MOTIF_OK;
}

}  // namespace

}  // namespace motif

using namespace motif;

extern "C" size_t motif_row_norm_bwd_workspace_bytes(int rows, int D, int layer) {
  if (rows < 1 || D < 1) return 0;
  return size_t(layer ? 2 : 1) * std::min(rows, kMaxGroups) * D * sizeof(float);
}

extern "C" int motif_row_norm_fwd(const void *x, int64_t x_rs, const void *w, const void *b, void *y, int64_t y_rs,
                                  float *rstd, float *mean, int rows, int D, float eps, int layer, int dtype, void *stream) {
  NormArgs a{};
  a.x = x, a.x_rs = x_rs, a.w = w, a.b = b, a.y = y, a.y_rs = y_rs, a.rstd = rstd, a.mean = mean;
  a.rows = rows, a.D = D, a.eps = eps;
  int rc = check_args(a, "row_norm_fwd");
  if (rc != MOTIF_OK) return rc;
  if (!y || (layer && rstd && !mean)) return set_error(MOTIF_ERR_INVALID, "row_norm_fwd: null pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MOTIF_F32: return wide(a, 4) ? launch_fwd<float, 4>(a, layer, s) : launch_fwd<float, 1>(a, layer, s);
    case MOTIF_BF16: return wide(a, 2) ? launch_fwd<bf16_t, 8>(a, layer, s) : launch_fwd<bf16_t, 1>(a, layer, s);
    case MOTIF_F16: return wide(a, 2) ? launch_fwd<f16_t, 8>(a, layer, s) : launch_fwd<f16_t, 1>(a, layer, s);
  }
  return set_error(MOTIF_ERR_UNSUPPORTED, "row_norm_fwd: unknown dtype");
}

extern "C" int motif_row_norm_bwd(const void *dy, int64_t dy_rs, const void *x, int64_t x_rs, const void *w,
                                  const float *rstd, const float *mean, void *dx, int64_t dx_rs, void *dw, void *db,
                                  int rows, int D, int layer, void *workspace, size_t workspace_bytes, int dtype,
                                  void *stream) {
  NormArgs a{};
  a.x = x, a.x_rs = x_rs, a.w = w, a.dy = dy, a.dy_rs = dy_rs, a.y = dx, a.y_rs = dx_rs;
  a.rstd = const_cast<float *>(rstd), a.mean = const_cast<float *>(mean);
  a.rows = rows, a.D = D, a.dw = dw, a.db = layer ? db : nullptr;
  int rc = check_args(a, "row_norm_bwd");
  if (rc != MOTIF_OK) return rc;
  if (!dy || !rstd || (layer && !mean)) return set_error(MOTIF_ERR_INVALID, "row_norm_bwd: null pointer");
  const bool params = a.dw || a.db;
  if (!dx && !params) return MOTIF_OK;
  if (params && (!workspace || workspace_bytes < motif_row_norm_bwd_workspace_bytes(rows, D, layer)))
    return set_error(MOTIF_ERR_INVALID, "row_norm_bwd: workspace too small");
  a.part = static_cast<float *>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MOTIF_F32: return wide(a, 4) ? launch_bwd<float, 4>(a, layer, params, s) : launch_bwd<float, 1>(a, layer, params, s);
    case MOTIF_BF16: return wide(a, 2) ? launch_bwd<bf16_t, 8>(a, layer, params, s) : launch_bwd<bf16_t, 1>(a, layer, params, s);
    case MOTIF_F16: return wide(a, 2) ? launch_bwd<f16_t, 8>(a, layer, params, s) : launch_bwd<f16_t, 1>(a, layer, params, s);
  }
  return set_error(MOTIF_ERR_UNSUPPORTED, "row_norm_bwd: unknown dtype");
}
