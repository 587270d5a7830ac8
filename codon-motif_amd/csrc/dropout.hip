// Dropout of a residual branch from a counter-based generator, its mask never stored:
//   y_e = residual_e + x_e keep_e / (1 - p),   dx_e = dy_e keep_e / (1 - p)
// Element e (its row-major index) is kept when word e mod 4 of Philox4x32-10 (J. Salmon et al.,
// "Parallel random numbers: as easy as 1, 2, 3", SC 2011) at the counter (e / 4 as two 32-bit
// words, 0, 0) under the 64-bit key `seed` is at least T = round(p 2^32).  The backward pass draws the
// same words again.  Computed in fp32, rounded once; a dropped element adds nothing, whatever it holds.
// T = 2^32 (p within 2^-33 of 1), which no word reaches, is a scale of 0: every element is dropped.
//
// Bound by memory (x, the residual and y once each) while the ten rounds, two 32 x 32 -> 64 bit products
// each for four elements, stay below it.  One thread draws for two (16-bit types) or one counter
// (fp32), whose elements are one 16-byte access.
#include "capi_internal.h"
#include "common.h"

#include <algorithm>

namespace motif {

namespace {

struct DropArgs {
  const void *x, *res;
  void *y;
  const int64_t *seed_dev;
  uint64_t seed;
  int64_t n;
  uint32_t threshold;
  float scale;
};

struct Words { uint32_t w[4]; };

__device__ __forceinline__ Words philox(uint64_t counter, uint64_t key) {
  uint32_t c0 = static_cast<uint32_t>(counter), c1 = static_cast<uint32_t>(counter >> 32), c2 = 0, c3 = 0;
  uint32_t k0 = static_cast<uint32_t>(key), k1 = static_cast<uint32_t>(key >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = static_cast<uint64_t>(c0) * 0xD2511F53u, b = static_cast<uint64_t>(c2) * 0xCD9E8D57u;
    c0 = static_cast<uint32_t>(b >> 32) ^ c1 ^ k0;
    c1 = static_cast<uint32_t>(b);
    c2 = static_cast<uint32_t>(a >> 32) ^ c3 ^ k1;
    c3 = static_cast<uint32_t>(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return {{c0, c1, c2, c3}};
}

// VEC: x, residual and y on 16-byte boundaries; the last n mod E elements one by one either way.
template <typename T, bool RES, bool VEC>
__global__ void __launch_bounds__(256) dropout_kernel(DropArgs a) {
  constexpr int E = 16 / sizeof(T);
  const uint64_t key = a.seed_dev ? static_cast<uint64_t>(*a.seed_dev) : a.seed;
  const bool some = a.scale != 0.f;
  const T *x = static_cast<const T *>(a.x), *res = static_cast<const T *>(a.res);
  T *y = static_cast<T *>(a.y);
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i * E < a.n; i += int64_t(gridDim.x) * 256) {
    const int64_t e0 = i * E;
    union Pack { uint4 u; T e[E]; } px, pr, py;
    const bool whole = VEC && e0 + E <= a.n;
    if (whole) {
      px.u = *reinterpret_cast<const uint4 *>(x + e0);
      if (RES) pr.u = *reinterpret_cast<const uint4 *>(res + e0);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e0 + e < a.n) {
          px.e[e] = x[e0 + e];
          if (RES) pr.e[e] = res[e0 + e];
        }
    }
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      const Words wd = philox(static_cast<uint64_t>(e0) / 4 + q, key);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int e = 4 * q + j;
        const bool keep = some && wd.w[j] >= a.threshold;
        const float xv = ld(&px.e[e]);
        float v;
        if (RES) {
          const float r = ld(&pr.e[e]);
          v = keep ? fmaf(xv, a.scale, r) : r;
        } else {
          v = keep ? xv * a.scale : 0.f;
        }
        st(&py.e[e], v);
      }
    }
    if (whole) {
      *reinterpret_cast<uint4 *>(y + e0) = py.u;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (e0 + e < a.n) y[e0 + e] = py.e[e];
    }
  }
}

template <typename T> int launch(const DropArgs &a, hipStream_t s) {
  constexpr int E = 16 / sizeof(T);
  const int64_t blocks = ((a.n + E - 1) / E + 255) / 256;
  const dim3 g(static_cast<unsigned>(std::min<int64_t>(blocks, 65536)));
  const bool vec = (reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.res) | reinterpret_cast<uintptr_t>(a.y)) % 16 == 0;
  if (a.res) {
    if (vec) dropout_kernel<T, true, true><<<g, 256, 0, s>>>(a);
    else dropout_kernel<T, true, false><<<g, 256, 0, s>>>(a);
  } else {
    if (vec) dropout_kernel<T, false, true><<<g, 256, 0, s>>>(a);
    else dropout_kernel<T, false, false><<<g, 256, 0, s>>>(a);
  }
  return check_launch("dropout_kernel");
}

}  // namespace

}  // namespace motif

using namespace motif;

extern "C" int motif_dropout_add(const void *x, const void *residual, void *y, int64_t n, uint32_t threshold, float scale,
                                 uint64_t seed, const int64_t *seed_dev, int dtype, void *stream) {
  if (n < 0 || (n > 0 && (!x || !y))) return set_error(MOTIF_ERR_INVALID, "dropout_add: null pointer or negative size");
  if (n == 0) return MOTIF_OK;
  const DropArgs a{x, residual, y, seed_dev, seed, n, threshold, scale};
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case MOTIF_F32: return launch<float>(a, s);
    case MOTIF_BF16: return launch<bf16_t>(a, s);
    case MOTIF_F16: return launch<f16_t>(a, s);
  }
  return set_error(MOTIF_ERR_UNSUPPORTED, "dropout_add: unknown dtype");
}
