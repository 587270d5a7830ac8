// Rows of a 4-bit key / value cache: written from the activations (motif_kv4_append) and read back
// (motif_kv4_read).
//
// A row of D features is D / 2 bytes of codes (feature 2 m in the low half of byte m, 2 m + 1 in the
// high half) and, for every group of min(32, D) features, a bf16 pair (scale, base):
//   base = bf16(min x), scale = bf16((max x - min x) / 15), code = rint((x - base) / scale) in 0 .. 15,
//   value = code * scale + base.
// Both ends of the range are held (a code for either), so features with an offset lose nothing; bf16
// keeps the inputs' range (fp32 features past bf16's largest number, 3.3895e38, count as that), and its rounding of base and scale (2^-9 of them) is small beside half a
// step (1 / 30 of the range).  The quotient is an IEEE division, so that a value exactly between two
// codes goes to the even one on every machine.  A group that holds an infinity or a NaN gets a NaN
// scale: its values read back NaN, no other group's do.  So does one whose max - min passes fp32's
// largest number.
//
// A lane takes 8 features (16 bytes of a 16-bit row, one 4-byte word of codes), a group 4 lanes (2 at
// head dim 16): minimum and maximum by lane exchanges, no LDS.  Bound by the rows' bytes where there are
// many, by the launch below some thousands: 192 rows 3.4 us to write and 2.8 to read, 24576 rows (8.3 MB
// either way) 5.9 and 4.8 us, of which 2.5 are a launch's own.
#include "capi_internal.h"
#include "chord_internal.h"
#include "common.h"

namespace motif {

namespace {

template <typename T> __device__ __forceinline__ void load8(const T *p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 u = *reinterpret_cast<const f32x4 *>(p), v = *reinterpret_cast<const f32x4 *>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[e] = u[e]; x[4 + e] = v[e]; }
  } else {
    const uint4 u = *reinterpret_cast<const uint4 *>(p);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const uint16_t b = static_cast<uint16_t>(w[e >> 1] >> (16 * (e & 1)));
      if constexpr (__is_same(T, bf16_t)) x[e] = bf16_to_f32(b);
      else x[e] = static_cast<float>(__builtin_bit_cast(f16_t, b));
    }
  }
}
template <typename T> __device__ __forceinline__ void store8(T *p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<f32x4 *>(p) = f32x4{x[0], x[1], x[2], x[3]};
    *reinterpret_cast<f32x4 *>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      uint16_t lo, hi;
      if constexpr (__is_same(T, bf16_t)) {
        lo = f32_to_bf16(x[2 * e]);
        hi = f32_to_bf16(x[2 * e + 1]);
      } else {  // (a base rounded to bf16 may pass the fp16 row's own extreme: held at the largest value)
        auto sat = [](float v) { return static_cast<f16_t>(v > 65504.f ? 65504.f : v < -65504.f ? -65504.f : v); };
        lo = __builtin_bit_cast(uint16_t, sat(x[2 * e]));
        hi = __builtin_bit_cast(uint16_t, sat(x[2 * e + 1]));
      }
      w[e] = lo | (static_cast<uint32_t>(hi) << 16);
    }
    *reinterpret_cast<uint4 *>(p) = uint4{w[0], w[1], w[2], w[3]};
  }
}

struct RowsArgs {
  const void *k; int64_t k_sb, k_sh, k_st;  // append: the new rows; read: (as void *) the destinations
  const void *v; int64_t v_sb, v_sh, v_st;
  KV4Args kv;
  const int *len_dev;  // device position of the first row, or null: pos
  int pos, capacity, n, Hkv;
  int64_t rows;  // B * Hkv * n
};

// blockIdx.y: 0 keys, 1 values
template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_append_kernel(RowsArgs a) {
  constexpr int LPR = D / 8, LPG = (D >= 32 ? 32 : D) / 8, G = D / (8 * LPG);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
  const int sub = threadIdx.x % LPR;
  const bool is_v = blockIdx.y != 0, valid = row < a.rows;
  const int64_t r = valid ? row : 0;
  const int t = static_cast<int>(r % a.n), h = static_cast<int>((r / a.n) % a.Hkv);
  const int64_t b = r / (static_cast<int64_t>(a.n) * a.Hkv);
  const T *src = is_v ? static_cast<const T *>(a.v) + b * a.v_sb + h * a.v_sh + t * a.v_st
                      : static_cast<const T *>(a.k) + b * a.k_sb + h * a.k_sh + t * a.k_st;
  float x[8];
  load8(src + 8 * sub, x);
  const int pos = (a.len_dev ? *a.len_dev : a.pos) + t;
  uint32_t pair;
  const uint32_t w = kv4_codes<8, LPG>(x, pair);
  if (!valid || pos < 0 || pos >= a.capacity) return;  // (never outside the slab)
  uint8_t *codes = const_cast<uint8_t *>(is_v ? a.kv.vc + b * a.kv.vc_sb + h * a.kv.vc_sh : a.kv.kc + b * a.kv.kc_sb + h * a.kv.kc_sh);
  uint32_t *pairs = const_cast<uint32_t *>(is_v ? a.kv.vp + b * a.kv.vp_sb + h * a.kv.vp_sh : a.kv.kp + b * a.kv.kp_sb + h * a.kv.kp_sh);
  *reinterpret_cast<uint32_t *>(codes + int64_t(pos) * (D / 2) + 4 * sub) = w;
  if (sub % LPG == 0) pairs[int64_t(pos) * G + sub / LPG] = pair;
}

template <typename T, int D>
__global__ void __launch_bounds__(256) kv4_read_kernel(RowsArgs a) {
  constexpr int LPR = D / 8, LPG = (D >= 32 ? 32 : D) / 8, G = D / (8 * LPG);
  const int64_t row = static_cast<int64_t>(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
  const int sub = threadIdx.x % LPR;
  if (row >= a.rows) return;
  const bool is_v = blockIdx.y != 0;
  const int t = static_cast<int>(row % a.n), h = static_cast<int>((row / a.n) % a.Hkv);
  const int64_t b = row / (static_cast<int64_t>(a.n) * a.Hkv), pos = a.pos + t;
  const uint8_t *codes = is_v ? a.kv.vc + b * a.kv.vc_sb + h * a.kv.vc_sh : a.kv.kc + b * a.kv.kc_sb + h * a.kv.kc_sh;
  const uint32_t *pairs = is_v ? a.kv.vp + b * a.kv.vp_sb + h * a.kv.vp_sh : a.kv.kp + b * a.kv.kp_sb + h * a.kv.kp_sh;
  const uint32_t w = *reinterpret_cast<const uint32_t *>(codes + pos * (D / 2) + 4 * sub), p = pairs[pos * G + sub / LPG];
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = fmaf(static_cast<float>((w >> (4 * e)) & 15u), kv4_scale(p), kv4_base(p));
  T *dst = is_v ? static_cast<T *>(const_cast<void *>(a.v)) + b * a.v_sb + h * a.v_sh + t * a.v_st
                : static_cast<T *>(const_cast<void *>(a.k)) + b * a.k_sb + h * a.k_sh + t * a.k_st;
  store8(dst + 8 * sub, x);
}

template <typename T, bool READ>
int launch_rows(const RowsArgs &a, int D, hipStream_t s) {
  const int64_t blocks = (a.rows * (D / 8) + 255) / 256;
  if (blocks > 0x7fffffff) return set_error(MOTIF_ERR_UNSUPPORTED, "kv4: too many rows");
  const dim3 grid(static_cast<unsigned>(blocks), 2), block(256);
  auto go = [&](auto d) {
    constexpr int kDim = decltype(d)::value;
    if constexpr (READ) kv4_read_kernel<T, kDim><<<grid, block, 0, s>>>(a);
    else kv4_append_kernel<T, kDim><<<grid, block, 0, s>>>(a);
  };
  if (D == 16) go(std::integral_constant<int, 16>());
  else if (D == 32) go(std::integral_constant<int, 32>());
  else if (D == 64) go(std::integral_constant<int, 64>());
  else go(std::integral_constant<int, 128>());
  return check_launch(READ ? "kv4_read_kernel" : "kv4_append_kernel");
}

template <bool READ>
int rows_entry(const char *what, RowsArgs a, int B, int D, int dtype, hipStream_t s) {
  const std::string name(what);
  if (B < 0 || a.n < 0 || a.Hkv <= 0 || a.capacity < 0) return set_error(MOTIF_ERR_INVALID, name + ": bad size");
  if (!kv4_head_dim(D)) return set_error(MOTIF_ERR_UNSUPPORTED, name + ": head_dim must be 16, 32, 64 or 128");
  if (dtype != MOTIF_F32 && dtype != MOTIF_BF16 && dtype != MOTIF_F16)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": dtype must be bf16, fp16 or fp32");
  if (!a.len_dev && (a.pos < 0 || static_cast<int64_t>(a.pos) + a.n > a.capacity))
    return set_error(MOTIF_ERR_INVALID, name + ": rows outside the cache");
  if (B == 0 || a.n == 0) return MOTIF_OK;
  if (const char *bad = kv4_check(a.kv, D)) return set_error(MOTIF_ERR_INVALID, name + ": " + bad);
  if (!a.k || !a.v) return set_error(MOTIF_ERR_INVALID, name + ": NULL pointer");
  const int64_t vec = dtype == MOTIF_F32 ? 4 : 8;
  if (((a.k_sb | a.k_sh | a.k_st | a.v_sb | a.v_sh | a.v_st) % vec) != 0 ||
      ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15) != 0)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": k / v need 16-byte aligned rows");
  a.rows = static_cast<int64_t>(B) * a.Hkv * a.n;
  if (dtype == MOTIF_BF16) return launch_rows<bf16_t, READ>(a, D, s);
  if (dtype == MOTIF_F16) return launch_rows<f16_t, READ>(a, D, s);
  return launch_rows<float, READ>(a, D, s);
}

}  // namespace

const char *kv4_check(const KV4Args &kv, int D) {
  if (!kv.kc || !kv.kp || !kv.vc || !kv.vp) return "NULL cache pointer";
  // (rows of codes are read in words)
  if (((reinterpret_cast<uintptr_t>(kv.kc) | reinterpret_cast<uintptr_t>(kv.kp) | reinterpret_cast<uintptr_t>(kv.vc) |
        reinterpret_cast<uintptr_t>(kv.vp)) & 3) != 0 ||
      ((kv.kc_sb | kv.kc_sh | kv.vc_sb | kv.vc_sh) & 3) != 0)
    return "cache rows must start on 4-byte boundaries";
  return nullptr;
}

}  // namespace motif

extern "C" int motif_kv4_append(const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st,
                                const void *v, int64_t v_sb, int64_t v_sh, int64_t v_st,
                                void *k_codes, int64_t kc_sb, int64_t kc_sh, void *k_params, int64_t kp_sb, int64_t kp_sh,
                                void *v_codes, int64_t vc_sb, int64_t vc_sh, void *v_params, int64_t vp_sb, int64_t vp_sh,
                                const int *position_dev, int position, int capacity, int B, int n, int Hkv, int D,
                                int dtype, void *stream) {
  using namespace motif;
  RowsArgs a{k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st,
             kv4_args(k_codes, kc_sb, kc_sh, k_params, kp_sb, kp_sh, v_codes, vc_sb, vc_sh, v_params, vp_sb, vp_sh),
             position_dev, position, capacity, n, Hkv, 0};
  return rows_entry<false>("kv4_append", a, B, D, dtype, static_cast<hipStream_t>(stream));
}

extern "C" int motif_kv4_read(const void *k_codes, int64_t kc_sb, int64_t kc_sh, const void *k_params, int64_t kp_sb,
                              int64_t kp_sh, const void *v_codes, int64_t vc_sb, int64_t vc_sh, const void *v_params,
                              int64_t vp_sb, int64_t vp_sh, void *k, int64_t k_sb, int64_t k_sh, int64_t k_st,
                              void *v, int64_t v_sb, int64_t v_sh, int64_t v_st,
                              int position, int capacity, int B, int n, int Hkv, int D, int dtype, void *stream) {
  using namespace motif;
  RowsArgs a{k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st,
             kv4_args(k_codes, kc_sb, kc_sh, k_params, kp_sb, kp_sh, v_codes, vc_sb, vc_sh, v_params, vp_sb, vp_sh),
             nullptr, position, capacity, n, Hkv, 0};
  return rows_entry<true>("kv4_read", a, B, D, dtype, static_cast<hipStream_t>(stream));
}
