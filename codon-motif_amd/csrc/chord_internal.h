// Shared between the Chord attention translation units.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "common.h"

namespace motif {

struct ChordArgs {
  const void *q; int64_t q_sb, q_sh, q_st;
  const void *k; int64_t k_sb, k_sh, k_st;
  const void *v; int64_t v_sb, v_sh, v_st;
  const float *alpha, *beta, *mu, *ssmax;
  const float *log_n; int64_t ln_sb, ln_st;
  void *out; int64_t o_sb, o_sh, o_st;
  float *lse;
  int B, H, Hkv, L, S, q_start;
  float scale, eps;
  const int32_t *cu;  // packed sequences (B == 1) or nullptr
  // split-K partials
  float *part;        // [B][Hkv][splits][L * group][D + 2]
  int splits;         // key-range splits (decode kernel)
  int nqc;            // row chunks per (batch, kv head) (decode kernel)
  // device cursor (decode kernels): when set, *len_dev positions are cached, the L
  // new keys sit at [*len_dev, *len_dev + L), S holds the cache capacity, and the
  // merge pass advances *len_dev by L
  int *len_dev;
  const float *log_tab;  // ln(1 .. n) when log_n is NULL: log_n[b, i] = log_tab[q_start + i]
  // sliding window (windowed kernels): a query at position p sees the keys j <= p with
  // j > p - window or j < sinks
  int window, sinks;
  // distances 0, -1, ... -(dist_n - 1) of each head: {x^beta, x^beta log2 x}, or null
  const float2 *dist;
  int dist_n;
};

// Longest window and most first tokens a launch takes (positions stay below it as well), so that
// no sum of two positions leaves 32 bits.
constexpr int kMaxWindow = 1 << 29;

// A 4-bit cache: for each (batch row, kv head) rows of D / 2 bytes (feature 2 m in the low half of
// byte m) and rows of D / min(32, D) bf16 pairs (scale, base), value = code * scale + base.
struct KV4Args {
  const uint8_t *kc; int64_t kc_sb, kc_sh;  // strides in bytes
  const uint32_t *kp; int64_t kp_sb, kp_sh;  // strides in pairs
  const uint8_t *vc; int64_t vc_sb, vc_sh;
  const uint32_t *vp; int64_t vp_sb, vp_sh;
};
inline KV4Args kv4_args(const void *kc, int64_t kc_sb, int64_t kc_sh, const void *kp, int64_t kp_sb, int64_t kp_sh,
                        const void *vc, int64_t vc_sb, int64_t vc_sh, const void *vp, int64_t vp_sb, int64_t vp_sh) {
  return {static_cast<const uint8_t *>(kc), kc_sb, kc_sh, static_cast<const uint32_t *>(kp), kp_sb, kp_sh,
          static_cast<const uint8_t *>(vc), vc_sb, vc_sh, static_cast<const uint32_t *>(vp), vp_sb, vp_sh};
}
inline bool kv4_head_dim(int D) { return D == 16 || D == 32 || D == 64 || D == 128; }
const char *kv4_check(const KV4Args &kv, int D);  // what is wrong with a cache's pointers, or null
// the two halves of a (scale, base) pair
__device__ __forceinline__ float kv4_scale(uint32_t p) { return __uint_as_float(p << 16); }
__device__ __forceinline__ float kv4_base(uint32_t p) { return __uint_as_float(p & 0xffff0000u); }

constexpr float kBf16Max = 0x1.fep+127f;
// A lane's N features of a row, LPG lanes to a group: their codes (4 bits each from the lowest on) and the
// group's pair.  Every lane of the group calls it.  Features past bf16's largest number M (fp32 ones only)
// count as M: with every |x| <= M = (1 - 2^-8) fp32's largest, neither the base's rounding nor 15 times
// the scale's (2^-8 of them) takes a value past fp32's range.
template <int N, int LPG> __device__ __forceinline__ uint32_t kv4_codes(float (&x)[N], uint32_t &pair) {
  float lo = INFINITY, hi = -INFINITY, bad = 0.f;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    bad = fmaf(x[e], 0.f, bad);  // NaN once any feature is not finite
    x[e] = __builtin_amdgcn_fmed3f(x[e], -kBf16Max, kBf16Max);
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
  }
#pragma unroll
  for (int off = 1; off < LPG; off <<= 1) {
    lo = fminf(lo, __shfl_xor(lo, off, 64));
    hi = fmaxf(hi, __shfl_xor(hi, off, 64));
    bad += __shfl_xor(bad, off, 64);
  }
  const bf16_t sb = f32_to_bf16((hi - lo) * (1.f / 15.f) + bad), bb = f32_to_bf16(lo);
  const float scale = bf16_to_f32(sb), base = bf16_to_f32(bb);
  pair = sb | (static_cast<uint32_t>(bb) << 16);
  uint32_t w = 0;
  if (scale > 0.f && scale < INFINITY) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float c = fminf(fmaxf(rintf(__fdiv_rn(x[e] - base, scale)), 0.f), 15.f);
      w |= static_cast<uint32_t>(c) << (4 * e);
    }
  }
  return w;
}

// The tiles of TS keys that queries at positions [first, ..], whose last key is end - 1, meet under a
// window: those of the first tokens, then those from the lowest key in a window on.  No tile holds a
// row that none of these queries sees (first tokens end at `se`, windows start at `lo`): what lies
// between may be anything.  A tile ends after its rows: keys behind them belong to another tile.
template <int TS> struct KeyWalk {
  int lo, se, end, ns, count;  // tiles of first tokens, all tiles
  __host__ __device__ KeyWalk(int first, int end_, int window, int sinks) : end(end_) {
    lo = first - window + 1;
    lo = lo > 0 ? lo : 0;
    se = sinks < end ? sinks : end;
    if (lo <= se) lo = se = 0;  // one run from the start
    ns = (se + TS - 1) / TS;
    count = ns + (end > lo ? (end - lo + TS - 1) / TS : 0);
  }
  __host__ __device__ int start(int i) const { return i < ns ? i * TS : lo + (i - ns) * TS; }
  __host__ __device__ int rows(int i) const {  // of tile i that may be read (none past the last tile)
    const int n = (i < ns ? se : end) - start(i);
    return n < 0 ? 0 : n < TS ? n : TS;
  }
};

// A tile of 64 features in LDS (the windowed prefill's and the backward's) is 32 rows of eight 16-byte pieces,
// piece c of row r at c ^ piece_swap(r): 16-byte reads of one piece of eight rows, transpose reads of 16
// features of four rows, and stores of four pieces of two rows in stage_row's order meet the banks alike.
// (Rows stored in their own order collide: 8.7M conflict cycles at 8192 tokens where 2.8M are left; so did the
// transpose reads with the swap's bits the other way round, 5.7M.)
__device__ __forceinline__ int piece_swap(int r) { return ((r & 3) << 1) | ((r >> 2) & 1); }
// The row that thread t of 128 stores pieces t % 4 and + 4 of
__device__ __forceinline__ int stage_row(int t) { const int r = t >> 2; return (r & ~3) | ((r & 1) << 1) | ((r >> 1) & 1); }
typedef short s16x4 __attribute__((ext_vector_type(4)));
// Lane l: feature l % 32 of keys 4 (l / 32) .. + 3, from the address of 4 features of key 4 (l / 32) + l % 16 / 4
// (16 (l / 16 % 2) + 4 (l % 4) on)
__device__ __forceinline__ uint2 ld_transposed(const bf16_t *p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)p));
}

// Keys and query start of a decode launch: from the host arguments, or from the
// device cursor (clamped so the window stays inside the capacity).
struct DecodeWindow { int S, q_start; };
__device__ __forceinline__ DecodeWindow decode_window(const ChordArgs &a) {
  if (!a.len_dev) return {min(a.S, a.q_start + a.L), a.q_start};
  const int cached = min(max(__builtin_amdgcn_readfirstlane(*a.len_dev), 0), a.S - a.L);
  return {cached + a.L, cached};
}

__device__ __forceinline__ float log_n_at(const ChordArgs &a, int b, int i, int q_start) {
  return a.log_n ? a.log_n[b * a.ln_sb + int64_t(i) * a.ln_st] : a.log_tab[q_start + i];
}

// Keys of a 32-key tile (bit k: key k) that are <= last, and > out or < first: one register for a lane's
// masks, a test per key.
__device__ __forceinline__ uint32_t keys_upto(int x) { return x < 0 ? 0u : x >= 31 ? ~0u : (2u << x) - 1u; }
__device__ __forceinline__ uint32_t seen_keys(int last, int out, int first) {
  return keys_upto(last) & (~keys_upto(out) | keys_upto(first - 1));
}

__device__ __forceinline__ float ggd_bias(float dist, float alpha, float beta, float mu, float eps) {
  // -alpha * (|d - mu| + eps)^beta, the power through exp2(beta * log2(.)).
  const float x = fabsf(dist - mu) + eps;
  return -alpha * fast_exp2(beta * fast_log2(x));
}

// The fp32-accumulating flash kernel (chord_wide.hip) for what the bf16 head-dim-64 kernel does
// not take: fp32, fp16 and bf16 at head dims 16, 32, 64, 128, padded batches.
bool chord_wide_serves(const ChordArgs &a);
int launch_chord_wide(const ChordArgs &a, int dtype, int D, hipStream_t s);
// The same kernel with a window (k / v rows), and over a 4-bit cache (`kv`; a.k / a.v unused),
// with the host's q_start or the device cursor (which the launch then advances).
int launch_chord_wide_window(const ChordArgs &a, int dtype, int D, hipStream_t s);
int launch_chord_wide_kv4(const ChordArgs &a, const KV4Args &kv, int dtype, int D, hipStream_t s);

// Few rows of bf16 at head dim 64 under a window ((H / Hkv) L <= 16): a.splits shares of the tiles, their
// partials (a.part) and a merge, or unsplit straight to out; the cursor, if any, advances.
bool chord_window_decode_serves(int H, int Hkv, int L, int D, int dtype);
int chord_window_splits(int B, int Hkv, int L, int S, int window, int sinks);
int launch_chord_window_decode(const ChordArgs &a, hipStream_t s);

// The same over a 4-bit cache (chord_kv4.hip; bf16 or fp16).
bool chord_kv4_serves(int H, int Hkv, int L, int D, int dtype);
int chord_kv4_splits(int B, int Hkv, int L, int S, int window, int sinks);
int launch_chord_kv4(const ChordArgs &a, const KV4Args &kv, int dtype, hipStream_t s);
// The merge of split partials (and the cursor's advance).
int launch_chord_merge(const ChordArgs &a, int dtype, int D, hipStream_t s);
// The cursor's advance alone (nothing without a cursor).
int launch_chord_advance(const ChordArgs &a, hipStream_t s);
int chord_cu_count();

// Chord decode over a device cursor, shared by the C-ABI entry points that take
// a caller workspace and those that use the library's own scratch.
// The body of motif_chord_decode (same arguments and status codes).
int chord_decode_run(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k_cache, int64_t k_sb, int64_t k_sh, int64_t k_st,
    const void *v_cache, int64_t v_sb, int64_t v_sh, int64_t v_st,
    int *length_dev, int capacity,
    const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st, const float *log_table, int log_table_len,
    void *out, int64_t o_sb, int64_t o_sh, int64_t o_st,
    int B, int H, int Hkv, int L, int D, float scale, float eps,
    void *workspace, size_t workspace_bytes, int dtype, void *stream);

}  // namespace motif
