// Cross entropy from hidden states in bf16 on v_mfma_f32_32x32x16_bf16: the three products of
// lce_internal.h.  A wave owns 128 x 64 of a product (8 matrix instructions for 6 LDS reads of 16 bytes a
// lane), four or eight waves a tile of 256 x 128 or 256 x 256.  Both sides go straight from memory to LDS (16 bytes
// a lane) in two or three stages of 32 or 64 k, one barrier a stage; LDS reads and writes meet no bank conflicts.
// What bounds them: at 4096 x 768 x 32000 z with its statistics reaches 850-910 TFLOP/s, with P 760-830, dX and dW 970-1020,
// where the library's bare products reach 920, 565 and 692.  Each stage's latency and the epilogues: matrix instructions are
// busy 52, 47 and 66% of the cycles, at a clock that falls to 1.75-2.1 GHz; the loads of dX and dW alone take 300 of 415 us, the
// matrix instructions without loads 330.
//
//   z = W X^T    left: 256 vocabulary rows, right: 128 or 256 tokens; a lane holds one token's scores, so a
//                row's maximum and sum are in-lane sums and one exchange
//   dX = P W     left: 256 tokens, right: 128 features
//   dW = P^T X   left: 256 vocabulary rows, right: 128 features
//
// P is laid out for both of its uses in blocks of 32 tokens x 16 vocabulary rows (1 KB): lane (t, h) of the
// product that makes it holds rows 8 (i / 4) + 4 h + i % 4, i < 8, of token t, and stores them as 16 bytes at
// place p(t, h) = (t + 32 h) ^ 4 h ^ 8 (block % 2).  dX reads those 16 bytes back as its operand (k in the
// order of i: the right side's rows are taken in the same order); dW reads four tokens' rows transposed
// (ds_read_tr16_b64: groups of 16 lanes give 4 tokens x 16 rows), the places keeping 4 tokens of both h, and
// of two blocks, in different banks.
#include "lce_internal.h"

#include <algorithm>

namespace motif {

namespace {

// The shapes of a workgroup: TM left rows (two waves over them, MB blocks of 32 each), TN right columns (64 a wave),
// BK k a stage, ST stages in LDS; PER of them on a CU.
template <int TM_, int TN_, int BK_, int ST_, int PER_> struct Shape {
  static constexpr int TM = TM_, TN = TN_, BK = BK_, ST = ST_, PER = PER_, MB = TM / 64, NW = 2 * (TN / 64), THREADS = 64 * NW;
  static constexpr int BOUND = PER * NW / 4;  // waves on a SIMD
  static constexpr int A_BYTES = TM * BK * 2, B_BYTES = TN * BK * 2, STAGE = A_BYTES + B_BYTES;
  static constexpr int LOADS = STAGE / 1024 / NW;  // 1 KB loads of a wave per stage
};
using Wide = Shape<256, 256, 64, 2, 1>;
using Narrow = Shape<256, 128, 32, 3, 2>;
using Three = Shape<256, 128, 32, 2, 3>;

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ uint2 read_tr(const char *p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
}

// 16 bytes a lane from buffer r at byte voff + soff into LDS at dst + 16 lane (dst the same for the wave).  The
// builtin for it makes the compiler wait for every load in flight before each transposed LDS read, which
// would empty the pipeline at every step; here `product` does all the waiting itself.  (m0 holds the place.  It is no
// register that the compiler keeps values in, which it warns of; said here, it sets m0 anew for whatever else may need it.)
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 make_rsrc(const void *p, int64_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return i32x4{static_cast<int>(a), static_cast<int>((a >> 32) & 0xffff), static_cast<int>(bytes), 0x00020000};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds(i32x4 r, uint32_t dst, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               ::"s"(dst), "v"(voff), "s"(r), "s"(soff) : "memory", "m0");
}
#pragma clang diagnostic pop
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ bf16x8 join(uint2 a, uint2 b) { return __builtin_bit_cast(bf16x8, uint4{a.x, a.y, b.x, b.y}); }

// R rows of BK k, k beside each other in memory (row stride ld): LDS row r is BK / 8 pieces of 16 bytes, piece c at
// c ^ swap(r): the LDS serves 16 lanes at a time, rows 0-3, 12-15, 20-23 and 24-27 or the others, from 64 banks,
// and no two of them may meet (r / 2 % 4 for rows of four pieces: half of the reads' cycles were conflicts).
template <typename C, int R> struct RowsK {
  static constexpr int NP = C::BK / 8, RL = 64 / NP, NJ = R / RL / C::NW;
  i32x4 buf;
  uint32_t off[NJ];
  int K;
  __device__ __forceinline__ static int swap(int r) { return NP == 4 ? (r >> 2) & 3 : (r >> 1) & 7; }
  __device__ __forceinline__ static int kc(int j) {  // first k of this lane's piece
    const int l = threadIdx.x & 63;
    return ((l % NP) ^ swap((wave_id() * NJ + j) * RL + l / NP)) * 8;
  }
  __device__ __forceinline__ RowsK(const bf16_t *p, int64_t ld, int rows, int K_) : K(K_) {
    const int l = threadIdx.x & 63, w = wave_id();
    const int n = min(rows, R);
    buf = make_rsrc(p, n > 0 ? ((n - 1) * ld + K) * 2 : 0);
#pragma unroll
    for (int j = 0; j < NJ; ++j) off[j] = static_cast<uint32_t>(((w * NJ + j) * RL + l / NP) * ld * 2 + kc(j) * 2);
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int w = wave_id();
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      load_lds(buf, dst + (w * NJ + j) * 1024, k0 + kc(j) < K ? off[j] : 0xfffffff0u, k0 * 2);
  }
  // operand of rows r0 .. r0 + 31 at k step s (16 k)
  __device__ __forceinline__ static bf16x8 frag(const char *src, int r0, int s) {
    const int l = threadIdx.x & 63, r = r0 + (l & 31), c = 2 * s + (l >> 5);
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(src + r * (C::BK * 2) + ((c ^ swap(r)) * 16)));
  }
};

// BK k rows of R columns (row stride ld): LDS row k is R / 8 pieces, piece c at c ^ swap(k).
__device__ __forceinline__ int tr_swap(int k) { return ((k & 1) << 2) | ((k & 2) ? 10 : 0); }
// FOLD: the rows are gone through a second time, from k = `fold` on.
template <typename C, int R, bool FOLD = false> struct ColsK {
  static constexpr int RP = 512 / R, NJ = C::BK / RP / C::NW;
  const bf16_t *p;
  int64_t ld;
  int cols, K, fold;
  uint32_t off[NJ];
  __device__ __forceinline__ ColsK(const bf16_t *p_, int64_t ld_, int cols_, int K_, int fold_ = 0)
      : p(p_), ld(ld_), cols(cols_), K(K_), fold(fold_) {
    const int l = threadIdx.x & 63, w = wave_id();
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int k = (w * NJ + j) * RP + l / (R / 8);
      off[j] = static_cast<uint32_t>(k * ld * 2 + ((l % (R / 8)) ^ tr_swap(k)) * 16);
    }
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    if (FOLD && k0 >= fold) k0 -= fold;
    const int w = wave_id(), n = min(K - k0, C::BK);
    const i32x4 buf = make_rsrc(p + int64_t(k0) * ld, ((n - 1) * ld + cols) * 2);
#pragma unroll
    for (int j = 0; j < NJ; ++j) load_lds(buf, dst + (w * NJ + j) * 1024, off[j], 0);
  }
  // operand of columns c0 .. c0 + 31, k in the order 8 (i / 4) + 4 h + i % 4
  __device__ __forceinline__ static bf16x8 frag(const char *src, int c0, int s) {
    const int l = threadIdx.x & 63, c = c0 + 16 * ((l >> 4) & 1) + 4 * (l & 3), k = 16 * s + 4 * (l >> 5) + ((l >> 2) & 3);
    const char *q = src + k * (R * 2) + (((c >> 3) ^ tr_swap(k)) * 16) + (c & 7) * 2;
    return join(read_tr(q), read_tr(q + 8 * R * 2));  // (swap(k + 8) = swap(k))
  }
};

// P's blocks as the left side of dX: 256 tokens x BK vocabulary rows, block (t / 32, v / 16) in order
template <typename C> struct PTokens {
  static constexpr int NB = C::BK / 16, NJ = 8 * NB / C::NW;
  const char *p;
  int nvc;
  uint32_t off[NJ];
  __device__ __forceinline__ PTokens(const void *p_, int t0, int vc) : nvc(vc / 16) {
    const int l = threadIdx.x & 63, w = wave_id();
    p = static_cast<const char *>(p_) + int64_t(t0 / 32) * nvc * 1024;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int q = w * NJ + j;
      off[j] = static_cast<uint32_t>(((q / NB) * nvc + q % NB) * 1024 + l * 16);
    }
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int w = wave_id();
    const i32x4 buf = make_rsrc(p + int64_t(k0 / 16) * 1024, (7 * nvc + NB) * 1024);
#pragma unroll
    for (int j = 0; j < NJ; ++j) load_lds(buf, dst + (w * NJ + j) * 1024, off[j], 0);
  }
  __device__ __forceinline__ static bf16x8 frag(const char *src, int r0, int s) {
    const int l = threadIdx.x & 63, q = (r0 >> 5) * NB + s;
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(src + q * 1024 + (l ^ ((l >> 5) << 2) ^ ((s & 1) << 3)) * 16));
  }
};

// ... as the left side of dW: 256 vocabulary rows x BK tokens (FOLD: from k = `fold` on the rows that hold remainders)
template <typename C, bool FOLD = false> struct PVocab {
  static constexpr int NJ = 16 * (C::BK / 32) / C::NW;
  const char *p;
  int nvc, fold;
  __device__ __forceinline__ PVocab(const void *p_, int r0, int vc, int fold_ = 0) : nvc(vc / 16), fold(fold_) {
    p = static_cast<const char *>(p_) + int64_t(r0 / 16) * 1024;
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int l = threadIdx.x & 63, w = wave_id();
    if (FOLD && k0 >= fold) k0 += kRestAt - fold;
    const i32x4 buf = make_rsrc(p + int64_t(k0 / 32) * nvc * 1024, ((C::BK / 32 - 1) * nvc + 16) * 1024);
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int q = w * NJ + j;
      load_lds(buf, dst + q * 1024, l * 16, ((q >> 4) * nvc + (q & 15)) * 1024);
    }
  }
  __device__ __forceinline__ static bf16x8 frag(const char *src, int r0, int s) {
    const int l = threadIdx.x & 63, g = (l >> 4) & 1, h = l & 1, t = 16 * (s & 1) + 4 * (l >> 5) + ((l >> 2) & 3);
    const int place = (t + 32 * h) ^ (h << 2) ^ (g << 3);
    const char *q = src + ((s >> 1) * 16 + (r0 >> 4) + g) * 1024 + ((l >> 1) & 1) * 8;
    return join(read_tr(q + place * 16), read_tr(q + (place ^ 8) * 16));
  }
};

// What bf16 b leaves of p (nothing of what is no finite number)
__device__ __forceinline__ bf16_t remainder(float p, uint32_t b) {
  return f32_to_bf16((b & 0x7f80u) == 0x7f80u ? 0.f : p - __uint_as_float(b << 16));
}

template <int MB> __device__ __forceinline__ void zero(f32x16 (&acc)[MB][2]) {
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mb][nb][i] = 0.f;
}

// One stage's products of a wave
template <typename C, typename A, typename B>
__device__ __forceinline__ void multiply(const char *sa, f32x16 (&acc)[C::MB][2]) {
  const int w = wave_id();
  const char *sb = sa + C::A_BYTES;
#pragma unroll
  for (int s = 0; s < C::BK / 16; ++s) {
    bf16x8 fa[C::MB], fb[2];
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) fb[nb] = B::frag(sb, 64 * (w >> 1) + 32 * nb, s);
#pragma unroll
    for (int mb = 0; mb < C::MB; ++mb) fa[mb] = A::frag(sa, C::TM / 2 * (w & 1) + 32 * mb, s);
#pragma unroll
    for (int mb = 0; mb < C::MB; ++mb)
#pragma unroll
      for (int nb = 0; nb < 2; ++nb)
        acc[mb][nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[mb], fb[nb], acc[mb][nb], 0, 0, 0);
  }
}

template <typename C, typename A, typename B>
__device__ __forceinline__ void product(const A &a, const B &b, int kb, int ke, char *lds, f32x16 (&acc)[C::MB][2]) {
  zero(acc);
  const int n = (ke - kb + C::BK - 1) / C::BK;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds));
  auto issue = [&](int i, uint32_t place) {
    a.issue(base + place, kb + i * C::BK);
    b.issue(base + place + C::A_BYTES, kb + i * C::BK);
  };
  for (int i = 0; i < C::ST - 1 && i < n; ++i) issue(i, i * C::STAGE);
  uint32_t at = 0, next = (C::ST - 1) * C::STAGE;  // places of stage i and of the one loaded beside it
  for (int i = 0; i < n; ++i) {
    // this wave has read stage i - 1 and its loads of stage i have landed (those of the later ones may fly, but for the last); then
    // all waves have, and the stage to load may take the place of i - 1
    if (C::ST > 2 && i + C::ST - 2 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((C::ST - 2) * C::LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + C::ST - 1 < n) issue(i + C::ST - 1, next);
    multiply<C, A, B>(lds + at, acc);
    next = at;
    at = at == (C::ST - 1) * C::STAGE ? 0 : at + C::STAGE;
  }
}

// Workgroups go to the eight XCDs in turn; give each XCD a run of tiles (its own L2 then holds the rows that
// neighbouring tiles share).
__device__ __forceinline__ int xcd_tile(int b, int n) {
  const int per = n >> 3, extra = n & 7, x = b & 7;
  return x * per + min(x, extra) + (b >> 3);
}
// Tile order: runs of `G` left tiles for each right tile, then the next right tile
struct TilePos { int m, n; };
__device__ __forceinline__ TilePos tile_at(int id, int nm, int nn, int G) {
  const int band = id / (G * nn), m0 = band * G, g = min(G, nm - m0), r = id - band * G * nn;
  return {m0 + r % g, r / g};
}

// z = W X^T of 256 vocabulary rows x TN tokens, then its statistics or P.  (Workgroups that stay and load the next
// tile's first stage beside an epilogue were no faster, 1113 against 1044 us for 15565 x 768 x 40960: the loop
// over tiles costs 70 registers.)
template <typename C, bool GRADS>
__global__ void __launch_bounds__(C::THREADS, C::BOUND) lce_z_kernel(LceArgs a, int nm, int nn) {
  __shared__ __align__(1024) char lds[C::ST * C::STAGE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int b = static_cast<int>(lce_block());  // (at most 2^14 x 2^16 tiles)
  if (b >= nm * nn) return;
  const TilePos at = tile_at(xcd_tile(b, nm * nn), nm, nn, 4);
  const int t0 = at.n * C::TN, v0 = (GRADS ? a.v0 : 0) + at.m * C::TM;
  if (t0 >= count) return;
  const RowsK<C, C::TM> A(static_cast<const bf16_t *>(a.w) + int64_t(v0) * a.ldw, a.ldw, a.V - v0, a.dk);
  const RowsK<C, C::TN> B(static_cast<const bf16_t *>(a.x) + int64_t(t0) * a.ldx, a.ldx, count - t0, static_cast<int>(a.ldx));
  f32x16 acc[C::MB][2];
  product<C>(A, B, 0, a.dk, lds, acc);
  const int l = threadIdx.x & 63, w = wave_id(), h = l >> 5;
  const int vw = v0 + C::TM / 2 * (w & 1), tw = t0 + 64 * (w >> 1);
  if (!GRADS) {
    lce_row_stats<C::MB, 2>(a, acc, vw, tw, count, 2 * at.m + (w & 1));
    return;
  }
  bool live[2];
  lce_row_grads<C::MB, 2>(a, acc, vw, tw, count, live);
  const int nvc = a.vc / 16;
  const bool few = count <= kFewRows;
  if (few && tw >= kRestAt) return;  // (behind the last row; the remainders of the first take these places)
  const int64_t rest = int64_t(kRestAt / 32) * nvc * 1024;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int mb = 0; mb < C::MB; ++mb)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        char *blk = static_cast<char *>(a.p) +
                    (int64_t(tw / 32 + nb) * nvc + (vw - a.v0) / 16 + 2 * mb + q) * 1024 + (l ^ (h << 2) ^ (q << 3)) * 16;
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[i] = static_cast<uint32_t>(f32_to_bf16(acc[mb][nb][8 * q + 2 * i])) |
                 (static_cast<uint32_t>(f32_to_bf16(acc[mb][nb][8 * q + 2 * i + 1])) << 16);
          if (!live[nb]) u[i] = 0;
        }
        *reinterpret_cast<uint4 *>(blk) = uint4{u[0], u[1], u[2], u[3]};
        if (!few || tw + 32 * nb >= kFewRows) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[i] = static_cast<uint32_t>(remainder(acc[mb][nb][8 * q + 2 * i], u[i] & 0xffffu)) |
                 (static_cast<uint32_t>(remainder(acc[mb][nb][8 * q + 2 * i + 1], u[i] >> 16)) << 16);
          if (!live[nb]) u[i] = 0;
        }
        *reinterpret_cast<uint4 *>(blk + rest) = uint4{u[0], u[1], u[2], u[3]};
      }
}

// dX: tile `at` of share `share` of the piece's vocabulary rows
template <typename C>
__device__ __forceinline__ void dx_tile(const LceArgs &a, TilePos at, int share, DxShares sh, char *lds) {
  const int t0 = at.m * C::TM, c0 = at.n * C::TN;
  const int steps = (a.vn + C::BK - 1) / C::BK, per = (steps + sh.n - 1) / sh.n;
  const int kb = share * per * C::BK, ke = min(a.vn, kb + per * C::BK);
  const PTokens<C> A(a.p, t0, a.vc);
  const ColsK<C, C::TN> B(static_cast<const bf16_t *>(a.w) + int64_t(a.v0) * a.ldw + c0, a.ldw, a.dk - c0, a.vn);
  f32x16 acc[4][2];
  product<C>(A, B, kb, ke, lds, acc);
  const int l = threadIdx.x & 63, w = wave_id(), h = l >> 5;
  float *out = a.dx_part + share * sh.rows * a.d;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int c = c0 + 64 * (w >> 1) + 32 * nb + (l & 31);
    if (c >= a.d) continue;
#pragma unroll
    for (int mb = 0; mb < 4; ++mb) {
      // (rows behind the last labelled one are the partial sums' own padding)
      float *o = out + int64_t(t0 + 128 * (w & 1) + 32 * mb + 4 * h) * a.d + c;
      if (!a.first) {
        float before[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) before[i] = o[int64_t(acc_row(i, 0)) * a.d];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[mb][nb][i] += before[i];
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) o[int64_t(acc_row(i, 0)) * a.d] = acc[mb][nb][i];
    }
  }
}

template <typename C, bool FEW>
__device__ __forceinline__ void dw_tile(const LceArgs &a, TilePos at, int count, char *lds) {
  const int r0 = at.m * C::TM, c0 = at.n * C::TN;
  const int fold = (count + C::BK - 1) / C::BK * C::BK;
  const PVocab<C, FEW> A(a.p, r0, a.vc, fold);
  const ColsK<C, C::TN, FEW> B(static_cast<const bf16_t *>(a.x) + c0, a.ldx, static_cast<int>(a.ldx) - c0, count, fold);
  f32x16 acc[4][2];
  product<C>(A, B, 0, FEW ? 2 * fold : count, lds, acc);
  const float f = lce_factor(a, count);
  const int l = threadIdx.x & 63, w = wave_id(), h = l >> 5;
  bf16_t *dw = static_cast<bf16_t *>(a.dw);
  const bool pairs = a.d % 2 == 0 && reinterpret_cast<uintptr_t>(dw) % 4 == 0;
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int c = c0 + 64 * (w >> 1) + 32 * nb + (l & 31);
#pragma unroll
      for (int i = 0; i < 16; i += 2) {
        // neighbouring lanes swap, so that each stores two columns of one of two rows
        const int r = r0 + 128 * (w & 1) + 32 * mb + acc_row(i, h);
        const float v0 = acc[mb][nb][i] * f, v1 = acc[mb][nb][i + 1] * f;
        if (pairs) {
          const float other = __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, l & 1 ? v0 : v1), 0xb1, 0xf, 0xf, true));
          const uint32_t u = static_cast<uint32_t>(f32_to_bf16(l & 1 ? other : v0)) |
                             (static_cast<uint32_t>(f32_to_bf16(l & 1 ? v1 : other)) << 16);
          if (r + (l & 1) < a.vn && c < a.d) *reinterpret_cast<uint32_t *>(dw + int64_t(a.v0 + r + (l & 1)) * a.d + (c & ~1)) = u;
        } else if (c < a.d) {
          if (r < a.vn) st(dw + int64_t(a.v0 + r) * a.d + c, v0);
          if (r + 1 < a.vn) st(dw + int64_t(a.v0 + r + 1) * a.d + c, v1);
        }
      }
    }
}

// Both products of a piece in one launch, so that neither's last round leaves the chip half idle: `ndx`
// workgroups for dX and then `ndw` for dW (multiples of 8), or the other way round where dW's sums are longer.
struct Grid { int xn, ndx, wm, wn, ndw; };
template <typename C>
__global__ void __launch_bounds__(C::THREADS, C::BOUND) lce_products_kernel(LceArgs a, Grid g) {
  __shared__ __align__(1024) char lds[C::ST * C::STAGE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count), b = blockIdx.x;
  const DxShares sh = lce_dx_shares(a, count);
  const bool dw_first = int64_t(count) * sh.n > a.vn;
  const int b_dx = dw_first ? b - g.ndw : b, b_dw = dw_first ? b : b - g.ndx;
  if (dw_first ? b_dx >= 0 : b_dw < 0) {
    const int xm = (count + C::TM - 1) / C::TM, tiles = xm * g.xn;
    if (b_dx >= tiles * sh.n) return;
    const int id = xcd_tile(b_dx, tiles * sh.n);
    dx_tile<C>(a, tile_at(id % tiles, xm, g.xn, 4), id / tiles, sh, lds);
  } else if (b_dw < g.wm * g.wn) {
    const TilePos at = tile_at(xcd_tile(b_dw, g.wm * g.wn), g.wm, g.wn, 4);
    if (count <= kFewRows) dw_tile<C, true>(a, at, count, lds);
    else dw_tile<C, false>(a, at, count, lds);
  }
}

template <typename T> T up(T a, int64_t b) { return static_cast<T>((a + b - 1) / b); }

// The tile of the logits' products.  256 x 256 moves the least through the caches, but its one workgroup a CU leaves the
// matrix instructions idle through its epilogue: for many tokens and long sums (4096 x 768 x 32000: 236 and 256 us for the
// two products where 256 x 128 take 255 and 271; 2111 tokens 136 and 149 against 134 and 144; 6000 x 256 x 32000: 150 and
// 92 against 135 and 88).  256 x 128: three workgroups to a CU with two stages each where two with three would not
// hold all of them at once (517 tokens: 42.6 against 45 us; 2000 x 100 x 40000: 46 against 54; 256 tokens the other way: 26.8
// against 24.7).  128 x 128 gained 4 us of 55 with 64 tokens and lost with 256 and more.
template <typename F> auto with_shape(int64_t N, int d, int64_t V, F &&f) {
  if (N >= 2560 && d >= 512) return f(Wide{});
  return up(V, Narrow::TM) * up(N, Narrow::TN) <= 2 * 256 ? f(Narrow{}) : f(Three{});
}

}  // namespace

bool lce_bf16_direct(const void *w, int64_t ldw, int d) {
  return d % 8 == 0 && ldw % 8 == 0 && ldw < (1 << 21) && reinterpret_cast<uintptr_t>(w) % 16 == 0;
}

int lce_bf16_parts(int V) { return 2 * up(V, 256); }

// Shares of a piece's vocabulary rows in dX: so many that none takes longer than the launch's work spread
// over the places (two workgroups per CU) does.  Each costs partial sums of N x d in fp32.
int lce_bf16_dx_splits(int64_t N, int d, int V, int vc) {
  const int64_t bk = Narrow::BK, tn = up(d, Narrow::TN), places = 512;
  const int64_t n = std::min(V, vc), steps = up(n, bk);
  const int64_t all = up(N, Narrow::TM) * tn * steps + up(n, Narrow::TM) * tn * up(N, bk);
  return static_cast<int>(std::min<int64_t>({int64_t(kMaxShares), steps, up(steps * places, all)}));
}

namespace {

template <bool GRADS> int z_launch(const LceArgs &a, hipStream_t s) {
  return with_shape(a.N, a.d, GRADS ? a.vn : a.V, [&](auto c) {
    using C = decltype(c);
    static_assert(C::TM == 256, "the vocabulary parts of the statistics");
    const int nm = up(GRADS ? a.vn : a.V, C::TM), nn = up(a.N, C::TN);
    lce_z_kernel<C, GRADS><<<lce_grid(int64_t(nm) * nn), C::THREADS, 0, s>>>(a, nm, nn);
    return check_launch("lce_z_kernel");
  });
}

}  // namespace

int launch_lce_bf16_stats(const LceArgs &a, hipStream_t s) { return z_launch<false>(a, s); }

int launch_lce_bf16_grads(const LceArgs &a, hipStream_t s) { return z_launch<true>(a, s); }

int launch_lce_bf16_products(const LceArgs &a, bool dx, bool dw, hipStream_t s) {
  using C = Narrow;
  const int xn = up(a.d, C::TN), wm = up(a.vn, C::TM);
  const Grid g{xn, dx ? up(a.dx_tiles * xn * a.dx_splits, 8) * 8 : 0, wm, xn, dw ? up(wm * xn, 8) * 8 : 0};
  lce_products_kernel<C><<<g.ndx + g.ndw, C::THREADS, 0, s>>>(a, g);
  return check_launch("lce_products_kernel");
}

}  // namespace motif
