// Cross entropy from hidden states in bf16 on v_mfma_f32_32x32x16_bf16: the three products of
// lce_internal.h, one workgroup of four waves to a tile of 256 x 128 (128 x 64 a wave: 8 matrix
// instructions for 6 LDS reads of 16 bytes a lane), 32 k at a time.  Both sides go straight from memory
// to LDS (16 bytes a lane), three stages deep, 72 KB, so that two workgroups share a CU and one's
// exponentials run beside the other's matrix instructions.
//
//   z = W X^T    left: 256 vocabulary rows, right: 128 tokens; a lane holds one token's scores, so a
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

constexpr int TM = 256, TN = 128, BK = 32, STAGES = 3;
constexpr int A_BYTES = TM * BK * 2, B_BYTES = TN * BK * 2, STAGE = A_BYTES + B_BYTES;
constexpr int LOADS = STAGE / 1024 / 4;  // 1 KB loads of a wave per stage

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

__device__ __forceinline__ uint2 read_tr(const char *p) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)p));
}

// 16 bytes a lane from buffer r at byte voff + soff into LDS at dst + 16 lane (dst the same for the wave).  The
// builtin for it makes the compiler wait for every load in flight before each transposed LDS read, which
// would empty the pipeline at every step; here `product` does all the waiting itself.  (m0 holds the place; nothing
// else in these kernels uses it.)
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 make_rsrc(const void *p, int64_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  return i32x4{static_cast<int>(a), static_cast<int>((a >> 32) & 0xffff), static_cast<int>(bytes), 0x00020000};
}
__device__ __forceinline__ void load_lds(i32x4 r, uint32_t dst, uint32_t voff, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               ::"s"(dst), "v"(voff), "s"(r), "s"(soff) : "memory");
}
__device__ __forceinline__ int wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
__device__ __forceinline__ bf16x8 join(uint2 a, uint2 b) { return __builtin_bit_cast(bf16x8, uint4{a.x, a.y, b.x, b.y}); }

// R rows of 32 k, k beside each other in memory (row stride ld): LDS row r is four 16-byte pieces, piece c at
// c ^ (r / 2 % 4) (eight rows' reads of one piece meet 128 bytes of banks once).
template <int R> struct RowsK {
  static constexpr int NJ = R * 64 / 1024 / 4;
  i32x4 buf;
  uint32_t off[NJ];
  int kc, K;
  __device__ __forceinline__ RowsK(const bf16_t *p, int64_t ld, int rows, int K_) : K(K_) {
    const int l = threadIdx.x & 63, w = wave_id();
    const int n = min(rows, R);
    buf = make_rsrc(p, n > 0 ? ((n - 1) * ld + K) * 2 : 0);
    kc = ((l & 3) ^ ((l >> 3) & 3)) * 8;
#pragma unroll
    for (int j = 0; j < NJ; ++j) off[j] = static_cast<uint32_t>(((w * NJ + j) * 16 + (l >> 2)) * ld * 2 + kc * 2);
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int w = wave_id();
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      load_lds(buf, dst + (w * NJ + j) * 1024, k0 + kc < K ? off[j] : 0xfffffff0u, k0 * 2);
  }
  // operand of rows r0 .. r0 + 31 at k step s (16 k)
  __device__ __forceinline__ static bf16x8 frag(const char *src, int r0, int s) {
    const int l = threadIdx.x & 63, r = r0 + (l & 31), c = 2 * s + (l >> 5);
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(src + r * 64 + ((c ^ ((r >> 1) & 3)) * 16)));
  }
};

// 32 k rows of R columns (row stride ld): LDS row k is R / 8 pieces, piece c at c ^ swap(k).
__device__ __forceinline__ int tr_swap(int k) { return ((k & 1) << 2) | ((k & 2) ? 10 : 0); }
template <int R> struct ColsK {
  static constexpr int NJ = R * 64 / 1024 / 4, RP = 512 / R;
  const bf16_t *p;
  int64_t ld;
  int cols, K;
  uint32_t off[NJ];
  __device__ __forceinline__ ColsK(const bf16_t *p_, int64_t ld_, int cols_, int K_) : p(p_), ld(ld_), cols(cols_), K(K_) {
    const int l = threadIdx.x & 63, w = wave_id();
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int k = (w * NJ + j) * RP + l / (R / 8);
      off[j] = static_cast<uint32_t>(k * ld * 2 + ((l % (R / 8)) ^ tr_swap(k)) * 16);
    }
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int w = wave_id(), n = min(K - k0, BK);
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

// P's blocks as the left side of dX: 256 tokens x 32 vocabulary rows, block (t / 32, v / 16) in order
struct PTokens {
  static constexpr int NJ = 4;
  const char *p;
  int nvc;
  uint32_t off[NJ];
  __device__ __forceinline__ PTokens(const void *p_, int t0, int vc) : nvc(vc / 16) {
    const int l = threadIdx.x & 63, w = wave_id();
    p = static_cast<const char *>(p_) + int64_t(t0 / 32) * nvc * 1024;
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int q = w * NJ + j;
      off[j] = static_cast<uint32_t>(((q >> 1) * nvc + (q & 1)) * 1024 + l * 16);
    }
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int w = wave_id();
    const i32x4 buf = make_rsrc(p + int64_t(k0 / 16) * 1024, (7 * nvc + 2) * 1024);
#pragma unroll
    for (int j = 0; j < NJ; ++j) load_lds(buf, dst + (w * NJ + j) * 1024, off[j], 0);
  }
  __device__ __forceinline__ static bf16x8 frag(const char *src, int r0, int s) {
    const int l = threadIdx.x & 63, q = (r0 >> 5) * 2 + s;
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const uint4 *>(src + q * 1024 + (l ^ ((l >> 5) << 2) ^ ((s & 1) << 3)) * 16));
  }
};

// ... as the left side of dW: 256 vocabulary rows x 32 tokens
struct PVocab {
  static constexpr int NJ = 4;
  const char *p;
  int nvc;
  __device__ __forceinline__ PVocab(const void *p_, int r0, int vc) : nvc(vc / 16) {
    p = static_cast<const char *>(p_) + int64_t(r0 / 16) * 1024;
  }
  __device__ __forceinline__ void issue(uint32_t dst, int k0) const {
    const int l = threadIdx.x & 63, w = wave_id();
    const i32x4 buf = make_rsrc(p + int64_t(k0 / 32) * nvc * 1024, 16 * 1024);
#pragma unroll
    for (int j = 0; j < NJ; ++j) load_lds(buf, dst + (w * NJ + j) * 1024, (w * NJ + j) * 1024 + l * 16, 0);
  }
  __device__ __forceinline__ static bf16x8 frag(const char *src, int r0, int s) {
    const int l = threadIdx.x & 63, g = (l >> 4) & 1, h = l & 1, t = 16 * s + 4 * (l >> 5) + ((l >> 2) & 3);
    const int place = (t + 32 * h) ^ (h << 2) ^ (g << 3);
    const char *q = src + ((r0 >> 4) + g) * 1024 + ((l >> 1) & 1) * 8;
    return join(read_tr(q + place * 16), read_tr(q + (place ^ 8) * 16));
  }
};

template <typename A, typename B>
__device__ __forceinline__ void product(const A &a, const B &b, int kb, int ke, char *lds, f32x16 (&acc)[4][2]) {
  const int w = wave_id();
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mb][nb][i] = 0.f;
  const int n = (ke - kb + BK - 1) / BK;
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char *)lds));
  auto issue = [&](int i, uint32_t place) {
    a.issue(base + place, kb + i * BK);
    b.issue(base + place + A_BYTES, kb + i * BK);
  };
  for (int i = 0; i < STAGES - 1 && i < n; ++i) issue(i, i * STAGE);
  uint32_t at = 0, next = (STAGES - 1) * STAGE;  // places of stage i and of the one loaded beside it
  for (int i = 0; i < n; ++i) {
    // this wave has read stage i - 1 and its loads of stage i have landed (those of i + 1 may fly); then all
    // waves have, and stage i + 2 may take the place of i - 1
    if (i + 1 < n) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LOADS) : "memory");
    else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (i + STAGES - 1 < n) issue(i + STAGES - 1, next);
    const char *sa = lds + at, *sb = sa + A_BYTES;
    next = at;
    at = at == (STAGES - 1) * STAGE ? 0 : at + STAGE;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 fa[4], fb[2];
#pragma unroll
      for (int nb = 0; nb < 2; ++nb) fb[nb] = B::frag(sb, 64 * (w >> 1) + 32 * nb, s);
#pragma unroll
      for (int mb = 0; mb < 4; ++mb) fa[mb] = A::frag(sa, 128 * (w & 1) + 32 * mb, s);
#pragma unroll
      for (int mb = 0; mb < 4; ++mb)
#pragma unroll
        for (int nb = 0; nb < 2; ++nb)
          acc[mb][nb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[mb], fb[nb], acc[mb][nb], 0, 0, 0);
    }
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

template <bool GRADS>
__global__ void __launch_bounds__(256, 2) lce_z_kernel(LceArgs a, int nm, int nn) {
  __shared__ __align__(1024) char lds[STAGES * STAGE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const TilePos at = tile_at(xcd_tile(blockIdx.x, gridDim.x), nm, nn, 4);
  const int t0 = at.n * TN, v0 = (GRADS ? a.v0 : 0) + at.m * TM;
  if (t0 >= count) return;
  const RowsK<TM> A(static_cast<const bf16_t *>(a.w) + int64_t(v0) * a.ldw, a.ldw, a.V - v0, a.d);
  const RowsK<TN> B(static_cast<const bf16_t *>(a.x) + int64_t(t0) * a.ldx, a.ldx, count - t0, static_cast<int>(a.ldx));
  f32x16 acc[4][2];
  product(A, B, 0, a.d, lds, acc);
  const int l = threadIdx.x & 63, w = wave_id(), h = l >> 5;
  const int vw = v0 + 128 * (w & 1), tw = t0 + 64 * (w >> 1);
  if (!GRADS) {
    lce_row_stats<4, 2>(a, acc, vw, tw, count, 2 * at.m + (w & 1));
    return;
  }
  lce_row_grads<4, 2>(a, acc, vw, tw, count);
  const int nvc = a.vc / 16;
#pragma unroll
  for (int nb = 0; nb < 2; ++nb)
#pragma unroll
    for (int mb = 0; mb < 4; ++mb)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          u[i] = static_cast<uint32_t>(f32_to_bf16(acc[mb][nb][8 * q + 2 * i])) |
                 (static_cast<uint32_t>(f32_to_bf16(acc[mb][nb][8 * q + 2 * i + 1])) << 16);
        char *blk = static_cast<char *>(a.p) +
                    (int64_t(tw / 32 + nb) * nvc + (vw - a.v0) / 16 + 2 * mb + q) * 1024;
        *reinterpret_cast<uint4 *>(blk + (l ^ (h << 2) ^ (q << 3)) * 16) = uint4{u[0], u[1], u[2], u[3]};
      }
}

// dX: tile `at` of share `share` of the piece's vocabulary rows (dx_splits shares, each with its own partial sums)
__device__ __forceinline__ void dx_tile(const LceArgs &a, TilePos at, int share, int count, char *lds) {
  const int t0 = at.m * TM, c0 = at.n * TN;
  if (t0 >= count) return;
  const int steps = (a.vn + BK - 1) / BK, per = (steps + a.dx_splits - 1) / a.dx_splits;
  const int kb = share * per * BK, ke = min(a.vn, kb + per * BK);
  const PTokens A(a.p, t0, a.vc);
  const ColsK<TN> B(static_cast<const bf16_t *>(a.w) + int64_t(a.v0) * a.ldw + c0, a.ldw, a.d - c0, a.vn);
  f32x16 acc[4][2];
  product(A, B, kb, ke, lds, acc);
  const int l = threadIdx.x & 63, w = wave_id(), h = l >> 5;
  float *out = a.dx_part + int64_t(share) * a.n_pad * a.d;
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

__device__ __forceinline__ void dw_tile(const LceArgs &a, TilePos at, int count, char *lds) {
  const int r0 = at.m * TM, c0 = at.n * TN;
  const PVocab A(a.p, r0, a.vc);
  const ColsK<TN> B(static_cast<const bf16_t *>(a.x) + c0, a.ldx, static_cast<int>(a.ldx) - c0, count);
  f32x16 acc[4][2];
  product(A, B, 0, count, lds, acc);
  const float f = lce_factor(a, count);
  const int l = threadIdx.x & 63, w = wave_id(), h = l >> 5;
#pragma unroll
  for (int mb = 0; mb < 4; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int c = c0 + 64 * (w >> 1) + 32 * nb + (l & 31);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = r0 + 128 * (w & 1) + 32 * mb + acc_row(i, h);
        if (r < a.vn && c < a.d) st(static_cast<bf16_t *>(a.dw) + int64_t(a.v0 + r) * a.d + c, acc[mb][nb][i] * f);
      }
    }
}

// Both products of a piece in one launch, so that neither's last round leaves the chip half idle: `ndx`
// workgroups (a multiple of 8) for dX, then dW's.
struct Grid { int xm, xn, ndx, wm, wn; };
__global__ void __launch_bounds__(256, 2) lce_products_kernel(LceArgs a, Grid g) {
  __shared__ __align__(1024) char lds[STAGES * STAGE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int b = blockIdx.x, tiles = g.xm * g.xn;
  if (b < g.ndx) {
    const int id = xcd_tile(b, g.ndx);
    if (id < tiles * a.dx_splits) dx_tile(a, tile_at(id % tiles, g.xm, g.xn, 4), id / tiles, count, lds);
  } else {
    dw_tile(a, tile_at(xcd_tile(b - g.ndx, gridDim.x - g.ndx), g.wm, g.wn, 4), count, lds);
  }
}

template <typename T> T up(T a, int b) { return (a + b - 1) / b; }

}  // namespace

bool lce_bf16_serves(const void *w, int64_t ldw, int d, int dtype) {
  return dtype == MOTIF_BF16 && d % 8 == 0 && ldw % 8 == 0 && ldw < (1 << 21) && reinterpret_cast<uintptr_t>(w) % 16 == 0;
}

int lce_bf16_parts(int V) { return 2 * up(V, TM); }

// Shares of a piece's vocabulary rows in dX: so many that none takes longer than the launch's work spread
// over 512 places (two workgroups per CU) does.  Each costs partial sums of N x d in fp32.
int lce_bf16_dx_splits(int64_t N, int d, int V, int vc) {
  const int64_t n = std::min(V, vc), tn = up(d, TN), steps = up(n, BK);
  const int64_t all = up(N, TM) * tn * steps + up(n, TM) * tn * up(N, BK);
  return static_cast<int>(std::min<int64_t>({int64_t(16), steps, (steps * 512 + all - 1) / all}));
}

int launch_lce_bf16_stats(const LceArgs &a, hipStream_t s) {
  const int nm = up(a.V, TM), nn = up(a.N, TN);
  lce_z_kernel<false><<<nm * nn, 256, 0, s>>>(a, nm, nn);
  return check_launch("lce_z_kernel (statistics)");
}

int launch_lce_bf16_grads(const LceArgs &a, hipStream_t s) {
  const int nm = up(a.vn, TM), nn = up(a.N, TN);
  lce_z_kernel<true><<<nm * nn, 256, 0, s>>>(a, nm, nn);
  return check_launch("lce_z_kernel (gradients)");
}

int launch_lce_bf16_products(const LceArgs &a, bool dx, bool dw, hipStream_t s) {
  Grid g{};
  g.xm = up(a.N, TM), g.xn = g.wn = up(a.d, TN), g.wm = up(a.vn, TM);
  g.ndx = dx ? up(g.xm * g.xn * a.dx_splits, 8) * 8 : 0;
  lce_products_kernel<<<g.ndx + (dw ? g.wm * g.wn : 0), 256, 0, s>>>(a, g);
  return check_launch("lce_products_kernel");
}

}  // namespace motif
