// Chord attention backward on bf16 MFMA (gfx950), head dim 64.
//
// For logits z_ij = c_i r_ij with r_ij = s q_i.k_j + b_h(j - i_abs), c_i = ssmax_h
// log_n[b, i], b_h(d) = -alpha_h (|d - mu_h| + eps)^beta_h, keys j <= i_abs, softmax
// P over keys and O = P V, the gradients of an upstream dO are
//   dP = dO V^T,  Delta_i = dO_i . O_i,  dZ = P * (dP - Delta),
//   dV = P^T dO,  dQ = s (c dZ) K,  dK = s (c dZ)^T Q,
//   d alpha_h = sum c dZ * (-(x^beta)),  d beta_h = sum c dZ * b ln x,
//   d mu_h = sum c dZ * alpha beta x^(beta-1) sign(d - mu),  d ssmax_h = sum log_n dZ r
// with x = |d - mu| + eps (the reference's backward: motif/ops/chord_attention.py:518-949,
// :1348-1470).  P is rebuilt from the forward's log-sum-exp (log2 units), as there.  s c dZ is
// rounded to bf16 as one operand in both kernels.
//
// chord_bwd_dq_kernel: one workgroup per (head, 128 queries, chunk of key tiles, batch
// row), a wave per 32 queries.  S^T = K Q^T and dP^T = V dO^T per 32-key tile on 32x32x16
// MFMAs (lane l owns query column l % 32, so the row values -- Delta, the log-sum-exp, c --
// are scalars per lane), dQ^T += K^T (s c dZ)^T from the same registers.  It also
// computes Delta (written for the second kernel) and partial sums of the four parameter
// gradients.
// chord_bwd_dkdv_kernel: one workgroup per (query head, 128 keys, chunk of query tiles,
// batch row), a wave per 32 keys (lane l owns key column l % 32): S = Q K^T, dP = dO V^T,
// dV^T += dO^T P, dK^T += Q^T (s c dZ).
// The causal loop of a block is cut into chunks of at most `cq` / `ckv` tiles so that no
// workgroup runs much longer than the average (the heaviest block otherwise sets the
// kernel's length); chunks write fp32 partials that chord_bwd_reduce_kernel sums in a
// fixed order (with one chunk and no GQA sharing the kernels write bf16 directly).
// Both loops keep two LDS tile buffers (one barrier per tile) and the next tile's global
// loads in registers.  The GGD bias (and, in the dQ kernel, its three parameter
// derivatives) come from per-wave windows over the 63 distances a 32 x 32 tile meets,
// evaluated in registers; tiles wholly below the causal diagonal skip the masks.
//
// Bound by VALU issue (a tile's 1024 scores take ~10 instructions each and one exp2, its 12 or 16
// MFMAs a third of that), so what is not per score is kept off the vector unit: tiles come through
// range-checked buffers with fixed lane offsets, accumulators sit in ordinary registers, the dK / dV
// kernel reads a query's four values as one row that the dQ kernel wrote.  B = 2, 12 heads, 2048
// tokens: dQ 73 -> 57 us, dK / dV 72 -> 62, reductions 26 (three launches) -> 14 (one).  Whole
// backward, back to back: that size 165 -> 131 us, 4096 tokens (3 kv heads) 282 -> 193, 1024 tokens
// 71 -> 45, 16 x 512 tokens 125 -> 88.  Tiles are held by rows alone and transposed as they are read: in
// a graph 2 x 2048 tokens 121 -> 118 us, 4096 181 -> 178.
//
// Under a window (WIN) both loops walk only the tiles that a block's windows and first tokens reach, and
// every block has about the same work, so nothing is cut but the queries that see a block's first tokens
// from behind its windows (plan_bwd_window).  The distances' powers come from a 64-bit table: in
// registers they took 20 instructions a score where 12 are left, and were the parameter gradients'
// largest error.  2 x 2048 tokens, 12 heads, window 512: dQ 43 us, dK / dV 37, reduction 4, table 3;
// 4001 tokens, 3 kv heads, window 1000: 68, 60, 10, 3.  At these lengths no unit is busy half of the time
// (4001 tokens: VALU 49% and 31% of the busy cycles, LDS 26% and 35%, MFMA 20%): 1.5 workgroups per CU,
// a wave or two per SIMD, each a chain of reads, products, exponentials and a barrier a tile.  P and P (dP -
// Delta) are rounded to bf16 where they enter the products for dQ, dK and dV, as in the causal kernels, since
// the matrix instructions' fp32 form would take 16 times as long (2.4e-3 off against 64 bits, where rounding the
// gradients alone gives 1.7e-3); the parameter sums take them in fp32.
#include <algorithm>
#include <string>
#include <type_traits>

#include "capi_internal.h"
#include "chord_internal.h"
#include "common.h"

namespace motif {

namespace {

constexpr int kBD = 64;    // head dim
constexpr int kT = 32;     // keys (dQ kernel) or queries (dK / dV kernel) per tile
constexpr int kBlk = 128;  // queries (dQ kernel) or keys (dK / dV kernel) per workgroup

struct ChordBwdArgs {
  const bf16_t *q; int64_t q_sb, q_sh, q_st;
  const bf16_t *k; int64_t k_sb, k_sh, k_st;
  const bf16_t *v; int64_t v_sb, v_sh, v_st;
  const bf16_t *o; int64_t o_sb, o_sh, o_st;
  const bf16_t *dout; int64_t d_sb, d_sh, d_st;
  const float *lse;  // [B][H][L], log2 units
  const float *alpha, *beta, *mu, *ssmax;
  const float *log_n; int64_t ln_sb, ln_st;
  bf16_t *dq; int64_t dq_sb, dq_sh, dq_st;
  bf16_t *dk; int64_t dk_sb, dk_sh, dk_st;
  bf16_t *dv; int64_t dv_sb, dv_sh, dv_st;
  float *dparam;  // [4][H]: d alpha, d beta, d mu, d ssmax
  // workspace
  float4 *rows;   // [B][H][L]: {log-sum-exp, Delta, c log2(e), c s} of a query
  float *pparam;  // [nsq][B][nqb][H][4] parameter partial sums
  float *pq;      // [nsq][B][H][L][64] dQ partials (nsq > 1)
  float *pk, *pv; // [nskv][H][B][S][64] dK / dV partials (unless kv_direct)
  int B, H, Hkv, L, S, q_start, nqb, nkb;
  int cq, nsq, ckv, nskv, kv_direct;
  float scale, eps;
  // window (WIN kernels): key blocks that hold first tokens, the chunks of `csink` query tiles behind
  // their windows, those chunks' partials [nsc][H][B][nsb * 128][64], and the key rows of pk / pv
  int window, sinks, nsb, nsc, csink, prows;
  float *pks, *pvs;
  const float2 *dist;  // [H][dist_n] {x^beta, x^beta log2 x} of distances 0, -1, .. (motif_chord_distances)
  const float *dmu;    // [H][dist_n] x^(beta - 1) sign
  int dist_n;
};

// Key tiles the dQ workgroup of query block qb visits, and query tiles the dK / dV
// workgroup of key block kb visits (first tile, end).
__host__ __device__ inline int dq_tiles(int qb, int L, int q_start) {
  const int last = std::min(L, qb * kBlk + kBlk) - 1;
  return (q_start + last + 1 + kT - 1) / kT;
}
__host__ __device__ inline int kv_first_tile(int kb, int q_start) { return std::max(0, kb * kBlk - q_start) / kT; }
// End of the query tiles whose windows reach key block kb.
__host__ __device__ inline int kv_window_end(int kb, int L, int q_start, int window) {
  const int last = kb * kBlk + kBlk - 1 + window - 1 - q_start;  // the last query that sees its last key
  return last < 0 ? 0 : std::min((L + kT - 1) / kT, last / kT + 1);
}

__device__ __forceinline__ f32x16 mma32(const bf16x8 &a, const bf16x8 &b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk2bf(float x0, float x1) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x0, x1}, bf16x2v));
}
__device__ __forceinline__ bf16x8 pack8(const float *x) {
  return __builtin_bit_cast(bf16x8, uint4{pk2bf(x[0], x[1]), pk2bf(x[2], x[3]), pk2bf(x[4], x[5]), pk2bf(x[6], x[7])});
}
__device__ __forceinline__ uint4 ld16(const bf16_t *p) { return *reinterpret_cast<const uint4 *>(p); }

// Tile staging by 128 threads t: row stage_row(t), 8-element pieces t & 3 and + 4 of a
// 32-row x 64 tile of [rows][64] bf16 rows, through a range-checked buffer that starts at the
// tile's first row (uniform) and ends at row `nrows` of the matrix: rows past it read 0 with no
// branch, and a tile costs two loads and its base.  The loads go to registers one tile ahead of the
// stores.  ANY: rows that share elements (an expanded gradient), run backwards or lie past the
// buffer's 32-bit offsets are told from those past the end by number, in kernels of their own (as
// a branch here, its loads made every tile wait for all in flight: 10% of the whole backward).
struct Stage2 { uint4 a, b; };
constexpr int64_t kBufStride = int64_t(1) << 25;  // 31 rows and a bit stay below 2^31 bytes
template <bool ANY>
struct StageSrc {
  const bf16_t *base;
  int64_t st;
  int nrows;
  uint32_t off;  // this thread's first piece
  __device__ __forceinline__ StageSrc(const bf16_t *p, int64_t s, int n, int t)
      : base(p), st(s), nrows(n), off(static_cast<uint32_t>((stage_row(t) * s + 8 * (t & 3)) * 2)) {}
  __device__ __forceinline__ Stage2 load(int row0) const { return load(row0, min(kT, nrows - row0)); }
  __device__ __forceinline__ Stage2 load(int row0, int rows) const {
    if constexpr (ANY) {
      const int r = stage_row(threadIdx.x & 127);
      const bf16_t *p = base + (row0 + r) * st + 8 * (threadIdx.x & 3);
      const uint4 z = {0u, 0u, 0u, 0u};
      return {r < rows ? ld16(p) : z, r < rows ? ld16(p + 32) : z};
    }
    const buf_t buf = make_buf(base + int64_t(row0) * st, rows > 0 ? static_cast<uint32_t>(((rows - 1) * st + kBD) * 2) : 0u);
    return {buf_ld16(buf, off), buf_ld16(buf, off + 64u)};
  }
};
// The pieces into the tile's rows.
__device__ __forceinline__ void stage_store(const Stage2 &g, int t, bf16_t *rows) {
  const int r = stage_row(t), o = r * kBD + 8 * ((t & 3) ^ piece_swap(r));
  *reinterpret_cast<uint4 *>(rows + o) = g.a;
  *reinterpret_cast<uint4 *>(rows + (o ^ 32)) = g.b;
}
// This lane's reads of a tile: row lane % 32, features 16 ds + 8 (lane / 32) .. + 7 (a product over
// features), and feature 32 dt + lane % 32 of rows 16 ks + 4 (lane / 32) .. + 3 and + 8 .. + 11 (over rows,
// in the order in which the accumulators hold them).
struct TileReads {
  int ro, to;
  __device__ __forceinline__ explicit TileReads(int lane) {
    const int lc = lane & 31, hh = lane >> 5, r = 4 * hh + ((lane & 15) >> 2);
    ro = lc * kBD + 8 * (hh ^ piece_swap(lc));
    to = r * kBD + 8 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ piece_swap(r)) + 4 * (lane & 1);
  }
  __device__ __forceinline__ bf16x8 row(const bf16_t *tile, int ds) const {
    return *reinterpret_cast<const bf16x8 *>(tile + (ro ^ (16 * ds)));
  }
  __device__ __forceinline__ bf16x8 col(const bf16_t *tile, int dt, int ks) const {
    const bf16_t *p = tile + (to ^ (32 * dt)) + 16 * ks * kBD;
    const uint2 a = ld_transposed(p), b = ld_transposed(p + 8 * kBD);
    return __builtin_bit_cast(bf16x8, uint4{a.x, a.y, b.x, b.y});
  }
};

// ------------------------------------------------------------------ dQ (+ Delta, parameter sums)
// WIN: with a window; MU: mu's gradient too (the layer's is frozen; it costs a window kernel 2 of 13
// instructions per score).
template <bool ANY, bool WIN, bool MU>
__global__ void __launch_bounds__(256) chord_bwd_dq_kernel(ChordBwdArgs a) {
  const int h = blockIdx.x, qb = a.nqb - 1 - static_cast<int>(blockIdx.y);  // heaviest blocks first
  const int b = blockIdx.z / a.nsq, chunk = blockIdx.z - b * a.nsq;
  const int kv_end = min(a.S, a.q_start + min(a.L, qb * kBlk + kBlk));
  // (a window's loop is one chunk, run over the tiles of the first tokens and of the block's windows)
  const KeyWalk<kT> walk(WIN ? a.q_start + qb * kBlk : 0, kv_end, WIN ? a.window : kMaxWindow, WIN ? a.sinks : 0);
  const int t_begin = WIN ? 0 : chunk * a.cq, t_end = WIN ? walk.count : min(dq_tiles(qb, a.L, a.q_start), t_begin + a.cq);
  if (!WIN && t_begin >= t_end) return;
  auto key_at = [&](int x) { return WIN ? walk.start(x) : x * kT; };
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 31, hh = lane >> 5;
  const int kvh = h / (a.H / a.Hkv);
  const int q0 = qb * kBlk + 32 * w;
  const int my_q = q0 + lc;
  const bool qv = my_q < a.L;
  // waves 0, 1 stage K, 2, 3 V; the first tile's loads go ahead of the rest
  const bool kside = w < 2;
  const StageSrc<ANY> src(kside ? a.k + b * a.k_sb + kvh * a.k_sh : a.v + b * a.v_sb + kvh * a.v_sh, kside ? a.k_st : a.v_st,
                     kv_end, tid & 127);
  auto load_tile = [&](int x) { return WIN ? src.load(walk.start(x), walk.rows(x)) : src.load(x * kT); };
  Stage2 stg = load_tile(t_begin);
  const int qr = min(my_q, a.L - 1);

  // this lane's query row: Q and dO as B operands (d = 16 ds + 8 hh .. +8), Delta
  const bf16_t *qrow = a.q + b * a.q_sb + h * a.q_sh + int64_t(qr) * a.q_st;
  const bf16_t *drow = a.dout + b * a.d_sb + h * a.d_sh + int64_t(qr) * a.d_st;
  const bf16_t *orow = a.o + b * a.o_sb + h * a.o_sh + int64_t(qr) * a.o_st;
  bf16x8 qreg[4], dreg[4];
  float dsum = 0.f;
#pragma unroll
  for (int ds = 0; ds < 4; ++ds) {
    qreg[ds] = __builtin_bit_cast(bf16x8, ld16(qrow + 16 * ds + 8 * hh));
    dreg[ds] = __builtin_bit_cast(bf16x8, ld16(drow + 16 * ds + 8 * hh));
    const bf16x8 ov = __builtin_bit_cast(bf16x8, ld16(orow + 16 * ds + 8 * hh));
#pragma unroll
    for (int t = 0; t < 8; ++t) dsum = fmaf(static_cast<float>(dreg[ds][t]), static_cast<float>(ov[t]), dsum);
  }
  {
    const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(dsum), __float_as_uint(dsum), false, false);
    dsum = __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
  }
  const float delta = dsum;
  const size_t ri = (static_cast<size_t>(b) * a.H + h) * a.L + my_q;
  const float lse2 = qv ? a.lse[ri] : 0.f;
  const float lam = a.log_n[b * a.ln_sb + int64_t(qr) * a.ln_st];
  const float sig = a.ssmax[h], al = a.alpha[h], be = a.beta[h], mu = a.mu[h];
  const float s = a.scale, c = sig * lam, cl = c * kLog2e, cs = c * s;
  if (!WIN && chunk == 0 && qv && hh == 0) a.rows[ri] = float4{lse2, delta, cl, cs};
  const int q_abs = a.q_start + my_q;
  const int wave_kv_end = a.q_start + min(a.L, q0 + 32);  // keys this wave sees: < wave_kv_end
  const int k_max = WIN ? min(q_abs, a.S - 1) : q_abs;    // this query's last key

  __shared__ __attribute__((aligned(16))) bf16_t sK[2][kT * kBD], sV[2][kT * kBD];  // the tile's rows
  const TileReads rd(lane);
  // per wave and distance: {b, d/d alpha, d/d beta, d/d mu}; WIN: {x^beta, x^beta log2 x, d x^beta / d x sign}
  using DistV = std::conditional_t<WIN && !MU, float2, float4>;
  __shared__ DistV sW[4][64];
  __shared__ float sRed[4][4];

  f32x16 dqacc[2];
  dqacc[0] = f32x16{};
  dqacc[1] = f32x16{};
  float sa = 0.f, sb = 0.f, sm = 0.f, ss = 0.f;
  // WIN: a row's sums of P and g = P (dP - Delta), and of both times r, x^beta, x^beta log2 x and mu's
  // factor, see below
  struct RowSums { float p, g, gs, ga, gb, gm, ps, pa, pb, pm; };
  RowSums sum = {};
  f32x16 pkacc[2];
  pkacc[0] = pkacc[1] = f32x16{};

  auto store_kv = [&](const Stage2 &g, int buf) { stage_store(g, tid & 127, kside ? sK[buf] : sV[buf]); };
  // WIN: this lane's entry of tile x's window, d = key - q_abs = key_at(x) - q_start - q0 - 31 + lane, loaded a
  // tile ahead (outside the table, where no query of the wave sees a key: zeros)
  const buf_t dbuf = make_buf(WIN ? a.dist + static_cast<size_t>(h) * a.dist_n : nullptr, WIN ? a.dist_n * 8u : 0u);
  const buf_t mbuf = make_buf(WIN ? a.dmu + static_cast<size_t>(h) * a.dist_n : nullptr, WIN && MU ? a.dist_n * 4u : 0u);
  auto dist_at = [&](int x) {
    const uint32_t i = static_cast<uint32_t>(a.q_start + q0 + 31 - lane - key_at(x));
    const uint32_t o = i < static_cast<uint32_t>(a.dist_n) ? i : 0x10000000u;
    const uint2 u = buf_ld8(dbuf, 8u * o);
    float4 r{__uint_as_float(u.x), __uint_as_float(u.y), 0.f, 0.f};
    if constexpr (MU) r.z = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(mbuf, 4u * o, 0, 0));
    return r;
  };
  float4 dnext{};
  if constexpr (WIN) dnext = dist_at(t_begin);
  store_kv(stg, 0);
  stg = load_tile(t_begin + 1);  // (past the last tile: zeros)
  __syncthreads();

  for (int kt = t_begin; kt < t_end; ++kt) {
    const int n0 = key_at(kt), buf = (kt - t_begin) & 1;
    if (kt + 1 < t_end) {  // the next tile into the other buffer (free since the last barrier)
      store_kv(stg, buf ^ 1);
      stg = load_tile(kt + 2);
    }
    const float4 dcur = dnext;
    if constexpr (WIN) dnext = dist_at(kt + 1);
    if (n0 < wave_kv_end && (!WIN || n0 + kT - 1 > a.q_start + q0 - a.window || n0 < a.sinks)) {
      // window entry j (lane j < 63): distance d = key - q_abs = n0 - q_start - q0 - 31 + j
      if constexpr (WIN && !MU) sW[w][lane] = float2{dcur.x, dcur.y};
      else if constexpr (WIN) sW[w][lane] = dcur;
      else {
        const int d = n0 - a.q_start - q0 - 31 + lane;
        const float x = fabsf(static_cast<float>(d) - mu) + a.eps;
        const float l2 = fast_log2(x);
        const float xb = fast_exp2(be * l2);
        const float bias = -al * xb;
        const float sgn = static_cast<float>(d) > mu ? 1.f : (static_cast<float>(d) < mu ? -1.f : 0.f);
        sW[w][lane] = d <= 0 ? float4{bias, -xb, bias * l2 * 0.6931471805599453f, al * be * xb * rcp_fast(x) * sgn}
                             : float4{0.f, 0.f, 0.f, 0.f};
      }
      // The wave reads other lanes' window entries below: LDS operations of a wave complete
      // in order, and the wave barrier keeps the compiler from moving those reads above
      // this store.
      __builtin_amdgcn_wave_barrier();
      f32x16 sacc = {}, pacc = {};
#pragma unroll
      for (int ds = 0; ds < 4; ++ds) {
        sacc = mma32(rd.row(sK[buf], ds), qreg[ds], sacc);
        pacc = mma32(rd.row(sV[buf], ds), dreg[ds], pacc);
      }
      float dz[16], pr[WIN ? 16 : 1];
      auto body = [&](auto masked) {
        uint32_t seen = 0u;  // WIN: the tile's keys that this query sees
        RowSums t;
        if constexpr (WIN && decltype(masked)::value)
          seen = qv ? seen_keys(min(k_max - n0, walk.rows(kt) - 1), q_abs - a.window - n0, a.sinks - n0) >> (4 * hh) : 0u;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kk = 8 * (r >> 2) + 4 * hh + (r & 3);
          const DistV wv = sW[w][kk - lc + 31];
          if constexpr (WIN) {
            const float rr = fmaf(-al, wv.x, s * sacc[r]);
            float p = fast_exp2(fmaf(cl, rr, -lse2));
            if constexpr (decltype(masked)::value) p = seen & (1u << (8 * (r >> 2) + (r & 3))) ? p : 0.f;
            const float g = p * (pacc[r] - delta);
            // a tile's sums on their own, then onto the row's: half the terms to round with
            auto add = [r](float &x, float f, float y) { x = r ? fmaf(f, y, x) : f * y; };
            t.p = r ? t.p + p : p;
            t.g = r ? t.g + g : g;
            add(t.gs, g, rr);
            add(t.ga, g, wv.x);
            add(t.gb, g, wv.y);
            add(t.ps, p, rr);
            add(t.pa, p, wv.x);
            add(t.pb, p, wv.y);
            if constexpr (MU) {
              add(t.gm, g, wv.z);
              add(t.pm, p, wv.z);
            }
            pr[r] = p;
            dz[r] = g;  // (c s goes onto the sum)
          } else {
            const float rr = fmaf(s, sacc[r], wv.x);
            float p = fast_exp2(fmaf(cl, rr, -lse2));
            if constexpr (decltype(masked)::value) p = (qv && n0 + kk <= q_abs) ? p : 0.f;
            const float g = p * (pacc[r] - delta);
            ss = fmaf(g, rr, ss);
            sa = fmaf(g, wv.y, sa);
            sb = fmaf(g, wv.z, sb);
            sm = fmaf(g, wv.w, sm);
            dz[r] = g * cs;  // (rounded to bf16 with its factor, as the dK / dV kernel rounds it)
          }
        }
        if constexpr (WIN) {
          sum.p += t.p, sum.g += t.g;
          sum.gs += t.gs, sum.ga += t.ga, sum.gb += t.gb;
          sum.ps += t.ps, sum.pa += t.pa, sum.pb += t.pb;
          if constexpr (MU) sum.gm += t.gm, sum.pm += t.pm;
        }
      };
      // every key of the tile at or before every query of the wave (and in its window), all queries valid
      if (n0 + kT - 1 <= a.q_start + q0 && q0 + 32 <= a.L &&
          (!WIN || (n0 + kT <= a.S && (n0 > a.q_start + q0 + 31 - a.window || n0 + kT <= a.sinks))))
        body(std::false_type{});
      else body(std::true_type{});
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const bf16x8 zb = pack8(dz + 8 * ks);
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
          const bf16x8 kto = rd.col(sK[buf], dt, ks);
          dqacc[dt] = mma32(kto, zb, dqacc[dt]);
          if constexpr (WIN) pkacc[dt] = mma32(kto, pack8(pr + 8 * ks), pkacc[dt]);
        }
      }
    }
    __syncthreads();  // this tile's reads done, the next tile's stores visible
  }

  // Delta = dO . O carries O's rounding (2^-8 of a term).  The sum over a row's keys of P (dP - Delta)
  // is 0, so what is left of it, rho, is the error of Delta: every sum of P (dP - Delta) x is put
  // right by rho times that of P x, and the second kernel is given Delta + rho.  The weights' own sum
  // takes the log-sum-exp's fp32 rounding (1e-6 of a weight) out of the parameter sums.  (2 x 2048
  // tokens, a window of 512, against 64 bits: dq and dk 4.6e-3 off without, 2.4e-3 with; alpha's
  // gradient 1e-2 and 1e-6.  Summed by tiles of r itself, ssmax's is 0.6e-6 off; one long sum of S and one
  // of x^beta, put together at the end, were 2.5e-6 off.)
  if constexpr (WIN) {
    auto both = [](float x) {  // over the two lane halves
      const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
      return __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
    };
    const float ps = both(sum.p), inv = ps > 0.f ? 1.f / ps : 0.f, r = both(sum.g) * inv;
    ss = fmaf(-r, sum.ps, sum.gs) * inv;                                    // r = s S + b, b = -alpha x^beta
    sa = -fmaf(-r, sum.pa, sum.ga) * inv;                                   // d b / d alpha
    sb = fmaf(-r, sum.pb, sum.gb) * inv * (-al * 0.6931471805599453f);      // d b / d beta = b ln x
    if constexpr (MU) sm = fmaf(-r, sum.pm, sum.gm) * inv * (al * be);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) dqacc[dt][i] = cs * fmaf(-r, pkacc[dt][i], dqacc[dt][i]);
    if (qv && hh == 0) a.rows[ri] = float4{lse2, delta + r, cl, cs};
  }

  if (qv) {
    if (a.nsq == 1) {
      bf16_t *dst = a.dq + b * a.dq_sb + h * a.dq_sh + int64_t(my_q) * a.dq_st;
#pragma unroll
      for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *reinterpret_cast<uint2 *>(dst + 32 * dt + 8 * q4 + 4 * hh) =
              uint2{pk2bf(dqacc[dt][4 * q4], dqacc[dt][4 * q4 + 1]), pk2bf(dqacc[dt][4 * q4 + 2], dqacc[dt][4 * q4 + 3])};
    } else {
      float *dst = a.pq + ((((static_cast<size_t>(chunk) * a.B + b) * a.H + h) * a.L) + my_q) * kBD;
#pragma unroll
      for (int dt = 0; dt < 2; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
          *reinterpret_cast<f32x4 *>(dst + 32 * dt + 8 * q4 + 4 * hh) =
              f32x4{dqacc[dt][4 * q4], dqacc[dt][4 * q4 + 1], dqacc[dt][4 * q4 + 2], dqacc[dt][4 * q4 + 3]};
    }
  }
  // parameter sums: d/d(bias) = c dZ, d/d ssmax = log_n dZ r
  float part[4] = {wave_sum(sa * c), wave_sum(sb * c), wave_sum(sm * c), wave_sum(ss * lam)};
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sRed[w][i] = part[i];
  }
  __syncthreads();
  if (tid < 4) {
    const float tot = sRed[0][tid] + sRed[1][tid] + sRed[2][tid] + sRed[3][tid];
    a.pparam[(((static_cast<size_t>(chunk) * a.B + b) * a.nqb + qb) * a.H + h) * 4 + tid] = tot;
  }
}

// ------------------------------------------------------------------ dK, dV
template <bool ANY, bool WIN>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) chord_bwd_dkdv_kernel(ChordBwdArgs a) {
  // WIN: first the chunks behind the windows of the blocks that hold first tokens (the longest loops)
  const int h = blockIdx.x, nsx = WIN ? a.nsb * a.nsc : 0;
  const bool behind = WIN && static_cast<int>(blockIdx.y) < nsx;
  const int kb = behind ? blockIdx.y / a.nsc : blockIdx.y - nsx;
  const int b = WIN ? blockIdx.z : blockIdx.z / a.nskv;
  const int chunk = !WIN ? blockIdx.z - b * a.nskv : behind ? blockIdx.y - kb * a.nsc : 0;
  const int qt_end = (a.L + kT - 1) / kT;
  int t_begin, t_end;
  if constexpr (WIN) {
    const int w_end = kv_window_end(kb, a.L, a.q_start, a.window);
    t_begin = behind ? max(w_end, kv_first_tile(kb, a.q_start)) + chunk * a.csink : kv_first_tile(kb, a.q_start);
    t_end = behind ? min(qt_end, t_begin + a.csink) : w_end;
    if (behind && t_begin >= t_end) return;
  } else {
    t_begin = kv_first_tile(kb, a.q_start) + chunk * a.ckv;
    t_end = min(qt_end, t_begin + a.ckv);
    // a chunk with no tiles writes nothing, except that direct writes must cover every key
    if (t_begin >= t_end && !(a.kv_direct && chunk == 0)) return;
  }
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lc = lane & 31, hh = lane >> 5;
  const int kvh = h / (a.H / a.Hkv);
  const int k0w = kb * kBlk + 32 * w;
  const int my_k = k0w + lc;
  const bool kvld = my_k < a.S;
  // waves 0, 1 stage Q, 2, 3 dO; threads 0-31 the row values; the first tile's loads go ahead of the rest
  const bool qside = w < 2;
  const size_t rbase = (static_cast<size_t>(b) * a.H + h) * a.L;
  const StageSrc<ANY> src(qside ? a.q + b * a.q_sb + h * a.q_sh : a.dout + b * a.d_sb + h * a.d_sh, qside ? a.q_st : a.d_st, a.L,
                     tid & 127);
  auto load_row = [&](int i0) {  // (queries past L: zeros, c = 0)
    const int n = min(kT, a.L - i0);
    return __builtin_bit_cast(float4, buf_ld16(make_buf(a.rows + rbase + i0, n > 0 ? n * 16u : 0u), 16u * (tid & (kT - 1))));
  };
  Stage2 stg = src.load(t_begin * kT);
  float4 rowv = load_row(t_begin * kT);
  const int kr = min(my_k, a.S - 1);

  const bf16_t *krow = a.k + b * a.k_sb + kvh * a.k_sh + int64_t(kr) * a.k_st;
  const bf16_t *vrow = a.v + b * a.v_sb + kvh * a.v_sh + int64_t(kr) * a.v_st;
  bf16x8 kreg[4], vreg[4];
#pragma unroll
  for (int ds = 0; ds < 4; ++ds) {
    kreg[ds] = __builtin_bit_cast(bf16x8, ld16(krow + 16 * ds + 8 * hh));
    vreg[ds] = __builtin_bit_cast(bf16x8, ld16(vrow + 16 * ds + 8 * hh));
  }

  __shared__ __attribute__((aligned(16))) bf16_t sQ[2][kT * kBD], sD[2][kT * kBD];  // Q and dO rows of the query tile
  const TileReads rd(lane);
  __shared__ float4 sRow[2][kT];  // per query: {lse2, Delta, c log2 e, c s}
  __shared__ float sW[4][64];     // per wave: the bias window

  f32x16 dkacc[2], dvacc[2];
  dkacc[0] = dkacc[1] = dvacc[0] = dvacc[1] = f32x16{};
  const float s = a.scale;
  const float sig = a.ssmax[h], al = a.alpha[h], be = a.beta[h], mu = a.mu[h];
  auto store_q = [&](const Stage2 &g, const float4 &rv, int buf) {
    stage_store(g, tid & 127, qside ? sQ[buf] : sD[buf]);
    if (tid < kT) sRow[buf][tid] = rv;
  };
  // WIN: this lane's entry of the window of query tile qt, distance k0w - q_start - 32 qt - 31 + lane
  const buf_t dbuf = make_buf(WIN ? a.dist + static_cast<size_t>(h) * a.dist_n : nullptr, WIN ? a.dist_n * 8u : 0u);
  auto dist_at = [&](int qt) {
    const uint32_t i = static_cast<uint32_t>(a.q_start + qt * kT + 31 - lane - k0w);
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                         dbuf, 8u * (i < static_cast<uint32_t>(a.dist_n) ? i : 0x10000000u), 0, 0));
  };
  float dnext = 0.f;
  if constexpr (WIN) dnext = dist_at(t_begin);
  store_q(stg, rowv, 0);
  stg = src.load((t_begin + 1) * kT);
  rowv = load_row((t_begin + 1) * kT);
  __syncthreads();

  for (int qt = t_begin; qt < t_end; ++qt) {
    const int i0 = qt * kT, buf = (qt - t_begin) & 1;
    if (qt + 1 < t_end) {  // the next tile into the other buffer (free since the last barrier)
      store_q(stg, rowv, buf ^ 1);
      stg = src.load(i0 + 2 * kT);
      rowv = load_row(i0 + 2 * kT);
    }
    const float dcur = dnext;
    if constexpr (WIN) dnext = dist_at(qt + 1);
    // a wave whose keys all lie past the tile's last query (or past S) skips it
    if (k0w < a.S && a.q_start + i0 + kT - 1 >= k0w &&
        (!WIN || k0w + kT - 1 > a.q_start + i0 - a.window || k0w < a.sinks)) {
      // window entry j: distance key - q_abs = k0w - q_start - i0 - 31 + j
      if constexpr (WIN) {
        sW[w][lane] = -al * dcur;
      } else {
        const int d = k0w - a.q_start - i0 - 31 + lane;
        const float x = fabsf(static_cast<float>(d) - mu) + a.eps;
        sW[w][lane] = d <= 0 ? -al * fast_exp2(be * fast_log2(x)) : 0.f;
      }
      // The wave reads other lanes' window entries below: LDS operations of a wave complete
      // in order, and the wave barrier keeps the compiler from moving those reads above
      // this store.
      __builtin_amdgcn_wave_barrier();
      f32x16 sacc = {}, pacc = {};
#pragma unroll
      for (int ds = 0; ds < 4; ++ds) {
        sacc = mma32(rd.row(sQ[buf], ds), kreg[ds], sacc);
        pacc = mma32(rd.row(sD[buf], ds), vreg[ds], pacc);
      }
      float pv[16], dz[16];
      // the tile's queries that see this lane's key: q_lo .. q_lo + q_n - 1 (one compare per element)
      const int q_lo = max(0, my_k - a.q_start - i0);
      const int q_hi = WIN && my_k >= a.sinks ? min(min(kT, a.L - i0), my_k + a.window - a.q_start - i0) : min(kT, a.L - i0);
      const uint32_t q_n = kvld ? max(0, q_hi - q_lo) : 0;
      auto body = [&](auto masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int qq = 8 * (r >> 2) + 4 * hh + (r & 3);
          const float4 rw = sRow[buf][qq];
          const float rr = fmaf(s, sacc[r], sW[w][lc - qq + 31]);
          float p = fast_exp2(fmaf(rw.z, rr, -rw.x));
          const bool ok = !decltype(masked)::value || static_cast<uint32_t>(qq - q_lo) < q_n;
          p = ok ? p : 0.f;
          pv[r] = p;
          dz[r] = p * (pacc[r] - rw.y) * rw.w;
          if constexpr (WIN) dz[r] = ok ? dz[r] : 0.f;  // (a row that no query sees may hold anything)
        }
      };
      // every key of the wave at or before every query of the tile (and in its window), all queries valid
      if (k0w + 31 <= a.q_start + i0 && i0 + kT <= a.L &&
          (!WIN || (k0w + kT <= a.S && (k0w > a.q_start + i0 + kT - 1 - a.window || k0w + kT <= a.sinks))))
        body(std::false_type{});
      else body(std::true_type{});
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const bf16x8 pb = pack8(pv + 8 * ks), zb = pack8(dz + 8 * ks);
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
          dvacc[dt] = mma32(rd.col(sD[buf], dt, ks), pb, dvacc[dt]);
          dkacc[dt] = mma32(rd.col(sQ[buf], dt, ks), zb, dkacc[dt]);
        }
      }
    }
    __syncthreads();  // this tile's reads done, the next tile's stores visible
  }

  if (!kvld) return;
  if (a.kv_direct && (!WIN || kb >= a.nsb)) {
    bf16_t *dk = a.dk + b * a.dk_sb + kvh * a.dk_sh + int64_t(my_k) * a.dk_st;
    bf16_t *dv = a.dv + b * a.dv_sb + kvh * a.dv_sh + int64_t(my_k) * a.dv_st;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const int d0 = 32 * dt + 8 * q4 + 4 * hh;
        *reinterpret_cast<uint2 *>(dk + d0) =
            uint2{pk2bf(dkacc[dt][4 * q4], dkacc[dt][4 * q4 + 1]), pk2bf(dkacc[dt][4 * q4 + 2], dkacc[dt][4 * q4 + 3])};
        *reinterpret_cast<uint2 *>(dv + d0) =
            uint2{pk2bf(dvacc[dt][4 * q4], dvacc[dt][4 * q4 + 1]), pk2bf(dvacc[dt][4 * q4 + 2], dvacc[dt][4 * q4 + 3])};
      }
    return;
  }
  const int rows = !WIN ? a.S : behind ? a.nsb * kBlk : a.prows;
  const size_t o = (((static_cast<size_t>(chunk) * a.H + h) * a.B + b) * rows + my_k) * kBD;
  float *pk = WIN && behind ? a.pks : a.pk, *pv = WIN && behind ? a.pvs : a.pv;
#pragma unroll
  for (int dt = 0; dt < 2; ++dt)
#pragma unroll
    for (int q4 = 0; q4 < 4; ++q4) {
      const int d0 = 32 * dt + 8 * q4 + 4 * hh;
      *reinterpret_cast<f32x4 *>(pk + o + d0) =
          f32x4{dkacc[dt][4 * q4], dkacc[dt][4 * q4 + 1], dkacc[dt][4 * q4 + 2], dkacc[dt][4 * q4 + 3]};
      *reinterpret_cast<f32x4 *>(pv + o + d0) =
          f32x4{dvacc[dt][4 * q4], dvacc[dt][4 * q4 + 1], dvacc[dt][4 * q4 + 2], dvacc[dt][4 * q4 + 3]};
    }
}

// dK / dV of kv head kvh = the sum over its GQA group's query heads and the chunks of the
// key's block, in that order, rounded to bf16; one thread per 4 elements.
__device__ __forceinline__ void reduce_kv(const ChordBwdArgs &a, int block) {
  const int64_t n4 = static_cast<int64_t>(a.B) * a.Hkv * a.S * (kBD / 4);
  const int64_t e = static_cast<int64_t>(block) * 256 + threadIdx.x;
  if (e >= n4) return;
  const int d0 = 4 * static_cast<int>(e % (kBD / 4));
  const int64_t rest = e / (kBD / 4);
  const int sk = static_cast<int>(rest % a.S);
  const int kvh = static_cast<int>((rest / a.S) % a.Hkv), b = static_cast<int>(rest / (static_cast<int64_t>(a.S) * a.Hkv));
  const int G = a.H / a.Hkv;
  const int qt_end = (a.L + kT - 1) / kT;
  const int nqt = max(0, qt_end - kv_first_tile(sk / kBlk, a.q_start));
  const int ns = (nqt + a.ckv - 1) / a.ckv;
  f32x4 ks = {0.f, 0.f, 0.f, 0.f}, vs = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < G; ++g)
    for (int c = 0; c < ns; ++c) {
      const size_t o = (((static_cast<size_t>(c) * a.H + kvh * G + g) * a.B + b) * a.S + sk) * kBD + d0;
      const f32x4 pk = *reinterpret_cast<const f32x4 *>(a.pk + o), pv = *reinterpret_cast<const f32x4 *>(a.pv + o);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ks[i] += pk[i];
        vs[i] += pv[i];
      }
    }
  bf16_t *dk = a.dk + b * a.dk_sb + kvh * a.dk_sh + int64_t(sk) * a.dk_st + d0;
  bf16_t *dv = a.dv + b * a.dv_sb + kvh * a.dv_sh + int64_t(sk) * a.dv_st + d0;
  *reinterpret_cast<uint2 *>(dk) = uint2{pk2bf(ks[0], ks[1]), pk2bf(ks[2], ks[3])};
  *reinterpret_cast<uint2 *>(dv) = uint2{pk2bf(vs[0], vs[1]), pk2bf(vs[2], vs[3])};
}

// The same for a window: the first a.prows keys' window partials (every key, or with kv_direct those
// of the blocks that hold first tokens), then the chunks behind those blocks' windows, in order.
__device__ __forceinline__ void reduce_kv_window(const ChordBwdArgs &a, int block) {
  const int rows = min(a.prows, a.S);
  const int64_t n4 = static_cast<int64_t>(a.B) * a.Hkv * rows * (kBD / 4);
  const int64_t e = static_cast<int64_t>(block) * 256 + threadIdx.x;
  if (e >= n4) return;
  const int d0 = 4 * static_cast<int>(e % (kBD / 4));
  const int64_t rest = e / (kBD / 4);
  const int sk = static_cast<int>(rest % rows);
  const int kvh = static_cast<int>((rest / rows) % a.Hkv), b = static_cast<int>(rest / (static_cast<int64_t>(rows) * a.Hkv));
  const int G = a.H / a.Hkv, kb = sk / kBlk, qt_end = (a.L + kT - 1) / kT;
  int ns = 0;
  if (kb < a.nsb) {
    const int first = max(kv_window_end(kb, a.L, a.q_start, a.window), kv_first_tile(kb, a.q_start));
    ns = (max(0, qt_end - first) + a.csink - 1) / a.csink;
  }
  f32x4 ks = {0.f, 0.f, 0.f, 0.f}, vs = {0.f, 0.f, 0.f, 0.f};
  for (int g = 0; g < G; ++g) {
    const int h = kvh * G + g;
    const size_t o = ((static_cast<size_t>(h) * a.B + b) * a.prows + sk) * kBD + d0;
    f32x4 pk = *reinterpret_cast<const f32x4 *>(a.pk + o), pv = *reinterpret_cast<const f32x4 *>(a.pv + o);
    for (int c = 0;; ++c) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ks[i] += pk[i];
        vs[i] += pv[i];
      }
      if (c == ns) break;
      const size_t oc = (((static_cast<size_t>(c) * a.H + h) * a.B + b) * (a.nsb * kBlk) + sk) * kBD + d0;
      pk = *reinterpret_cast<const f32x4 *>(a.pks + oc);
      pv = *reinterpret_cast<const f32x4 *>(a.pvs + oc);
    }
  }
  bf16_t *dk = a.dk + b * a.dk_sb + kvh * a.dk_sh + int64_t(sk) * a.dk_st + d0;
  bf16_t *dv = a.dv + b * a.dv_sb + kvh * a.dv_sh + int64_t(sk) * a.dv_st + d0;
  *reinterpret_cast<uint2 *>(dk) = uint2{pk2bf(ks[0], ks[1]), pk2bf(ks[2], ks[3])};
  *reinterpret_cast<uint2 *>(dv) = uint2{pk2bf(vs[0], vs[1]), pk2bf(vs[2], vs[3])};
}

// dQ = the sum over the chunks of the query's block, in order, rounded to bf16.
__device__ __forceinline__ void reduce_q(const ChordBwdArgs &a, int block) {
  const int64_t n4 = static_cast<int64_t>(a.B) * a.H * a.L * (kBD / 4);
  const int64_t e = static_cast<int64_t>(block) * 256 + threadIdx.x;
  if (e >= n4) return;
  const int d0 = 4 * static_cast<int>(e % (kBD / 4));
  const int64_t rest = e / (kBD / 4);
  const int i = static_cast<int>(rest % a.L);
  const int h = static_cast<int>((rest / a.L) % a.H), b = static_cast<int>(rest / (static_cast<int64_t>(a.L) * a.H));
  const int ns = (dq_tiles(i / kBlk, a.L, a.q_start) + a.cq - 1) / a.cq;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < ns; ++c) {
    const f32x4 p = *reinterpret_cast<const f32x4 *>(
        a.pq + (((static_cast<size_t>(c) * a.B + b) * a.H + h) * a.L + i) * kBD + d0);
#pragma unroll
    for (int t = 0; t < 4; ++t) acc[t] += p[t];
  }
  bf16_t *dst = a.dq + b * a.dq_sb + h * a.dq_sh + int64_t(i) * a.dq_st + d0;
  *reinterpret_cast<uint2 *>(dst) = uint2{pk2bf(acc[0], acc[1]), pk2bf(acc[2], acc[3])};
}

// dparam[k][h] = the sum of the dQ workgroups' partials (batch rows, query blocks, chunks):
// one wave per (k, h), lanes over (batch row, query block) in a fixed order.
template <bool WIN>
__device__ __forceinline__ void reduce_param(const ChordBwdArgs &a, int t) {
  const int h = t % a.H, k = t / a.H, lane = threadIdx.x & 63;
  float acc = 0.f;
  for (int e = lane; e < a.B * a.nqb; e += 64) {
    const int b = e / a.nqb, qb = e - b * a.nqb;
    const int ns = WIN ? 1 : (dq_tiles(qb, a.L, a.q_start) + a.cq - 1) / a.cq;
    for (int c = 0; c < ns; ++c) acc += a.pparam[(((static_cast<size_t>(c) * a.B + b) * a.nqb + qb) * a.H + h) * 4 + k];
  }
  acc = wave_sum(acc);
  if (lane == 0) a.dparam[k * a.H + h] = acc;
}

// Every reduction in one launch (three apart took 12.5 + 7.7 + 4.7 us at B = 2, 12 heads, 2048
// tokens, most of it launch and tail): workgroups [0, nkv) dK / dV, then nq of dQ, then one of four
// waves per four parameter sums.
template <bool WIN>
__global__ void __launch_bounds__(256) chord_bwd_reduce_kernel(ChordBwdArgs a, int nkv, int nq) {
  const int block = blockIdx.x;
  if (block < nkv) return WIN ? reduce_kv_window(a, block) : reduce_kv(a, block);
  if (block < nkv + nq) return reduce_q(a, block - nkv);
  const int t = 4 * (block - nkv - nq) + (threadIdx.x >> 6);
  if (t < 4 * a.H) reduce_param<WIN>(a, t);
}

}  // namespace

// Chunk sizes: about as many full chunks over the whole causal loop as the kernel's workgroups fit
// on the chip at once (dQ: three per CU, dK / dV: two; blocks end in shorter chunks, so the counts
// aimed at lie below 768 and 512), at least 6 tiles each and at most 8 chunks per block.  Swept at
// 12 heads (the two kernels and the reductions in a loop, us; 1024 chunks of at least 16 tiles against
// these): 2 x 2048 tokens 141 -> 117, 4096 tokens (3 kv heads) 209 -> 186, 1024 tokens 57 -> 47, 700
// tokens 57 -> 42.
// A cut saves the tiles by which it shortens the longest block (1.25 us each on a CU of its own) and
// costs each chunk's fp32 partial rows, written and read again: it is made where there are at most
// `worth` chunks per tile saved.  Cut and whole measured side by side at 519 (dQ) and 399 (dK / dV)
// sizes of 4 to 16 heads, 1 to 64 sequences and 64 to 4096 tokens: the rule takes the faster form or
// one within 5% (dQ; worth 62), 7% (dK / dV, 42) and 8% (heads that share a kv head, whose partials
// are written either way: 52).  Always cutting lost up to 31% where the launch filled the chip by
// itself; 12 heads, us, cut / by the rule (and with the 1024-chunk plan): 16 x 512 tokens 104 / 87
// (122), 8 x 512 75 / 60 (70), 16 x 256 59 / 42 (48).
struct BwdPlan {
  int nqb, nkb, cq, nsq, ckv, nskv;
  bool kv_direct;
  size_t off_param, off_pq, off_pk, off_pv, bytes;
};

static BwdPlan plan_bwd(int B, int H, int Hkv, int L, int S, int q_start) {
  BwdPlan p{};
  p.nqb = (L + kBlk - 1) / kBlk;
  p.nkb = (S + kBlk - 1) / kBlk;
  const int qt_end = (L + kT - 1) / kT;
  auto chunking = [&](int nblocks, auto tiles, int target, int worth, int &csize, int &ns) {
    int64_t total = 0, chunks = 0;
    int maxt = 0;
    for (int i = 0; i < nblocks; ++i) {
      total += tiles(i);
      maxt = std::max(maxt, tiles(i));
    }
    csize = static_cast<int>(std::max<int64_t>({6, (total * B * H + target - 1) / target, (maxt + 7) / 8}));
    for (int i = 0; i < nblocks; ++i) chunks += (tiles(i) + csize - 1) / csize;
    if (chunks * B * H > int64_t(worth) * (maxt - csize)) csize = std::max(csize, maxt);
    ns = std::max(1, (maxt + csize - 1) / csize);
  };
  chunking(p.nqb, [&](int qb) { return dq_tiles(qb, L, q_start); }, 640, 62, p.cq, p.nsq);
  chunking(p.nkb, [&](int kb) { return std::max(0, qt_end - kv_first_tile(kb, q_start)); }, 384, H == Hkv ? 42 : 52, p.ckv,
           p.nskv);
  p.kv_direct = H == Hkv && p.nskv == 1;
  auto al = [](size_t x) { return (x + 255) / 256 * 256; };
  size_t off = al(static_cast<size_t>(B) * H * L * sizeof(float4));  // the query rows' values
  p.off_param = off;
  off += al(static_cast<size_t>(p.nsq) * B * p.nqb * H * 4 * sizeof(float));
  p.off_pq = off;
  if (p.nsq > 1) off += al(static_cast<size_t>(p.nsq) * B * H * L * kBD * sizeof(float));
  p.off_pk = p.off_pv = off;
  if (!p.kv_direct) {
    const size_t kvp = al(static_cast<size_t>(p.nskv) * H * B * S * kBD * sizeof(float));
    p.off_pv = off + kvp;
    off += 2 * kvp;
  }
  p.bytes = off;
  return p;
}

// The windowed backward: one chunk per query block and per key block (every block's loop is about as
// long as its window), and for the blocks that hold first tokens chunks of the queries behind.
struct WinBwdPlan {
  int nqb, nkb, nsb, nsc, csink, prows;
  bool kv_direct;
  size_t off_param, off_pk, off_pv, off_pks, off_pvs, bytes;
};

static WinBwdPlan plan_bwd_window(int B, int H, int Hkv, int L, int S, int q_start, int window, int sinks) {
  WinBwdPlan p{};
  p.nqb = (L + kBlk - 1) / kBlk;
  p.nkb = (S + kBlk - 1) / kBlk;
  p.nsb = (std::min(sinks, S) + kBlk - 1) / kBlk;
  const int qt_end = (L + kT - 1) / kT;
  int most = 0;  // query tiles behind a window that see first tokens
  for (int kb = 0; kb < p.nsb; ++kb)
    most = std::max(most, qt_end - std::max(kv_window_end(kb, L, q_start, window), kv_first_tile(kb, q_start)));
  // chunks about as long as a window's loop, at most 16 of them and no more than make 2048 workgroups, eight per
  // CU: each is a copy of the blocks' fp32 partials (at 8192 tokens, 12 heads, every second of them a first
  // token, 16 are 403 MB, 5 are 126)
  const int64_t blocks = static_cast<int64_t>(p.nsb) * H * B;
  const int cap = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(16, 2048 / std::max<int64_t>(1, blocks))));
  p.csink = std::max({8, (window + kBlk) / kT, (most + cap - 1) / cap});
  p.nsc = (most + p.csink - 1) / p.csink;
  p.kv_direct = H == Hkv;
  p.prows = p.kv_direct ? p.nsb * kBlk : S;
  auto al = [](size_t x) { return (x + 255) / 256 * 256; };
  size_t off = al(static_cast<size_t>(B) * H * L * sizeof(float4));
  p.off_param = off;
  off += al(static_cast<size_t>(B) * p.nqb * H * 4 * sizeof(float));
  const size_t row = static_cast<size_t>(H) * B * kBD * sizeof(float);
  p.off_pk = off;
  p.off_pv = off += al(row * p.prows);
  p.off_pks = off += al(row * p.prows);
  p.off_pvs = off += al(row * p.nsc * p.nsb * kBlk);
  p.bytes = off + al(row * p.nsc * p.nsb * kBlk);
  return p;
}

}  // namespace motif

extern "C" size_t motif_chord_bwd_workspace_bytes(int B, int H, int Hkv, int L, int S, int q_start) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || L < 0 || S < 0 || q_start < 0) return 0;
  return motif::plan_bwd(B, H, Hkv, L, S, q_start).bytes + 16;  // (up to 15 to align an odd base)
}

extern "C" int motif_chord_bwd(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st,
    const void *v, int64_t v_sb, int64_t v_sh, int64_t v_st,
    const void *out, int64_t o_sb, int64_t o_sh, int64_t o_st,
    const void *dout, int64_t d_sb, int64_t d_sh, int64_t d_st,
    const float *lse, const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st,
    void *dq, int64_t dq_sb, int64_t dq_sh, int64_t dq_st,
    void *dk, int64_t dk_sb, int64_t dk_sh, int64_t dk_st,
    void *dv, int64_t dv_sb, int64_t dv_sh, int64_t dv_st,
    float *dparam, int B, int H, int Hkv, int L, int S, int D, int q_start, float scale, float eps,
    void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  using namespace motif;
  if (B < 0 || H <= 0 || Hkv <= 0 || L < 0 || S < 0 || H % Hkv != 0)
    return set_error(MOTIF_ERR_INVALID, "chord_bwd: bad sizes");
  if (dtype != MOTIF_BF16 || D != kBD)
    return set_error(MOTIF_ERR_UNSUPPORTED, "chord_bwd: bf16 with head_dim 64 only");
  if (q_start < 0 || static_cast<int64_t>(q_start) + L > S)
    return set_error(MOTIF_ERR_INVALID, "chord_bwd: need 0 <= q_start and q_start + L <= S");
  if (!dparam) return set_error(MOTIF_ERR_INVALID, "chord_bwd: NULL pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (B == 0 || S == 0) {  // (L <= S) nothing to differentiate: zero parameter gradients
    ChordBwdArgs z{};
    z.H = H;
    z.cq = 1;
    z.dparam = dparam;
    chord_bwd_reduce_kernel<false><<<dim3(H), dim3(256), 0, s>>>(z, 0, 0);
    return check_launch("chord_bwd_reduce_kernel");
  }
  if (!q || !k || !v || !out || !dout || !lse || !alpha || !beta || !mu || !ssmax || !log_n || !dq || !dk || !dv)
    return set_error(MOTIF_ERR_INVALID, "chord_bwd: NULL pointer");
  const int64_t st = q_sb | q_sh | q_st | k_sb | k_sh | k_st | v_sb | v_sh | v_st | o_sb | o_sh | o_st | d_sb | d_sh |
                     d_st | dq_sb | dq_sh | dq_st | dk_sb | dk_sh | dk_st | dv_sb | dv_sh | dv_st;
  const uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dout) |
                       reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv);
  if ((st & 7) != 0 || (al & 15) != 0) return set_error(MOTIF_ERR_UNSUPPORTED, "chord_bwd: need 16-byte aligned rows");
  const BwdPlan pl = plan_bwd(B, H, Hkv, L, S, q_start);
  const size_t pad = -reinterpret_cast<uintptr_t>(workspace) & 15;  // (the size asked for holds it)
  if (!workspace || workspace_bytes < pl.bytes + pad)
    return set_error(MOTIF_ERR_INVALID, "chord_bwd: workspace too small (need " + std::to_string(pl.bytes + pad) + " bytes)");
  ChordBwdArgs a;
  a.q = static_cast<const bf16_t *>(q); a.q_sb = q_sb; a.q_sh = q_sh; a.q_st = q_st;
  a.k = static_cast<const bf16_t *>(k); a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v = static_cast<const bf16_t *>(v); a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  a.o = static_cast<const bf16_t *>(out); a.o_sb = o_sb; a.o_sh = o_sh; a.o_st = o_st;
  a.dout = static_cast<const bf16_t *>(dout); a.d_sb = d_sb; a.d_sh = d_sh; a.d_st = d_st;
  a.lse = lse; a.alpha = alpha; a.beta = beta; a.mu = mu; a.ssmax = ssmax;
  a.log_n = log_n; a.ln_sb = ln_sb; a.ln_st = ln_st;
  a.dq = static_cast<bf16_t *>(dq); a.dq_sb = dq_sb; a.dq_sh = dq_sh; a.dq_st = dq_st;
  a.dk = static_cast<bf16_t *>(dk); a.dk_sb = dk_sb; a.dk_sh = dk_sh; a.dk_st = dk_st;
  a.dv = static_cast<bf16_t *>(dv); a.dv_sb = dv_sb; a.dv_sh = dv_sh; a.dv_st = dv_st;
  a.dparam = dparam;
  char *ws = static_cast<char *>(workspace) + pad;
  a.rows = reinterpret_cast<float4 *>(ws);
  a.pparam = reinterpret_cast<float *>(ws + pl.off_param);
  a.pq = reinterpret_cast<float *>(ws + pl.off_pq);
  a.pk = reinterpret_cast<float *>(ws + pl.off_pk);
  a.pv = reinterpret_cast<float *>(ws + pl.off_pv);
  a.B = B; a.H = H; a.Hkv = Hkv; a.L = L; a.S = S; a.q_start = q_start;
  a.nqb = pl.nqb; a.nkb = pl.nkb;
  a.cq = pl.cq; a.nsq = pl.nsq; a.ckv = pl.ckv; a.nskv = pl.nskv; a.kv_direct = pl.kv_direct ? 1 : 0;
  a.scale = scale; a.eps = eps;
  bool any = false;  // (a single row's stride is not used)
  for (int64_t x : {q_st, d_st}) any |= L > 1 && (x < kBD || x >= kBufStride);
  for (int64_t x : {k_st, v_st}) any |= S > 1 && (x < kBD || x >= kBufStride);
  int rc = MOTIF_OK;
  if (L > 0) {  // with no queries dK and dV are zero (the dK / dV pass below writes them)
    (any ? chord_bwd_dq_kernel<true, false, true> : chord_bwd_dq_kernel<false, false, true>)<<<dim3(H, pl.nqb, B * pl.nsq), dim3(256), 0, s>>>(a);
    if ((rc = check_launch("chord_bwd_dq_kernel"))) return rc;
  }
  (any ? chord_bwd_dkdv_kernel<true, false> : chord_bwd_dkdv_kernel<false, false>)<<<dim3(H, pl.nkb, B * pl.nskv), dim3(256), 0, s>>>(a);
  if ((rc = check_launch("chord_bwd_dkdv_kernel"))) return rc;
  auto blocks = [](int64_t rows) { return static_cast<int>((rows * (kBD / 4) + 255) / 256); };
  const int nkv = pl.kv_direct ? 0 : blocks(static_cast<int64_t>(B) * Hkv * S);
  const int nq = L > 0 && pl.nsq > 1 ? blocks(static_cast<int64_t>(B) * H * L) : 0;
  chord_bwd_reduce_kernel<false><<<dim3(nkv + nq + H), dim3(256), 0, s>>>(a, nkv, nq);
  if ((rc = check_launch("chord_bwd_reduce_kernel"))) return rc;
  return MOTIF_OK;
}

extern "C" size_t motif_chord_window_bwd_workspace_bytes(int B, int H, int Hkv, int L, int S, int q_start, int window,
                                                         int sinks) {
  using namespace motif;
  if (B <= 0 || H <= 0 || Hkv <= 0 || L < 0 || S < 0 || q_start < 0 || window < 1 || sinks < 0) return 0;
  if (std::max<int64_t>(S, static_cast<int64_t>(q_start) + L) >= kMaxWindow) return 0;
  return plan_bwd_window(B, H, Hkv, L, S, q_start, std::min(window, kMaxWindow), std::min(sinks, kMaxWindow)).bytes + 16;
}

extern "C" int motif_chord_window_bwd(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st,
    const void *v, int64_t v_sb, int64_t v_sh, int64_t v_st,
    const void *out, int64_t o_sb, int64_t o_sh, int64_t o_st,
    const void *dout, int64_t d_sb, int64_t d_sh, int64_t d_st,
    const float *lse, const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st,
    void *dq, int64_t dq_sb, int64_t dq_sh, int64_t dq_st,
    void *dk, int64_t dk_sb, int64_t dk_sh, int64_t dk_st,
    void *dv, int64_t dv_sb, int64_t dv_sh, int64_t dv_st,
    float *dparam, int B, int H, int Hkv, int L, int S, int D, int q_start, float scale, float eps,
    int window, int sinks, int need_mu, const float *distances, int distances_len,
    void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  using namespace motif;
  if (B < 0 || H <= 0 || Hkv <= 0 || L < 0 || S < 0 || H % Hkv != 0)
    return set_error(MOTIF_ERR_INVALID, "chord_window_bwd: bad sizes");
  if (dtype != MOTIF_BF16 || D != kBD)
    return set_error(MOTIF_ERR_UNSUPPORTED, "chord_window_bwd: bf16 with head_dim 64 only");
  if (q_start < 0 || window < 1 || sinks < 0)
    return set_error(MOTIF_ERR_INVALID, "chord_window_bwd: need q_start >= 0, window >= 1 and sinks >= 0");
  if (std::max<int64_t>(S, static_cast<int64_t>(q_start) + L) >= kMaxWindow || B > 65535)
    return set_error(MOTIF_ERR_UNSUPPORTED, "chord_window_bwd: sequence too long or too many batch rows");
  window = std::min(window, kMaxWindow);
  sinks = std::min(sinks, kMaxWindow);
  if (!dparam) return set_error(MOTIF_ERR_INVALID, "chord_window_bwd: NULL pointer");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (B == 0 || S == 0 || L == 0) {  // nothing to differentiate: zero parameter gradients (dq, dk, dv: the caller's)
    ChordBwdArgs z{};
    z.H = H;
    z.cq = 1;
    z.dparam = dparam;
    chord_bwd_reduce_kernel<true><<<dim3(H), dim3(256), 0, s>>>(z, 0, 0);
    return check_launch("chord_bwd_reduce_kernel");
  }
  if (!q || !k || !v || !out || !dout || !lse || !alpha || !beta || !mu || !ssmax || !log_n || !dq || !dk || !dv || !distances)
    return set_error(MOTIF_ERR_INVALID, "chord_window_bwd: NULL pointer");
  if (distances_len < motif_chord_distances_len(L, q_start, window, sinks) || distances_len >= (1 << 28))
    return set_error(MOTIF_ERR_INVALID, "chord_window_bwd: distance table too short (or too long)");
  const int64_t st = q_sb | q_sh | q_st | k_sb | k_sh | k_st | v_sb | v_sh | v_st | o_sb | o_sh | o_st | d_sb | d_sh |
                     d_st | dq_sb | dq_sh | dq_st | dk_sb | dk_sh | dk_st | dv_sb | dv_sh | dv_st;
  const uintptr_t al = reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dout) |
                       reinterpret_cast<uintptr_t>(dq) | reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv);
  if ((st & 7) != 0 || (al & 15) != 0) return set_error(MOTIF_ERR_UNSUPPORTED, "chord_window_bwd: need 16-byte aligned rows");
  const WinBwdPlan pl = plan_bwd_window(B, H, Hkv, L, S, q_start, window, sinks);
  if (pl.nkb + pl.nsb * pl.nsc > 65535)
    return set_error(MOTIF_ERR_UNSUPPORTED, "chord_window_bwd: sequence too long");
  const size_t pad = -reinterpret_cast<uintptr_t>(workspace) & 15;  // (the size asked for holds it)
  if (!workspace || workspace_bytes < pl.bytes + pad)
    return set_error(MOTIF_ERR_INVALID, "chord_window_bwd: workspace too small (need " + std::to_string(pl.bytes + pad) + " bytes)");
  ChordBwdArgs a{};
  a.q = static_cast<const bf16_t *>(q); a.q_sb = q_sb; a.q_sh = q_sh; a.q_st = q_st;
  a.k = static_cast<const bf16_t *>(k); a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v = static_cast<const bf16_t *>(v); a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  a.o = static_cast<const bf16_t *>(out); a.o_sb = o_sb; a.o_sh = o_sh; a.o_st = o_st;
  a.dout = static_cast<const bf16_t *>(dout); a.d_sb = d_sb; a.d_sh = d_sh; a.d_st = d_st;
  a.lse = lse; a.alpha = alpha; a.beta = beta; a.mu = mu; a.ssmax = ssmax;
  a.log_n = log_n; a.ln_sb = ln_sb; a.ln_st = ln_st;
  a.dq = static_cast<bf16_t *>(dq); a.dq_sb = dq_sb; a.dq_sh = dq_sh; a.dq_st = dq_st;
  a.dk = static_cast<bf16_t *>(dk); a.dk_sb = dk_sb; a.dk_sh = dk_sh; a.dk_st = dk_st;
  a.dv = static_cast<bf16_t *>(dv); a.dv_sb = dv_sb; a.dv_sh = dv_sh; a.dv_st = dv_st;
  a.dparam = dparam;
  char *ws = static_cast<char *>(workspace) + pad;
  a.rows = reinterpret_cast<float4 *>(ws);
  a.pparam = reinterpret_cast<float *>(ws + pl.off_param);
  a.pk = reinterpret_cast<float *>(ws + pl.off_pk);
  a.pv = reinterpret_cast<float *>(ws + pl.off_pv);
  a.B = B; a.H = H; a.Hkv = Hkv; a.L = L; a.S = S; a.q_start = q_start;
  a.nqb = pl.nqb; a.nkb = pl.nkb;
  a.nsq = a.nskv = 1; a.kv_direct = pl.kv_direct ? 1 : 0;
  a.dist = reinterpret_cast<const float2 *>(distances);
  a.dmu = distances + 2 * static_cast<size_t>(H) * distances_len;
  a.dist_n = distances_len;
  a.window = window; a.sinks = sinks; a.nsb = pl.nsb; a.nsc = pl.nsc; a.csink = pl.csink; a.prows = pl.prows;
  a.pks = reinterpret_cast<float *>(ws + pl.off_pks);
  a.pvs = reinterpret_cast<float *>(ws + pl.off_pvs);
  a.scale = scale; a.eps = eps;
  bool any = false;  // (a single row's stride is not used)
  for (int64_t x : {q_st, d_st}) any |= L > 1 && (x < kBD || x >= kBufStride);
  for (int64_t x : {k_st, v_st}) any |= S > 1 && (x < kBD || x >= kBufStride);
  int rc = MOTIF_OK;
  const dim3 grid_q(H, pl.nqb, B);
  if (any) (need_mu ? chord_bwd_dq_kernel<true, true, true> : chord_bwd_dq_kernel<true, true, false>)<<<grid_q, dim3(256), 0, s>>>(a);
  else (need_mu ? chord_bwd_dq_kernel<false, true, true> : chord_bwd_dq_kernel<false, true, false>)<<<grid_q, dim3(256), 0, s>>>(a);
  if ((rc = check_launch("chord_bwd_dq_kernel"))) return rc;
  (any ? chord_bwd_dkdv_kernel<true, true> : chord_bwd_dkdv_kernel<false, true>)<<<dim3(H, pl.nkb + pl.nsb * pl.nsc, B), dim3(256), 0, s>>>(a);
  if ((rc = check_launch("chord_bwd_dkdv_kernel"))) return rc;
  const int64_t red = static_cast<int64_t>(B) * Hkv * std::min(pl.prows, S) * (kBD / 4);
  const int nkv = static_cast<int>((red + 255) / 256);
  chord_bwd_reduce_kernel<true><<<dim3(nkv + H), dim3(256), 0, s>>>(a, nkv, 0);
  return check_launch("chord_bwd_reduce_kernel");
}
