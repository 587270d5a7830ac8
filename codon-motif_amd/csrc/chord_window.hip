// Chord attention under a sliding window with visible first tokens (gfx950): the bf16 head-dim-64
// prefill kernel, and the entry points of the windowed and the 4-bit forwards with the choice of
// kernel.  A query at position p sees the keys j <= p with j > p - window or j < sinks; a row that
// sees none gives zeros.
//
// chord_window_kernel: flash attention whose key loop visits the tiles that hold first tokens and
// those that the block's windows reach, and no others.  With a window every query block has the same
// work, so the workgroups are small and even: PARTS (two or four) parts of two waves, a part taking its run of the
// 32-key tiles.  A wave owns 32 score columns (16 queries of two heads that share a kv head, or 32 of
// one head): S^T = K Q^T on v_mfma_f32_32x32x16_bf16, lane l column l % 32, register r of lane half h
// key 8 (r / 4) + 4 h + r % 4; P^T enters O^T += V^T P^T from the same registers, V transposed in that
// key order as it is read from LDS.  K / V tiles are double buffered in LDS, one barrier a tile, the tile after next in
// registers.  The distance bias, the diagonal and the window's edge are one value per distance: 47
// (two heads) or 63 distances meet in a tile, 32 of them new, so each lane evaluates one per tile
// (-inf where the distance is masked) into its wave's LDS row, and the score accumulators start from
// it.  Tiles with first tokens are masked by key instead.  The row sums take P before its rounding to
// bf16, so that the log-sum-exp the backward rebuilds P from is exact to fp32; P and Q K^T's operands are
// the bf16 that the matrix instructions take (P's rounding, 2^-9 in the mean of a weight, is the
// output's own).
// Bound by VALU issue: a score takes some ten instructions and an exponential at a quarter of the rate,
// three times its matrix instructions' time (8192 tokens, window 2048: the vector unit issues in 64% of
// the busy cycles, LDS is read or written in 43%, the matrix unit works in 23%), which puts the floor of
// this form at 2.5 times the products'.  12 heads on 3 kv heads: 4096 tokens, window 1024 32 us (350 TFLOP/s of visible pairs; a
// large library product 1190), 8192 and 2048 97 us (470); as chord_wide_kernel 113 and 349.  16 packed
// sequences of 115 to 528 tokens 16 us in one launch (one by one 301).
#include <algorithm>
#include <string>

#include "capi_internal.h"
#include "chord_internal.h"
#include "common.h"

namespace motif {

namespace {

constexpr int kBD = 64;    // head dim
constexpr int kT = 32;     // keys per tile

__device__ __forceinline__ f32x16 mma32(const bf16x8 &a, const bf16x8 &b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pk2bf(float x0, float x1) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x0, x1}, bf16x2v));
}

// x^beta and its derivatives' factors at distances d = 0, -1, .. of a head, x = |d - mu| + eps:
// dist[h][-d] = {x^beta, x^beta log2 x}, dmu[h][-d] = x^(beta - 1) sign(d - mu).  In 64 bits and rounded
// once: through fp32 log2 and exp2 the power is 3e-7 off, which the scaled logits turn into 1e-5 of a
// weight, and the parameter gradients are small differences of sums over weights.  At distance x = 0 (eps 0, mu
// a whole number) x^beta log2 x is taken as 0, its limit beside a beta
// above 0, and x^0 as 1.
__global__ void __launch_bounds__(256) chord_distance_kernel(const float *beta, const float *mu, float eps, float2 *dist,
                                                             float *dmu, int n) {
  const int h = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const double e = -static_cast<double>(i) - mu[h], x = fabs(e) + eps, l = log2(x);
  const double p = beta[h] == 0.f ? 1. : exp2(beta[h] * l);
  const size_t o = static_cast<size_t>(h) * n + i;
  dist[o] = float2{static_cast<float>(p), x == 0. && beta[h] >= 0.f ? 0.f : static_cast<float>(p * l)};
  dmu[o] = e == 0. ? 0.f : static_cast<float>(e > 0. ? p / x : -p / x);
}

template <int HPW, int PARTS, bool TAB>  // query heads per workgroup (of one kv head), key parts, distances from a.dist
__global__ void __launch_bounds__(128 * PARTS) __attribute__((amdgpu_waves_per_eu(4, 4))) chord_window_kernel(ChordArgs a) {
  constexpr int RH = HPW >= 2 ? 2 : 1;  // heads per wave
  constexpr int RQ = 32 / RH;           // queries per wave
  constexpr int HGW = HPW / RH;         // head groups per part
  constexpr int QW = (2 / HGW) * RQ;    // queries per workgroup
  constexpr int kWin = kT + RQ;         // bias row of a head (>= 31 + RQ entries)
  const int tid = threadIdx.x, lane = tid & 63;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int part = wv >> 1, w = wv & 1;
  const int htid = tid & 127;  // thread inside the part
  const int lc = lane & 31, hh = lane >> 5;
  const int hg = blockIdx.x, sq = blockIdx.z;

  int batch = sq, tok0 = 0, Lq = a.L, Skv = a.S, q_start = a.q_start;
  if (a.cu) {  // a packed sequence
    batch = 0; tok0 = a.cu[sq]; Lq = a.cu[sq + 1] - tok0; Skv = Lq; q_start = 0;
  }
  const int qb0 = blockIdx.y * QW;
  if (qb0 >= Lq) return;

  const int head0 = hg * HPW + (w % HGW) * RH;  // the wave's first head
  const int cq = lc % RQ, head = head0 + lc / RQ;
  const int kvh = (hg * HPW) / (a.H / a.Hkv);
  const int q0 = qb0 + (w / HGW) * RQ, my_q = q0 + cq, q_last = q0 + RQ - 1;
  const bool q_valid = my_q < Lq;
  const int kv_end = min(Skv, q_start + min(Lq, qb0 + QW));
  const KeyWalk<kT> walk(q_start + qb0, kv_end, a.window, a.sinks);
  const int nsteps = (walk.count + PARTS - 1) / PARTS;
  const int t_first = part * nsteps, t_count = max(0, min(nsteps, walk.count - t_first));
  const int wave_kv_end = min(Skv, q_start + min(Lq, q0 + RQ));

  const bf16_t *kp = static_cast<const bf16_t *>(a.k) + batch * a.k_sb + kvh * a.k_sh + int64_t(tok0) * a.k_st;
  const bf16_t *vp = static_cast<const bf16_t *>(a.v) + batch * a.v_sb + kvh * a.v_sh + int64_t(tok0) * a.v_st;

  // logit = a_row acc with acc = rho q.k + kappa GGD, rho = sign(ssmax log_n scale) (0 when scale is 0), kappa =
  // sign(ssmax log_n) / |scale| (sign(ssmax log_n) when scale is 0), a_row = |ssmax log_n scale| (|ssmax log_n|);
  // p = exp2(A (acc - m)), A = log2e a_row > 0 so that a masked key's -inf stays one.  (The bias rows,
  // which the wave's queries share, hold sign(ssmax) only: see `neg`.)
  const float ssm = a.ssmax[head], sg = ssm < 0.f ? -1.f : 1.f;
  const float lnv = a.log_n ? a.log_n[batch * a.ln_sb + int64_t(tok0 + min(my_q, Lq - 1)) * a.ln_st]
                            : a.log_tab[q_start + min(my_q, Lq - 1)];
  const bool neg = q_valid && lnv < 0.f;
  const uint64_t any_neg = __ballot(neg);
  const float sgr = neg ? -sg : sg, rho = a.scale > 0.f ? sgr : a.scale < 0.f ? -sgr : 0.f;
  const float A = q_valid ? fmaxf(fabsf(ssm) * (a.scale != 0.f ? fabsf(a.scale) : 1.f) * fabsf(lnv) * kLog2e, 1e-30f) : 1.f;

  bf16x8 qreg[4];  // rho Q^T, the B operand: features 16 ds + 8 hh .. of this lane's row
  {
    const bf16_t *qrow = static_cast<const bf16_t *>(a.q) + batch * a.q_sb + head * a.q_sh + int64_t(tok0 + min(my_q, Lq - 1)) * a.q_st;
#pragma unroll
    for (int ds = 0; ds < 4; ++ds) {
      uint4 u = *reinterpret_cast<const uint4 *>(qrow + 16 * ds + 8 * hh);
      if (rho < 0.f) { u.x ^= 0x80008000u; u.y ^= 0x80008000u; u.z ^= 0x80008000u; u.w ^= 0x80008000u; }
      if (rho == 0.f || !q_valid) u = uint4{0u, 0u, 0u, 0u};
      qreg[ds] = __builtin_bit_cast(bf16x8, u);
    }
  }

  constexpr int kTile = kT * kBD;
  constexpr int kStage = PARTS * 2 * 2 * kTile, kMerge = (PARTS - 1) * 2 * 32 * 64 * 2;  // in bf16 elements
  __shared__ __attribute__((aligned(16))) bf16_t sKV[kStage > kMerge ? kStage : kMerge];
  __shared__ float sB[2 * PARTS][RH * kWin > 128 ? RH * kWin : 128];
  auto sK = [&](int buf) { return sKV + (part * 2 + buf) * 2 * kTile; };
  auto sV = [&](int buf) { return sKV + (part * 2 + buf) * 2 * kTile + kTile; };

  // Bias rows: entry j of a head is distance key - q_abs = n0 - q_start - q0 - (RQ - 1) + j.  Lane l
  // (head l / 32 of two) holds entry RQ - 1 + l % 32 of its tile in `bnew`; the first RQ - 1 entries are
  // the last ones of the tile before (`bold`, 32 distances less), evaluated anew where that tile is not
  // the one before or was masked by key.
  const int bh = RH == 2 ? lane >> 5 : 0;
  const float gal = a.alpha[head0 + bh], gbe = a.beta[head0 + bh], gmu = a.mu[head0 + bh];
  const float gka = (a.ssmax[head0 + bh] < 0.f ? -1.f : 1.f) / (a.scale != 0.f ? fabsf(a.scale) : 1.f);
  const buf_t dbuf = make_buf(a.dist, TAB ? static_cast<uint32_t>(a.H) * static_cast<uint32_t>(a.dist_n) * 8u : 0u);
  const uint32_t dhead = static_cast<uint32_t>(head0 + bh) * static_cast<uint32_t>(a.dist_n);
  auto eval = [&](int n0, int d) {  // for the tile from key n0 on
    const bool ok = d <= 0 && (d > -a.window || n0 < a.sinks);
    float bias;
    if constexpr (TAB) {  // (a masked distance may lie past the table: entry 0 is read instead)
      bias = -gal * __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                        dbuf, 8u * (dhead + static_cast<uint32_t>(ok ? -d : 0)), 0, 0));
    } else {
      bias = ggd_bias(static_cast<float>(d), gal, gbe, gmu, a.eps);
    }
    return ok ? gka * bias : -INFINITY;
  };
  const int d0 = lc - q_start - q0;
  float *bw = &sB[wv][bh * kWin];
  auto store_bias = [&](float bnew, float bold) {
    bw[RQ - 1 + lc] = bnew;
    if (lc >= kT + 1 - RQ) bw[RQ - 1 + lc - kT] = bold;
  };
  // this lane's entries for keys 8 q4 + 4 hh + (0..3): j = 8 q4 + p + 4 hh - cq + RQ - 1
  const float *bwr = &sB[wv][(lc / RQ) * kWin] + 4 * hh - cq + RQ - 1;

  // Staging by the part's 128 threads: row stage_row(htid), pieces htid % 4 and + 4
  uint4 kst[2], vst[2];
  const int srow = stage_row(htid);
  const uint32_t koff = static_cast<uint32_t>((srow * a.k_st + (htid & 3) * 8) * 2);
  const uint32_t voff = static_cast<uint32_t>((srow * a.v_st + (htid & 3) * 8) * 2);
  const int sto = srow * kBD + 8 * ((htid & 3) ^ piece_swap(srow));
  auto load_tile = [&](int x) {  // (rows past the tile's own read zeros)
    const int n0 = walk.start(x), rows = walk.rows(x);
    const buf_t kr = make_buf(kp + int64_t(n0) * a.k_st, rows > 0 ? static_cast<uint32_t>(((rows - 1) * a.k_st + kBD) * 2) : 0u);
    const buf_t vr = make_buf(vp + int64_t(n0) * a.v_st, rows > 0 ? static_cast<uint32_t>(((rows - 1) * a.v_st + kBD) * 2) : 0u);
    kst[0] = buf_ld16(kr, koff);
    kst[1] = buf_ld16(kr, koff + 64u);
    vst[0] = buf_ld16(vr, voff);
    vst[1] = buf_ld16(vr, voff + 64u);
  };
  auto store_tile = [&](int buf) {
    bf16_t *kd = sK(buf), *vd = sV(buf);
    *reinterpret_cast<uint4 *>(kd + sto) = kst[0];
    *reinterpret_cast<uint4 *>(kd + (sto ^ 32)) = kst[1];
    *reinterpret_cast<uint4 *>(vd + sto) = vst[0];
    *reinterpret_cast<uint4 *>(vd + (sto ^ 32)) = vst[1];
  };
  // this lane's reads: K row lc, pieces 2 ds + hh; V^T, keys 4 hh + lane % 16 / 4 (+ 8, + 16), features
  // 16 (lane / 16 % 2) + 4 (lane % 4) (+ 32) on
  const int ko = lc * kBD + 8 * (hh ^ piece_swap(lc));
  const int vrow = 4 * hh + ((lane & 15) >> 2), vpiece = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const int vo = vrow * kBD + 8 * (vpiece ^ piece_swap(vrow)) + 4 * (lane & 1);

  float m_run = -INFINITY, l_run = 0.f;  // per column (m: acc units; l: this lane's share)
  f32x16 oacc[2] = {f32x16{}, f32x16{}};  // O^T rows d = 32 dt + 8 (r / 4) + 4 hh + r % 4, column lc

  load_tile(t_first);
  store_tile(0);
  float bnew = eval(walk.start(t_first), walk.start(t_first) + d0);
  store_bias(bnew, eval(walk.start(t_first), walk.start(t_first) + d0 - kT));
  load_tile(t_first + 1);
  __syncthreads();

  for (int i = 0; i < nsteps; ++i) {
    const int n0 = walk.start(t_first + i), nn = walk.start(t_first + i + 1), buf = i & 1;
    // the next tile's new distances ahead of this tile's work
    float bold = bnew;
    bnew = eval(nn, nn + d0);
    if (nn != n0 + kT || n0 < a.sinks) bold = eval(nn, nn + d0 - kT);
    if (i < t_count && n0 < wave_kv_end && (n0 + kT - 1 > q_start + q0 - a.window || n0 < a.sinks)) {
      f32x16 acc;
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
#pragma unroll
        for (int p4 = 0; p4 < 4; ++p4) acc[4 * q4 + p4] = bwr[8 * q4 + p4];
      if (any_neg) {  // (a factor log_n below 0, no logarithm of a count: the bias's sign turned, masked keys kept so)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = neg && acc[r] != -INFINITY ? -acc[r] : acc[r];
      }
#pragma unroll
      for (int ds = 0; ds < 4; ++ds) {
        const bf16x8 kop = *reinterpret_cast<const bf16x8 *>(sK(buf) + (ko ^ (16 * ds)));
        acc = mma32(kop, qreg[ds], acc);
      }
      // by key: tiles of first tokens at the window's edge, and the end of the keys
      if ((n0 < a.sinks && n0 + kT > a.sinks && n0 <= q_start + q_last - a.window) || n0 + kT > Skv) {
        const uint32_t seen =
            seen_keys(walk.rows(t_first + i) - 1, q_start + my_q - a.window - n0, a.sinks - n0) >> (4 * hh);
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[r] = seen & (1u << (8 * (r >> 2) + (r & 3))) ? acc[r] : -INFINITY;
      }
      float mx = acc[0];
#pragma unroll
      for (int r = 1; r < 16; ++r) mx = fmaxf(mx, acc[r]);
      {
        const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(s32[0]), __uint_as_float(s32[1]));
      }
      // the running max moves only when a tile passes it by more than 8 (log2 units), so p <= 2^8
      const bool grow = A * (mx - m_run) > 8.f || m_run == -INFINITY;
      const float m_new = grow ? mx : m_run;
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      if (__builtin_amdgcn_read_exec() & __ballot(grow)) {
        const float resc = m_run == -INFINITY ? 0.f : fast_exp2(A * (m_run - m_use));
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          oacc[0][r] *= resc;
          oacc[1][r] *= resc;
        }
        l_run *= resc;
      }
      m_run = m_new;
      const float nb = -A * m_use;
#pragma unroll
      for (int hk = 0; hk < 2; ++hk) {
        uint32_t pw[4];
        float ps[2] = {0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float p0 = fast_exp2(fmaf(acc[8 * hk + 2 * e], A, nb)), p1 = fast_exp2(fmaf(acc[8 * hk + 2 * e + 1], A, nb));
          ps[0] += p0;
          ps[1] += p1;
          pw[e] = pk2bf(p0, p1);
        }
        l_run += ps[0] + ps[1];
        const bf16x8 pb = __builtin_bit_cast(bf16x8, uint4{pw[0], pw[1], pw[2], pw[3]});
#pragma unroll
        for (int dt = 0; dt < 2; ++dt) {
          const bf16_t *vp = sV(buf) + (vo ^ (32 * dt)) + 16 * hk * kBD;
          const uint2 v0 = ld_transposed(vp), v1 = ld_transposed(vp + 8 * kBD);
          oacc[dt] = mma32(__builtin_bit_cast(bf16x8, uint4{v0.x, v0.y, v1.x, v1.y}), pb, oacc[dt]);
        }
      }
    }
    // the next tile's bias rows (this wave's own; its reads above come first) and rows into LDS (the
    // other buffer, last read before the previous barrier), the tile after into flight
    store_bias(bnew, bold);
    store_tile(buf ^ 1);
    load_tile(t_first + i + 2);
    __syncthreads();
  }

  {
    const auto s32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_run), __float_as_uint(l_run), false, false);
    l_run = __uint_as_float(s32[0]) + __uint_as_float(s32[1]);
  }

  // Merge: parts 1 .. leave O^T over the tiles and (l, m) in their bias rows; part 0 writes the rows.
  float *mo = reinterpret_cast<float *>(sKV) + lane;
  if (part > 0) {
    float *dst = mo + ((part - 1) * 2 + w) * 32 * 64;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      dst[r * 64] = oacc[0][r];
      dst[(16 + r) * 64] = oacc[1][r];
    }
    sB[wv][lane] = l_run;
    sB[wv][64 + lane] = m_run;
  }
  __syncthreads();
  if (part == 0 && q_valid) {
    float m = m_run;
#pragma unroll
    for (int p = 1; p < PARTS; ++p) m = fmaxf(m, sB[2 * p + w][64 + lane]);
    float f[PARTS];
    f[0] = m_run == -INFINITY ? 0.f : fast_exp2(A * (m_run - m));
    float l = l_run * f[0];
#pragma unroll
    for (int p = 1; p < PARTS; ++p) {
      const float mp = sB[2 * p + w][64 + lane];
      f[p] = mp == -INFINITY ? 0.f : fast_exp2(A * (mp - m));
      l = fmaf(sB[2 * p + w][lane], f[p], l);
    }
    const float inv = 1.f / fmaxf(l, 1e-20f);
    bf16_t *op = static_cast<bf16_t *>(a.out) + batch * a.o_sb + head * a.o_sh + int64_t(tok0 + my_q) * a.o_st;
#pragma unroll
    for (int dt = 0; dt < 2; ++dt)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        float o[4];
#pragma unroll
        for (int p4 = 0; p4 < 4; ++p4) {
          const int r = 4 * q4 + p4;
          float x = oacc[dt][r] * f[0];
#pragma unroll
          for (int p = 1; p < PARTS; ++p) x = fmaf(mo[(((p - 1) * 2 + w) * 32 + 16 * dt + r) * 64], f[p], x);
          o[p4] = x * inv;
        }
        *reinterpret_cast<uint2 *>(op + 32 * dt + 8 * q4 + 4 * hh) = uint2{pk2bf(o[0], o[1]), pk2bf(o[2], o[3])};
      }
    if (a.lse && hh == 0)
      a.lse[(static_cast<size_t>(batch) * a.H + head) * a.L + tok0 + my_q] = A * (m == -INFINITY ? 0.f : m) + fast_log2(l);
  }
}

// Key parts of a workgroup: four where the blocks are at most three for every two CUs and a block's tiles at
// least 12, so that the parts shorten its chain by more than they cost to join.  Measured, us, 12 heads,
// two parts / four: 3 kv heads, 512 tokens (96 blocks), a window of 512 11.7 / 10.1; 1024 (192) 256 9.3 / 9.2,
// 1024 19.1 / 15.2; 1500 (282) 600 16.2 / 14.9; 2048 (384) 256 11.6 / 12.6, 1024 24.1 / 21.5; 3000 (564) 1024
// 27.9 / 27.7; 4096 (768) 1024 32.1 / 34.9; 300 (57) 128 7.2 / 7.7; 12 kv heads, 1024 (192) 512 12.9 / 11.1, 2048
// (384) 512 17.2 / 16.1.  One part: 8192 tokens, 1024 63.5 (two: 56.7), 2 x 2048 25.3 (20.8).
template <int HPW>
int launch_window_h(const ChordArgs &a, int nseq, int max_len, hipStream_t s) {
  constexpr int kQ = HPW == 4 ? 16 : HPW == 2 ? 32 : 64;
  const dim3 grid(a.H / HPW, (max_len + kQ - 1) / kQ, nseq);
  const int64_t blocks = int64_t(grid.x) * grid.y * grid.z;
  const int keys = std::min(a.cu ? max_len : std::min(a.S, a.q_start + a.L), a.window + kQ + std::min(a.sinks, kMaxWindow / 2));
  if (2 * blocks <= 3 * chord_cu_count() && keys >= 12 * kT)
    (a.dist ? chord_window_kernel<HPW, 4, true> : chord_window_kernel<HPW, 4, false>)<<<grid, dim3(512), 0, s>>>(a);
  else
    (a.dist ? chord_window_kernel<HPW, 2, true> : chord_window_kernel<HPW, 2, false>)<<<grid, dim3(256), 0, s>>>(a);
  return check_launch("chord_window_kernel");
}

int launch_window(const ChordArgs &a, int nseq, int max_len, hipStream_t s) {
  const int group = a.H / a.Hkv;
  if (group % 4 == 0) return launch_window_h<4>(a, nseq, max_len, s);
  if (group % 2 == 0) return launch_window_h<2>(a, nseq, max_len, s);
  return launch_window_h<1>(a, nseq, max_len, s);
}

// Distances that the queries of a call meet: those of a window, or with first tokens all of them.
int distance_count(int L, int q_start, int window, int sinks) { return sinks > 0 ? q_start + L : std::min(window, q_start + L); }

// Everything the three forward entries share: sizes, types, pointers, alignment; fills a.
struct Call {
  const char *name;
  const void *q; int64_t q_sb, q_sh, q_st;
  const float *alpha, *beta, *mu, *ssmax, *log_n; int64_t ln_sb, ln_st;
  const float *log_table; int log_table_len;
  void *out; int64_t o_sb, o_sh, o_st;
  float *lse;
  int *length_dev;
  int B, H, Hkv, L, S, D, q_start;
  float scale, eps;
  int window, sinks, dtype;
};

int fill(const Call &c, ChordArgs &a) {
  const std::string name(c.name);
  if (c.B < 0 || c.H <= 0 || c.Hkv <= 0 || c.L < 0 || c.S < 0 || c.q_start < 0 || c.H % c.Hkv)
    return set_error(MOTIF_ERR_INVALID, name + ": bad size or negative q_start");
  if (!kv4_head_dim(c.D)) return set_error(MOTIF_ERR_UNSUPPORTED, name + ": head_dim must be 16, 32, 64 or 128");
  if (c.dtype != MOTIF_BF16 && c.dtype != MOTIF_F32 && c.dtype != MOTIF_F16)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": dtype must be bf16, fp16 or fp32");
  if (c.window < 1 || c.sinks < 0) return set_error(MOTIF_ERR_INVALID, name + ": need window >= 1 and sinks >= 0");
  if (std::max<int64_t>(c.S, static_cast<int64_t>(c.q_start) + c.L) >= kMaxWindow || c.B > 65535 || c.L > 65535 * 32)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": sequence too long or too many batch rows");
  a = ChordArgs{};
  a.q = c.q; a.q_sb = c.q_sb; a.q_sh = c.q_sh; a.q_st = c.q_st;
  a.alpha = c.alpha; a.beta = c.beta; a.mu = c.mu; a.ssmax = c.ssmax;
  a.log_n = c.log_n; a.ln_sb = c.ln_sb; a.ln_st = c.ln_st; a.log_tab = c.log_table;
  a.out = c.out; a.o_sb = c.o_sb; a.o_sh = c.o_sh; a.o_st = c.o_st;
  a.lse = c.lse;
  a.B = c.B; a.H = c.H; a.Hkv = c.Hkv; a.L = c.L; a.S = c.S; a.q_start = c.q_start;
  a.scale = c.scale; a.eps = c.eps;
  a.splits = a.nqc = 1;
  a.len_dev = c.length_dev;
  a.window = std::min(c.window, kMaxWindow);
  a.sinks = std::min(c.sinks, kMaxWindow);
  if (c.B == 0 || c.L == 0) return MOTIF_OK;
  if (c.S == 0) return set_error(MOTIF_ERR_INVALID, name + ": empty key cache");
  if (!c.q || !c.alpha || !c.beta || !c.mu || !c.ssmax || !c.out)
    return set_error(MOTIF_ERR_INVALID, name + ": NULL pointer");
  if (c.length_dev && c.S < c.L) return set_error(MOTIF_ERR_INVALID, name + ": capacity below the query count");
  if (!c.log_n && (!c.log_table || c.log_table_len < std::max(c.S, c.q_start + c.L)))
    return set_error(MOTIF_ERR_INVALID, name + ": log_n is NULL and the log table is too short");
  const int64_t vec = c.dtype == MOTIF_F32 ? 4 : 8;
  if (((c.q_st | c.o_st | c.q_sh | c.o_sh | c.q_sb | c.o_sb) % vec) != 0 ||
      ((reinterpret_cast<uintptr_t>(c.q) | reinterpret_cast<uintptr_t>(c.out)) & 15) != 0)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": q/out need 16-byte aligned rows");
  if (c.L == 1) a.q_st = c.D;  // (the stride of a single row is not used)
  return MOTIF_OK;
}

int fill_rows(const Call &c, ChordArgs &a, const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st, const void *v,
              int64_t v_sb, int64_t v_sh, int64_t v_st) {
  const std::string name(c.name);
  a.k = k; a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
  a.v = v; a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
  if (!k || !v) return set_error(MOTIF_ERR_INVALID, name + ": NULL pointer");
  const int64_t vec = c.dtype == MOTIF_F32 ? 4 : 8;
  if (((k_st | v_st | k_sh | v_sh | k_sb | v_sb) % vec) != 0 ||
      ((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) != 0)
    return set_error(MOTIF_ERR_UNSUPPORTED, name + ": k/v need 16-byte aligned rows");
  if (c.S == 1) a.k_st = a.v_st = c.D;
  // 32-bit offsets inside a tile of rows
  for (int64_t st : {a.q_st, a.k_st, a.v_st})
    if (st < 0 || st >= (int64_t(1) << 24)) return set_error(MOTIF_ERR_UNSUPPORTED, name + ": row stride out of range");
  return MOTIF_OK;
}

}  // namespace

}  // namespace motif

using namespace motif;

extern "C" int motif_chord_window_fwd(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k, int64_t k_sb, int64_t k_sh, int64_t k_st,
    const void *v, int64_t v_sb, int64_t v_sh, int64_t v_st,
    const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st, const float *log_table, int log_table_len,
    void *out, int64_t o_sb, int64_t o_sh, int64_t o_st, float *lse,
    int *length_dev, int B, int H, int Hkv, int L, int S, int D, int q_start, float scale, float eps,
    int window, int sinks, const float *distances, int distances_len, const int32_t *cu_seqlens, int nseq, int max_seqlen,
    void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  const Call c{"chord_window_fwd", q, q_sb, q_sh, q_st, alpha, beta, mu, ssmax, log_n, ln_sb, ln_st, log_table,
               log_table_len, out, o_sb, o_sh, o_st, lse, length_dev, B, H, Hkv, L, S, D, q_start, scale, eps,
               window, sinks, dtype};
  ChordArgs a;
  int rc = fill(c, a);
  if (rc || B == 0 || L == 0) return rc;
  if ((rc = fill_rows(c, a, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st))) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (cu_seqlens) {
    if (B != 1 || S != L || q_start || nseq < 0 || nseq > 65535 || max_seqlen < 0 || max_seqlen > L)
      return set_error(MOTIF_ERR_INVALID, "chord_window_fwd: packed sequences need B == 1, S == L, q_start 0 and sizes within L");
    if (dtype != MOTIF_BF16 || D != kBD || length_dev || lse || distances || !log_n || max_seqlen > 65535 * 16)
      return set_error(MOTIF_ERR_UNSUPPORTED, "chord_window_fwd: packed sequences need bf16, head_dim 64 and host positions");
    a.cu = cu_seqlens;
    return nseq && max_seqlen ? launch_window(a, nseq, max_seqlen, st) : MOTIF_OK;
  }
  if (chord_window_decode_serves(H, Hkv, L, D, dtype) && !lse) {
    a.splits = chord_window_splits(B, Hkv, L, S, window, sinks);
    if (a.splits > 1) {
      const size_t need = motif_chord_window_workspace_bytes(B, H, Hkv, L, S, D, window, sinks, dtype);
      if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3))
        return set_error(MOTIF_ERR_INVALID, "chord_window_fwd: workspace too small (need " + std::to_string(need) + " bytes) or not aligned");
      a.part = static_cast<float *>(workspace);
    }
    return launch_chord_window_decode(a, st);
  }
  if (distances && distances_len < distance_count(L, q_start, window, sinks))
    return set_error(MOTIF_ERR_INVALID, "chord_window_fwd: distance table too short");
  a.dist = reinterpret_cast<const float2 *>(distances);
  a.dist_n = distances_len;
  if (static_cast<int64_t>(H) * distances_len >= (int64_t(1) << 29)) a.dist = nullptr;  // (past 32-bit offsets: evaluated)
  if (dtype == MOTIF_BF16 && D == kBD && !length_dev && L <= 65535 * 16) return launch_window(a, B, L, st);
  return launch_chord_wide_window(a, dtype, D, st);
}

extern "C" int motif_chord_distances_len(int L, int q_start, int window, int sinks) {
  if (L <= 0 || q_start < 0 || window < 1 || sinks < 0 || static_cast<int64_t>(q_start) + L >= kMaxWindow) return 0;
  return distance_count(L, q_start, window, sinks);
}

extern "C" int motif_chord_distances(const float *beta, const float *mu, int H, int n, float eps, float *out, void *stream) {
  if (H < 0 || n < 0 || H > 65535) return set_error(MOTIF_ERR_INVALID, "chord_distances: bad size");
  if (H == 0 || n == 0) return MOTIF_OK;
  if (!beta || !mu || !out) return set_error(MOTIF_ERR_INVALID, "chord_distances: NULL pointer");
  if (reinterpret_cast<uintptr_t>(out) & 7) return set_error(MOTIF_ERR_INVALID, "chord_distances: out must be 8-byte aligned");
  chord_distance_kernel<<<dim3((n + 255) / 256, H), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
      beta, mu, eps, reinterpret_cast<float2 *>(out), out + 2 * static_cast<size_t>(H) * n, n);
  return check_launch("chord_distance_kernel");
}

extern "C" size_t motif_chord_window_workspace_bytes(int B, int H, int Hkv, int L, int S, int D, int window, int sinks,
                                                     int dtype) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || L <= 0 || S <= 0 || window < 1 || sinks < 0 ||
      !chord_window_decode_serves(H, Hkv, L, D, dtype))
    return 0;
  const int sp = chord_window_splits(B, Hkv, L, S, window, sinks);
  return sp > 1 ? static_cast<size_t>(B) * H * L * sp * (D + 2) * sizeof(float) : 0;
}

extern "C" size_t motif_chord_kv4_workspace_bytes(int B, int H, int Hkv, int L, int S, int D, int window, int sinks,
                                                  int dtype) {
  if (B <= 0 || H <= 0 || Hkv <= 0 || H % Hkv || L <= 0 || S <= 0 || window < 1 || sinks < 0 ||
      !chord_kv4_serves(H, Hkv, L, D, dtype))
    return 0;
  const int sp = chord_kv4_splits(B, Hkv, L, S, window, sinks);
  return sp > 1 ? static_cast<size_t>(B) * H * L * sp * (D + 2) * sizeof(float) : 0;
}

extern "C" int motif_chord_kv4_fwd(
    const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st,
    const void *k_codes, int64_t kc_sb, int64_t kc_sh, const void *k_params, int64_t kp_sb, int64_t kp_sh,
    const void *v_codes, int64_t vc_sb, int64_t vc_sh, const void *v_params, int64_t vp_sb, int64_t vp_sh,
    const float *alpha, const float *beta, const float *mu, const float *ssmax,
    const float *log_n, int64_t ln_sb, int64_t ln_st, const float *log_table, int log_table_len,
    void *out, int64_t o_sb, int64_t o_sh, int64_t o_st,
    int *length_dev, int B, int H, int Hkv, int L, int S, int D, int q_start, float scale, float eps,
    int window, int sinks, void *workspace, size_t workspace_bytes, int dtype, void *stream) {
  const Call c{"chord_kv4_fwd", q, q_sb, q_sh, q_st, alpha, beta, mu, ssmax, log_n, ln_sb, ln_st, log_table,
               log_table_len, out, o_sb, o_sh, o_st, nullptr, length_dev, B, H, Hkv, L, S, D, q_start, scale, eps,
               window, sinks, dtype};
  ChordArgs a;
  int rc = fill(c, a);
  if (rc || B == 0 || L == 0) return rc;
  const KV4Args kv = kv4_args(k_codes, kc_sb, kc_sh, k_params, kp_sb, kp_sh, v_codes, vc_sb, vc_sh, v_params, vp_sb, vp_sh);
  if (const char *bad = kv4_check(kv, D)) return set_error(MOTIF_ERR_INVALID, std::string("chord_kv4_fwd: ") + bad);
  if (a.q_st < 0 || a.q_st >= (int64_t(1) << 24)) return set_error(MOTIF_ERR_UNSUPPORTED, "chord_kv4_fwd: row stride out of range");
  hipStream_t st = static_cast<hipStream_t>(stream);
  // more rows, fp32 and other head dims: the fp32-accumulating flash kernel, which expands the codes
  if (!chord_kv4_serves(H, Hkv, L, D, dtype)) return launch_chord_wide_kv4(a, kv, dtype, D, st);
  a.splits = chord_kv4_splits(B, Hkv, L, S, window, sinks);
  if (a.splits > 1) {
    const size_t need = motif_chord_kv4_workspace_bytes(B, H, Hkv, L, S, D, window, sinks, dtype);
    if (!workspace || workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 3))
      return set_error(MOTIF_ERR_INVALID, "chord_kv4_fwd: workspace too small (need " + std::to_string(need) + " bytes) or not aligned");
    a.part = static_cast<float *>(workspace);
  }
  return launch_chord_kv4(a, kv, dtype, st);
}
