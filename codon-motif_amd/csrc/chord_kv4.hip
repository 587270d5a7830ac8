// Chord attention of a few query rows over a 4-bit cache (kv4.hip has the format), bf16 and fp16,
// head dim 64: split over the keys, the codes multiplied as they are held.
//
// With codes n and a (scale, base) pair per key and 32-feature group,
//   q . k = sum_g scale_g (q . n)_g + base_g (sum of q)_g,   O = sum_j p_j scale_jg n_j + p_j base_jg,
// so no key or value is ever expanded: codes enter v_mfma_f32_16x16x32 as the 16-bit numbers 128 + n
// (bf16; a mask and an or per pair, exact, and 128 times the other operand's sum is taken out in
// fp32) or n (fp16), the key's scale is applied to the score product, the value's to the weight.
//
// A workgroup is four waves over one kv head's rows and a range of the keys, or up to twelve over all of
// them (chord_kv4_splits); a wave step is 64 keys (5 KB), staged by buffer-to-LDS loads one step ahead, so a wave's loads fly while it computes.
// Key 16 g + 4 t + i of a step is row 4 g + i of score tile t, which leaves lane group g its own 16
// keys; ds_read_b64_tr_b4 gives a lane one feature of those 16 keys, the operand of O^T += V^T P^T.
// The MFMA has 16 columns, the rows of a step are few: U = 16 / rows copies of the query rows sit in
// the columns, copy u with zeros but for the tiles t of its own, so one accumulator holds the scores
// of U tiles and every lane's softmax work is on scores of its own (4 a step at U = 4, where columns
// of padding would make it 16).  The weights enter the second product masked the same way, and
// the copies' outputs are added in the wave, the waves' through LDS.  The weights are rounded to bf16 with the value's scale
// (fp16: to two bf16, 17 bits, as fp16's range would not hold the product).
// What the offset of 128 leaves when it is taken out again is fp32's rounding of 136 times the weighted scales,
// some 2^-24 136 of them: up to 1e-5 where codes span 0 .. 3.5, against 0.1 for half a code.
// Bound by VALU issue (codes to operands 112 of some 280 instructions a step, the bias's logarithm and
// exponential and the softmax's at a quarter of the rate): 64 sequences of 4097 keys, 12 heads on 3, 63 MB
// of cache in 18.8 us (3.3 TB/s); the bf16 rows of the same cache are 201 MB, 40 us.  One sequence of 300
// keys 6.5 us; 32 x 2 fp16 rows, window 4000 of 8190 keys, 19.7 us with the merge.  Without the matrix instructions (chord_wide_kernel) 592 us.
#include <algorithm>
#include <string>

#include "capi_internal.h"
#include "chord_internal.h"
#include "common.h"

namespace motif {

namespace {

constexpr int kD = 64, kStep = 64;  // head dim, keys per wave step
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
typedef float f32x2v __attribute__((ext_vector_type(2)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t pk2bf(float x0, float x1) {
  return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2v){x0, x1}, bf16x2v));
}
// The mask of a pair of codes, in a register: as a constant it and the bits or'ed in are two literals, which
// take two instructions where v_and_or_b32 takes one (64 of 340 vector instructions of a step).
__device__ __forceinline__ uint32_t pair_mask() {
  uint32_t m = 0x000f000fu;
  asm("" : "+v"(m));
  return m;
}
// 8 codes to an MFMA operand: pairs (n0, n4), (n1, n5), (n2, n6), (n3, n7), bf16 128 + n (m: pair_mask())
__device__ __forceinline__ uint4 codes_bf16(uint32_t w, uint32_t m) {
  constexpr uint32_t b = 0x43004300u;
  return uint4{(w & m) | b, ((w >> 4) & m) | b, ((w >> 8) & m) | b, ((w >> 12) & m) | b};
}
// the same as fp16 n (1024 + n less 1024)
__device__ __forceinline__ uint4 codes_f16(uint32_t w, uint32_t m) {
  auto one = [m](uint32_t x) {
    const f16x2 v = __builtin_bit_cast(f16x2, (x & m) | 0x64006400u) - f16x2{1024, 1024};
    return __builtin_bit_cast(uint32_t, v);
  };
  return uint4{one(w), one(w >> 4), one(w >> 8), one(w >> 12)};
}
__device__ __forceinline__ float max_g(float x) {  // over the four lane groups of 16
  auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
  s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float sum_g(float x) {
  x += __shfl_xor(x, 32, 64);
  return x + __shfl_xor(x, 16, 64);
}

// over the U columns c % (16 / U) of 16 lanes
template <int N> __device__ __forceinline__ float row_ror(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x120 + N, 0xf, 0xf, false));
}
template <int U> __device__ __forceinline__ float sum_copies(float x) {
  x += row_ror<8>(x);
  return U == 4 ? x + row_ror<4>(x) : x;
}
template <int U> __device__ __forceinline__ float max_copies(float x) {
  x = fmaxf(x, row_ror<8>(x));
  return U == 4 ? fmaxf(x, row_ror<4>(x)) : x;
}

template <typename T, int U, int NW>  // NW: waves of a workgroup
__global__ void __launch_bounds__(64 * NW) chord_kv4_kernel(ChordArgs a, KV4Args kv) {
  constexpr int RC = 16 / U, TPL = 4 / U, NK = 4 * TPL;  // rows, tiles and keys of a lane
  constexpr bool kBf = sizeof(T) == 2 && __is_same(T, bf16_t);
  constexpr int kHalves = kBf ? 1 : 2;  // fp16 weights as two bf16 (17 bits; fp16's range would not hold p scale)
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g = lane >> 4;
  const int u = c16 / RC, r = c16 % RC;
  const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
  const int group = a.H / a.Hkv, rows = a.L * group;
  const bool row_ok = r < rows;
  const int head = kvh * group + (row_ok ? r % group : 0), qi = row_ok ? r / group : 0;
  const DecodeWindow cur = decode_window(a);
  const int q_start = cur.q_start, k_end = min(cur.S, q_start + a.L);
  const int q_abs = row_ok ? q_start + qi : -1;

  // q in the codes' pair order, and its sums over a scale's features
  uint4 q[2];
  float qs[2];
  {
    const T *qr = static_cast<const T *>(a.q) + b * a.q_sb + head * a.q_sh + int64_t(qi) * a.q_st + 8 * g;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint4 x = *reinterpret_cast<const uint4 *>(qr + 32 * p);
      if (!row_ok) x = uint4{0u, 0u, 0u, 0u};
      q[p] = uint4{(x.x & 0xffffu) | (x.z << 16), (x.x >> 16) | (x.z & 0xffff0000u),
                   (x.y & 0xffffu) | (x.w << 16), (x.y >> 16) | (x.w & 0xffff0000u)};
      const uint32_t ws[4] = {x.x, x.y, x.z, x.w};
      float s = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint16_t h = static_cast<uint16_t>(ws[e >> 1] >> (16 * (e & 1)));
        if constexpr (kBf) s += bf16_to_f32(h);
        else s += static_cast<float>(__builtin_bit_cast(f16_t, h));
      }
      qs[p] = sum_g(s);
    }
  }
  uint4 qm[U][2];  // the copies' operands: q in the columns of copy u, zeros elsewhere
#pragma unroll
  for (int v = 0; v < U; ++v)
#pragma unroll
    for (int p = 0; p < 2; ++p) qm[v][p] = u == v ? q[p] : uint4{0u, 0u, 0u, 0u};
  uint32_t pmask[2];  // this lane's weights in the second product's tile pairs
#pragma unroll
  for (int t2 = 0; t2 < 2; ++t2)
    pmask[t2] = U == 1 ? ~0u : U == 2 ? (u == t2 ? ~0u : 0u) : (u >> 1) == t2 ? ((u & 1) ? 0xffff0000u : 0xffffu) : 0u;

  const float mul = row_ok ? a.ssmax[head] * log_n_at(a, b, qi, q_start) : 0.f;
  const float c_qk = mul * a.scale * kLog2e, c_b = -mul * kLog2e * a.alpha[head];
  const float gbe = a.beta[head], gmu = a.mu[head];

  const KeyWalk<kStep> walk(q_start, k_end, a.window, a.sinks);
  const int per = (walk.count + a.splits - 1) / a.splits;
  const int x_end = min(walk.count, (split + 1) * per);

  // per wave: codes of 64 keys and values (2 KB each) and their pairs (512 bytes each, written as 1 KB)
  constexpr int kWave = 2 * 2048 + 2 * 1024;
  constexpr int kRow = kD + 4, kMerge = NW * RC * (kRow + 4) * 4;
  __shared__ __attribute__((aligned(16))) uint8_t smem[NW * kWave > kMerge ? NW * kWave : kMerge];
  uint8_t *sk = smem + w * kWave, *sv = sk + 2048, *skp = sv + 2048, *svp = skp + 1024;
  const uint8_t *kc = kv.kc + b * kv.kc_sb + kvh * kv.kc_sh, *vc = kv.vc + b * kv.vc_sb + kvh * kv.vc_sh;
  const uint32_t *kp = kv.kp + b * kv.kp_sb + kvh * kv.kp_sh, *vp = kv.vp + b * kv.vp_sb + kvh * kv.vp_sh;
  // 16-byte pieces in LDS: key 16 a + x's half h at 32 a + ((2 x + h) ^ 8 (a % 2)); value row's half h at
  // 2 row + (h ^ (row / 8 % 2)): the operand reads below meet each bank as seldom as they can
  uint32_t ko[2], vo[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int s = 64 * j + lane, ka = s >> 5;
    ko[j] = 16u * (32 * ka + ((s & 31) ^ (8 * (ka & 1))));
    vo[j] = 16u * (s ^ ((s >> 4) & 1));
  }
  const uint32_t po = lane < 32 ? 16u * lane : 0x40000000u;
  auto stage = [&](int x) {
    const int n0 = walk.start(x);
    const uint32_t n = static_cast<uint32_t>(walk.rows(x));
    const buf_t kb = make_buf(kc + int64_t(n0) * 32, n * 32u), vb = make_buf(vc + int64_t(n0) * 32, n * 32u);
    const buf_t kpb = make_buf(kp + int64_t(n0) * 2, n * 8u), vpb = make_buf(vp + int64_t(n0) * 2, n * 8u);
    buf_ld16_lds<2>(kb, sk, ko[0], 0);
    buf_ld16_lds<2>(kb, sk + 1024, ko[1], 0);
    buf_ld16_lds<2>(kpb, skp, po, 0);
    buf_ld16_lds<2>(vb, sv, vo[0], 0);
    buf_ld16_lds<2>(vb, sv + 1024, vo[1], 0);
    buf_ld16_lds<2>(vpb, svp, po, 0);
  };
  // this lane's reads: score tile t's row c16 is key 16 (c16 / 4) + 4 t + c16 % 4, words g and 4 + g
  const int ka = c16 >> 2;
  auto k_at = [&](int t, int p) {
    return reinterpret_cast<const uint32_t *>(sk + 16 * (32 * ka + ((2 * (4 * t + (c16 & 3)) + p) ^ (8 * (ka & 1)))))[g];
  };
  auto v_at = [&](int ft) {  // feature 16 ft + c16 of keys 16 g ..: lane's row 16 g + c16, 8 bytes
    const uint8_t *p = sv + 32 * (16 * g + c16) + 16 * ((ft >> 1) ^ ((c16 >> 3) & 1)) + 8 * (ft & 1);
    return __builtin_amdgcn_ds_read_tr4_b64_v2i32((__attribute__((address_space(3))) i32x2 *)p);
  };

  const uint32_t nib = pair_mask();
  float m = -INFINITY, l = 0.f, ob[2] = {0.f, 0.f};
  f32x4 o[4];
#pragma unroll
  for (int ft = 0; ft < 4; ++ft) o[ft] = f32x4{0.f, 0.f, 0.f, 0.f};
  f32x4 c0[2];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const float c = kBf ? -128.f * qs[p] : 0.f;
    c0[p] = f32x4{c, c, c, c};
  }

  int x = split * per + w;
  if (x < x_end) stage(x);
  for (; x < x_end; x += NW) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this step's rows are in LDS
    uint32_t kw[4][2];
    i32x2 vw[4];
    uint4 kq[2 * TPL], vq[2 * TPL];  // pairs of this lane's keys, two keys each
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int p = 0; p < 2; ++p) kw[t][p] = k_at(t, p);
#pragma unroll
    for (int ft = 0; ft < 4; ++ft) vw[ft] = v_at(ft);
#pragma unroll
    for (int j = 0; j < 2 * TPL; ++j) {
      kq[j] = *reinterpret_cast<const uint4 *>(skp + 8 * (16 * g + NK * u) + 16 * j);
      vq[j] = *reinterpret_cast<const uint4 *>(svp + 8 * (16 * g + NK * u) + 16 * j);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // and out of it again
    const int n0 = walk.start(x);
    if (x + NW < x_end) stage(x + NW);
    __builtin_amdgcn_sched_barrier(0);

    f32x4 acc[TPL][2];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int tt = 0; tt < TPL; ++tt) {
        acc[tt][p] = c0[p];
#pragma unroll
        for (int v = 0; v < U; ++v) {
          if constexpr (kBf)
            acc[tt][p] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, codes_bf16(kw[v * TPL + tt][p], nib)),
                                                                 __builtin_bit_cast(bf16x8, qm[v][p]), acc[tt][p], 0, 0, 0);
          else
            acc[tt][p] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, codes_f16(kw[v * TPL + tt][p], nib)),
                                                                __builtin_bit_cast(f16x8, qm[v][p]), acc[tt][p], 0, 0, 0);
        }
      }
    const int key0 = n0 + 16 * g + NK * u;  // this lane's keys: key0 + e
    float z[NK], mx = -INFINITY;
#pragma unroll
    for (int e = 0; e < NK; ++e) {
      const uint4 pr = kq[e >> 1];
      const uint32_t p0 = e & 1 ? pr.z : pr.x, p1 = e & 1 ? pr.w : pr.y;
      const float s = fmaf(kv4_scale(p0), acc[e >> 2][0][e & 3], kv4_base(p0) * qs[0]) +
                      fmaf(kv4_scale(p1), acc[e >> 2][1][e & 3], kv4_base(p1) * qs[1]);
      const float d = fabsf(static_cast<float>(key0 + e - q_abs) - gmu) + a.eps;
      z[e] = fmaf(s, c_qk, c_b * fast_exp2(gbe * fast_log2(d)));
    }
    // the step's last keys, the diagonal, the window's edges: by key (their values' pairs may hold anything)
    const int n_end = n0 + walk.rows(x);
    const bool masked = n0 + kStep - 1 > q_start || n0 + kStep > k_end || (n0 <= q_start + a.L - 1 - a.window && n0 + kStep > a.sinks);
    if (masked) {
#pragma unroll
      for (int e = 0; e < NK; ++e) {
        const int key = key0 + e;
        const bool ok = (key <= q_abs) & (key < n_end) & ((key > q_abs - a.window) | (key < a.sinks));
        z[e] = ok ? z[e] : -INFINITY;
        uint4 &pr = vq[e >> 1];
        if (e & 1) { pr.z = ok ? pr.z : 0u; pr.w = ok ? pr.w : 0u; }
        else { pr.x = ok ? pr.x : 0u; pr.y = ok ? pr.y : 0u; }
      }
    }
#pragma unroll
    for (int e = 0; e < NK; ++e) mx = fmaxf(mx, z[e]);
    mx = max_g(mx);  // (the lanes of one column share its outputs' scale)
    const float m_new = fmaxf(m, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
    if (__ballot(m_new > m)) {
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - m_use);
      l *= f;
      ob[0] *= f;
      ob[1] *= f;
#pragma unroll
      for (int ft = 0; ft < 4; ++ft) o[ft] *= f;
      m = m_new;
    }
    float p[NK];
#pragma unroll
    for (int e = 0; e < NK; ++e) {
      p[e] = fast_exp2(z[e] - m_use);
      l += p[e];
    }
    uint4 vA[4][2];
#pragma unroll
    for (int ft = 0; ft < 4; ++ft)
#pragma unroll
      for (int t2 = 0; t2 < 2; ++t2) vA[ft][t2] = codes_bf16(static_cast<uint32_t>(t2 ? vw[ft].y : vw[ft].x), nib);
#pragma unroll
    for (int gr = 0; gr < 2; ++gr) {
      float ps[NK];
#pragma unroll
      for (int e = 0; e < NK; ++e) {
        const uint4 pr = vq[e >> 1];
        const uint32_t pg = gr ? (e & 1 ? pr.w : pr.y) : (e & 1 ? pr.z : pr.x);
        ps[e] = p[e] * kv4_scale(pg);
        ob[gr] = fmaf(p[e], fmaf(8.f, kv4_scale(pg), kv4_base(pg)), ob[gr]);
      }
#pragma unroll
      for (int hv = 0; hv < kHalves; ++hv) {
        // word (t2, i): weights of tiles 2 t2 and 2 t2 + 1, key i; at U = 4 both halves hold this lane's
        // one tile and the mask keeps its own
        constexpr int kW = U == 1 ? 2 : 1;
        uint32_t pk[kW][4];
#pragma unroll
        for (int t2 = 0; t2 < kW; ++t2)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float lo = ps[U == 4 ? i : 8 * t2 + i], hi = ps[U == 4 ? i : 8 * t2 + 4 + i];
            pk[t2][i] = pk2bf(lo, hi);
            // 136 of every 128 + n out again (n - 8 is what the rounded weight multiplies, the 8 with the base)
            constexpr float c = U == 4 ? -68.f : -136.f;
            const bf16x2v cc = {static_cast<__bf16>(c), static_cast<__bf16>(c)};
            ob[gr] = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2v, pk[t2][i]), cc, ob[gr], false);
            if (hv + 1 < kHalves) {  // what the first half leaves
              ps[U == 4 ? i : 8 * t2 + i] -= __uint_as_float(pk[t2][i] << 16);
              if (U != 4) ps[8 * t2 + 4 + i] -= __uint_as_float(pk[t2][i] & 0xffff0000u);
            }
          }
#pragma unroll
        for (int t2 = 0; t2 < 2; ++t2) {
          const uint32_t *s = pk[U == 1 ? t2 : 0];
          const uint4 pb = {s[0] & pmask[t2], s[1] & pmask[t2], s[2] & pmask[t2], s[3] & pmask[t2]};
#pragma unroll
          for (int f2 = 0; f2 < 2; ++f2)
            o[2 * gr + f2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, vA[2 * gr + f2][t2]),
                                                                     __builtin_bit_cast(bf16x8, pb), o[2 * gr + f2], 0, 0, 0);
        }
      }
    }
  }

  l = sum_g(l);
  ob[0] = sum_g(ob[0]);
  ob[1] = sum_g(ob[1]);
  if constexpr (U > 1) {  // the copies of a row, columns RC apart, to one
    const float M = max_copies<U>(m), f = m == -INFINITY ? 0.f : fast_exp2(m - M);
    l = sum_copies<U>(l * f);
    ob[0] = sum_copies<U>(ob[0] * f);
    ob[1] = sum_copies<U>(ob[1] * f);
#pragma unroll
    for (int ft = 0; ft < 4; ++ft)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[ft][i] = sum_copies<U>(o[ft][i] * f);
    m = M;
  }
  __syncthreads();  // every wave's staged rows are read
  float *so = reinterpret_cast<float *>(smem), *sm = so + NW * RC * kRow;  // [wave][row][feature], [wave][row][m, l, ..]
  if (u == 0) {
    if (g == 0) *reinterpret_cast<f32x4 *>(sm + 4 * (RC * w + r)) = f32x4{m, l, ob[0], ob[1]};
#pragma unroll
    for (int ft = 0; ft < 4; ++ft) *reinterpret_cast<f32x4 *>(so + (RC * w + r) * kRow + 16 * ft + 4 * g) = o[ft];
  }
  __syncthreads();
  for (int e = tid; e < RC * kD; e += 64 * NW) {
    const int rr = e / kD, d = e % kD;
    if (rr >= rows) continue;
    float M = -INFINITY;
#pragma unroll
    for (int c = 0; c < NW; ++c) M = fmaxf(M, sm[4 * (RC * c + rr)]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float ov = 0.f, Ls = 0.f;
#pragma unroll
    for (int c = 0; c < NW; ++c) {
      const f32x4 st4 = *reinterpret_cast<const f32x4 *>(sm + 4 * (RC * c + rr));
      const float f = fast_exp2(st4[0] - Mu);
      ov = fmaf(so[(RC * c + rr) * kRow + d] + (d < 32 ? st4[2] : st4[3]), f, ov);
      Ls = fmaf(st4[1], f, Ls);
    }
    if (a.part) {
      float *pp = a.part + (((static_cast<size_t>(b) * a.Hkv + kvh) * a.splits + split) * rows + rr) * (kD + 2);
      pp[d] = ov;
      if (d == 0) { pp[kD] = M; pp[kD + 1] = Ls; }
    } else {
      const int hh = kvh * group + rr % group, ii = rr / group;
      st(static_cast<T *>(a.out) + b * a.o_sb + hh * a.o_sh + int64_t(ii) * a.o_st + d, ov / fmaxf(Ls, 1e-20f));
    }
  }
}

// waves of an unsplit call: what the registers let a CU hold
constexpr int waves_of(int U) { return U == 1 ? 8 : 12; }

template <typename T, int U>
int launch_u(const ChordArgs &a, const KV4Args &kv, hipStream_t s) {
  const dim3 grid(a.splits, a.Hkv, a.B);
  if (a.part) chord_kv4_kernel<T, U, 4><<<grid, dim3(256), 0, s>>>(a, kv);
  else chord_kv4_kernel<T, U, waves_of(U)><<<grid, dim3(64 * waves_of(U)), 0, s>>>(a, kv);
  return check_launch("chord_kv4_kernel");
}

template <typename T>
int launch_t(const ChordArgs &a, const KV4Args &kv, int rows, hipStream_t s) {
  if (rows <= 4) return launch_u<T, 4>(a, kv, s);
  if (rows <= 8) return launch_u<T, 2>(a, kv, s);
  return launch_u<T, 1>(a, kv, s);
}

}  // namespace

bool chord_kv4_serves(int H, int Hkv, int L, int D, int dtype) {
  return D == kD && (dtype == MOTIF_BF16 || dtype == MOTIF_F16) && (H / Hkv) * static_cast<int64_t>(L) <= 16;
}

// Key ranges of a call, 1: one workgroup of up to 12 waves per kv head and nothing to merge.  Measured (a
// tenth more than they take now), us, 4 query heads per kv head, one token, unsplit / 4 / 8 ranges (and their merge): 3 kv heads (one sequence)
// over 1000 keys 9.4 / 8.7 / 8.9, 2000 12.2 / 10.2 / 10.6, 4097 19.4 / 13.7 / 12.8, 8000 31.5 / 17.6 / 14.3;
// 48 (16 sequences) 4097 19.9 / 14.7 / 16.0, 8000 31.7 / 19.0 / 18.8; 96 4097 20.1 / 17.8 / 18.5, 8000
// 32.6 / 24.3 / 23.1; 192 (64 sequences) 2000 13.4 / 15.3 / 21.7, 4097 21.4 / 22.2 / 29.1, 8000 34.4 /
// 30.8 / 38.7.  (Up to 1280 keys a second launch would cost the host more than it saves the device.)
int chord_kv4_splits(int B, int Hkv, int L, int S, int window, int sinks) {
  const int64_t keys = std::min<int64_t>(S, std::min<int64_t>(window, S) + L + std::min(sinks, S) + 2 * kStep);
  const int64_t steps = (keys + kStep - 1) / kStep, heads = int64_t(B) * Hkv;
  if (steps <= 20) return 1;
  if (heads >= 160) return steps > 96 ? 4 : 1;
  return steps > 96 || (heads < 32 && steps > 48) ? 8 : 4;
}

int launch_chord_kv4(const ChordArgs &a, const KV4Args &kv, int dtype, hipStream_t s) {
  const int rows = a.L * (a.H / a.Hkv);
  const int rc = dtype == MOTIF_BF16 ? launch_t<bf16_t>(a, kv, rows, s) : launch_t<f16_t>(a, kv, rows, s);
  if (rc) return rc;
  return a.part ? launch_chord_merge(a, dtype, kD, s) : launch_chord_advance(a, s);
}

}  // namespace motif
