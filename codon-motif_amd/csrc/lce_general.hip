// Cross entropy from hidden states for fp32 inputs, on v_mfma_f32_32x32x2_f32.  One product,
// C = A B^T over k, in four uses: z = W X^T (row statistics, or P), dX = P W, dW = P^T X.  A
// workgroup of four waves owns 64 x 64 of C (32 x 32 a wave) and stages 32 k of both sides in LDS, k outermost,
// twice: one place is filled, from registers loaded a step before, while the other is multiplied.  The matrix
// instruction (64 cycles for two k) bounds it, so LDS reads of single words suffice.  (128 x 128 were slower
// at every size: 512 x 1024 x 8192, dW 125 against 94 us.)  dX and dW share a launch (189 against 203 us there; 27 against 37
// for 271 x 256 x 5003).  What is reached: 88-95 TFLOP/s at 2048 x 768 x 8192, where a large library product reaches
// 154; a wave per SIMD and workgroup, its chain of one accumulator and its barriers leave the rest.
// Sums run over 512 k at a time, which are then added (one chain over a vocabulary of 5000 lost a bit of dX: 1.3e-6
// off where this is 6e-7).
#include "lce_internal.h"

#include <algorithm>

namespace motif {

namespace {

constexpr int TM = 64, BK = 32, LD = TM + 4, SIZE = BK * LD;
constexpr int kChain = 512;

// TM rows x BK k of an operand: element (m, k) at p[m ld + k] (KIN) or p[k ld + m]; zero outside.  VEC: 16 bytes a load,
// through a range-checked buffer (rows on 16-byte boundaries, k_max a multiple of 4 where KIN).
template <bool KIN, bool VEC> struct Side {
  static constexpr int E = VEC ? 4 : 1, N = 8 / E, ROW = (KIN ? BK : TM) / E;  // accesses of a thread, and along memory
  const float *p;
  int64_t ld;
  int m_max, k_max;  // elements from p on
  float r[8];
  __device__ __forceinline__ static int along(int i) { return (threadIdx.x + 256 * i) % ROW * E; }
  __device__ __forceinline__ static int across(int i) { return (threadIdx.x + 256 * i) / ROW; }
  __device__ __forceinline__ void load(int k0) {
    if (VEC) {
      const int n = KIN ? min(m_max, TM) : min(k_max - k0, BK);
      const buf_t b = make_buf(KIN ? p : p + k0 * ld, n > 0 ? static_cast<uint32_t>(((n - 1) * ld + (KIN ? k_max : min(m_max, TM))) * 4) : 0u);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int k = k0 + along(i);
        const uint32_t off = static_cast<uint32_t>((across(i) * ld + (KIN ? k : along(i))) * 4);
        const uint4 u = buf_ld16(b, !KIN || k < k_max ? off : 0xfffffff0u);
        r[4 * i] = __uint_as_float(u.x), r[4 * i + 1] = __uint_as_float(u.y);
        r[4 * i + 2] = __uint_as_float(u.z), r[4 * i + 3] = __uint_as_float(u.w);
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int m = KIN ? across(i) : along(i), k = k0 + (KIN ? along(i) : across(i));
        r[i] = m < m_max && k < k_max ? p[KIN ? int64_t(m) * ld + k : int64_t(k) * ld + m] : 0.f;
      }
    }
  }
  __device__ __forceinline__ void store(float *s) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float *q = s + (KIN ? along(i) * LD + across(i) : across(i) * LD + along(i));
      if (KIN || !VEC) {
#pragma unroll
        for (int e = 0; e < E; ++e) q[e * LD] = r[E * i + e];
      } else {
        *reinterpret_cast<f32x4 *>(q) = f32x4{r[E * i], r[(E * i + 1) % 8], r[(E * i + 2) % 8], r[(E * i + 3) % 8]};
      }
    }
  }
};

// C of the workgroup's tile over k in [kb, ke), this wave's 32 x 32 in sum[0][0]
template <typename SA, typename SB>
__device__ __forceinline__ void product(SA &A, SB &B, int kb, int ke, float *lds, f32x16 (&sum)[1][1]) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  f32x16 acc;
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i] = sum[0][0][i] = 0.f;
  if (kb >= ke) return;
  A.load(kb);
  B.load(kb);
  A.store(lds);
  B.store(lds + SIZE);
  int at = 0;
  for (int k0 = kb; k0 < ke; k0 += BK) {
    const bool more = k0 + BK < ke;
    if (more) {
      A.load(k0 + BK);
      B.load(k0 + BK);
    }
    __syncthreads();
    const float *pa = lds + at + 32 * (w & 1) + (l & 31), *pb = lds + at + SIZE + 32 * (w >> 1) + (l & 31);
#pragma unroll
    for (int k = 0; k < BK; k += 2)
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(pa[(k + h) * LD], pb[(k + h) * LD], acc, 0, 0, 0);
    if ((k0 - kb) % kChain == kChain - BK || !more)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sum[0][0][i] += acc[i];
        acc[i] = 0.f;
      }
    // (the other place was last read before this step's barrier)
    at ^= 2 * SIZE;
    if (more) {
      A.store(lds + at);
      B.store(lds + at + SIZE);
    }
  }
}

// z of TM vocabulary rows and TM tokens, then their statistics or P
template <bool VEC, bool GRADS>
__global__ void __launch_bounds__(256) lce_general_z_kernel(LceArgs a) {
  __shared__ __align__(16) float lds[4 * SIZE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int t0 = blockIdx.x * TM, v0 = (GRADS ? a.v0 : 0) + blockIdx.y * TM;
  if (t0 >= count) return;
  Side<true, VEC> A{static_cast<const float *>(a.w) + int64_t(v0) * a.ldw, a.ldw, a.V - v0, a.d};
  Side<true, VEC> B{static_cast<const float *>(a.x) + int64_t(t0) * a.ldx, a.ldx, count - t0, a.d};
  f32x16 acc[1][1];
  product(A, B, 0, a.d, lds, acc);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  const int vw = v0 + 32 * (w & 1), tw = t0 + 32 * (w >> 1);
  if (!GRADS) {
    lce_row_stats<1, 1>(a, acc, vw, tw, count, 2 * blockIdx.y + (w & 1));
    return;
  }
  bool live[1];
  lce_row_grads<1, 1>(a, acc, vw, tw, count, live);
  if (!live[0]) return;
  float *p = static_cast<float *>(a.p) + int64_t(tw + (l & 31)) * a.vc + (vw - a.v0);
#pragma unroll
  for (int i = 0; i < 16; i += 4)
    *reinterpret_cast<f32x4 *>(p + acc_row(i, h)) = f32x4{acc[0][0][i], acc[0][0][i + 1], acc[0][0][i + 2], acc[0][0][i + 3]};
}

// Both products of a piece in one launch: `ndx` workgroups for dX (token tile, column tile, share of the vocabulary rows,
// the first fastest), then dW's (vocabulary tile, column tile).
template <bool VEC>
__global__ void __launch_bounds__(256) lce_general_products_kernel(LceArgs a, int tt, int vt, int ndx) {
  __shared__ __align__(16) float lds[4 * SIZE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  f32x16 acc[1][1];
  if (static_cast<int>(blockIdx.x) < ndx) {  // dX [tokens, d] += P W over the piece
    const int ct = (a.d + TM - 1) / TM, b = blockIdx.x;
    const int t0 = b % tt * TM, c0 = b / tt % ct * TM, share = b / tt / ct;
    if (t0 >= count) return;
    const int steps = (a.vn + BK - 1) / BK, per = (steps + a.dx_splits - 1) / a.dx_splits;
    const int kb = min(a.vn, share * per * BK), ke = min(a.vn, kb + per * BK);
    // (P holds zeros behind the piece)
    Side<true, VEC> A{static_cast<const float *>(a.p) + int64_t(t0) * a.vc, a.vc, count - t0, (a.vn + 3) & ~3};
    Side<false, VEC> B{static_cast<const float *>(a.w) + int64_t(a.v0) * a.ldw + c0, a.ldw, a.d - c0, a.vn};
    product(A, B, kb, ke, lds, acc);
    const int c = c0 + 32 * (w >> 1) + (l & 31);
    if (c >= a.d) return;
    float *out = a.dx_part + int64_t(share) * a.n_pad * a.d + c;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int t = t0 + 32 * (w & 1) + acc_row(i, h);
      if (t < count) {
        float *o = out + int64_t(t) * a.d;
        *o = a.first ? acc[0][0][i] : *o + acc[0][0][i];
      }
    }
    return;
  }
  // dW rows of the piece = P^T X
  const int b = blockIdx.x - ndx, r0 = b % vt * TM, c0 = b / vt * TM;
  Side<false, VEC> A{static_cast<const float *>(a.p) + r0, a.vc, a.vn - r0, count};
  Side<false, VEC> B{static_cast<const float *>(a.x) + c0, a.ldx, a.d - c0, count};
  product(A, B, 0, count, lds, acc);
  const float f = lce_factor(a, count);
  const int c = c0 + 32 * (w >> 1) + (l & 31);
  if (c >= a.d) return;
  float *out = static_cast<float *>(a.dw) + int64_t(a.v0) * a.d + c;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int r = r0 + 32 * (w & 1) + acc_row(i, h);
    if (r < a.vn) out[int64_t(r) * a.d] = acc[0][0][i] * f;
  }
}

unsigned tiles(int n) { return static_cast<unsigned>((n + TM - 1) / TM); }

// 16 bytes a load where the vocabulary's rows allow it (the labelled rows and P are laid out for it)
bool wide_rows(const LceArgs &a) {
  return a.d % 4 == 0 && a.ldw % 4 == 0 && a.ldw < (1 << 21) && reinterpret_cast<uintptr_t>(a.w) % 16 == 0;
}

}  // namespace

int lce_general_parts(int V) { return 2 * static_cast<int>(tiles(V)); }

// Shares of a piece's vocabulary rows: rounds of two workgroups to a CU (0.8 us a step of 32) against the partial sums'
// traffic (4 TB/s).
int lce_general_dx_splits(int64_t N, int d, int V, int vc) {
  const int64_t t = (N + TM - 1) / TM * tiles(d), steps = (std::min(V, vc) + BK - 1) / BK;
  int best = 1;
  double least = 0;
  for (int s = 1; s <= 16 && s <= steps; ++s) {
    const double cost = double((t * s + 511) / 512) * double((steps + s - 1) / s) * 0.8 + double(s) * N * d * 8 / 4e6;
    if (s == 1 || cost < least) best = s, least = cost;
  }
  return best;
}

int launch_lce_general_stats(const LceArgs &a, hipStream_t s) {
  const dim3 g(tiles(a.N), tiles(a.V));
  if (wide_rows(a)) lce_general_z_kernel<true, false><<<g, 256, 0, s>>>(a);
  else lce_general_z_kernel<false, false><<<g, 256, 0, s>>>(a);
  return check_launch("lce_general_z_kernel (statistics)");
}

int launch_lce_general_grads(const LceArgs &a, hipStream_t s) {
  const dim3 g(tiles(a.N), tiles(a.vn));
  if (wide_rows(a)) lce_general_z_kernel<true, true><<<g, 256, 0, s>>>(a);
  else lce_general_z_kernel<false, true><<<g, 256, 0, s>>>(a);
  return check_launch("lce_general_z_kernel (gradients)");
}

int launch_lce_general_products(const LceArgs &a, bool dx, bool dw, hipStream_t s) {
  const int tt = static_cast<int>(tiles(a.N)), vt = static_cast<int>(tiles(a.vn)), ct = static_cast<int>(tiles(a.d));
  const int ndx = dx ? tt * ct * a.dx_splits : 0;
  const dim3 g(ndx + (dw ? vt * ct : 0));
  if (wide_rows(a)) lce_general_products_kernel<true><<<g, 256, 0, s>>>(a, tt, vt, ndx);
  else lce_general_products_kernel<false><<<g, 256, 0, s>>>(a, tt, vt, ndx);
  return check_launch("lce_general_products_kernel");
}

}  // namespace motif
