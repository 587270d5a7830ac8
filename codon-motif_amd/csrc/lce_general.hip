// Cross entropy from hidden states on the fp32 matrix instructions (v_mfma_f32_32x32x2_f32): fp32
// inputs, and bf16 ones whose rows the bf16 kernels cannot load 16 bytes at a time.  One product,
// C = A B^T over k, in four uses: z = W X^T (row statistics, or P), dX = P W, dW = P^T X.  A
// workgroup of four waves owns 128 x 128 of C (64 x 64 a wave) and stages 16 k of both sides in LDS
// as fp32, k outermost, the next 16 in registers meanwhile; the matrix instruction (64 cycles for two
// k) bounds it, so LDS reads of single words suffice.
#include "lce_internal.h"

namespace motif {

namespace {

constexpr int TM = 128, BK = 16, LD = TM + 4;

// 128 rows x 16 k of an operand: element (m, k) at p[m ld + k] (KIN) or p[k ld + m]; zero outside.
template <typename T, bool KIN> struct Side {
  const T *p;
  int64_t ld;
  int m_max, k_max;  // elements from p on
  float r[8];
  __device__ __forceinline__ void load(int k0) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = KIN ? (t >> 4) + 16 * i : t & 127, k = k0 + (KIN ? t & 15 : (t >> 7) + 2 * i);
      r[i] = m < m_max && k < k_max ? ld_(KIN ? int64_t(m) * ld + k : int64_t(k) * ld + m) : 0.f;
    }
  }
  __device__ __forceinline__ float ld_(int64_t e) const { return motif::ld(p + e); }
  __device__ __forceinline__ void store(float *s) const {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      s[KIN ? (t & 15) * LD + (t >> 4) + 16 * i : ((t >> 7) + 2 * i) * LD + (t & 127)] = r[i];
  }
};

template <typename SA, typename SB>
__device__ __forceinline__ void product(SA &A, SB &B, int K, float *sa, float *sb, f32x16 (&acc)[2][2]) {
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mb][nb][i] = 0.f;
  A.load(0);
  B.load(0);
  const float *pa = sa + 64 * (w & 1) + (l & 31), *pb = sb + 64 * (w >> 1) + (l & 31);
  for (int k0 = 0; k0 < K; k0 += BK) {
    __syncthreads();
    A.store(sa);
    B.store(sb);
    __syncthreads();
    if (k0 + BK < K) {
      A.load(k0 + BK);
      B.load(k0 + BK);
    }
#pragma unroll
    for (int k = 0; k < BK; k += 2) {
      const int o = (k + h) * LD;
      const float a0 = pa[o], a1 = pa[o + 32], b0 = pb[o], b1 = pb[o + 32];
      acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a0, b0, acc[0][0], 0, 0, 0);
      acc[0][1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a0, b1, acc[0][1], 0, 0, 0);
      acc[1][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a1, b0, acc[1][0], 0, 0, 0);
      acc[1][1] = __builtin_amdgcn_mfma_f32_32x32x2f32(a1, b1, acc[1][1], 0, 0, 0);
    }
  }
}

// z of 128 vocabulary rows and 128 tokens, then their statistics or P
template <typename T, bool GRADS>
__global__ void __launch_bounds__(256) lce_general_z_kernel(LceArgs a) {
  __shared__ float sa[BK * LD], sb[BK * LD];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int t0 = blockIdx.y * TM, v0 = (GRADS ? a.v0 : 0) + blockIdx.x * TM;
  if (t0 >= count) return;
  Side<T, true> A{static_cast<const T *>(a.w) + int64_t(v0) * a.ldw, a.ldw, a.V - v0, a.d};
  Side<T, true> B{static_cast<const T *>(a.x) + int64_t(t0) * a.ldx, a.ldx, count - t0, a.d};
  f32x16 acc[2][2];
  product(A, B, a.d, sa, sb, acc);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  const int vw = v0 + 64 * (w & 1), tw = t0 + 64 * (w >> 1);
  if (!GRADS) {
    lce_row_stats<2, 2>(a, acc, vw, tw, count, 2 * blockIdx.x + (w & 1));
    return;
  }
  lce_row_grads<2, 2>(a, acc, vw, tw, count);
  float *p = static_cast<float *>(a.p) + (vw - a.v0);
#pragma unroll
  for (int nb = 0; nb < 2; ++nb) {
    const int t = tw + 32 * nb + (l & 31);
    if (t >= count) continue;
#pragma unroll
    for (int mb = 0; mb < 2; ++mb)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 v = {acc[mb][nb][i], acc[mb][nb][i + 1], acc[mb][nb][i + 2], acc[mb][nb][i + 3]};
        *reinterpret_cast<f32x4 *>(p + int64_t(t) * a.vc + 32 * mb + acc_row(i, h)) = v;
      }
  }
}

// dX [tokens, d] += P W over the piece
template <typename T>
__global__ void __launch_bounds__(256) lce_general_dx_kernel(LceArgs a) {
  __shared__ float sa[BK * LD], sb[BK * LD];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int t0 = blockIdx.y * TM, c0 = blockIdx.x * TM;
  if (t0 >= count) return;
  Side<float, true> A{static_cast<const float *>(a.p) + int64_t(t0) * a.vc, a.vc, count - t0, a.vn};
  Side<T, false> B{static_cast<const T *>(a.w) + int64_t(a.v0) * a.ldw + c0, a.ldw, a.d - c0, a.vn};
  f32x16 acc[2][2];
  product(A, B, a.vn, sa, sb, acc);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int c = c0 + 64 * (w >> 1) + 32 * nb + (l & 31);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = t0 + 64 * (w & 1) + 32 * mb + acc_row(i, h);
        if (t < count && c < a.d) {
          float *o = a.dx_part + int64_t(t) * a.d + c;
          *o = a.first ? acc[mb][nb][i] : *o + acc[mb][nb][i];
        }
      }
    }
}

// dW rows of the piece = P^T X
template <typename T>
__global__ void __launch_bounds__(256) lce_general_dw_kernel(LceArgs a) {
  __shared__ float sa[BK * LD], sb[BK * LD];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int r0 = blockIdx.y * TM, c0 = blockIdx.x * TM;
  Side<float, false> A{static_cast<const float *>(a.p) + r0, a.vc, a.vn - r0, count};
  Side<T, false> B{static_cast<const T *>(a.x) + c0, a.ldx, a.d - c0, count};
  f32x16 acc[2][2];
  product(A, B, count, sa, sb, acc);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
#pragma unroll
  for (int mb = 0; mb < 2; ++mb)
#pragma unroll
    for (int nb = 0; nb < 2; ++nb) {
      const int c = c0 + 64 * (w >> 1) + 32 * nb + (l & 31);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = r0 + 64 * (w & 1) + 32 * mb + acc_row(i, h);
        if (r < a.vn && c < a.d) st(static_cast<T *>(a.dw) + int64_t(a.v0 + r) * a.d + c, acc[mb][nb][i]);
      }
    }
}

dim3 tiles(int x, int y) { return dim3((x + TM - 1) / TM, (y + TM - 1) / TM); }

template <typename T> void z_launch(const LceArgs &a, bool grads, hipStream_t s) {
  if (grads)
    lce_general_z_kernel<T, true><<<tiles(a.vn, a.N), 256, 0, s>>>(a);
  else
    lce_general_z_kernel<T, false><<<tiles(a.V, a.N), 256, 0, s>>>(a);
}

}  // namespace

int lce_general_parts(int V) { return 2 * ((V + TM - 1) / TM); }

int launch_lce_general_stats(const LceArgs &a, int dtype, hipStream_t s) {
  if (dtype == MOTIF_F32) z_launch<float>(a, false, s);
  else z_launch<bf16_t>(a, false, s);
  return check_launch("lce_general_z_kernel (statistics)");
}

int launch_lce_general_grads(const LceArgs &a, int dtype, hipStream_t s) {
  if (dtype == MOTIF_F32) z_launch<float>(a, true, s);
  else z_launch<bf16_t>(a, true, s);
  return check_launch("lce_general_z_kernel (gradients)");
}

int launch_lce_general_dx(const LceArgs &a, int dtype, hipStream_t s) {
  const dim3 g = tiles(a.d, a.N);
  if (dtype == MOTIF_F32) lce_general_dx_kernel<float><<<g, 256, 0, s>>>(a);
  else lce_general_dx_kernel<bf16_t><<<g, 256, 0, s>>>(a);
  return check_launch("lce_general_dx_kernel");
}

int launch_lce_general_dw(const LceArgs &a, int dtype, hipStream_t s) {
  const dim3 g = tiles(a.d, a.vn);
  if (dtype == MOTIF_F32) lce_general_dw_kernel<float><<<g, 256, 0, s>>>(a);
  else lce_general_dw_kernel<bf16_t><<<g, 256, 0, s>>>(a);
  return check_launch("lce_general_dw_kernel");
}

}  // namespace motif
