// Cross entropy from hidden states for fp32 inputs, on v_mfma_f32_32x32x2_f32.  One product,
// C = A B^T over k, in four uses: z = W X^T (row statistics, or P), dX = P W, dW = P^T X.  A
// workgroup of four waves owns 64 x 64 or 128 x 128 of C and stages 32 or 16 k of both sides in LDS
// as fp32, k outermost, the next ones in registers meanwhile; the matrix instruction (64 cycles for two
// k) bounds it, so LDS reads of single words suffice.  Sums run over 512 k at a time, which are then added (one
// chain over a vocabulary of 5000 lost a bit of dX: 1.3e-6 off where this is 7e-7).
#include "lce_internal.h"

#include <algorithm>

namespace motif {

namespace {

// Tiles of TM x TM, TM = 64 MB: one or two blocks of 32 a side for each of the four waves.
template <int MB> struct Tile {
  static constexpr int TM = 64 * MB, BK = 2048 / TM, LD = TM + 4, SIZE = BK * LD;
};
constexpr int kChain = 512;  // k summed after each other

// TM rows x BK k of an operand: element (m, k) at p[m ld + k] (KIN) or p[k ld + m]; zero outside.
template <int MB, bool KIN> struct Side {
  using X = Tile<MB>;
  const float *p;
  int64_t ld;
  int m_max, k_max;  // elements from p on
  float r[8];
  __device__ __forceinline__ static int m_of(int i) { return KIN ? threadIdx.x / X::BK + 256 / X::BK * i : threadIdx.x % X::TM; }
  __device__ __forceinline__ static int k_of(int i) { return KIN ? threadIdx.x % X::BK : threadIdx.x / X::TM + 256 / X::TM * i; }
  __device__ __forceinline__ void load(int k0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int m = m_of(i), k = k0 + k_of(i);
      r[i] = m < m_max && k < k_max ? p[KIN ? int64_t(m) * ld + k : int64_t(k) * ld + m] : 0.f;
    }
  }
  __device__ __forceinline__ void store(float *s) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[k_of(i) * X::LD + m_of(i)] = r[i];
  }
};

template <int MB, typename SA, typename SB>
__device__ __forceinline__ void product(SA &A, SB &B, int kb, int ke, float *sa, float *sb, f32x16 (&sum)[MB][MB]) {
  using X = Tile<MB>;
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  f32x16 acc[MB][MB];
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < MB; ++nb)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[mb][nb][i] = sum[mb][nb][i] = 0.f;
  if (kb >= ke) return;
  A.load(kb);
  B.load(kb);
  const float *pa = sa + 32 * MB * (w & 1) + (l & 31), *pb = sb + 32 * MB * (w >> 1) + (l & 31);
  for (int k0 = kb; k0 < ke; k0 += X::BK) {
    __syncthreads();
    A.store(sa);
    B.store(sb);
    __syncthreads();
    if (k0 + X::BK < ke) {
      A.load(k0 + X::BK);
      B.load(k0 + X::BK);
    }
#pragma unroll
    for (int k = 0; k < X::BK; k += 2) {
      float fa[MB], fb[MB];
#pragma unroll
      for (int b = 0; b < MB; ++b) fa[b] = pa[(k + h) * X::LD + 32 * b], fb[b] = pb[(k + h) * X::LD + 32 * b];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < MB; ++nb)
          acc[mb][nb] = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[mb], fb[nb], acc[mb][nb], 0, 0, 0);
    }
    if ((k0 - kb) % kChain == kChain - X::BK || k0 + X::BK >= ke)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int nb = 0; nb < MB; ++nb)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            sum[mb][nb][i] += acc[mb][nb][i];
            acc[mb][nb][i] = 0.f;
          }
  }
}

// z of TM vocabulary rows and TM tokens, then their statistics or P
template <int MB, bool GRADS>
__global__ void __launch_bounds__(256) lce_general_z_kernel(LceArgs a) {
  using X = Tile<MB>;
  __shared__ float sa[X::SIZE], sb[X::SIZE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int t0 = blockIdx.y * X::TM, v0 = (GRADS ? a.v0 : 0) + blockIdx.x * X::TM;
  if (t0 >= count) return;
  Side<MB, true> A{static_cast<const float *>(a.w) + int64_t(v0) * a.ldw, a.ldw, a.V - v0, a.d};
  Side<MB, true> B{static_cast<const float *>(a.x) + int64_t(t0) * a.ldx, a.ldx, count - t0, a.d};
  f32x16 acc[MB][MB];
  product<MB>(A, B, 0, a.d, sa, sb, acc);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  const int vw = v0 + 32 * MB * (w & 1), tw = t0 + 32 * MB * (w >> 1);
  if (!GRADS) {
    lce_row_stats<MB, MB>(a, acc, vw, tw, count, 2 * blockIdx.x + (w & 1));
    return;
  }
  bool live[MB];
  lce_row_grads<MB, MB>(a, acc, vw, tw, count, live);
  float *p = static_cast<float *>(a.p) + (vw - a.v0);
#pragma unroll
  for (int nb = 0; nb < MB; ++nb) {
    const int t = tw + 32 * nb + (l & 31);
    if (!live[nb]) continue;
#pragma unroll
    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const f32x4 v = {acc[mb][nb][i], acc[mb][nb][i + 1], acc[mb][nb][i + 2], acc[mb][nb][i + 3]};
        *reinterpret_cast<f32x4 *>(p + int64_t(t) * a.vc + 32 * mb + acc_row(i, h)) = v;
      }
  }
}

// Share blockIdx.z of dX [tokens, d] += P W over the piece
template <int MB>
__global__ void __launch_bounds__(256) lce_general_dx_kernel(LceArgs a) {
  using X = Tile<MB>;
  __shared__ float sa[X::SIZE], sb[X::SIZE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int t0 = blockIdx.y * X::TM, c0 = blockIdx.x * X::TM;
  if (t0 >= count) return;
  const int steps = (a.vn + X::BK - 1) / X::BK, per = (steps + a.dx_splits - 1) / a.dx_splits;
  const int kb = min(a.vn, int(blockIdx.z) * per * X::BK), ke = min(a.vn, kb + per * X::BK);
  Side<MB, true> A{static_cast<const float *>(a.p) + int64_t(t0) * a.vc, a.vc, count - t0, a.vn};
  Side<MB, false> B{static_cast<const float *>(a.w) + int64_t(a.v0) * a.ldw + c0, a.ldw, a.d - c0, a.vn};
  f32x16 acc[MB][MB];
  product<MB>(A, B, kb, ke, sa, sb, acc);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
  float *out = a.dx_part + int64_t(blockIdx.z) * a.n_pad * a.d;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < MB; ++nb) {
      const int c = c0 + 32 * MB * (w >> 1) + 32 * nb + (l & 31);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int t = t0 + 32 * MB * (w & 1) + 32 * mb + acc_row(i, h);
        if (t < count && c < a.d) {
          float *o = out + int64_t(t) * a.d + c;
          *o = a.first ? acc[mb][nb][i] : *o + acc[mb][nb][i];
        }
      }
    }
}

// dW rows of the piece = P^T X
template <int MB>
__global__ void __launch_bounds__(256) lce_general_dw_kernel(LceArgs a) {
  using X = Tile<MB>;
  __shared__ float sa[X::SIZE], sb[X::SIZE];
  const int count = __builtin_amdgcn_readfirstlane(*a.count);
  const int r0 = blockIdx.y * X::TM, c0 = blockIdx.x * X::TM;
  Side<MB, false> A{static_cast<const float *>(a.p) + r0, a.vc, a.vn - r0, count};
  Side<MB, false> B{static_cast<const float *>(a.x) + c0, a.ldx, a.d - c0, count};
  f32x16 acc[MB][MB];
  product<MB>(A, B, 0, count, sa, sb, acc);
  const float f = lce_factor(a, count);
  const int l = threadIdx.x & 63, w = threadIdx.x >> 6, h = l >> 5;
#pragma unroll
  for (int mb = 0; mb < MB; ++mb)
#pragma unroll
    for (int nb = 0; nb < MB; ++nb) {
      const int c = c0 + 32 * MB * (w >> 1) + 32 * nb + (l & 31);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int r = r0 + 32 * MB * (w & 1) + 32 * mb + acc_row(i, h);
        if (r < a.vn && c < a.d) static_cast<float *>(a.dw)[int64_t(a.v0 + r) * a.d + c] = acc[mb][nb][i] * f;
      }
    }
}

// Tiles of 64 until tiles of 128 give two workgroups to every CU (301 rows, 256 features, 5003 words: the
// three products 39, 40 and 597 us with 128, see the table's case for now).
bool small(int x, int y, int z = 1) { return int64_t((x + 127) / 128) * ((y + 127) / 128) * z < 512; }
template <int MB> dim3 tiles(int x, int y, int z = 1) {
  return dim3((x + Tile<MB>::TM - 1) / Tile<MB>::TM, (y + Tile<MB>::TM - 1) / Tile<MB>::TM, z);
}

}  // namespace

int lce_general_parts(int V, int N) {
  const int tm = small(V, N) ? 64 : 128;
  return 2 * ((V + tm - 1) / tm);
}

// Shares of a piece's vocabulary rows: until 512 workgroups of 64 x 64, each with 128 rows at least
int lce_general_dx_splits(int64_t N, int d, int V, int vc) {
  const int64_t t = ((N + 63) / 64) * ((d + 63) / 64);
  const int most = (std::min(V, vc) + 127) / 128;
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>({512 / t, int64_t(most), int64_t(16)})));
}

int launch_lce_general_stats(const LceArgs &a, hipStream_t s) {
  if (small(a.V, a.N)) lce_general_z_kernel<1, false><<<tiles<1>(a.V, a.N), 256, 0, s>>>(a);
  else lce_general_z_kernel<2, false><<<tiles<2>(a.V, a.N), 256, 0, s>>>(a);
  return check_launch("lce_general_z_kernel (statistics)");
}

int launch_lce_general_grads(const LceArgs &a, hipStream_t s) {
  if (small(a.vn, a.N)) lce_general_z_kernel<1, true><<<tiles<1>(a.vn, a.N), 256, 0, s>>>(a);
  else lce_general_z_kernel<2, true><<<tiles<2>(a.vn, a.N), 256, 0, s>>>(a);
  return check_launch("lce_general_z_kernel (gradients)");
}

int launch_lce_general_dx(const LceArgs &a, hipStream_t s) {
  if (small(a.d, a.N, a.dx_splits)) lce_general_dx_kernel<1><<<tiles<1>(a.d, a.N, a.dx_splits), 256, 0, s>>>(a);
  else lce_general_dx_kernel<2><<<tiles<2>(a.d, a.N, a.dx_splits), 256, 0, s>>>(a);
  return check_launch("lce_general_dx_kernel");
}

int launch_lce_general_dw(const LceArgs &a, hipStream_t s) {
  if (small(a.d, a.vn)) lce_general_dw_kernel<1><<<tiles<1>(a.d, a.vn), 256, 0, s>>>(a);
  else lce_general_dw_kernel<2><<<tiles<2>(a.d, a.vn), 256, 0, s>>>(a);
  return check_launch("lce_general_dw_kernel");
}

}  // namespace motif
