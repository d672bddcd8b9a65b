// op_gemm.h — C[i][j] = sum_c A(i, c) B(j, c) with the linear layer's epilogue, for every size, stride and alignment.
#pragma once
#include "op_common.h"

namespace vdbk {

struct GemmParams {
  const void* a; long long lda;
  const void* b; long long ldb;
  long long m, n, k;
  void* y; long long ldy;
  const void* bias; const void* residual; long long ldr;
  void* z;
  float* partial;      // split contraction: [splits][m][n]
  long long k_split;   // contraction values per split (a multiple of the K step)
  int vec_a, vec_b;    // rows start on 16-byte borders
};

template <typename T>
__device__ __forceinline__ T to_elem(float x) { return (T)x; }

// One value of the epilogue: sum -> bias -> (z) -> activation -> residual -> y
template <typename T, int ACT>
__device__ __forceinline__ void store_one(const GemmParams& p, long long i, long long j, float s, float bias) {
  s += bias;
  if (p.z) ((T*)p.z)[i * p.n + j] = (T)s;
  s = act_value<ACT>(s);
  if (p.residual) s += (float)((const T*)p.residual)[i * p.ldr + j];
  ((T*)p.y)[i * p.ldy + j] = (T)s;
}

// ---- any shape -----------------------------------------------------------------------------------------------------
// 128 x 128 (or 64 x 64) outputs per block of four waves, each wave a quarter; operands go through registers into LDS
// as [row][c] with 16 bytes of padding, elements outside the operands as zeros.  The fallback of the kernels below:
// what they require of sizes and alignment does not hold here.
template <typename T, bool AT, bool BT, int ACT, bool SPLIT, int BM>
__global__ __launch_bounds__(256) void gemm_any_kernel(const GemmParams p) {
  using E = Elem<T>;
  using vec = typename E::vec;
  constexpr int V = E::kVec, BK = 4 * 2 * V, LD = BK + V, W = BM / 64;   // W x W 32x32 tiles per wave
  __shared__ __align__(16) T sa[BM * LD];
  __shared__ __align__(16) T sb[BM * LD];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const long long i0 = (long long)blockIdx.x * BM, j0 = (long long)blockIdx.y * BM;
  const long long c0 = SPLIT ? (long long)blockIdx.z * p.k_split : 0;
  const long long c1 = SPLIT ? (c0 + p.k_split < p.k ? c0 + p.k_split : p.k) : p.k;
  f32x16 acc[W][W] = {};

  auto stage = [&](T* s, const T* g, long long ld, bool tr, bool vec_ok, long long r0, long long r_end, long long cc) {
    constexpr int kChunks = BM * BK / V;
    for (int t = tid; t < kChunks; t += 256) {
      T x[V];
      if (!tr) {
        const int r = t / (BK / V), c = (t % (BK / V)) * V;
        const long long gr = r0 + r, gc = cc + c;
        if (vec_ok && gr < r_end && gc + V <= c1) {
          *(vec*)&s[r * LD + c] = *(const vec*)(g + gr * ld + gc);
          continue;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = gr < r_end && gc + e < c1 ? g[gr * ld + gc + e] : (T)0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) s[r * LD + c + e] = x[e];
      } else {
        const int c = t / (BM / V), r = (t % (BM / V)) * V;
        const long long gr = r0 + r, gc = cc + c;
        if (vec_ok && gr + V <= r_end && gc < c1) {
          *(vec*)x = *(const vec*)(g + gc * ld + gr);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) x[e] = gr + e < r_end && gc < c1 ? g[gc * ld + gr + e] : (T)0.f;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) s[(r + e) * LD + c] = x[e];
      }
    }
  };

  const int wi = (wave >> 1) * 32 * W, wj = (wave & 1) * 32 * W;
  for (long long cc = c0; cc < c1; cc += BK) {
    __syncthreads();
    stage(sa, (const T*)p.a, p.lda, AT, p.vec_a, i0, p.m, cc);
    stage(sb, (const T*)p.b, p.ldb, BT, p.vec_b, j0, p.n, cc);
    __syncthreads();
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      vec fa[W], fb[W];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        fa[w] = *(const vec*)&sa[(wi + w * 32 + (lane & 31)) * LD + ks * 2 * V + (lane >> 5) * V];
        fb[w] = *(const vec*)&sb[(wj + w * 32 + (lane & 31)) * LD + ks * 2 * V + (lane >> 5) * V];
      }
#pragma unroll
      for (int a = 0; a < W; ++a)
#pragma unroll
        for (int b = 0; b < W; ++b) E::mma(fa[a], fb[b], acc[a][b]);
    }
  }
#pragma unroll
  for (int a = 0; a < W; ++a)
#pragma unroll
    for (int b = 0; b < W; ++b) {
      const long long j = j0 + wj + b * 32 + (lane & 31);
      if (j >= p.n) continue;
      const float bias = !SPLIT && p.bias ? (float)((const T*)p.bias)[j] : 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const long long i = i0 + wi + a * 32 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5);
        if (i >= p.m) continue;
        if constexpr (SPLIT) p.partial[((long long)blockIdx.z * p.m + i) * p.n + j] = acc[a][b][r];
        else store_one<T, ACT>(p, i, j, acc[a][b][r], bias);
      }
    }
}

// The join of a split contraction: the parts in order, then the epilogue.  Memory-bound: splits * m * n * 4 bytes.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void gemm_join_kernel(const GemmParams p, int splits) {
  const long long mn = p.m * p.n;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < mn; t += (long long)gridDim.x * 256) {
    float s = 0.f;
    for (int z = 0; z < splits; ++z) s += p.partial[(long long)z * mn + t];
    const long long i = t / p.n, j = t - i * p.n;
    store_one<T, ACT>(p, i, j, s, p.bias ? (float)((const T*)p.bias)[j] : 0.f);
  }
}

// ---- activation gradient and column sums -------------------------------------------------------------------------------
// Block (x, y): columns x * 64 .., rows of part y; four waves take rows in turn, one column per lane.  Column sums: 32-bit
// within a part, the parts joined in order by col_join_kernel.
template <typename T, int ACT>
__global__ __launch_bounds__(256) void act_grad_kernel(const T* __restrict__ dy, long long lddy, const T* __restrict__ z, T* __restrict__ dz,
                                                       float* __restrict__ part, long long m, long long n, long long rows_per_part) {
  __shared__ float red[4][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long long j = (long long)blockIdx.x * 64 + lane;
  const long long r0 = (long long)blockIdx.y * rows_per_part, r1 = r0 + rows_per_part < m ? r0 + rows_per_part : m;
  float s = 0.f;
  if (j < n)
    for (long long i = r0 + wave; i < r1; i += 4) {
      float g = (float)dy[i * lddy + j];
      if constexpr (ACT != 0) {
        g *= act_slope<ACT>((float)z[i * n + j]);
        if (dz) dz[i * n + j] = (T)g;
      }
      s += g;
    }
  if (!part) return;
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && j < n) part[(long long)blockIdx.y * n + j] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

template <typename T>
__global__ __launch_bounds__(256) void col_join_kernel(const float* __restrict__ part, int parts, long long n, T* __restrict__ db) {
  const long long j = (long long)blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  double s = 0.0;
  for (int i = 0; i < parts; ++i) s += part[(long long)i * n + j];
  db[j] = (T)(float)s;
}

}  // namespace vdbk
