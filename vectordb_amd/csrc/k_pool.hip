// k_pool.hip — mean pooling of packed token rows to unit vectors, forward and backward.  Memory-bound: each row once.
#include <algorithm>
#include "op_common.h"
#include "ops.h"

namespace vdbk {
namespace {

constexpr float kTiny = 1e-12f;   // the smallest norm a row is divided by

__device__ __forceinline__ float block_sum(float x, float* red) {
  for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
  for (int w = 0; w < (int)(blockDim.x >> 6); ++w) s += red[w];
  return s;
}

// Block: one sequence.  The row's 16-byte pieces (VEC) or values go to neighbouring threads; what is left of the block takes further
// rows at once, whose sums are joined in LDS, in order.  1024 texts of 3 to 128 rows of 768 bf16: 100 MB.
template <typename T, bool VEC, int THREADS>
__global__ __launch_bounds__(THREADS) void mean_pool_kernel(const T* __restrict__ h, long long ld, const int64_t* __restrict__ offsets, long long total,
                                                            int dim, int normalize, float* __restrict__ y, float* __restrict__ inv_norm) {
  constexpr int V = VEC ? Elem<T>::kVec : 1;
  typedef T piece __attribute__((ext_vector_type(V)));
  __shared__ float red[THREADS / 64];
  __shared__ float join[THREADS * V];
  const long long b = blockIdx.x;
  const long long r0 = seq_edge(offsets, b, total);
  long long r1 = seq_edge(offsets, b + 1, total);
  if (r1 < r0) r1 = r0;
  const int rows = (int)(r1 - r0);
  const float f = rows ? 1.f / (float)rows : 0.f;
  const int pieces = dim / V;
  y += b * dim;
  float sq = 0.f;
  for (int p0 = 0; p0 < pieces; p0 += THREADS) {
    const int n = pieces - p0 < THREADS ? pieces - p0 : THREADS, groups = THREADS / n, group = threadIdx.x / n, c = p0 + threadIdx.x % n;
    float s[V] = {};
    if (group < groups) {
      const T* at = h + (r0 + group) * ld + (long long)c * V;
      const long long step = groups * ld;
      int r = group;
      for (; r + 3 * groups < rows; r += 4 * groups, at += 4 * step) {
        const piece x0 = *(const piece*)at, x1 = *(const piece*)(at + step), x2 = *(const piece*)(at + 2 * step), x3 = *(const piece*)(at + 3 * step);
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += ((float)x0[e] + (float)x1[e]) + ((float)x2[e] + (float)x3[e]);
      }
      for (; r < rows; r += groups, at += step) {
        const piece x0 = *(const piece*)at;
#pragma unroll
        for (int e = 0; e < V; ++e) s[e] += (float)x0[e];
      }
    }
    if (groups > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < V; ++e) join[e * THREADS + threadIdx.x] = s[e];
      __syncthreads();
    }
    if (group == 0) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        for (int k = 1; k < groups; ++k) s[e] += join[e * THREADS + k * n + threadIdx.x];
        s[e] *= f;
        y[(long long)c * V + e] = s[e];
        sq += s[e] * s[e];
      }
    }
  }
  if (!normalize) return;
  const float norm = sqrtf(block_sum(sq, red)), inv = 1.f / (norm < kTiny ? kTiny : norm);      // NaN stays: the vector's, and the gradient's
  for (int p0 = 0; p0 < pieces; p0 += THREADS) {       // the values that this thread wrote
    const int n = pieces - p0 < THREADS ? pieces - p0 : THREADS, c = p0 + threadIdx.x;
    if ((int)threadIdx.x < n)
#pragma unroll
      for (int e = 0; e < V; ++e) y[(long long)c * V + e] *= inv;
  }
  if (inv_norm && threadIdx.x == 0) inv_norm[b] = inv;
}

// block: 32 rows of one sequence.  With y = m / |m|: dm = (dy - y (y.dy)) / |m|; below the smallest norm y = m / 1e-12 and
// dm = dy / 1e-12.  Each row gets dm / len.
template <typename T>
__global__ __launch_bounds__(256) void mean_pool_backward_kernel(const float* __restrict__ dy, const float* __restrict__ y, const float* __restrict__ inv_norm,
                                                                 const int64_t* __restrict__ offsets, long long n_seqs, long long total, long long dim,
                                                                 int normalize, T* __restrict__ dh) {
  __shared__ float red[4];
  const Slot s = find_slot(offsets, n_seqs, total, 32, blockIdx.x);
  if (s.b < 0) return;
  const long long r0 = s.begin + (long long)s.tile * 32, r1 = r0 + 32 < s.end ? r0 + 32 : s.end;
  if (s.b == n_seqs) {
    for (long long t = threadIdx.x; t < (r1 - r0) * dim; t += 256) dh[r0 * dim + t] = (T)0.f;
    return;
  }
  dy += s.b * dim;
  y += s.b * dim;
  float inv = 1.f, dot = 0.f;
  if (normalize) {
    inv = inv_norm[s.b];
    float x = 0.f;
    for (long long c = threadIdx.x; c < dim; c += 256) x += dy[c] * y[c];
    x = block_sum(x, red);
    if (inv < 1.f / kTiny) dot = x;
  }
  const float f = inv / (float)(s.end - s.begin);
  for (long long c = threadIdx.x; c < dim; c += 256) {
    const T g = (T)((dy[c] - (dot != 0.f ? y[c] * dot : 0.f)) * f);
    for (long long r = r0; r < r1; ++r) dh[r * dim + c] = g;
  }
}

template <typename T>
hipError_t pool(const PoolArgs& a) {
  const bool vec = ((uintptr_t)a.hidden & 15) == 0 && a.dim % Elem<T>::kVec == 0 && a.ld % Elem<T>::kVec == 0;
  // few texts: more threads a text, for more rows under way
  auto go = [&](auto kernel, int threads) {
    kernel<<<(unsigned)a.n_seqs, threads, 0, a.st>>>((const T*)a.hidden, a.ld, a.offsets, a.total, (int)a.dim, a.normalize, a.y, a.inv_norm);
  };
  if (a.n_seqs < 512) vec ? go(mean_pool_kernel<T, true, 1024>, 1024) : go(mean_pool_kernel<T, false, 1024>, 1024);
  else vec ? go(mean_pool_kernel<T, true, 256>, 256) : go(mean_pool_kernel<T, false, 256>, 256);
  return hipGetLastError();
}
template <typename T>
hipError_t pool_backward(const PoolArgs& a) {
  mean_pool_backward_kernel<T><<<(unsigned)n_slots(a.total, a.n_seqs, 32), 256, 0, a.st>>>(a.dy, a.y, a.inv_norm, a.offsets, a.n_seqs, a.total, a.dim,
                                                                                          a.normalize, (T*)a.dhidden);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mean_pool(int dtype, const PoolArgs& a) {
  return dtype == 0 ? pool<float>(a) : dtype == 1 ? pool<__bf16>(a) : pool<_Float16>(a);
}
hipError_t launch_mean_pool_backward(int dtype, const PoolArgs& a) {
  return dtype == 0 ? pool_backward<float>(a) : dtype == 1 ? pool_backward<__bf16>(a) : pool_backward<_Float16>(a);
}

}  // namespace vdbk
