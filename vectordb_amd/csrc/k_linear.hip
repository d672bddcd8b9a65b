// k_linear.hip — launches of the linear layer's products, forward and backward.
#include <algorithm>
#include "op_gemm.h"
#include "ops.h"

namespace vdbk {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// A contraction is split over blocks when the output alone would leave most compute units idle and each part still is
// long enough to pay for writing and joining its fp32 outputs.
int split_count(int64_t m, int64_t n, int64_t k) {
  const int64_t tiles = std::max<int64_t>(1, cdiv(m, 128) * cdiv(n, 128));
  if (tiles >= 128) return 1;
  return (int)std::max<int64_t>(1, std::min<int64_t>({512 / tiles, k / 512, 64}));
}

template <typename T, bool AT, bool BT, int ACT>
hipError_t launch_any(const GemmArgs& a, GemmParams p) {
  const int splits = split_count(a.m, a.n, a.k);
  const int64_t step = 8 * Elem<T>::kVec;
  p.k_split = std::max(step, cdiv(cdiv(a.k, splits), step) * step);
  const int parts = (int)std::max<int64_t>(1, cdiv(a.k, p.k_split));
  const bool split = parts > 1 && a.partial_bytes >= (int64_t)parts * a.m * a.n * 4;
  const bool big = a.m > 64 && a.n > 64;
  const int64_t bm = big ? 128 : 64;
  const dim3 grid((unsigned)cdiv(a.m, bm), (unsigned)cdiv(a.n, bm), split ? parts : 1);
  if (split) {
    if (big) gemm_any_kernel<T, AT, BT, 0, true, 128><<<grid, 256, 0, a.st>>>(p);
    else gemm_any_kernel<T, AT, BT, 0, true, 64><<<grid, 256, 0, a.st>>>(p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    gemm_join_kernel<T, ACT><<<(unsigned)std::min<int64_t>(cdiv(a.m * a.n, 256), 4096), 256, 0, a.st>>>(p, parts);
  } else if (big) {
    gemm_any_kernel<T, AT, BT, ACT, false, 128><<<grid, 256, 0, a.st>>>(p);
  } else {
    gemm_any_kernel<T, AT, BT, ACT, false, 64><<<grid, 256, 0, a.st>>>(p);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(const GemmArgs& a) {
  GemmParams p{};
  p.a = a.a; p.lda = a.lda; p.b = a.b; p.ldb = a.ldb; p.m = a.m; p.n = a.n; p.k = a.k;
  p.y = a.y; p.ldy = a.ldy; p.bias = a.bias; p.residual = a.residual; p.ldr = a.ldr; p.z = a.z; p.partial = a.partial;
  auto aligned = [](const void* q, int64_t ld) { return ((uintptr_t)q & 15) == 0 && ld % Elem<T>::kVec == 0; };
  p.vec_a = aligned(a.a, a.lda); p.vec_b = aligned(a.b, a.ldb);
  if (a.a_t) return launch_any<T, true, true, 0>(a, p);     // weight gradient
  if (a.b_t) return launch_any<T, false, true, 0>(a, p);    // input gradient
  switch (a.act) {
    case 1: return launch_any<T, false, false, 1>(a, p);
    case 2: return launch_any<T, false, false, 2>(a, p);
    case 3: return launch_any<T, false, false, 3>(a, p);
    default: return launch_any<T, false, false, 0>(a, p);
  }
}

template <typename T, int ACT>
hipError_t act_grad(const ActGradArgs& a) {
  const int parts = act_grad_parts(a.m, a.n);
  const int64_t rows = cdiv(a.m, parts);
  const dim3 grid((unsigned)cdiv(a.n, 64), (unsigned)parts);
  act_grad_kernel<T, ACT><<<grid, 256, 0, a.st>>>((const T*)a.dy, a.lddy, (const T*)a.z, (T*)a.dz, a.db ? a.partial : nullptr, a.m, a.n, rows);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.db) return e;
  col_join_kernel<T><<<(unsigned)cdiv(a.n, 256), 256, 0, a.st>>>(a.partial, parts, a.n, (T*)a.db);
  return hipGetLastError();
}

template <typename T>
hipError_t act_grad_t(const ActGradArgs& a) {
  switch (a.act) {
    case 1: return act_grad<T, 1>(a);
    case 2: return act_grad<T, 2>(a);
    case 3: return act_grad<T, 3>(a);
    default: return act_grad<T, 0>(a);
  }
}

}  // namespace

int64_t gemm_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k) {
  (void)dtype;
  const int s = split_count(m, n, k);
  return s > 1 ? (int64_t)s * m * n * 4 : 0;
}

hipError_t launch_gemm(int dtype, const GemmArgs& a) {
  return dtype == 0 ? launch_t<float>(a) : dtype == 1 ? launch_t<__bf16>(a) : launch_t<_Float16>(a);
}

int act_grad_parts(int64_t m, int64_t n) {
  const int64_t cols = cdiv(n, 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(m, 16), cdiv(2048, cols), 512}));
}

hipError_t launch_act_grad(int dtype, const ActGradArgs& a) {
  return dtype == 0 ? act_grad_t<float>(a) : dtype == 1 ? act_grad_t<__bf16>(a) : act_grad_t<_Float16>(a);
}

}  // namespace vdbk
