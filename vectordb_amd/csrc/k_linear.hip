// k_linear.hip — launches of the linear layer's products, forward and backward.
#include <algorithm>
#include "op_gemm.h"
#include "ops.h"

namespace vdbk {
namespace {

int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Which kernel serves a product: one rule on sizes and alignment, for the launch and for the size of its scratch.
//   any    a row or a width that is no whole number of 16-byte pieces;
//   few    (forward) fewer than 64 tiles of 64 x 64: there a block a tile leaves most of the chip idle.  200 x 768 from 768 in
//          bf16: 48 tiles 7.0 us, few 5.1; 14 x 2304: 36 tiles 6.6, few 4.6; but 480 x 768: 96 tiles 6.6, few 9.6;
//   64     64 x 64 tiles: fp32, bound by its matrix rate, where the smaller tiles fill the chip evenly (next line), and 16-bit
//          products with fewer than 160 tiles of 128 x 128 (1000 x 776 from 776: 7.6 us against 10.2);
//   96     fp32, 96 x 64 tiles where they spread more evenly: the time goes by the fullest compute unit.  64 x 64 gives some units
//          five tiles where the mean is 4.5, 96 x 64 gives each three: 6144 x 768 from 768 61 us, 64 x 64 69, 128 x 64 80;
//          6144 x 768 from 2048 149 and 172; 1536 x 1024 from 1024 34 and 40; 1999 x 640 from 640 24 and 28;
//   128    up to 512 tiles of 256 x 256 (8192 x 1536 from 768: 25 us; 256 x 256 25.6, 64 x 64 31);
//   256    from there on, forward only: L2 to LDS moves 14.5 TB/s over the chip, which 128 x 128 tiles of 16-bit values need in full
//          (49152 x 2304 from 768: 184 us against 187; 8192 x 8192 from 8192: 907 us against 1192).
// 16-bit blocks stay and walk over tiles (128 x 128: 212 us against 226 with a block a tile); fp32 ones do not (49152 x 768 from 768:
// 454 us against 513).
// A contraction is split over blocks when the output alone would leave compute units idle: for weight gradients, whose contraction is
// the batch (1536 x 768 from 8192 tokens: 30 us and 9 to join, unsplit 64), for less than 64 tiles (fp32, whose steps take longer, 128:
// 480 x 768 from 768 17 us, whole 20), and for long contractions on less than 256 (1000 x 768 from 2304: fp32 41 us, whole 53; bf16
// 18 and 20); each part is at least eight steps long.  Elsewhere joining costs what the shorter parts save (1536 x 1024 from 1024
// in bf16 in two parts: 20 us, whole 10; 1000 x 776 from 776 in fp32: 26, whole 21).
enum Kernel { kAny, kFew, k64, k96, k128, k256 };
struct Plan { Kernel kernel; int parts; int64_t k_split; };

Plan plan_of(int dtype, bool a_t, bool b_t, bool whole, int64_t m, int64_t n, int64_t k) {
  const int64_t step = dtype == 0 ? 32 : 64;
  Plan p{kAny, 1, std::max<int64_t>(k, 1)};
  auto tiles = [&](int64_t s) { return cdiv(m, s) * cdiv(n, s); };
  const int64_t t128 = std::max<int64_t>(1, tiles(128)), t64 = std::max<int64_t>(1, tiles(64));
  if (whole && k > 0) {
    if (!a_t && !b_t && t64 < 64) { p.kernel = kFew; return p; }
    if (!a_t && !b_t && dtype != 0 && tiles(256) >= 512) { p.kernel = k256; return p; }
  }
  const bool may_split = a_t || t64 < (dtype == 0 ? 128 : 64) || (k >= 2048 && t64 < 256);
  const int64_t parts128 = may_split ? std::min<int64_t>({512 / t128, k / (8 * step), 64}) : 1;
  const int64_t parts64 = may_split ? std::min<int64_t>({1024 / t64, k / (8 * step), 64}) : 1;
  int64_t parts;
  if (whole && k > 0) {
    p.kernel = dtype != 0 && t128 * std::max<int64_t>(1, parts128) >= 160 ? k128 : k64;
    parts = p.kernel == k128 ? (t128 >= 256 ? 1 : parts128) : (t64 >= 512 ? 1 : parts64);
    if (dtype == 0 && !a_t && parts <= 1 && cdiv(cdiv(m, 96) * cdiv(n, 64), 256) * 96 < cdiv(t64, 256) * 64) p.kernel = k96;
  } else {
    parts = t128 >= 128 ? 1 : parts128;
  }
  if (parts > 1) {
    p.k_split = cdiv(cdiv(k, parts), step) * step;
    p.parts = (int)cdiv(k, p.k_split);
  }
  return p;
}

template <typename T, bool AT, bool BT, int ACT, bool SPLIT, int BM, int BN, int WGI, int WGJ, int MINW>
void tile(const GemmArgs& a, const GemmParams& p, int parts, int64_t resident) {
  const int64_t ti = cdiv(a.m, BM), tj = cdiv(a.n, BN);
  const dim3 grid((unsigned)(SPLIT ? ti * tj : std::min({ti * tj, resident, (int64_t)1 << 22})), (unsigned)parts);
  gemm_tile_kernel<T, AT, BT, ACT, SPLIT, BM, BN, WGI, WGJ, MINW><<<grid, WGI * WGJ * 64, 0, a.st>>>(p, (int)ti, (int)tj);
}

template <typename T, bool AT, bool BT, int ACT>
hipError_t launch_with(const GemmArgs& a, GemmParams p, const Plan& plan) {
  const bool split = plan.parts > 1;
  switch (plan.kernel) {
    case kFew:
      if constexpr (!AT && !BT) {
        const unsigned cols = (unsigned)cdiv(a.n, 16);
        if (a.m <= 16) gemm_few_kernel<T, ACT, 1><<<dim3(cols, 1), 512, 0, a.st>>>(p);
        else if (a.m <= 32) gemm_few_kernel<T, ACT, 2><<<dim3(cols, 1), 512, 0, a.st>>>(p);
        else gemm_few_kernel<T, ACT, 4><<<dim3(cols, (unsigned)cdiv(a.m, 64)), 512, 0, a.st>>>(p);
      }
      return hipGetLastError();
    case k64: {
      const int64_t ti64 = cdiv(a.m, 64) * cdiv(a.n, 64);
      if (split) tile<T, AT, BT, 0, true, 64, 64, 2, 2, 4>(a, p, plan.parts, 0);
      else tile<T, AT, BT, ACT, false, 64, 64, 2, 2, 4>(a, p, 1, sizeof(T) == 4 ? ti64 : 1024);
      break;
    }
    case k96:
      if constexpr (sizeof(T) == 4 && !AT) tile<T, AT, BT, ACT, false, 96, 64, 2, 2, 4>(a, p, 1, cdiv(a.m, 96) * cdiv(a.n, 64));
      break;
    case k128:
      if constexpr (sizeof(T) == 2) {
        if (split) tile<T, AT, BT, 0, true, 128, 128, 4, 2, 4>(a, p, plan.parts, 0);
        else tile<T, AT, BT, ACT, false, 128, 128, 4, 2, 4>(a, p, 1, 512);
      }
      break;
    case k256:
      if constexpr (sizeof(T) == 2 && !AT && !BT) tile<T, AT, BT, ACT, false, 256, 256, 2, 4, 2>(a, p, 1, 256);
      break;
    case kAny: {
      const bool big = a.m > 64 && a.n > 64;
      const int64_t bm = big ? 128 : 64;
      const dim3 grid((unsigned)cdiv(a.m, bm), (unsigned)cdiv(a.n, bm), plan.parts);
      if (split) {
        if (big) gemm_any_kernel<T, AT, BT, 0, true, 128><<<grid, 256, 0, a.st>>>(p);
        else gemm_any_kernel<T, AT, BT, 0, true, 64><<<grid, 256, 0, a.st>>>(p);
      } else if (big) {
        gemm_any_kernel<T, AT, BT, ACT, false, 128><<<grid, 256, 0, a.st>>>(p);
      } else {
        gemm_any_kernel<T, AT, BT, ACT, false, 64><<<grid, 256, 0, a.st>>>(p);
      }
      break;
    }
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !split) return e;
  gemm_join_kernel<T, ACT><<<(unsigned)std::min<int64_t>(cdiv(a.m * a.n, 256), 4096), 256, 0, a.st>>>(p, plan.parts);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_t(int dtype, const GemmArgs& a) {
  constexpr int64_t V = Elem<T>::kVec;
  GemmParams p{};
  p.a = a.a; p.lda = a.lda; p.b = a.b; p.ldb = a.ldb; p.m = a.m; p.n = a.n; p.k = a.k;
  p.y = a.y; p.ldy = a.ldy; p.bias = a.bias; p.residual = a.residual; p.ldr = a.ldr; p.z = a.z; p.partial = a.partial;
  auto at = [](const void* q, uintptr_t bytes) { return ((uintptr_t)q & (bytes - 1)) == 0; };
  p.vec_a = at(a.a, 16) && a.lda % V == 0;
  p.vec_b = at(a.b, 16) && a.ldb % V == 0;
  const uintptr_t four = 4 * sizeof(T);
  p.vec_y = a.n % 4 == 0 && a.ldy % 4 == 0 && at(a.y, four) && at(a.z, four) && at(a.bias, four) && at(a.partial, 16) &&
            (!a.residual || (a.ldr % 4 == 0 && at(a.residual, four)));
  if (p.vec_y && a.n % 8 == 0 && a.ldy % 8 == 0 && at(a.y, 16) && at(a.z, 16)) p.vec_y = 2;
  p.stream = a.m * a.n * (int64_t)sizeof(T) > (32 << 20);
  // whole pieces along each operand's dense dimension, and tile offsets that fit 32 bits
  const int64_t far = (int64_t)1 << 31;
  const bool whole = p.vec_a && p.vec_b && (a.a_t ? a.m : a.k) % V == 0 && (a.b_t ? a.n : a.k) % V == 0 &&
                     a.lda < far / 1024 && a.ldb < far / 1024;
  const Plan plan = plan_of(dtype, a.a_t, a.b_t, whole, a.m, a.n, a.k);
  p.k_split = plan.k_split;
  if (plan.parts > 1 && a.partial_bytes < (int64_t)plan.parts * a.m * a.n * 4) return hipErrorInvalidValue;
  if (a.a_t) return launch_with<T, true, true, 0>(a, p, plan);     // weight gradient
  if (a.b_t) return launch_with<T, false, true, 0>(a, p, plan);    // input gradient
  switch (a.act) {
    case 1: return launch_with<T, false, false, 1>(a, p, plan);
    case 2: return launch_with<T, false, false, 2>(a, p, plan);
    case 3: return launch_with<T, false, false, 3>(a, p, plan);
    default: return launch_with<T, false, false, 0>(a, p, plan);
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
  col_join_kernel<T><<<(unsigned)cdiv(a.n, 32), 256, 0, a.st>>>(a.partial, parts, a.n, (T*)a.db);
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

int64_t gemm_workspace_bytes(int dtype, bool a_t, bool b_t, int64_t m, int64_t n, int64_t k) {
  // alignment is not known here: room for either choice
  const int p = plan_of(dtype, a_t, b_t, true, m, n, k).parts, q = plan_of(dtype, a_t, b_t, false, m, n, k).parts;
  const int parts = std::max(p, q);
  return parts > 1 ? (int64_t)parts * m * n * 4 : 0;
}

hipError_t launch_gemm(int dtype, const GemmArgs& a) {
  return dtype == 0 ? launch_t<float>(dtype, a) : dtype == 1 ? launch_t<__bf16>(dtype, a) : launch_t<_Float16>(dtype, a);
}

int act_grad_parts(int64_t m, int64_t n) {
  const int64_t cols = cdiv(n, 64);
  return (int)std::max<int64_t>(1, std::min<int64_t>({cdiv(m, 16), cdiv(2048, cols), 512}));
}

hipError_t launch_act_grad(int dtype, const ActGradArgs& a) {
  return dtype == 0 ? act_grad_t<float>(a) : dtype == 1 ? act_grad_t<__bf16>(a) : act_grad_t<_Float16>(a);
}

}  // namespace vdbk
