// op_common.h — what the encoder operators' kernels share: the three element types with their matrix instructions
// and roundings, the activations, and the search for a packed sequence.
//
// Matrix-instruction operand layouts used throughout (64 lanes, l = lane):
//   32x32 tiles  A: row l & 31, B: column l & 31, C: column l & 31, rows (r & 3) + 8 (r >> 2) + 4 (l >> 5), r = 0..15
//   16-bit       one instruction contracts 16: lane half l >> 5 holds 8 consecutive values
//   fp32         one instruction contracts 2: lane half l >> 5 holds one value
// The contraction index may be permuted freely as long as A and B agree; the kernels use that to feed one product's
// C registers to the next as an operand without moving them between lanes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#pragma clang diagnostic ignored "-Winline-asm"   // m0 on a clobber list (it is reserved; nothing else in these kernels uses it)

namespace vdbk {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x2 __attribute__((ext_vector_type(2)));

// kVec: elements in 16 bytes; Frag: what one lane holds of an operand for kDepth = 2 kVec contracted values.
template <typename T> struct Elem;
template <> struct Elem<float> {
  static constexpr int kVec = 4;
  typedef f32x4 vec;
  // eight contracted values as four instructions: half 0 holds values 0..3, half 1 values 4..7
  static __device__ __forceinline__ void mma(vec a, vec b, f32x16& c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
  }
};
template <> struct Elem<__bf16> {
  static constexpr int kVec = 8;
  typedef bf16x8 vec;
  static __device__ __forceinline__ void mma(vec a, vec b, f32x16& c) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<_Float16> {
  static constexpr int kVec = 8;
  typedef f16x8 vec;
  static __device__ __forceinline__ void mma(vec a, vec b, f32x16& c) { c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

constexpr float kLog2e = 1.4426950408889634f;

// ---- direct loads to LDS ------------------------------------------------------------------------------------------
// 64 lanes x 16 bytes from sbase + voff to LDS lds_dst + 16 lane; waited for by hand (the compiler does not see the load).
__device__ __forceinline__ void lds_load16(const void* sbase, unsigned voff, unsigned lds_dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "s"(lds_dst) : "memory", "m0");
}
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory"); }

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// ---- activations and their slopes, fp32 -----------------------------------------------------------------------
// The normal distribution's integral Phi(z), and exp(-z^2 / 2).  fp32 operands: erff.  16-bit operands: Abramowitz and Stegun's
// rational form 7.1.26 of erf (error at most 1.5e-7, a hundredth of half a bf16 or a five-hundredth of half an fp16 step of 1), about
// twelve instructions: with erff inlined the epilogue of a 128 x 128 tile spilled 97 registers.
template <typename T> __device__ __forceinline__ float normal_cdf(float z, float& bell) {
  bell = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
  if constexpr (sizeof(T) == 4) return 0.5f * (1.f + erff(z * 0.70710678118654752f));
  const float t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * 0.70710678118654752f * fabsf(z));
  const float tail = 0.5f * bell * t * (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
  return z < 0.f ? tail : 1.f - tail;
}
template <typename T, int ACT> __device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == 1) { float bell; return z * normal_cdf<T>(z, bell); }
  if constexpr (ACT == 2) {   // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
    const float u = 0.79788456080286536f * (z + 0.044715f * z * z * z);
    const float d = 1.f + __expf(-2.f * u);
    return sizeof(T) == 4 ? z / d : z * __builtin_amdgcn_rcpf(d);
  }
  if constexpr (ACT == 3) return z > 0.f ? z : (z != z ? z : 0.f);
  return z;
}
template <typename T, int ACT> __device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == 1) {
    float bell;
    const float cdf = normal_cdf<T>(z, bell);
    return cdf + (bell == 0.f ? 0.f : z * 0.3989422804014327f * bell);   // a kept sum of -inf: 0 * inf stays out
  }
  if constexpr (ACT == 2) {
    const float c = 0.79788456080286536f, u = c * (z + 0.044715f * z * z * z);
    const float s = 1.f / (1.f + __expf(-2.f * u));   // (1 + tanh u) / 2; its derivative by u is 2 s (1 - s)
    // a z whose square overflows has s (1 - s) = 0: keep 0 * inf out
    const float t = s * (1.f - s);
    return s + (t == 0.f ? 0.f : z * 2.f * t * c * (1.f + 3.f * 0.044715f * z * z));
  }
  if constexpr (ACT == 3) return z > 0.f ? 1.f : 0.f;
  return 1.f;
}

// ---- packed sequences --------------------------------------------------------------------------------------------
// Sequence b's rows, whatever the device memory holds: inside [0, total], never of negative length.
__device__ __forceinline__ long long seq_edge(const int64_t* offsets, long long b, long long total) {
  if (b == 0) return 0;
  const long long o = offsets[b];
  return o < 0 ? 0 : o > total ? total : o;
}

// Work slots over packed sequences, without a list made on the host: sequence b's tiles of `tile` rows take the slots
// from floor(begin_b / tile) + b on.  ceil(len / tile) <= floor(end / tile) - floor(begin / tile) + 1, so the slots of
// two sequences never meet; n_slots = floor(total / tile) + n_seqs + 1 covers every sequence and, as one more, the rows
// behind the last (b = n_seqs).  One wave finds the sequence of a slot with a 64-way search: two rounds for 4096 texts.
struct Slot { long long begin, end; long long b; int tile; };   // tile: index of the tile inside the sequence; b = -1: none
__host__ __device__ __forceinline__ long long n_slots(long long total, long long n_seqs, int tile) { return total / tile + n_seqs + 1; }

__device__ __forceinline__ Slot find_slot(const int64_t* __restrict__ offsets, long long n_seqs, long long total, int tile, long long slot) {
  const int lane = threadIdx.x & 63;
  // the largest b in [0, n_seqs] with floor(begin_b / tile) + b <= slot; lo always satisfies it (b = 0 has slot 0)
  long long lo = 0, hi = n_seqs + 1;   // answer in [lo, hi)
  int edge = 0, last = 0;              // lane's edge of the last round, and the lane of the answer: total is below 2^31
  bool near = false;                   // the lane behind it holds the answer's end
  while (hi - lo > 1) {
    const long long step = (hi - lo + 63) >> 6;
    const long long b = lo + (long long)lane * step;
    edge = b < hi ? (int)seq_edge(offsets, b, total) : 0;
    const bool ok = b < hi && (b == lo || edge / tile + b <= slot);
    const unsigned long long m = __ballot(ok);
    // contents may be unordered: take the leading run of lanes that hold, which lane 0 always does
    last = m == ~0ull ? 63 : __builtin_ctzll(~m) - 1;
    near = step == 1 && last < 63 && lo + last + 1 < hi;
    lo += (long long)last * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  Slot s;
  s.b = lo;
  if (near) {                          // one dependent load less
    s.begin = __builtin_amdgcn_readlane(edge, last);
    s.end = __builtin_amdgcn_readlane(edge, last + 1);
  } else {
    s.begin = seq_edge(offsets, lo, total);
    s.end = lo == n_seqs ? total : seq_edge(offsets, lo + 1, total);
  }
  if (s.end < s.begin) s.end = s.begin;
  const long long t = slot - (s.begin / tile + lo);
  if (t < 0 || t * tile >= s.end - s.begin) { s.b = -1; s.tile = 0; } else s.tile = (int)t;
  return s;
}

}  // namespace vdbk
