// op_attn.h — self-attention over packed sequences with a learned relative position bias, forward and backward.
//
//   s_ij = scale q_i.k_j + table[bucket(j - i)][h],  p = softmax_j(s),  o_i = sum_j p_ij v_j
//   ds = p (do v^T - rowsum(do o));  dq = scale ds k,  dk = scale ds^T q,  dv = p^T do,  dtable = bucket sums of ds
//
// The bias depends on j - i alone and is constant beyond the last bucket's first distance R, so a block keeps ONE line of
// 2R + 1 values for its head in LDS (log2 units) instead of any [len][len] matrix; a 32x32 tile wholly beyond R needs no
// look-up at all.  Softmax runs in base 2 with a running maximum and sum, both fp32.
//
// Every product is arranged so that its C registers are the next product's operand (op_common.h): the forward pass and dq
// compute s^T with the keys in the registers and one query per lane, dk / dv compute s with the queries in the registers.
#pragma once
#include "attn_lines.h"
#include "op_common.h"
#include "ops.h"

namespace vdbk {

struct AttnParams {
  const void *q, *k, *v; long long ld_t, ld_h;
  const void* table; int n_buckets;
  const int64_t* offsets; long long n_seqs, total;
  int heads, d; float scale;
  void* out; void* rest; float* lse;
  const void* dout; void *dq, *dk, *dv; long long gld_t, gld_h;
  float* delta; float* from; float* fix; const unsigned* peak; float* part;   // peak: [2][heads][n_seqs] largest |dout| and |v| (fp16 only)
  const i32x4* order;   // the tiled backward kernels' places, longest sequences first, or nullptr
  int vec;        // q, k, v, out, dout, gradients: 16-byte rows
  int reach;      // R
  Buckets bk;
};

__device__ __forceinline__ int bucket_of(const Buckets& bk, int e) {
  const int n = e < 0 ? -e : e;
  int b = n;
  if (n >= bk.near) {
    b = bk.near;
    for (int i = 0; i < bk.n_steps; i += 8) {
#pragma unroll
      for (int u = 0; u < 8; ++u) b += n >= bk.step[i + u];     // behind the last: never
    }
  }
  return b + (e > 0 ? bk.half : 0);
}

// The tiled kernels let the bias enter a product that is scaled afterwards, as bias / scale: with a scale far from 1 that quotient leaves
// the 32-bit range (100 / 1e-37) or its normal part, and the bias would be lost.  Then the general kernels serve, which add it behind the
// scaling.
__host__ __device__ __forceinline__ bool even_scale(float s) { return s >= 1e-18f && s <= 1e18f; }
// What the bias b is in such a product, c = scale log2(e).  Finite values stay within what the product with c can hold: a row of the
// type's lowest value has a softmax.  NaN stays.
__device__ __forceinline__ float start_value(float b, float scale, float c) {
  const float most = 3e38f / fmaxf(c, 1.f), x = b / scale;
  return __builtin_isinf(b) ? b : x > most ? most : x < -most ? -most : x;
}

// line[R + e] for |e| <= R: what a tile's sums start from, as in the tiled kernels (scores_any); bias(e) * log2(e) where the scale is not even
template <typename T>
__device__ __forceinline__ void make_line(float* line, const AttnParams& p, int head) {
  const float c = p.scale * kLog2e;
  for (int t = threadIdx.x; t <= 2 * p.reach; t += blockDim.x) {
    const float b = (float)((const T*)p.table)[(long long)bucket_of(p.bk, t - p.reach) * p.heads + head];
    float x = b * kLog2e;
    if (__builtin_isinf(x) && !__builtin_isinf(b)) x = b < 0.f ? -3.4028234e38f : 3.4028234e38f;
    line[t] = even_scale(p.scale) ? start_value(b, p.scale, c) : x;
  }
}

// Rows whose scores lie beyond 2^10 (all of a row's biases are some mask's great number) take a slower, exact way through exp2(s - m):
// - s is rounded before m is taken away.  Fused, scale x - m keeps the product's exact tail, and half a step of a number like 1e38 is far
//   beyond any exponent.
// - The kept lse = m + log2(sum) has no room for log2(sum) there (at the type's lowest value p would be 1 instead of 1 / len): the backward
//   pass takes such rows' greatest score and sum once more, and keeps the two apart (`from` and `fix`, which is never 0; lse and 0 for other rows).  Both from
//   its own scores, so that no other kernel's rounding of numbers like 1e12 enters.
// The tiled kernels do so in a branch ahead of the exponentials that turns a tile's x into (s - m) / c, so that what every tile runs
// through stays as it is: with a second form of the exponentials in the loop, 16 x 384 tokens in fp32 took 107 us instead of 85.
__device__ __forceinline__ bool is_great(float x) { return fabsf(x) > 1024.f && fabsf(x) < INFINITY; }

// A row's greatest score and log2 of its sum of exp2(s - greatest), one s after the other; half a row a lane
struct RowSum {
  float top = -INFINITY, sum = 0.f;
  __device__ __forceinline__ void add(float s) {
    if (s > top) { sum = sum * __builtin_amdgcn_exp2f(top - s) + 1.f; top = s; }
    else if (s != -INFINITY) sum += __builtin_amdgcn_exp2f(s - top);       // NaN stays
  }
  __device__ __forceinline__ void join() {
    const float top2 = __shfl_xor(top, 32, 64), sum2 = __shfl_xor(sum, 32, 64), m = fmaxf(top, top2);
    sum = (sum == 0.f ? 0.f : sum * __builtin_amdgcn_exp2f(top - m)) + (sum2 == 0.f ? 0.f : sum2 * __builtin_amdgcn_exp2f(top2 - m));
    top = m;
  }
};

// fp16 operands: p <= 1 would lose bits below 2^-14 and vanish below 2^-25 (beside a key of nearly all the weight, or 1 / len of a text of
// 20 thousand tokens); as 2^15 p it keeps them down to 2^-29.  The sums carry the factor too, dv and ds are freed of it.
template <typename T> constexpr bool kLifted = sizeof(T) == 2 && !__is_same(T, __bf16);
template <typename T> constexpr float kLift = kLifted<T> ? 15.f : 0.f;      // log2
template <typename T> constexpr float kUnlift = kLifted<T> ? 1.f / 32768.f : 1.f;

// ROWS rows of one head into LDS: [ROWS][DP + V], or transposed [DP][ROWS + V]; zeros beyond `valid` rows and d columns.
template <typename T, int DP, int ROWS, bool PLAIN, bool TRANS>
__device__ __forceinline__ void stage_rows(T* s, T* st, const T* g, long long ld, int valid, int d, int vec_ok, int threads) {
  constexpr int V = Elem<T>::kVec;
  using vec = typename Elem<T>::vec;
  for (int t = threadIdx.x; t < ROWS * (DP / V); t += threads) {
    const int r = t / (DP / V), c = (t % (DP / V)) * V;
    T x[V];
    if (vec_ok && r < valid && c + V <= d) {
      *(vec*)x = *(const vec*)(g + r * ld + c);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = r < valid && c + e < d ? g[r * ld + c + e] : (T)0.f;
    }
    if constexpr (PLAIN) *(vec*)&s[r * (DP + V) + c] = *(vec*)x;
    if constexpr (TRANS) {
#pragma unroll
      for (int e = 0; e < V; ++e) st[(c + e) * (ROWS + V) + r] = x[e];
    }
  }
}

// One row's operand registers for contractions over the head dimension: piece s holds columns 2 V s + V half ..
template <typename T, int DP>
__device__ __forceinline__ void load_row_frags(typename Elem<T>::vec (&f)[DP / (2 * Elem<T>::kVec)], const T* row, bool there, int d, int vec_ok) {
  constexpr int V = Elem<T>::kVec;
  using vec = typename Elem<T>::vec;
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int s = 0; s < DP / (2 * V); ++s) {
    const int c = s * 2 * V + half * V;
    if (vec_ok && there && c + V <= d) f[s] = *(const vec*)(row + c);
    else {
      vec x;
#pragma unroll
      for (int e = 0; e < V; ++e) x[e] = there && c + e < d ? row[c + e] : (T)0.f;
      f[s] = x;
    }
  }
}

// 32 LDS rows (plain layout) times a row operand in registers, added to c: C rows = the LDS rows, C column = the lane's row
template <typename T, int DP>
__device__ __forceinline__ f32x16 rows_times(const T* s, const typename Elem<T>::vec (&f)[DP / (2 * Elem<T>::kVec)], f32x16 c = {}) {
  constexpr int V = Elem<T>::kVec;
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < DP / (2 * V); ++i)
    Elem<T>::mma(*(const typename Elem<T>::vec*)&s[(lane & 31) * (DP + V) + i * 2 * V + (lane >> 5) * V], f[i], c);
  return c;
}

// acc[db] += X^T p for X = 32 rows in LDS, transposed layout [DP][32 + V], and p a 32x32 tile in C registers (rows = X's rows):
// C rows = head dimension db * 32 .., C column = p's column.
template <typename T, int DP>
__device__ __forceinline__ void trans_times(f32x16 (&acc)[DP / 32], const T* st, const f32x16& p) {
  constexpr int V = Elem<T>::kVec, LD = 32 + V;
  using vec = typename Elem<T>::vec;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  if constexpr (V == 4) {
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      vec b = {p[4 * g], p[4 * g + 1], p[4 * g + 2], p[4 * g + 3]};
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) Elem<T>::mma(*(const vec*)&st[(db * 32 + (lane & 31)) * LD + 8 * g + 4 * half], b, acc[db]);
    }
  } else {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      vec b;
#pragma unroll
      for (int e = 0; e < 8; ++e) b[e] = (T)p[8 * g + e];
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) {
        const T* r = &st[(db * 32 + (lane & 31)) * LD + 16 * g + 4 * half];
        vec a;
        *(i32x2*)&a = *(const i32x2*)r;
        *((i32x2*)&a + 1) = *(const i32x2*)(r + 8);
        Elem<T>::mma(a, b, acc[db]);
      }
    }
  }
}

// A scaled sum as it is stored, or (LOW) what that rounding left of it
template <typename T, bool LOW> __device__ __forceinline__ T rounded(float x) {
  const T t = (T)x;
  return LOW ? (T)(x - (float)t) : t;
}

// C registers [DP / 32] with C column = a token row: store columns [0, d) of that row, scaled
template <typename T, int DP, bool LOW = false>
__device__ __forceinline__ void store_cols(T* row, const f32x16 (&acc)[DP / 32], float f, int d, int vec_ok) {
  const int half = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int db = 0; db < DP / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = db * 32 + 8 * g + 4 * half;
      T x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = rounded<T, LOW>(acc[db][4 * g + e] * f);
      if (vec_ok && c + 4 <= d) {
        if constexpr (sizeof(T) == 2) *(i32x2*)(row + c) = *(i32x2*)x; else *(i32x4*)(row + c) = *(i32x4*)x;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (c + e < d) row[c + e] = x[e];
      }
    }
}

template <typename T>
__device__ __forceinline__ void zero_rows(T* base, long long ld, long long first, long long last, int d) {
  const long long n = (last - first) * d;
  for (long long t = threadIdx.x; t < n; t += blockDim.x) base[(first + t / d) * ld + t % d] = (T)0.f;
}

// Scores in log2 units of a 32x32 tile, the LDS rows s against the lane's row f, with the keys in the rows and the lane's query as the
// column, or the other way round; e0 = (first key - first query) of the tile.  The same sums in the same order as in the tiled kernels, which
// may have made the other pass (fp32 heads of 128): the bias is what a tile's sums start from, beyond R it is added behind the product.
template <typename T, int DP, bool KEYS_IN_ROWS>
__device__ __forceinline__ f32x16 scores_any(const T* s, const typename Elem<T>::vec (&f)[DP / (2 * Elem<T>::kVec)], float c, const float* line, int reach, int e0, bool even) {
  const int lane = threadIdx.x & 63;
  f32x16 x;
  if (tile_is_far(e0, reach)) {
    const float b = line[e0 > 0 ? 2 * reach : 0], shift = even ? b * c : b;
    x = rows_times<T, DP>(s, f);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], c, shift);
    return x;
  }
  f32x16 bias;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5), col = lane & 31;
    int e = e0 + (KEYS_IN_ROWS ? row - col : col - row);
    e = e > reach ? reach : e < -reach ? -reach : e;
    bias[r] = line[reach + e];
  }
  if (even) {
    x = rows_times<T, DP>(s, f, bias);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] *= c;
  } else {
    x = rows_times<T, DP>(s, f);
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = __builtin_fmaf(x[r], c, bias[r]);
  }
  return x;
}

// ---- forward, any width, stride and alignment ---------------------------------------------------------------------------
// Block: one slot of NW * 32 queries of one head; each wave 32 queries, one per lane column; key tiles of 32 through LDS.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void attention_any_kernel(const AttnParams p) {
  constexpr int V = Elem<T>::kVec, BQ = NW * 32;
  __shared__ __align__(16) T sk[32 * (DP + V)];
  __shared__ __align__(16) T sv[DP * (32 + V)];
  extern __shared__ float line[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = blockIdx.x % p.heads;
  const Slot s = find_slot(p.offsets, p.n_seqs, p.total, BQ, blockIdx.x / p.heads);
  if (s.b < 0) return;
  const long long hd = (long long)p.heads * p.d;
  if (s.b == p.n_seqs) {
    const long long r0 = s.begin + (long long)s.tile * BQ, r1 = r0 + BQ < s.end ? r0 + BQ : s.end;
    zero_rows((T*)p.out + (long long)head * p.d, hd, r0, r1, p.d);
    return;
  }
  const int len = (int)(s.end - s.begin);
  const int i0 = s.tile * BQ + wave * 32, i = i0 + (lane & 31);
  make_line<T>(line, p, head);
  const T* kb = (const T*)p.k + s.begin * p.ld_t + head * p.ld_h;
  const T* vb = (const T*)p.v + s.begin * p.ld_t + head * p.ld_h;
  typename Elem<T>::vec fq[DP / (2 * V)];
  load_row_frags<T, DP>(fq, (const T*)p.q + (s.begin + i) * p.ld_t + head * p.ld_h, i < len, p.d, p.vec);
  const float c = p.scale * kLog2e;
  const bool even = even_scale(p.scale);
  float m = -INFINITY, l = 0.f;
  f32x16 acc[DP / 32] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    __syncthreads();
    stage_rows<T, DP, 32, true, false>(sk, nullptr, kb + j0 * p.ld_t, p.ld_t, len - j0, p.d, p.vec, NW * 64);
    stage_rows<T, DP, 32, false, true>(nullptr, sv, vb + j0 * p.ld_t, p.ld_t, len - j0, p.d, p.vec, NW * 64);
    __syncthreads();
    if (i0 >= len) continue;
    f32x16 t = scores_any<T, DP, true>(sk, fq, c, line, p.reach, j0 - i0, even);
    if (j0 + 32 > len) {
#pragma unroll
      for (int r = 0; r < 16; ++r) if (j0 + (r & 3) + 8 * (r >> 2) + 4 * (lane >> 5) >= len) t[r] = -INFINITY;
    }
    float top = t[0];
#pragma unroll
    for (int r = 1; r < 16; ++r) top = fmaxf(top, t[r]);
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float m1 = fmaxf(m, top), ms = m1 == -INFINITY ? 0.f : m1;   // a row of -inf alone: p = 0, not NaN
    const float fade = __builtin_amdgcn_exp2f(m - ms);
    l *= fade;
#pragma unroll
    for (int r = 0; r < 16; ++r) { t[r] = __builtin_amdgcn_exp2f(t[r] - ms + kLift<T>); l += t[r]; }
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] *= fade;
    trans_times<T, DP>(acc, sv, t);
    m = m1;
  }
  if (i >= len) return;
  l += __shfl_xor(l, 32, 64);
  const bool left = l > 0.f || l != l;
  if (!left) {                       // nothing is left of the row: zeros, whatever v holds
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) acc[db] = f32x16{};
  }
  const float f = left ? 1.f / l : 0.f;
  store_cols<T, DP>((T*)p.out + (s.begin + i) * hd + (long long)head * p.d, acc, f, p.d, p.vec);
  if (p.rest) store_cols<T, DP, true>((T*)p.rest + (s.begin + i) * hd + (long long)head * p.d, acc, f, p.d, p.vec);
  // +inf where nothing was left of the row: the backward pass' exp2(s - lse) is 0 there
  if (p.lse && lane < 32) p.lse[(long long)head * p.total + s.begin + i] = left ? m + (log2f(l) - kLift<T>) : INFINITY;
}

// ---- whole 16-byte pieces and head widths of 32, 64 and 128 ----------------------------------------------------------------
// Rows of one head in LDS: D values, 16-byte pieces, moved by XOR.  For reads along the row (kRow: 32 rows x 16 bytes at one place)
// the row number spreads the pieces over all banks; for transposed reads (kCol: 4 rows x 64 bytes, or fp32 words of rows 4 apart)
// it moves whole 64- or 128-byte groups.
enum Order { kRow, kCol };
template <typename T, int D, Order O> struct Rows {
  static constexpr int V = Elem<T>::kVec, C = D / V;        // pieces of a row
  using vec = typename Elem<T>::vec;
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (O == kRow) return C >= 16 ? row & 15 : C == 8 ? (row >> 1) & 7 : (row >> 2) & 3;
    else if constexpr (sizeof(T) == 4) return C >= 16 ? (row >> 2 & 1) << 3 : 0;
    else return C >= 16 ? (row & 3) << 2 : C == 8 ? (row >> 1 & 1) << 2 : 0;
  }
  // operand piece i (of D / 2V) for contractions over D: row r0 + lane & 31, r0 a multiple of 32
  static __device__ __forceinline__ vec along(const T* s, int r0, int i) {
    const int lane = threadIdx.x & 63, l = lane & 31;
    return *(const vec*)(s + (r0 + l) * D + (((2 * i + (lane >> 5)) ^ swz(l)) * V));
  }
  // operand for contractions over 4 V rows from r0 in the order of C registers, columns c0 + lane & 31
  static __device__ __forceinline__ vec across(const T* s, int r0, int c0) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    vec x;
    if constexpr (sizeof(T) == 4) {
      const int l = lane & 31;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int row = 4 * half + e;                        // r0 is a multiple of 8
        x[e] = s[(r0 + row) * D + ((((c0 + l) >> 2) ^ swz(row)) << 2) + (l & 3)];
      }
    } else {
      const int i = lane & 15, row = 4 * half + (i >> 2), piece = (c0 >> 3) + ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);   // r0 is a multiple of 16
      const T* at = s + (r0 + row) * D + ((piece ^ swz(row)) << 3) + (i & 1) * 4;
      *(s16x4*)&x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)at);
      *((s16x4*)&x + 1) = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + 8 * D));      // swz(row + 8) = swz(row)
    }
    return x;
  }
  // N rows from g on to LDS by direct loads.  Rows past `left` repeat the last one there is, or (ZEROS) are zeros, written by the lanes
  // that would have loaded them: what is multiplied by a p of 0 there may not be an infinity.
  template <int N, int THREADS, bool ZEROS = false> static __device__ __forceinline__ void load(T* s, const T* g, long long ld, int left) {
    constexpr int kPieces = N * C / THREADS;
    static_assert(N * C % THREADS == 0, "whole turns");
    const unsigned dst = (unsigned)(size_t)(__attribute__((address_space(3))) void*)s + (unsigned)__builtin_amdgcn_readfirstlane((threadIdx.x >> 6) << 10);
    if (ZEROS && left < N) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const int L = i * THREADS + threadIdx.x, row = L / C;
        if (row < left) lds_load16(g, (unsigned)(((unsigned)row * (unsigned)ld + (unsigned)(((L % C) ^ swz(row)) * V)) * (unsigned)sizeof(T)), dst + i * (THREADS * 16));
        else *(i32x4*)((char*)s + L * 16) = i32x4{0, 0, 0, 0};
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int L = i * THREADS + threadIdx.x, row = L / C, r = ZEROS || row < left ? row : left - 1;
      lds_load16(g, (unsigned)(((unsigned)r * (unsigned)ld + (unsigned)(((L % C) ^ swz(row)) * V)) * (unsigned)sizeof(T)), dst + i * (THREADS * 16));
    }
  }
};

// acc[db] (C rows = columns db * 32 .. of D, C column = p's column) += X^T p, X = the 32 LDS rows from r0
template <typename T, int D>
__device__ __forceinline__ void add_across(f32x16 (&acc)[D / 32], const T* s, int r0, const f32x16& p) {
  using vec = typename Elem<T>::vec;
  constexpr int kStep = sizeof(T) == 4 ? 8 : 16;
#pragma unroll
  for (int g = 0; g < 32 / kStep; ++g) {
    vec b;
#pragma unroll
    for (int e = 0; e < kStep / 2; ++e) b[e] = (T)p[g * (kStep / 2) + e];
#pragma unroll
    for (int db = 0; db < D / 32; ++db) Elem<T>::mma(Rows<T, D, kCol>::across(s, r0 + g * kStep, db * 32), b, acc[db]);
  }
}

// line[start_at(R, e)] = bias(e) / scale, |e| <= R + kMargin: the start value of a tile's sums, so that a tile near the diagonal costs a
// look-up a score and no arithmetic.  Only the distances that a text of this length meets are filled in (around: its length and
// a tile; a far tile, which takes its bias from an end of the line, is met only where all of it is).  VOTE: -> whether any thread says so.
template <typename T, bool VOTE = false>
__device__ __forceinline__ bool make_start_line(float* line, const AttnParams& p, int head, float c, int around, bool vote = false) {
  __shared__ float tab[128];
  for (int t = threadIdx.x; t < p.n_buckets; t += blockDim.x) tab[t] = start_value((float)((const T*)p.table)[(long long)t * p.heads + head], p.scale, c);
  if constexpr (VOTE) vote = __builtin_amdgcn_readfirstlane(__syncthreads_or(vote)); else __syncthreads();
  const int middle = start_zero(p.reach), w = around < middle ? around : middle;
  for (int t = middle - w + threadIdx.x; t <= middle + w; t += blockDim.x) line[t] = tab[bucket_of(p.bk, t - middle)];
  return vote;
}

// Waits for what the compiler has loaded into x, here: left to itself it waits where x is used first, inside the loop over tiles, and
// that wait counts the direct loads under way there, which it does not know of.
template <typename X> __device__ __forceinline__ void settle(X& x) { asm volatile("" : "+v"(x)); }

// The block's place: contiguous runs of (head, slot) per XCD, so that the blocks that read one sequence's keys share an L2; inside
// its run an XCD takes the places `hop` apart (a prime that divides no run's length).  Blocks go to compute units in turn, and in
// order the empty slots (one in four where every text has 384 tokens) would all fall to the same units: 16 x 384 tokens, 12 heads,
// fp32, left a quarter of the chip idle.
__device__ __forceinline__ unsigned xcd_run(unsigned n, unsigned hop) {
  const unsigned x = blockIdx.x & 7, q = blockIdx.x >> 3, run = (n >> 3) + (x < (n & 7));
  return x * (n >> 3) + (x < (n & 7) ? x : (n & 7)) + (unsigned)((unsigned long long)q * hop % run);
}

// A 32x32 tile of scores: the LDS rows from r0 against the lane's row f.  Near the diagonal the sums start from the line (start[row]);
// a far tile's start from nothing, without sixteen moves, and its one bias is returned for the caller to add behind the product.
template <typename T, int D, typename ROWS, int SIGN>
__device__ __forceinline__ float scores(f32x16& x, const T* s, int r0, const typename Elem<T>::vec (&f)[D / (2 * Elem<T>::kVec)], int e0, const AttnParams& p,
                                        const float* line, const float* start) {
  constexpr int N = D / (2 * Elem<T>::kVec);
  float shift = 0.f;
  const bool is_far = tile_is_far(e0, p.reach);
  if (__builtin_amdgcn_readfirstlane(is_far)) {
    shift = line[e0 > 0 ? start_span(p.reach) - 1 : 0];
    f32x16 none = {};
    Elem<T>::mma(ROWS::along(s, r0, 0), f[0], none);
    x = none;
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) x[r] = start[SIGN * ((r & 3) + 8 * (r >> 2))];
    Elem<T>::mma(ROWS::along(s, r0, 0), f[0], x);
  }
#pragma unroll
  for (int i = 1; i < N; ++i) Elem<T>::mma(ROWS::along(s, r0, i), f[i], x);
  return shift;
}

// C registers -> D / 32 column blocks of the wave's 32 rows, through LDS of the wave's own, as whole rows
template <typename T, int D, bool LOW = false>
__device__ __forceinline__ void store_turned(T* mine, T* dst, long long ld, const f32x16 (&acc)[D / 32], float f, int rows) {
  using R = Rows<T, D, kRow>;
  typedef T vec4 __attribute__((ext_vector_type(4)));
  const int lane = threadIdx.x & 63, half = lane >> 5, l = lane & 31;
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = db * 32 + 8 * g + 4 * half;
      vec4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = rounded<T, LOW>(acc[db][4 * g + e] * f);
      *(vec4*)(mine + l * D + (((c / R::V) ^ R::swz(l)) * R::V) + (c & (R::V - 1))) = o;
    }
  asm volatile("" ::: "memory");       // a wave's LDS operations keep their order
#pragma unroll
  for (int i = 0; i < 32 * R::C / 64; ++i) {
    const int L = i * 64 + lane, row = L / R::C, c = L % R::C;
    const i32x4 v = *(const i32x4*)(mine + row * D + ((c ^ R::swz(row)) * R::V));
    if (row < rows) *(i32x4*)(dst + row * ld + c * R::V) = v;
  }
  asm volatile("" ::: "memory");
}

// sum += a + b: of the values as the product with v takes them, two by one instruction where there is one
template <typename T> __device__ __forceinline__ void add_pair(float& sum, float a, float b) {
  typedef T pair __attribute__((ext_vector_type(2)));
  if constexpr (__is_same(T, __bf16)) sum = __builtin_amdgcn_fdot2_f32_bf16(pair{(T)a, (T)b}, pair{(T)1.f, (T)1.f}, sum, false);
  else if constexpr (__is_same(T, _Float16)) sum = __builtin_amdgcn_fdot2(pair{(T)a, (T)b}, pair{(T)1.f, (T)1.f}, sum, false);
  else sum += a + b;
}

// Block: one slot of NW * 32 queries of one head, 32 queries a wave, one per lane column; key tiles of 64 (fp32 and blocks of two
// waves: 32, which lets more blocks share a compute unit: 512 texts of 3 to 64 tokens took 20 us, with 64 keys 25), the next one under
// way while one is multiplied.  Per score: one product-and-add, one exponential, half a maximum, one sum, half a conversion; the
// running sums are rescaled only when a maximum has moved.
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, 2) void attention_kernel(const AttnParams p, unsigned slots, unsigned hop) {
  constexpr int BQ = NW * 32, KT = sizeof(T) == 4 || NW == 2 ? 32 : 64, V = Elem<T>::kVec;
  using KR = Rows<T, D, kRow>;
  using VR = Rows<T, D, kCol>;
  __shared__ __align__(1024) T buf[2][2][KT * D];          // [turn][k, v]
  extern __shared__ float line[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l = lane & 31;
  const unsigned at = xcd_run(slots * p.heads, hop);
  const int head = at / slots;
  const Slot s = find_slot(p.offsets, p.n_seqs, p.total, BQ, at % slots);
  if (s.b < 0) return;
  const long long hd = (long long)p.heads * D;
  if (s.b == p.n_seqs) {
    const long long r0 = s.begin + (long long)s.tile * BQ, r1 = r0 + BQ < s.end ? r0 + BQ : s.end;
    zero_rows((T*)p.out + (long long)head * D, hd, r0, r1, D);
    return;
  }
  const int len = (int)(s.end - s.begin), tiles = (len + KT - 1) / KT;
  const int i0 = s.tile * BQ + wave * 32;
  const T* kb = (const T*)p.k + s.begin * p.ld_t + head * p.ld_h;
  const T* vb = (const T*)p.v + s.begin * p.ld_t + head * p.ld_h;
  auto issue = [&](int t) {
    const int left = len - t * KT;
    KR::template load<KT, NW * 64>(buf[t & 1][0], kb + (long long)t * KT * p.ld_t, p.ld_t, left);
    VR::template load<KT, NW * 64, true>(buf[t & 1][1], vb + (long long)t * KT * p.ld_t, p.ld_t, left);
  };
  issue(0);
  typename Elem<T>::vec fq[D / (2 * V)];
  {
    const int i = i0 + l < len ? i0 + l : len - 1;
    const T* q = (const T*)p.q + (s.begin + i) * p.ld_t + head * p.ld_h + half * V;
#pragma unroll
    for (int x = 0; x < D / (2 * V); ++x) fq[x] = *(const typename Elem<T>::vec*)(q + x * 2 * V);
  }
  const float c = p.scale * kLog2e;
  make_start_line<T>(line, p, head, c, len + KT);
  const float* mid = line + start_at(p.reach, 4 * half - l);      // mid[e0 + row] = start value of row (+ 4 half), column l
#pragma unroll
  for (int x = 0; x < D / (2 * V); ++x) settle(fq[x]);
  float m = -INFINITY, base = 0.f, sum = 0.f;
  bool great = false;                  // some row of the wave has a great maximum
  f32x16 acc[D / 32] = {};
  for (int t = 0; t < tiles; ++t) {
    wait_loads<0>();
    __syncthreads();
    if (t + 1 < tiles) issue(t + 1);
    if (i0 >= len) continue;
    const T* sk = buf[t & 1][0];
    const T* sv = buf[t & 1][1];
    const int j0 = t * KT;
    f32x16 x[KT / 32];
    float shift[KT / 32];                // a far tile's bias, added behind the product
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      const int e0 = j0 + u * 32 - i0;
      shift[u] = c * scores<T, D, KR, 1>(x[u], sk, u * 32, fq, e0, p, line, mid + e0);
      if (j0 + u * 32 + 32 > len) {
        if (j0 + u * 32 >= len) shift[u] = 0.f;      // no key there meets a far bias, which may be NaN or infinite
#pragma unroll
        for (int r = 0; r < 16; ++r) if (j0 + u * 32 + (r & 3) + 8 * (r >> 2) + 4 * half >= len) x[u][r] = -INFINITY;
      }
      float high = x[u][0];
#pragma unroll
      for (int r = 1; r < 16; ++r) high = fmaxf(high, x[u][r]);
      top = fmaxf(top, __builtin_fmaf(high, c, shift[u]));
    }
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    if (__any(top > m) || great) {
      const float m1 = fmaxf(m, top), fade = __builtin_amdgcn_exp2f(m - (m1 == -INFINITY ? 0.f : m1));
      m = m1;
      base = m == -INFINITY ? 0.f : m;       // a row of -inf alone: p = 0, not NaN
      sum *= fade;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) acc[db] *= fade;
      great = __any(is_great(m));
      if (__builtin_expect(great, 0)) {
        const float back = 1.f / c;
#pragma unroll
        for (int u = 0; u < KT / 32; ++u) {
#pragma unroll
          for (int r = 0; r < 16; ++r) x[u][r] = (__builtin_fmaf(x[u][r], c, shift[u]) - base + kLift<T>) * back;
          shift[u] = 0.f;
        }
        base = kLift<T>;
      }
    }
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      const float off = shift[u] - base + kLift<T>;
#pragma unroll
      for (int r = 0; r < 16; ++r) x[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[u][r], c, off));
#pragma unroll
      for (int r = 0; r < 16; r += 2) add_pair<T>(sum, x[u][r], x[u][r + 1]);
      add_across<T, D>(acc, sv, u * 32, x[u]);
    }
  }
  __syncthreads();
  if (i0 >= len) return;
  sum += __shfl_xor(sum, 32, 64);
  const bool any = sum > 0.f || sum != sum;
  if (!any) {                        // nothing is left of the row: zeros, whatever v holds
#pragma unroll
    for (int db = 0; db < D / 32; ++db) acc[db] = f32x16{};
  }
  T* mine = &buf[0][0][0] + wave * (32 * D);
  const float f = any ? 1.f / sum : 0.f;
  store_turned<T, D>(mine, (T*)p.out + (s.begin + i0) * hd + (long long)head * D, hd, acc, f, len - i0);
  if (p.rest) store_turned<T, D, true>(mine, (T*)p.rest + (s.begin + i0) * hd + (long long)head * D, hd, acc, f, len - i0);
  if (p.lse && lane < 32 && i0 + l < len) p.lse[(long long)head * p.total + s.begin + i0 + l] = any ? m + (__log2f(sum) - kLift<T>) : INFINITY;
}

// A 32x32 tile's sums by distance, keys in the registers.  Register r's key is row(r) and a lane's query 16 b + c, so shifting the 16
// lanes of a row by s = row & 15 brings distances row - 16 b - c that are alike but for a multiple of 16 to one lane: what stays
// inside belongs to 16 (row >> 4) - 16 b - c, what is pushed out and comes in again at the other end to 16 more.  Two shifted
// additions a register (one instruction each) into three sums; the middle one's halves go to the outer two; and two additions to
// the half's line in LDS, where a lane meets only its own residue of 32 (tiles begin at multiples of 32), so that plain reads and
// writes serve.  64 texts of 16 to 384 tokens, 12 heads: the dq kernel without bucket sums took 49 us, with these 59; with one LDS
// atomic a score it took 296 (an LDS float atomic of a wave holds the LDS about 190 cycles).
template <int CTRL> __device__ __forceinline__ float shifted(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));     // 0 where nothing comes in
}
template <int R> __device__ __forceinline__ void add_shifted(float (&sum)[3], const f32x16& x) {
  if constexpr (R < 16) {
    constexpr int row = (R & 3) + 8 * (R >> 2), k = row >> 4, s = row & 15;
    if constexpr (s == 0) {
      sum[k] += x[R];
    } else {
      sum[k] += shifted<0x100 + s>(x[R]);              // lane c gets lane c + s
      sum[k + 1] += shifted<0x110 + 16 - s>(x[R]);     // lane c gets lane c + s - 16
    }
    add_shifted<R + 1>(sum, x);
  }
}
__device__ __forceinline__ void add_diagonals(float* mine, int reach, int e0, const f32x16& x) {
  const int l = threadIdx.x & 31, half = (threadIdx.x & 63) >> 5;
  float sum[3] = {};
  add_shifted<0>(sum, x);
  const float other = __shfl_xor(sum[1], 16, 64);      // distance 16 - (l ^ 16): -l for l below 16, else 32 - l
  float* at = mine + sums_at(reach, e0, half, l);
  at[0] += sum[0] + (l < 16 ? other : 0.f);
  at[32] += sum[2] + (l < 16 ? 0.f : other);
}

// part[t] = bucket t's sum of the lines hist [lines][span] by distance and of what lies beyond R (far): the lines joined in order,
// then eight lanes per bucket.
__device__ __forceinline__ void fold_buckets(const AttnParams& p, float* hist, const float (*far)[2], int lines, int span, float* part) {
  __syncthreads();
  for (int t = threadIdx.x; t < span; t += blockDim.x) {
    float x = hist[t];
    for (int w = 1; w < lines; ++w) x += hist[w * span + t];
    hist[t] = x;
  }
  __syncthreads();
  const int sub = threadIdx.x & 7, zero = sums_zero(p.reach);
  for (int t = threadIdx.x >> 3; t < ((p.n_buckets + 7) & ~7); t += blockDim.x >> 3) {
    float x = 0.f;
    if (t < p.n_buckets) {
      const int low = t % p.bk.half, side = t / p.bk.half;
      const int n0 = low <= p.bk.near ? low : p.bk.step[low - p.bk.near - 1];
      const int n1 = low + 1 == p.bk.half ? zero : low + 1 <= p.bk.near ? low + 1 : p.bk.step[low - p.bk.near];
      for (int n = (side && n0 == 0 ? 1 : n0) + sub; n < n1; n += 8) x += hist[zero + (side ? n : -n)];
      if (sub == 0 && low + 1 == p.bk.half) for (int w = 0; w < lines / 2; ++w) x += far[w][side];
    }
    for (int k = 1; k < 8; k <<= 1) x += __shfl_xor(x, k, 64);
    if (sub == 0 && t < p.n_buckets) part[t] = x;
  }
}

// ---- backward -------------------------------------------------------------------------------------------------------------
// delta[h][t] = sum_d dout (out + rest) (the general kernels'; attention_dq_kernel has its own); fp16 also the largest |dout| and |v|
// of each sequence and head (bits of non-negative floats order like integers, so the atomic maximum does not depend on the order
// of arrival).
template <typename T, bool PEAK>
__global__ __launch_bounds__(256) void attention_delta_kernel(const AttnParams p, unsigned* peak) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int head = blockIdx.x % p.heads;
  const Slot s = find_slot(p.offsets, p.n_seqs, p.total, 32, blockIdx.x / p.heads);
  if (s.b < 0 || s.b == p.n_seqs) return;
  float po = 0.f, pv = 0.f;
  for (int r = wave; r < 32; r += 4) {
    const long long t = s.begin + (long long)s.tile * 32 + r;
    if (t >= s.end) break;
    const T* o = (const T*)p.out + (t * p.heads + head) * p.d;
    const T* g = (const T*)p.dout + (t * p.heads + head) * p.d;
    const T* v = (const T*)p.v + t * p.ld_t + head * p.ld_h;
    float x = 0.f;
    for (int c = lane; c < p.d; c += 64) {
      x += ((float)o[c] + (p.rest ? (float)((const T*)p.rest)[(t * p.heads + head) * p.d + c] : 0.f)) * (float)g[c];
      if (PEAK) { po = fmaxf(po, fabsf((float)g[c])); pv = fmaxf(pv, fabsf((float)v[c])); }
    }
    for (int k = 32; k; k >>= 1) x += __shfl_xor(x, k, 64);
    if (lane == 0) p.delta[(long long)head * p.total + t] = x;
  }
  if (PEAK) {
    for (int k = 32; k; k >>= 1) { po = fmaxf(po, __shfl_xor(po, k, 64)); pv = fmaxf(pv, __shfl_xor(pv, k, 64)); }
    if (lane == 0) {
      atomicMax(peak + (long long)head * p.n_seqs + s.b, __float_as_uint(po));
      atomicMax(peak + ((long long)p.heads + head) * p.n_seqs + s.b, __float_as_uint(pv));
    }
  }
}

static __global__ void fill_zero_kernel(unsigned* x, long long n) {
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) x[i] = 0;
}

// fp16 has five exponent bits: ds of a long row (p ~ 1 / len) times a small gradient would fall among its subnormals.
// A power of two per sequence and head lifts it: |ds| <= 2 d max|dout| max|v| stays below 2^15.
template <typename T>
__device__ __forceinline__ float ds_lift(const AttnParams& p, int head, long long b) {
  if constexpr (sizeof(T) == 2 && !__is_same(T, __bf16)) {
    const float po = __uint_as_float(p.peak[(long long)head * p.n_seqs + b]), pv = __uint_as_float(p.peak[((long long)p.heads + head) * p.n_seqs + b]);
    const float bound = 2.f * (float)p.d * po * pv;
    if (!(bound > 0.f) || bound > 1e30f || bound < 1e-30f) return 1.f;
    return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(ldexpf(1.f, 14 - ilogbf(bound)))));     // one value a block; waited for here
  } else {
    return 1.f;
  }
}

// dq and the block's part of dtable: like the forward pass, with ds^T in the place of p^T.
// The bucket sums: each half of a wave adds its tile's ds by distance into a line of its own in LDS; tiles beyond R go into two
// registers.  One block's lines are folded into buckets in a fixed order, and the blocks' buckets by attention_dtable_kernel.
template <typename T, int DP, int NW, bool DTABLE>
__global__ __launch_bounds__(NW * 64) void attention_dq_any_kernel(const AttnParams p) {
  constexpr int V = Elem<T>::kVec, BQ = NW * 32;
  __shared__ __align__(16) T sk[32 * (DP + V)];
  __shared__ __align__(16) T skt[DP * (32 + V)];
  __shared__ __align__(16) T sv[32 * (DP + V)];
  __shared__ float far[NW][2];
  extern __shared__ float line[];                      // 2R + 1, then NW * 2 lines of sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int head = blockIdx.x % p.heads;
  const long long slot = blockIdx.x / p.heads;
  const Slot s = find_slot(p.offsets, p.n_seqs, p.total, BQ, slot);
  float* part = p.part + (slot * p.heads + head) * p.n_buckets;
  if (s.b < 0 || s.b == p.n_seqs) {
    if (s.b >= 0) {
      const long long r0 = s.begin + (long long)s.tile * BQ, r1 = r0 + BQ < s.end ? r0 + BQ : s.end;
      zero_rows((T*)p.dq + head * p.gld_h, p.gld_t, r0, r1, p.d);
    }
    if constexpr (DTABLE) for (int t = threadIdx.x; t < p.n_buckets; t += NW * 64) part[t] = 0.f;
    return;
  }
  const int len = (int)(s.end - s.begin);
  const int i0 = s.tile * BQ + wave * 32, i = i0 + (lane & 31);
  const int reach = p.reach, span = sums_span(reach);
  float* hist = line + 2 * reach + 1;
  make_line<T>(line, p, head);
  if constexpr (DTABLE) for (int t = threadIdx.x; t < NW * 2 * span; t += NW * 64) hist[t] = 0.f;
  float* mine = hist + (wave * 2 + half) * span;
  const T* kb = (const T*)p.k + s.begin * p.ld_t + head * p.ld_h;
  const T* vb = (const T*)p.v + s.begin * p.ld_t + head * p.ld_h;
  const long long hd = (long long)p.heads * p.d;
  typename Elem<T>::vec fq[DP / (2 * V)], fg[DP / (2 * V)];
  load_row_frags<T, DP>(fq, (const T*)p.q + (s.begin + i) * p.ld_t + head * p.ld_h, i < len, p.d, p.vec);
  load_row_frags<T, DP>(fg, (const T*)p.dout + (s.begin + i) * hd + (long long)head * p.d, i < len, p.d, p.vec);
  float lse = i < len ? p.lse[(long long)head * p.total + s.begin + i] : INFINITY;
  const float delta = i < len ? p.delta[(long long)head * p.total + s.begin + i] : 0.f;
  const float lift = ds_lift<T>(p, head, s.b);
  const float c = p.scale * kLog2e;
  const bool even = even_scale(p.scale);
  float fix = 0.f;
  if (__builtin_amdgcn_readfirstlane(__syncthreads_or(is_great(lse)))) {
    RowSum row;
    for (int j0 = 0; j0 < len; j0 += 32) {
      __syncthreads();
      stage_rows<T, DP, 32, true, false>(sk, nullptr, kb + j0 * p.ld_t, p.ld_t, len - j0, p.d, p.vec, NW * 64);
      __syncthreads();
      const f32x16 t = scores_any<T, DP, true>(sk, fq, c, line, reach, j0 - i0, even);
#pragma unroll
      for (int r = 0; r < 16; ++r) if (j0 + (r & 3) + 8 * (r >> 2) + 4 * half < len) row.add(t[r]);
    }
    row.join();
    if (is_great(lse)) { lse = row.top; fix = log2f(row.sum) + 1e-30f; }
  }
  if (lane < 32 && i < len) { p.from[(long long)head * p.total + s.begin + i] = lse; p.fix[(long long)head * p.total + s.begin + i] = fix; }
  float below = 0.f, above = 0.f;
  f32x16 acc[DP / 32] = {};
  for (int j0 = 0; j0 < len; j0 += 32) {
    __syncthreads();
    stage_rows<T, DP, 32, true, true>(sk, skt, kb + j0 * p.ld_t, p.ld_t, len - j0, p.d, p.vec, NW * 64);
    stage_rows<T, DP, 32, true, false>(sv, nullptr, vb + j0 * p.ld_t, p.ld_t, len - j0, p.d, p.vec, NW * 64);
    __syncthreads();
    if (i0 >= len) continue;
    const int e0 = j0 - i0;
    f32x16 t = scores_any<T, DP, true>(sk, fq, c, line, reach, e0, even);
    const f32x16 dp = rows_times<T, DP>(sv, fg);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int j = j0 + (r & 3) + 8 * (r >> 2) + 4 * half;
      const float w = j < len && i < len ? __builtin_amdgcn_exp2f(t[r] - lse - fix) : 0.f;      // what is not there meets any bias
      t[r] = w == 0.f ? 0.f : w * (dp[r] - delta);
    }
    if constexpr (DTABLE) {
      if (tile_is_far(e0, reach)) {
        float x = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) x += t[r];
        if (e0 > 0) above += x; else below += x;
      } else {
        add_diagonals(mine, reach, e0, t);
      }
    }
    if (lift != 1.f) t *= lift;
    trans_times<T, DP>(acc, skt, t);
  }
  if (i < len) store_cols<T, DP>((T*)p.dq + (s.begin + i) * p.gld_t + head * p.gld_h, acc, p.scale / lift, p.d, p.vec);
  if constexpr (DTABLE) {
    for (int k = 32; k; k >>= 1) { below += __shfl_xor(below, k, 64); above += __shfl_xor(above, k, 64); }
    if (lane == 0) { far[wave][0] = below; far[wave][1] = above; }
    fold_buckets(p, hist, far, NW * 2, span, part);
  }
}

// dk and dv: block = NW * 32 keys of one head, one key per lane column; query tiles of 32 through LDS.
template <typename T, int DP, int NW>
__global__ __launch_bounds__(NW * 64) void attention_dkv_any_kernel(const AttnParams p) {
  constexpr int V = Elem<T>::kVec, BQ = NW * 32;
  __shared__ __align__(16) T sq[32 * (DP + V)];
  __shared__ __align__(16) T sqt[DP * (32 + V)];
  __shared__ __align__(16) T sg[32 * (DP + V)];
  __shared__ __align__(16) T sgt[DP * (32 + V)];
  __shared__ __align__(16) float sl[32], sd[32], sf[32];
  extern __shared__ float line[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
  const int head = blockIdx.x % p.heads;
  const Slot s = find_slot(p.offsets, p.n_seqs, p.total, BQ, blockIdx.x / p.heads);
  if (s.b < 0) return;
  if (s.b == p.n_seqs) {
    const long long r0 = s.begin + (long long)s.tile * BQ, r1 = r0 + BQ < s.end ? r0 + BQ : s.end;
    zero_rows((T*)p.dk + head * p.gld_h, p.gld_t, r0, r1, p.d);
    zero_rows((T*)p.dv + head * p.gld_h, p.gld_t, r0, r1, p.d);
    return;
  }
  const int len = (int)(s.end - s.begin);
  const int j0 = s.tile * BQ + wave * 32, j = j0 + (lane & 31);
  make_line<T>(line, p, head);
  const long long hd = (long long)p.heads * p.d;
  typename Elem<T>::vec fk[DP / (2 * V)], fv[DP / (2 * V)];
  load_row_frags<T, DP>(fk, (const T*)p.k + (s.begin + j) * p.ld_t + head * p.ld_h, j < len, p.d, p.vec);
  load_row_frags<T, DP>(fv, (const T*)p.v + (s.begin + j) * p.ld_t + head * p.ld_h, j < len, p.d, p.vec);
  const T* qb = (const T*)p.q + s.begin * p.ld_t + head * p.ld_h;
  const T* gb = (const T*)p.dout + s.begin * hd + (long long)head * p.d;
  const float* lse = p.from + (long long)head * p.total + s.begin;
  const float* delta = p.delta + (long long)head * p.total + s.begin;
  const float* fix = p.fix + (long long)head * p.total + s.begin;
  const float lift = ds_lift<T>(p, head, s.b), down = lift * kUnlift<T>;
  const float c = p.scale * kLog2e;
  const bool even = even_scale(p.scale);
  f32x16 ak[DP / 32] = {}, av[DP / 32] = {};
  for (int i0 = 0; i0 < len; i0 += 32) {
    __syncthreads();
    stage_rows<T, DP, 32, true, true>(sq, sqt, qb + i0 * p.ld_t, p.ld_t, len - i0, p.d, p.vec, NW * 64);
    stage_rows<T, DP, 32, true, true>(sg, sgt, gb + i0 * hd, hd, len - i0, p.d, p.vec, NW * 64);
    if (threadIdx.x < 32) {
      sl[threadIdx.x] = i0 + (int)threadIdx.x < len ? lse[i0 + threadIdx.x] : INFINITY;
      sd[threadIdx.x] = i0 + (int)threadIdx.x < len ? delta[i0 + threadIdx.x] : 0.f;
      sf[threadIdx.x] = i0 + (int)threadIdx.x < len ? fix[i0 + threadIdx.x] : 0.f;
    }
    __syncthreads();
    if (j0 >= len) continue;
    f32x16 t = scores_any<T, DP, false>(sq, fk, c, line, p.reach, j0 - i0, even);
    const f32x16 dp = rows_times<T, DP>(sg, fv);
    f32x16 ds;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = (r & 3) + 8 * (r >> 2) + 4 * half;
      t[r] = i0 + row < len ? __builtin_amdgcn_exp2f(t[r] - sl[row] - sf[row] + kLift<T>) : 0.f;      // a query that is not there meets any bias
      ds[r] = t[r] == 0.f ? 0.f : t[r] * (dp[r] - sd[row]);
    }
    trans_times<T, DP>(av, sgt, t);
    if (down != 1.f) ds *= down;
    trans_times<T, DP>(ak, sqt, ds);
  }
  if (j >= len) return;
  store_cols<T, DP>((T*)p.dk + (s.begin + j) * p.gld_t + head * p.gld_h, ak, p.scale / lift, p.d, p.vec);
  store_cols<T, DP>((T*)p.dv + (s.begin + j) * p.gld_t + head * p.gld_h, av, kUnlift<T>, p.d, p.vec);
}

// ---- backward, whole 16-byte pieces and head widths of 32, 64 and 128 -------------------------------------------------------
// The places of the tiled backward kernels, longest sequences first: [slots] of (begin, end, sequence, tile), then the rows behind the
// last sequence, then nothing (-1).  A block's time goes by its sequence's length, and blocks that begin in the sequences' own order
// leave the chip waiting for the long ones that began last: 64 texts of 16 to 384 tokens, 12 heads of 64, bf16: 121 us for the
// backward pass, 111 with this; fp32 516 and 409.  One block; a sequence's place is the tiles of all that come ahead of it, counted
// by 4 to 16 threads.
constexpr int kMaxOrdered = 256;
__global__ __launch_bounds__(1024) static void attention_order_kernel(const int64_t* __restrict__ offsets, int n_seqs, long long total, int tile,
                                                                      int slots, i32x4* __restrict__ order) {
  __shared__ int begin[kMaxOrdered], first[kMaxOrdered], used;
  __shared__ int2 size[kMaxOrdered];                   // rows and tiles
  const int b = threadIdx.x;
  if (b == 0) used = 0;
  if (b < n_seqs) {
    const int r0 = (int)seq_edge(offsets, b, total), r1 = (int)seq_edge(offsets, b + 1, total), len = r1 > r0 ? r1 - r0 : 0;
    begin[b] = r0;
    size[b] = make_int2(len, (len + tile - 1) / tile);
  }
  const int end = (int)seq_edge(offsets, n_seqs, total);
  __syncthreads();
  const int share = n_seqs <= 64 ? 4 : n_seqs <= 128 ? 3 : 2;      // log2 of the threads that count for one sequence
  const int mine = threadIdx.x >> share;
  if (mine < n_seqs) {
    const int2 me = size[mine];
    int at = 0;
#pragma unroll 4
    for (int o = threadIdx.x & ((1 << share) - 1); o < n_seqs; o += 1 << share) {
      const int2 x = size[o];
      at += x.x > me.x || (x.x == me.x && o < mine) ? x.y : 0;
    }
    for (int k = 1; k < 1 << share; k <<= 1) at += __shfl_xor(at, k, 64);
    first[mine] = at;
    if ((threadIdx.x & ((1 << share) - 1)) == 0) atomicMax(&used, at + me.y);
  }
  __syncthreads();
  // unordered offsets can ask for more places than there are: the bounds hold whatever they say
  for (int s = threadIdx.x >> 4; s < n_seqs; s += 64)
    for (int t = threadIdx.x & 15; t < size[s].y && first[s] + t < slots; t += 16) order[first[s] + t] = i32x4{begin[s], begin[s] + size[s].x, s, t};
  for (int at = used + threadIdx.x; at < slots; at += 1024) {
    const int t = at - used;
    order[at] = (long long)t * tile < total - end ? i32x4{end, (int)total, n_seqs, t} : i32x4{0, 0, -1, 0};
  }
}

// A block's head and place
__device__ __forceinline__ Slot place_of(const AttnParams& p, unsigned slots, unsigned hop, int tile, int& head, unsigned& slot) {
  if (p.order) {
    slot = blockIdx.x / p.heads;
    head = blockIdx.x % p.heads;
    const i32x4 o = p.order[slot];
    return Slot{__builtin_amdgcn_readfirstlane(o[0]), __builtin_amdgcn_readfirstlane(o[1]), __builtin_amdgcn_readfirstlane(o[2]),
                __builtin_amdgcn_readfirstlane(o[3])};
  }
  const unsigned at = xcd_run(slots * p.heads, hop);
  head = at / slots;
  slot = at % slots;
  return find_slot(p.offsets, p.n_seqs, p.total, tile, slot);
}

// dq and the block's bucket sums.  Each wave: 32 queries, one per lane column; key tiles of 64 through LDS.  k is read along its
// rows (scores) and across them (ds k): one copy in LDS, in the order of the transposed reads, serves both - the reads along it
// meet two by two on a bank.  64 texts of 16 to 384 tokens, 12 heads of 64, bf16: 53 us, 0.30 PFLOP/s, 19 vector instructions a
// score: bound by their issue and by the latency of a chain a tile.
template <typename T, int D, int NW, bool DTABLE>
__global__ __launch_bounds__(NW * 64, D == 128 ? 1 : 2) void attention_dq_kernel(const AttnParams p, unsigned slots, unsigned hop) {
  constexpr int BQ = NW * 32, KT = 64, V = Elem<T>::kVec;
  using R = Rows<T, D, kCol>;
  using RV = Rows<T, D, kRow>;
  __shared__ __align__(1024) T buf[2][2][KT * D];          // [turn][k, v]
  __shared__ float far[NW][2];
  extern __shared__ float line[];                          // start values, then NW * 2 lines of sums
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l = lane & 31;
  int head;
  unsigned slot;
  const Slot s = place_of(p, slots, hop, BQ, head, slot);
  float* part = p.part + ((long long)slot * p.heads + head) * p.n_buckets;
  if (s.b < 0 || s.b == p.n_seqs) {
    if (s.b >= 0) {
      const long long r0 = s.begin + (long long)s.tile * BQ, r1 = r0 + BQ < s.end ? r0 + BQ : s.end;
      zero_rows((T*)p.dq + head * p.gld_h, p.gld_t, r0, r1, D);
    }
    if constexpr (DTABLE) for (int t = threadIdx.x; t < p.n_buckets; t += NW * 64) part[t] = 0.f;
    return;
  }
  const int len = (int)(s.end - s.begin), tiles = (len + KT - 1) / KT;
  const int i0 = s.tile * BQ + wave * 32;
  const int reach = p.reach, span = sums_span(reach);
  const T* kb = (const T*)p.k + s.begin * p.ld_t + head * p.ld_h;
  const T* vb = (const T*)p.v + s.begin * p.ld_t + head * p.ld_h;
  auto issue = [&](int t) {
    const int left = len - t * KT;
    R::template load<KT, NW * 64>(buf[t & 1][0], kb + (long long)t * KT * p.ld_t, p.ld_t, left);
    RV::template load<KT, NW * 64>(buf[t & 1][1], vb + (long long)t * KT * p.ld_t, p.ld_t, left);
  };
  issue(0);
  const long long hd = (long long)p.heads * D;
  using vec = typename Elem<T>::vec;
  vec fq[D / (2 * V)], fg[D / (2 * V)];
  const int i = i0 + l < len ? i0 + l : len - 1;
  {
    const T* q = (const T*)p.q + (s.begin + i) * p.ld_t + head * p.ld_h + half * V;
    const T* g = (const T*)p.dout + (s.begin + i) * hd + (long long)head * D + half * V;
#pragma unroll
    for (int x = 0; x < D / (2 * V); ++x) { fq[x] = *(const vec*)(q + x * 2 * V); fg[x] = *(const vec*)(g + x * 2 * V); }
  }
  const long long row = (long long)head * p.total + s.begin + i;
  float lse = i0 + l < len ? p.lse[row] : INFINITY;
  float delta = 0.f;                 // dout . out, for this kernel and, through memory, for dk
  {
    const T* o = (const T*)p.out + (s.begin + i) * hd + (long long)head * D + half * V;
#pragma unroll
    for (int x = 0; x < D / (2 * V); ++x) {
      const vec fo = *(const vec*)(o + x * 2 * V);
      vec fr = {};
      if (p.rest) fr = *(const vec*)((const T*)p.rest + (o - (const T*)p.out) + x * 2 * V);
#pragma unroll
      for (int e = 0; e < V; ++e) delta += ((float)fo[e] + (float)fr[e]) * (float)fg[x][e];
    }
    delta += __shfl_xor(delta, 32, 64);
    if (lane < 32 && i0 + l < len) p.delta[row] = delta;
  }
  const float lift = ds_lift<T>(p, head, s.b);
  const float c = p.scale * kLog2e;
  float* hist = line + start_span(reach);
  const bool great = make_start_line<T, true>(line, p, head, c, len + KT, is_great(lse));
  if constexpr (DTABLE) for (int t = threadIdx.x; t < NW * 2 * span; t += NW * 64) hist[t] = 0.f;
  const float* mid = line + start_at(reach, 4 * half - l);
  float* mine = hist + (wave * 2 + half) * span;
#pragma unroll
  for (int x = 0; x < D / (2 * V); ++x) { settle(fq[x]); settle(fg[x]); }
  float less = delta;
  settle(lse);
  settle(less);
  float fix = 0.f;
  if (__builtin_expect(great, 0)) {
    RowSum all;
    for (int t = 0; t < tiles; ++t) {
      wait_loads<0>();
      __syncthreads();
      if (t + 1 < tiles) issue(t + 1);
      if (i0 >= len) continue;
#pragma unroll 1
      for (int u = 0; u < KT / 32; ++u) {
        const int j0 = t * KT + u * 32, e0 = j0 - i0;
        if (j0 >= len) break;
        f32x16 x;
        const float bias = c * scores<T, D, R, 1>(x, buf[t & 1][0], u * 32, fq, e0, p, line, mid + e0);
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (j0 + (r & 3) + 8 * (r >> 2) + 4 * half < len) all.add(__builtin_fmaf(x[r], c, bias));
      }
    }
    all.join();
    if (is_great(lse)) { lse = all.top; fix = log2f(all.sum) + 1e-30f; }
    __syncthreads();                 // the last tile is read: its place may be loaded again
    issue(0);
  }
  if (lane < 32 && i0 + l < len) { p.from[row] = lse; p.fix[row] = fix; }
  const float from = -lse;
  const bool seldom = great || __builtin_amdgcn_readfirstlane(i0 + 32 > len);
  float below = 0.f, above = 0.f;
  f32x16 acc[D / 32] = {};
  for (int t = 0; t < tiles; ++t) {
    wait_loads<0>();
    __syncthreads();
    if (t + 1 < tiles) issue(t + 1);
    if (i0 >= len) continue;
    const T* sk = buf[t & 1][0];
    const T* sv = buf[t & 1][1];
#pragma unroll
    for (int u = 0; u < KT / 32; ++u) {
      const int j0 = t * KT + u * 32, e0 = j0 - i0;
      if (j0 >= len) break;
      const bool is_far = tile_is_far(e0, reach);
      f32x16 x, dp = {};
      float shift = c * scores<T, D, R, 1>(x, sk, u * 32, fq, e0, p, line, mid + e0);
#pragma unroll
      for (int y = 0; y < D / (2 * V); ++y) Elem<T>::mma(RV::along(sv, u * 32, y), fg[y], dp);
      if (__builtin_expect(seldom, 0)) {
        if (i0 + l >= len) {           // a query that is not there meets any bias, NaN and infinities too
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = -INFINITY;
        }
        if (great) {
          const float back = 1.f / c;
#pragma unroll
          for (int r = 0; r < 16; ++r) x[r] = (__builtin_fmaf(x[r], c, shift) + from - fix) * back;
        }
      }
      shift = great ? 0.f : shift + from;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], c, shift));
        x[r] = w == 0.f ? 0.f : w * (dp[r] - less);       // a forbidden place may hold anything
      }
      if (j0 + 32 > len) {
#pragma unroll
        for (int r = 0; r < 16; ++r) if (j0 + (r & 3) + 8 * (r >> 2) + 4 * half >= len) x[r] = 0.f;
      }
      if constexpr (DTABLE) {
        if (is_far) {
          float y = 0.f;
#pragma unroll
          for (int r = 0; r < 16; ++r) y += x[r];
          if (e0 > 0) above += y; else below += y;
        } else {
          add_diagonals(mine, reach, e0, x);
        }
      }
      if (lift != 1.f) x *= lift;
      add_across<T, D>(acc, sk, u * 32, x);
    }
  }
  __syncthreads();
  if (i0 < len) store_turned<T, D>(&buf[0][0][0] + wave * (32 * D), (T*)p.dq + (s.begin + i0) * p.gld_t + head * p.gld_h, p.gld_t, acc, p.scale / lift, len - i0);
  if constexpr (DTABLE) {
    for (int k = 32; k; k >>= 1) { below += __shfl_xor(below, k, 64); above += __shfl_xor(above, k, 64); }
    if (lane == 0) { far[wave][0] = below; far[wave][1] = above; }
    fold_buckets(p, hist, far, NW * 2, span, part);
  }
}

// dk and dv: each wave 32 keys, one per lane column; query tiles of 64 through LDS, q and dout once, in the order of the
// transposed reads.  The two halves of a tile one after the other: held together they cost registers, 63 us
// instead of 58 at the size above, 52 with the longest texts first, 58 with what great rows and absent places need (0.35 PFLOP/s).
template <typename T, int D, int NW>
__global__ __launch_bounds__(NW * 64, D == 128 ? 1 : 2) void attention_dkv_kernel(const AttnParams p, unsigned slots, unsigned hop) {
  constexpr int BQ = NW * 32, QT = 64, V = Elem<T>::kVec;
  using R = Rows<T, D, kCol>;
  using vec = typename Elem<T>::vec;
  __shared__ __align__(1024) T buf[2][2][QT * D];       // [turn][q, dout]
  __shared__ __align__(16) float stat[2][4][QT];             // [turn][lse, delta]; a text with great rows: [0, delta, lse, fix]
  extern __shared__ float line[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5, l = lane & 31;
  int head;
  unsigned slot;
  const Slot s = place_of(p, slots, hop, BQ, head, slot);
  if (s.b < 0) return;
  if (s.b == p.n_seqs) {
    const long long r0 = s.begin + (long long)s.tile * BQ, r1 = r0 + BQ < s.end ? r0 + BQ : s.end;
    zero_rows((T*)p.dk + head * p.gld_h, p.gld_t, r0, r1, D);
    zero_rows((T*)p.dv + head * p.gld_h, p.gld_t, r0, r1, D);
    return;
  }
  const int len = (int)(s.end - s.begin), tiles = (len + QT - 1) / QT;
  const int j0 = s.tile * BQ + wave * 32;
  const long long hd = (long long)p.heads * D;
  const T* qb = (const T*)p.q + s.begin * p.ld_t + head * p.ld_h;
  const T* gb = (const T*)p.dout + s.begin * hd + (long long)head * D;
  const float* lse = p.from + (long long)head * p.total + s.begin;
  const float* delta = p.delta + (long long)head * p.total + s.begin;
  const float* fix = p.fix + (long long)head * p.total + s.begin;
  float next_lse = 0.f, next_delta = 0.f, next_fix = 0.f;    // thread x < QT: of query x of the tile under way
  bool great = false;                        // some query of the text has a fix
  auto issue = [&](int t) {
    const int left = len - t * QT;
    R::template load<QT, NW * 64>(buf[t & 1][0], qb + (long long)t * QT * p.ld_t, p.ld_t, left);
    R::template load<QT, NW * 64, true>(buf[t & 1][1], gb + (long long)t * QT * hd, hd, left);
    if (threadIdx.x < QT) {
      const bool there = (int)threadIdx.x < left;
      next_lse = there ? lse[t * QT + threadIdx.x] : INFINITY;
      next_delta = there ? delta[t * QT + threadIdx.x] : 0.f;
      next_fix = great && there ? fix[t * QT + threadIdx.x] : 0.f;
    }
  };
  issue(0);
  vec fk[D / (2 * V)], fv[D / (2 * V)];
  {
    const long long j = s.begin + (j0 + l < len ? j0 + l : len - 1);
    const T* k = (const T*)p.k + j * p.ld_t + head * p.ld_h + half * V;
    const T* v = (const T*)p.v + j * p.ld_t + head * p.ld_h + half * V;
#pragma unroll
    for (int x = 0; x < D / (2 * V); ++x) { fk[x] = *(const vec*)(k + x * 2 * V); fv[x] = *(const vec*)(v + x * 2 * V); }
  }
  const float lift = ds_lift<T>(p, head, s.b), down = lift * kUnlift<T>;
  const float c = p.scale * kLog2e;
#pragma unroll 4
  for (int i = threadIdx.x; i < len; i += NW * 64) great |= fix[i] != 0.f;
  great = make_start_line<T, true>(line, p, head, c, len + QT, great);
  if (great && threadIdx.x < QT) next_fix = (int)threadIdx.x < len ? fix[threadIdx.x] : 0.f;
  const float* mid = line + start_at(p.reach, l - 4 * half);        // mid[e0 - row]: column l is the key, the rows are queries
#pragma unroll
  for (int x = 0; x < D / (2 * V); ++x) { settle(fk[x]); settle(fv[x]); }
  f32x16 ak[D / 32] = {}, av[D / 32] = {};
  for (int t = 0; t < tiles; ++t) {
    if (threadIdx.x < QT) {
      stat[t & 1][0][threadIdx.x] = great ? 0.f : next_lse;
      stat[t & 1][1][threadIdx.x] = next_delta;
      if (great) { stat[t & 1][2][threadIdx.x] = next_lse; stat[t & 1][3][threadIdx.x] = next_fix; }
    }
    wait_loads<0>();
    __syncthreads();
    if (t + 1 < tiles) issue(t + 1);
    if (j0 >= len) continue;
    const T* sq = buf[t & 1][0];
    const T* sg = buf[t & 1][1];
#pragma unroll 1
    for (int u = 0; u < QT / 32; ++u) {
      if (t * QT + u * 32 >= len) break;
      const int e0 = j0 - t * QT - u * 32;
      f32x16 x, dp = {};
      float shift = c * scores<T, D, R, -1>(x, sq, u * 32, fk, e0, p, line, mid + e0);
#pragma unroll
      for (int y = 0; y < D / (2 * V); ++y) Elem<T>::mma(R::along(sg, u * 32, y), fv[y], dp);
      if (__builtin_expect(great || t * QT + u * 32 + 32 > len, 0)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int row = u * 32 + (r & 3) + 8 * (r >> 2) + 4 * half;
          if (great) x[r] = (__builtin_fmaf(x[r], c, shift) - stat[t & 1][2][row] - stat[t & 1][3][row] + kLift<T>) * (1.f / c);
          if (t * QT + row >= len) x[r] = -INFINITY;       // a query that is not there meets any bias, NaN and infinities too
        }
      }
      shift = great ? 0.f : shift + kLift<T>;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 ls = *(const f32x4*)&stat[t & 1][0][u * 32 + 8 * g + 4 * half], dl = *(const f32x4*)&stat[t & 1][1][u * 32 + 8 * g + 4 * half];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          x[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[r], c, shift - ls[e]));
          dp[r] = x[r] == 0.f ? 0.f : x[r] * (dp[r] - dl[e]);       // a forbidden place may hold anything
        }
      }
      add_across<T, D>(av, sg, u * 32, x);
      if (down != 1.f) dp *= down;
      add_across<T, D>(ak, sq, u * 32, dp);
    }
  }
  __syncthreads();
  if (j0 >= len) return;
  // 32 rows at a time through the wave's part of LDS
  T* mine = &buf[0][0][0] + wave * (32 * D);
  store_turned<T, D>(mine, (T*)p.dk + (s.begin + j0) * p.gld_t + head * p.gld_h, p.gld_t, ak, p.scale / lift, len - j0);
  store_turned<T, D>(mine, (T*)p.dv + (s.begin + j0) * p.gld_t + head * p.gld_h, p.gld_t, av, kUnlift<T>, len - j0);
}

// dtable[t][h] = the slots' parts in order, in 64 bits: block = one head and bucket
template <typename T>
__global__ __launch_bounds__(256) void attention_dtable_kernel(const float* __restrict__ part, long long slots, int heads, int n_buckets, T* __restrict__ dtable) {
  __shared__ double red[256];
  const int t = blockIdx.x % n_buckets, head = blockIdx.x / n_buckets;
  double x = 0.0;
  for (long long s = threadIdx.x; s < slots; s += 256) x += part[(s * heads + head) * n_buckets + t];
  red[threadIdx.x] = x;
  __syncthreads();
  for (int k = 128; k; k >>= 1) {
    if ((int)threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) dtable[(long long)t * heads + head] = (T)(float)red[0];
}

}  // namespace vdbk
