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
  int stream;          // the output is larger than the L2s hold: its stores pass them by (49152 x 2304 from 768: 184 us against 199)
  int vec_y;           // neighbouring outputs (and residuals, z, partial sums) can move 1: four at once, 2: 16-bit ones eight at once, too
};

template <typename T>
__device__ __forceinline__ T to_elem(float x) { return (T)x; }

// One value of the epilogue: sum -> bias -> (z) -> activation -> residual -> y
template <typename T, int ACT>
__device__ __forceinline__ void store_one(const GemmParams& p, long long i, long long j, float s, float bias) {
  s += bias;
  if (p.z) ((T*)p.z)[i * p.n + j] = (T)s;
  s = act_value<T, ACT>(s);
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

// ---- whole 16-byte pieces: tiles through LDS by direct loads -------------------------------------------------------------
// BM x BN outputs per block of WGI x WGJ waves; a K step is 128 bytes of every operand row (64 16-bit or 32 fp32 values), two
// steps in LDS.  Loads go straight to LDS, 16 bytes a lane.  A step has two halves of fragments: while the first half is
// multiplied the second is read; then, behind the one barrier, the step's slot is free - the step after next is sent for into
// it - and the next step's first half is read while the second half is multiplied.  The sequence of steps runs on from one
// tile of a block into the next, so a tile's outputs are written while the next tile's first two steps arrive.
// The product is computed transposed (rows of C = j): a lane then holds four neighbouring j of one i.
//
// An operand [row][c] ("along": the contracted index is dense) is laid out as 128-byte rows, its 16-byte pieces moved by
// XOR with (row >> 1) & 7, so that the 16 rows x 16 bytes of a fragment read cover all LDS banks.  An operand [c][row]
// ("across") keeps that order; 16-bit fragments come out of ds_read_b64_tr_b16, which hands lane l of 16 the column l of four
// rows, fp32 ones by single words; the XOR moves 64-byte groups so that the rows read together are on different banks.
//
// Edges: rows past the end repeat the last (never stored); contracted values past the end are zeros written by the lane that
// would have loaded them.
// 16x16 tiles: one 16-byte fragment contracts 32 (16-bit: one instruction) or 16 (fp32: four) values
template <typename T> struct Frag16;
template <> struct Frag16<float> {
  static constexpr int kIns = 4;
  static __device__ __forceinline__ void mma(f32x4 a, f32x4 b, f32x4& c, int i) { c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0); }
};
template <> struct Frag16<__bf16> {
  static constexpr int kIns = 1;
  static __device__ __forceinline__ void mma(bf16x8 a, bf16x8 b, f32x4& c, int) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Frag16<_Float16> {
  static constexpr int kIns = 1;
  static __device__ __forceinline__ void mma(f16x8 a, f16x8 b, f32x4& c, int) { c = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};

template <typename T, bool ACROSS, int ROWS, int THREADS>
struct TileOperand {
  static constexpr int V = Elem<T>::kVec, KB = 8 * V, kPieces = ROWS * 8 / THREADS;   // pieces of 16 bytes per thread and step
  static constexpr int kChunksRow = ACROSS ? ROWS / V : 8;                           // 16-byte pieces per LDS row
  static_assert(ROWS * 8 % THREADS == 0 && THREADS % 128 == 0 && (!ACROSS || (ROWS & (ROWS - 1)) == 0), "whole pieces; the XOR stays inside a row");
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (!ACROSS) return (row >> 1) & 7;
    else if constexpr (sizeof(T) == 4) return ((row >> 2) & 3) << 2;
    else if constexpr (ROWS >= 128) return ((row & 3) << 2) | ((row >> 3 & 1) << 1);
    else return ((row >> 1 & 1) << 2) | ((row >> 3 & 1) << 1);
  }
  unsigned off[kPieces];     // byte offsets from the step's base
  int c0;                    // first contracted value of this thread's pieces inside a step (across: its LDS row of piece 0)
  // rows: how many of the tile's rows exist (at least one piece's worth)
  __device__ __forceinline__ void init(long long ld, long long rows) {
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int L = i * THREADS + t, row = L / kChunksRow, chunk = (L % kChunksRow) ^ swizzle(row);
      if constexpr (!ACROSS) {
        const long long r = row < rows ? row : rows - 1;
        off[i] = (unsigned)((r * ld + chunk * V) * (long long)sizeof(T));
        c0 = chunk * V;      // the same for every piece: the threads cover a multiple of 16 rows
      } else {
        const long long r = chunk * V + V <= rows ? chunk * V : rows - V;
        off[i] = (unsigned)(((long long)row * ld + r) * (long long)sizeof(T));
        c0 = t / kChunksRow;
      }
    }
  }
  static __device__ __forceinline__ const T* base(const T* g, long long ld, long long row0, long long c) { return ACROSS ? g + c * ld + row0 : g + row0 * ld + c; }
  static constexpr int kRowsPerPiece = THREADS / kChunksRow;   // across: LDS rows between two pieces of a thread
  // left: contracted values from this step's first on
  __device__ __forceinline__ void load(const T* b, unsigned lds, T* slot, long long left) const {
    const unsigned wave_dst = lds + (unsigned)__builtin_amdgcn_readfirstlane((threadIdx.x >> 6) << 10);
    if (left >= KB) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) lds_load16(b, off[i], wave_dst + i * (THREADS * 16));
    } else {
#pragma unroll
      for (int i = 0; i < kPieces; ++i) {
        const bool there = ACROSS ? c0 + i * kRowsPerPiece < left : c0 + V <= left;
        if (there) lds_load16(b, off[i], wave_dst + i * (THREADS * 16));
        else *(i32x4*)((char*)slot + i * (THREADS * 16) + threadIdx.x * 16) = i32x4{0, 0, 0, 0};
      }
    }
  }
  // Fragment of the 16 rows from r0 (a multiple of 16) for sub-step s (0 or 1).  The XOR is written in lane numbers: of the row
  // that a lane reads only those bits enter it, and the compiler then keeps one address for all r0 and s (along) or all s (across).
  static __device__ __forceinline__ typename Elem<T>::vec frag(const T* slot, int r0, int s) {
    const int lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
    using vec = typename Elem<T>::vec;
    if constexpr (!ACROSS) {
      const int at = l * 128 + ((g ^ ((l >> 1) & 3)) << 4) + (l & 8 ? 64 : 0);     // sub-step 0; sub-step 1 is 64 bytes to the other side
      return *(const vec*)((const char*)slot + r0 * 128 + (s ? at ^ 64 : at));
    } else if constexpr (sizeof(T) == 4) {
      vec x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = s * 16 + g * 4 + e;
        x[e] = slot[c * ROWS + ((((r0 + l) >> 2) ^ (g << 2)) << 2) + (l & 3)];
      }
      return x;
    } else {
      vec x;
      const int swz = ROWS >= 128 ? ((l >> 2) << 2) | ((g & 1) << 1) : ((l >> 3) << 2) | ((g & 1) << 1);
      const T* at = slot + (g * 8 + (l >> 2)) * ROWS + ((((r0 >> 3) + ((l & 3) >> 1)) ^ swz) << 3) + (l & 1) * 4;
#pragma unroll
      for (int e = 0; e < 2; ++e) *((s16x4*)&x + e) = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + (s * 32 + e * 4) * ROWS));
      return x;
    }
  }
};

template <typename T, bool AT, bool BT, int ACT, bool SPLIT, int BM, int BN, int WGI, int WGJ, int MINW>
__global__ __launch_bounds__(WGI * WGJ * 64, MINW) void gemm_tile_kernel(const GemmParams p, int tiles_i, int tiles_j) {
  constexpr int kThreads = WGI * WGJ * 64;
  using OA = TileOperand<T, AT, BM, kThreads>;
  using OB = TileOperand<T, BT, BN, kThreads>;
  constexpr int KB = OA::KB, kSlotA = BM * 128, kSlot = (BM + BN) * 128, WI = BM / WGI / 16, WJ = BN / WGJ / 16;   // 16x16 tiles of a wave
  constexpr int kRow = WJ * 32;                                                // bytes of a wave's 16-bit output row
  __shared__ __align__(1024) char smem[2 * kSlot];
  __shared__ __align__(16) char turn[sizeof(T) == 2 && !SPLIT ? WGI * WGJ * 16 * kRow : 16];
  const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) void*)smem;
  // Blocks go to the eight XCDs in turn; each XCD gets a contiguous run of tiles, j fastest: a run walks down the rows of A
  // with all of B in its L2.  A block takes every (gridDim.x / 8)-th tile of its XCD's run.
  const unsigned n_tiles = (unsigned)tiles_i * tiles_j, x = blockIdx.x & 7, run = (n_tiles >> 3) + (x < (n_tiles & 7));
  const unsigned run0 = x * (n_tiles >> 3) + (x < (n_tiles & 7) ? x : (n_tiles & 7)), stride = (gridDim.x + 7 - x) >> 3;
  const long long cc0 = SPLIT ? (long long)blockIdx.y * p.k_split : 0;
  const long long cc1 = SPLIT ? (cc0 + p.k_split < p.k ? cc0 + p.k_split : p.k) : p.k;
  const int steps = (int)((cc1 - cc0 + KB - 1) / KB);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, g = lane >> 4, l = lane & 15;
  const int wi = (wave / WGJ) * (BM / WGI), wj = (wave % WGJ) * (BN / WGJ);
  // the step that is sent for next
  OA oa;
  OB ob;
  const T *ba = nullptr, *bb = nullptr;
  unsigned lq = blockIdx.x >> 3;
  int ls = 0, slot = 0;
  auto aim = [&]() {
    const unsigned tile = run0 + lq;
    const long long i0 = (long long)(tile / tiles_j) * BM, j0 = (long long)(tile % tiles_j) * BN;
    oa.init(p.lda, p.m - i0);
    ob.init(p.ldb, p.n - j0);
    ba = OA::base((const T*)p.a, p.lda, i0, cc0);
    bb = OB::base((const T*)p.b, p.ldb, j0, cc0);
  };
  auto issue = [&]() {
    if (lq >= run) return;
    const int at = slot * kSlot;
    const long long left = cc1 - cc0 - (long long)ls * KB;
    oa.load(ba, lds0 + at, (T*)(smem + at), left);
    ob.load(bb, lds0 + at + kSlotA, (T*)(smem + at + kSlotA), left);
    slot ^= 1;
    ba += AT ? (long long)KB * p.lda : KB;
    bb += BT ? (long long)KB * p.ldb : KB;
    if (++ls == steps) {
      ls = 0;
      lq += stride;
      if (lq < run) aim();
    }
  };
  if (lq >= run) return;
  unsigned q = lq;
  aim();
  issue();
  issue();
  wait_loads<0>();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // zeros of a last step, written by this wave
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  bool waited = true;             // the next step has landed, as far as this wave's loads go
  int use = 0;
  for (; q < run; q += stride) {
  const unsigned tile = run0 + q;
  const long long ti0 = (long long)(tile / tiles_j) * BM, tj0 = (long long)(tile % tiles_j) * BN;
  const bool more = q + stride < run;
  f32x4 acc[WJ][WI] = {};
  // fp32: the residual is fetched ahead of the sums (16 registers a lane).  All blocks end at about the same time there, and reading it
  // at the end stood open: 6144 x 768 from 768 72 us.
  constexpr bool kAhead = sizeof(T) == 4 && !SPLIT && !AT && !BT;
  f32x4 ahead[kAhead ? WJ : 1][kAhead ? WI : 1] = {};
  if constexpr (kAhead) {
    if (p.residual && p.vec_y) {
#pragma unroll
      for (int j = 0; j < WJ; ++j)
#pragma unroll
        for (int i = 0; i < WI; ++i) {
          const long long ii = ti0 + wi + i * 16 + l, jj = tj0 + wj + j * 16 + g * 4;
          if (ii < p.m && jj < p.n) ahead[j][i] = *(const f32x4*)((const T*)p.residual + ii * p.ldr + jj);
        }
    }
  }
  typename Elem<T>::vec fa[WI], fb[WJ];
  auto read = [&](int h) {
    const T* sa = (const T*)(smem + use * kSlot);
    const T* sb = (const T*)(smem + use * kSlot + kSlotA);
#pragma unroll
    for (int i = 0; i < WI; ++i) fa[i] = OA::frag(sa, wi + i * 16, h);
#pragma unroll
    for (int j = 0; j < WJ; ++j) fb[j] = OB::frag(sb, wj + j * 16, h);
  };
  auto multiply = [&]() {
#pragma unroll
    for (int e = 0; e < Frag16<T>::kIns; ++e)      // outermost: neighbouring instructions do not wait for each other's sums
#pragma unroll
      for (int j = 0; j < WJ; ++j)
#pragma unroll
        for (int i = 0; i < WI; ++i) Frag16<T>::mma(fb[j], fa[i], acc[j][i], e);
  };
  for (int s = 0; s < steps; ++s) {
    read(0);
    multiply();
    read(1);
    if (s + 1 < steps || more) {
      if (!waited) wait_loads<0>();
      waited = false;
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // this wave's reads of the slot, and its zeros
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      issue();
    }
    use ^= 1;
    multiply();
  }
  // C rows = j: lane (g, l) holds j = 4 g .. 4 g + 3 of the 16, i = l
  typedef T vec4 __attribute__((ext_vector_type(4)));
  auto finish = [&](f32x4 v, const float (&bias)[4], long long ii, long long jj, vec4& z, const f32x4& res) {   // whole groups of four
    vec4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += bias[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) z[e] = (T)v[e];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = act_value<T, ACT>(v[e]);
    if constexpr (kAhead) {
      v += res;
    } else if (p.residual) {
      const vec4 r = *(const vec4*)((const T*)p.residual + ii * p.ldr + jj);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += (float)r[e];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
    return o;
  };
  auto bias_of = [&](long long jj, float (&bias)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) bias[e] = !SPLIT && p.bias && jj + e < p.n ? (float)((const T*)p.bias)[jj + e] : 0.f;
  };
  // 16-bit outputs: a lane's four are 8 bytes of a row, 32 bytes with its neighbours', and stores of such pieces stand at half
  // the rate of whole lines.  Each wave turns 16 rows of its tile at a time in LDS of its own: 16-byte pieces, moved by XOR so
  // that neither the writes nor the reads meet on a bank, and stores of WJ * 32 bytes of a row.
  if constexpr (!SPLIT && sizeof(T) == 2) {
    if (p.vec_y == 2) {
      constexpr int kChunks = WJ * 2, kShift = kChunks >= 16 ? 0 : kChunks == 8 ? 1 : 2, kPerRead = 64 / kChunks;   // rows a read covers
      char* mine = turn + wave * (16 * kRow);
      vec4 bias4[WJ];
#pragma unroll
      for (int j = 0; j < WJ; ++j) {
        const long long jj = tj0 + wj + j * 16 + g * 4;
        bias4[j] = p.bias && jj < p.n ? *(const vec4*)((const T*)p.bias + jj) : vec4{};
      }
      const int my_row = lane / kChunks, my_c = lane % kChunks;
      const long long jj_out = tj0 + wj + my_c * 8, ii_out = ti0 + wi + my_row;
      const int rows_left = jj_out < p.n ? (int)(p.m - ii_out < BM ? p.m - ii_out : BM) : 0;
      // the steps under way are waited for ahead of the first store: stores share the counter, and a wait behind them would
      // stand until they are written
      if (more) { wait_loads<0>(); waited = true; }
      for (int pass = p.z ? 0 : 1; pass < 2; ++pass) {
        const long long ld = pass == 0 ? p.n : p.ldy;
        T* dst = (T*)(pass == 0 ? p.z : p.y) + ii_out * ld + jj_out;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
#pragma unroll
          for (int j = 0; j < WJ; ++j) {
            f32x4 v = acc[j][i];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += (float)bias4[j][e];
            if (pass) {
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = act_value<T, ACT>(v[e]);
              if (p.residual) {
                const long long ii = ti0 + wi + i * 16 + l, jj = tj0 + wj + j * 16 + g * 4;
                if (ii < p.m && jj < p.n) {
                  const vec4 r = *(const vec4*)((const T*)p.residual + ii * p.ldr + jj);
#pragma unroll
                  for (int e = 0; e < 4; ++e) v[e] += (float)r[e];
                }
              }
            }
            vec4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
            *(vec4*)(mine + l * kRow + ((((j * 2 + (g >> 1)) ^ ((l >> kShift) & (kChunks - 1))) << 4) | ((g & 1) << 3))) = o;
          }
          asm volatile("" ::: "memory");     // a wave's LDS operations keep their order
#pragma unroll
          for (int r = 0; r < 16; r += kPerRead) {
            const int row = r + my_row;
            const i32x4 v = *(const i32x4*)(mine + row * kRow + ((my_c ^ ((row >> kShift) & (kChunks - 1))) << 4));
            if (i * 16 + r < rows_left) {
              if (p.stream) __builtin_nontemporal_store(v, (i32x4*)(dst + (i * 16 + r) * ld));
              else *(i32x4*)(dst + (i * 16 + r) * ld) = v;
            }
          }
          asm volatile("" ::: "memory");
        }
      }
      continue;
    }
  }
  if (more) { wait_loads<0>(); waited = true; }
#pragma unroll
  for (int j = 0; j < WJ; ++j) {
    const long long jj = tj0 + wj + j * 16 + g * 4;
    if (jj >= p.n) continue;
    const bool whole = p.vec_y && jj + 4 <= p.n;
    float bias[4];
    bias_of(jj, bias);
#pragma unroll
    for (int i = 0; i < WI; ++i) {
      const long long ii = ti0 + wi + i * 16 + l;
      if (ii >= p.m) continue;
      if constexpr (SPLIT) {
        float* at = p.partial + ((long long)blockIdx.y * p.m + ii) * p.n + jj;
        if (whole) *(f32x4*)at = acc[j][i];
        else {
#pragma unroll
          for (int e = 0; e < 4; ++e) if (jj + e < p.n) at[e] = acc[j][i][e];
        }
      } else if (whole) {
        vec4 z;
        const vec4 o = finish(acc[j][i], bias, ii, jj, z, ahead[kAhead ? j : 0][kAhead ? i : 0]);
        if (p.z) *(vec4*)((T*)p.z + ii * p.n + jj) = z;
        *(vec4*)((T*)p.y + ii * p.ldy + jj) = o;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (jj + e < p.n) store_one<T, ACT>(p, ii, jj + e, acc[j][i][e], bias[e]);
      }
    }
  }
  }
}

// ---- few rows ----------------------------------------------------------------------------------------------------------------
// 16 MT rows of A x 16 rows of B per block; its eight waves take the contracted values in turn, fragments straight from global
// memory (each element of B is used by one block only, LDS would not save a read), and join their sums in LDS, in order.  Bound by
// the latency of a few loads in flight at once: 14 x 2304 from 768 in bf16 is 3.5 MB of weights.
template <typename T, int ACT, int MT>
__global__ __launch_bounds__(512) void gemm_few_kernel(const GemmParams p) {
  using vec = typename Elem<T>::vec;
  constexpr int V = Elem<T>::kVec, KS = 4 * V;           // contracted values of one fragment
  __shared__ __align__(16) float sums[8][MT * 16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, l = lane & 15;
  const long long j0 = (long long)blockIdx.x * 16, i0 = (long long)blockIdx.y * (16 * MT);
  const T* b = (const T*)p.b + (j0 + l < p.n ? j0 + l : p.n - 1) * p.ldb + g * V;
  const T* a[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) a[t] = (const T*)p.a + (i0 + t * 16 + l < p.m ? i0 + t * 16 + l : p.m - 1) * p.lda + g * V;
  f32x4 acc[MT] = {};
#pragma unroll 3
  for (long long c = (long long)wave * KS; c < p.k; c += 8 * KS) {
    const bool there = c + g * V < p.k;                  // k is a multiple of V
    vec fb = {}, fa[MT] = {};
    if (there) {
      fb = *(const vec*)(b + c);
#pragma unroll
      for (int t = 0; t < MT; ++t) fa[t] = *(const vec*)(a[t] + c);
    }
#pragma unroll
    for (int e = 0; e < Frag16<T>::kIns; ++e)
#pragma unroll
      for (int t = 0; t < MT; ++t) Frag16<T>::mma(fa[t], fb, acc[t], e);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) sums[wave][t * 16 + g * 4 + e][l] = acc[t][e];
  __syncthreads();
  for (int t = threadIdx.x; t < MT * 256; t += 512) {
    const int r = t >> 4, c = t & 15;
    const long long i = i0 + r, j = j0 + c;
    if (i >= p.m || j >= p.n) continue;
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) s += sums[w][r][c];
    store_one<T, ACT>(p, i, j, s, p.bias ? (float)((const T*)p.bias)[j] : 0.f);
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
        const float slope = act_slope<T, ACT>((float)z[i * n + j]);
        g = ACT == 3 && slope == 0.f ? 0.f : g * slope;      // relu lets nothing through, an infinity or NaN neither
        if (dz) dz[i * n + j] = (T)g;
      }
      s += g;
    }
  if (!part) return;
  red[wave][lane] = s;
  __syncthreads();
  if (wave == 0 && j < n) part[(long long)blockIdx.y * n + j] = (red[0][lane] + red[1][lane]) + (red[2][lane] + red[3][lane]);
}

// 32 columns a block; eight threads a column take the parts in turn and are joined in order, in 64 bits
template <typename T>
__global__ __launch_bounds__(256) void col_join_kernel(const float* __restrict__ part, int parts, long long n, T* __restrict__ db) {
  __shared__ double red[8][32];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  const long long j = (long long)blockIdx.x * 32 + c;
  double s = 0.0;
  if (j < n)
    for (int i = g; i < parts; i += 8) s += part[(long long)i * n + j];
  red[g][c] = s;
  __syncthreads();
  if (g || j >= n) return;
  for (int i = 1; i < 8; ++i) s += red[i][c];
  db[j] = (T)(float)s;
}

}  // namespace vdbk
