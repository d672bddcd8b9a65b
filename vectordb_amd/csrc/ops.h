// ops.h — host-side seams of the encoder operators (include/vdb_ops.h): the C ABI in ops_api.hip sees only these.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vdbk {

// C[i][j] = sum_c A(i, c) B(j, c), fp32 sums.  A(i, c) = a[i * lda + c], or a[c * lda + i] with a_t; B likewise.
struct GemmArgs {
  const void* a; int64_t lda; bool a_t;
  const void* b; int64_t ldb; bool b_t;
  int64_t m, n, k;
  void* y; int64_t ldy;                 // element type of the operands
  const void* bias;                     // [n] or nullptr
  int act;
  const void* residual; int64_t ldr;    // [m][n] or nullptr
  void* z;                              // [m][n] dense, the sum before the activation, or nullptr
  float* partial; int64_t partial_bytes;   // scratch for a contraction split over blocks
  hipStream_t st;
};
int64_t gemm_workspace_bytes(int dtype, bool a_t, bool b_t, int64_t m, int64_t n, int64_t k);
hipError_t launch_gemm(int dtype, const GemmArgs& a);

// dz = dy act'(z) (dz dense [m][n]; skipped when act is none) and db = column sums of dy act'(z)
struct ActGradArgs {
  const void* dy; int64_t lddy; const void* z; int act; int64_t m, n;
  void* dz; void* db;                   // each may be nullptr
  float* partial;                       // [act_grad_parts(m, n)][n]
  hipStream_t st;
};
int act_grad_parts(int64_t m, int64_t n);
hipError_t launch_act_grad(int dtype, const ActGradArgs& a);

constexpr int kMaxSteps = 64;           // VDB_OP_MAX_BUCKETS / 2
// Smallest distance of bucket near + 1 + i; distances below `near` are buckets of their own.
struct Buckets { int half, near, n_steps; int step[kMaxSteps]; };
struct AttnArgs {
  const void *q, *k, *v; int64_t ld_t, ld_h;
  const void* table; int n_buckets; Buckets bk;
  const int64_t* offsets; int64_t n_seqs, total;
  int heads, d; float scale;
  void* out; void* rest; float* lse;     // rest: what the rounding of out left, or nullptr
  // backward
  const void* dout; void *dq, *dk, *dv; int64_t gld_t, gld_h; void* dtable;
  float* delta; float* from; float* fix; float* gscale; float* part; void* order;    // workspace pieces
  hipStream_t st;
};
hipError_t launch_attention(int dtype, const AttnArgs& a);
int64_t attention_backward_workspace(int dtype, int64_t n_seqs, int64_t total, int heads, int d, int n_buckets);
hipError_t launch_attention_backward(int dtype, AttnArgs a, char* ws);

struct PoolArgs {
  const void* hidden; int64_t ld; const int64_t* offsets; int64_t n_seqs, total, dim; int normalize;
  float* y; float* inv_norm;
  const float* dy; void* dhidden;
  hipStream_t st;
};
hipError_t launch_mean_pool(int dtype, const PoolArgs& a);
hipError_t launch_mean_pool_backward(int dtype, const PoolArgs& a);

void set_last_error(const char* msg);   // what vdb_last_error(NULL) returns on this thread (vdb_api.hip)

}  // namespace vdbk
