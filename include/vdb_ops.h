/*
 * vdb_ops.h — C ABI of the text encoder's operators (libvdb_hip.so, beside vdb.h).
 *
 * The reference embeds its texts with sentence-transformers' all-mpnet-base-v2 (src/vectordb.py:13-69,
 * src/config.py:36), a transformer encoder whose attention carries a learned relative position bias.  These are the
 * operators such an encoder is made of, forward and backward, on token rows packed WITHOUT padding:
 *
 *   rows      [total][...]  one row per token, sequence after sequence
 *   offsets   int64 [n_seqs + 1] in DEVICE memory: sequence b owns rows [offsets[b], offsets[b+1]).  offsets[0] is taken
 *             as 0; values are clamped into [0, total] and to non-negative lengths, so that no contents make a kernel
 *             leave its buffers (a descending list gives unspecified results).  Rows behind the last sequence get zeros.
 *
 * Conventions are vdb.h's: 0 or a negative vdb_status, message from vdb_last_error(NULL); the caller owns every buffer
 * (the *_workspace_bytes functions size the scratch; it may be reused as soon as the work on the stream is done, and two
 * calls that may overlap need two); nothing is allocated, no call waits for the device, and every launch can be captured
 * into a HIP graph.  All pointers are device memory on `device`, the stream is one of that device's; the calling
 * thread's current device is left as it was.  Element strides (ld*) are in elements; the last dimension is contiguous.
 * Outputs and scratch must not overlap inputs.  A failed call's error is reported by its status alone, the runtime's last error is cleared.
 * Limits: m up to 2^29; n, k and dim up to 2^20; (total / 32 + n_seqs + 1) times the heads below 2^24.
 * Results do not depend on the order in which blocks run: there is no floating-point atomic between two of them.
 */
#ifndef VDB_OPS_H
#define VDB_OPS_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum vdb_op_dtype { VDB_OP_F32 = 0, VDB_OP_BF16 = 1, VDB_OP_F16 = 2 };
enum vdb_op_act { VDB_ACT_NONE = 0, VDB_ACT_GELU = 1, VDB_ACT_GELU_TANH = 2, VDB_ACT_RELU = 3 };

#define VDB_OP_MAX_HEAD_DIM 128
#define VDB_OP_MAX_BUCKETS 128
#define VDB_OP_MAX_DISTANCE 512

/* y[m][n] = act(x[m][k] w[n][k]^T + bias[n]) + residual[m][n], summed in 32 bits, rounded once.
 * bias, residual and z may be NULL; z [m][n] dense receives the sum before the activation (what the backward pass needs
 * when act is not VDB_ACT_NONE).  m may be 0.  workspace: vdb_op_linear_workspace_bytes (may be 0 bytes / NULL). */
int64_t vdb_op_linear_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k);
int vdb_op_linear_dev(int device, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                      const void* residual, int64_t ldr, void* y, int64_t ldy, void* z, int64_t m, int64_t n, int64_t k,
                      int act, void* workspace, int64_t workspace_bytes, void* stream);

/* Gradients of the above for dy [m][n]: dz = dy act'(z); dx = dz w; dw = dz^T x; db = the column sums of dz.  Each of
 * dx [m][k], dw [n][k], db [n] (dense) may be NULL.  z: what the forward pass wrote (NULL for VDB_ACT_NONE).  dz is
 * rounded to the operands' type before the two products (they run on matrix instructions of that type), db sums it
 * before that rounding.  The residual's gradient is dy itself. */
int64_t vdb_op_linear_backward_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k, int act);
int vdb_op_linear_backward_dev(int device, int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w,
                               int64_t ldw, const void* z, void* dx, void* dw, void* db, int64_t m, int64_t n, int64_t k,
                               int act, void* workspace, int64_t workspace_bytes, void* stream);

/* Self-attention over packed sequences with a learned relative position bias:
 *   p = softmax_j(scale q_i.k_j + table[bucket(j - i)][h]),  out_i = sum_j p v_j      (i, j places in one sequence)
 * bucket(e), with half = n_buckets/2, near = half/2, n = |e|: n below near, else near + the number of i in 1..half-near-1
 * with n >= near (max_distance/near)^(i/(half-near)) (compared in whole numbers); + half where e > 0.  This is the
 * bidirectional bucketing of the reference's embedding model (32 buckets, max_distance 128).
 * A bias of -inf forbids its distances; a row that is left nothing gives zeros, one whose biases are all the same finite number, so great
 * that the scores vanish beside it in 32 bits, an even softmax.  Scales outside [1e-18, 1e18] take the general kernels.
 * q, k, v: token stride ld_t, head stride ld_h, dense head rows of head_dim.  out: dense [total][heads][head_dim].
 * Kept for the backward pass, each may be NULL: lse fp32 [heads][total], log2 of the softmax denominators; rest, of out's type and
 * shape, what the rounding of out left (16-bit types: the gradients need rowsum(dout out) closer than that rounding). */
int vdb_op_attention_dev(int device, int dtype, const void* q, const void* k, const void* v, int64_t ld_t, int64_t ld_h,
                         const void* table, int n_buckets, int max_distance, const int64_t* offsets, int64_t n_seqs,
                         int64_t total, int heads, int head_dim, float scale, void* out, void* rest, float* lse, void* stream);

/* Gradients for dout (dense, like out): dq, dk, dv (strides gld_t, gld_h) and dtable [n_buckets][heads] (dense; NULL = not
 * wanted).  ds = p (dout v^T - rowsum(dout (out + rest))) is rounded to the operands' type before the products with k and q. */
int64_t vdb_op_attention_backward_workspace_bytes(int dtype, int64_t n_seqs, int64_t total, int heads, int head_dim, int n_buckets);
int vdb_op_attention_backward_dev(int device, int dtype, const void* q, const void* k, const void* v, int64_t ld_t, int64_t ld_h,
                                  const void* table, int n_buckets, int max_distance, const int64_t* offsets, int64_t n_seqs,
                                  int64_t total, int heads, int head_dim, float scale, const void* out, const void* rest, const float* lse,
                                  const void* dout, void* dq, void* dk, void* dv, int64_t gld_t, int64_t gld_h, void* dtable,
                                  void* workspace, int64_t workspace_bytes, void* stream);

/* y[b] = mean of the hidden rows of sequence b, fp32 [n_seqs][dim], divided by max(its 2-norm, 1e-12) if normalize != 0:
 * what sentence-transformers' mean pooling and Normalize give, and what the store takes (vdb_add_dev).  A sequence
 * without rows gives zeros.  inv_norm (may be NULL): fp32 [n_seqs], 1 / max(norm, 1e-12), kept for the backward pass. */
int vdb_op_mean_pool_dev(int device, int dtype, const void* hidden, int64_t ld, const int64_t* offsets, int64_t n_seqs,
                         int64_t total, int64_t dim, int normalize, float* y, float* inv_norm, void* stream);
/* dhidden [total][dim] (dense) for dy fp32 [n_seqs][dim]. */
int vdb_op_mean_pool_backward_dev(int device, int dtype, const float* dy, const float* y, const float* inv_norm,
                                  const int64_t* offsets, int64_t n_seqs, int64_t total, int64_t dim, int normalize,
                                  void* dhidden, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* VDB_OPS_H */
