// ops_api.hip — C ABI of the encoder operators (include/vdb_ops.h): argument checks, scratch layout, launches.
#include <cmath>
#include <string>
#include "../../include/vdb.h"
#include "../../include/vdb_ops.h"
#include "ops.h"

using namespace vdbk;

namespace {

// a launch has fewer than 2^32 threads along a dimension: 2^24 blocks of 256
constexpr int64_t kMaxRows = (int64_t)1 << 29, kMaxWidth = (int64_t)1 << 20, kMaxBlocks = ((int64_t)1 << 24) - 1;

int bad(int code, const char* what) {
  set_last_error(what);
  return code;
}
int hip_fail(const char* where, hipError_t e) {
  char msg[256];
  snprintf(msg, sizeof msg, "%s: %s", where, hipGetErrorString(e));
  (void)hipGetLastError();     // reported here: the next launch on this thread, whoever's, must not find it again
  return bad(e == hipErrorOutOfMemory ? VDB_ERR_MEMORY : VDB_ERR_DEVICE, msg);
}
#define NEED(cond, what) do { if (!(cond)) return bad(VDB_ERR_ARG, what); } while (0)

// The call's device for its duration; the caller's current device comes back.
struct OnDevice {
  int before = -1; hipError_t err;
  explicit OnDevice(int device) {
    err = hipGetDevice(&before);
    if (err == hipSuccess && before != device) err = hipSetDevice(device);
    else if (err == hipSuccess) before = -1;
  }
  ~OnDevice() { if (before >= 0) (void)hipSetDevice(before); }
};
#define ON_DEVICE(where) \
  OnDevice on(device); \
  if (on.err != hipSuccess) return hip_fail(where, on.err)

int64_t pad256(int64_t x) { return (x + 255) / 256 * 256; }
int elem_size(int dtype) { return dtype == VDB_OP_F32 ? 4 : 2; }
bool known(int dtype) { return dtype >= VDB_OP_F32 && dtype <= VDB_OP_F16; }
bool widths(int64_t m, int64_t n, int64_t k) { return m >= 0 && m <= kMaxRows && n >= 1 && n <= kMaxWidth && k >= 1 && k <= kMaxWidth; }

// n^wide >= near^(wide - i) max_distance^i, in whole numbers of as many 32-bit digits as it takes
struct Big {
  uint32_t d[72]; int n = 1;
  Big() { d[0] = 1; }
  void times(uint32_t f) {
    uint64_t c = 0;
    for (int i = 0; i < n; ++i) { c += (uint64_t)d[i] * f; d[i] = (uint32_t)c; c >>= 32; }
    if (c) d[n++] = (uint32_t)c;
  }
  bool at_least(const Big& o) const {
    if (n != o.n) return n > o.n;
    for (int i = n - 1; i >= 0; --i) if (d[i] != o.d[i]) return d[i] > o.d[i];
    return true;
  }
};
Buckets make_buckets(int n_buckets, int max_distance) {
  thread_local Buckets b{};
  thread_local int have_buckets = 0, have_distance = 0;
  if (have_buckets == n_buckets && have_distance == max_distance) return b;   // a model asks for one set, layer after layer
  have_buckets = n_buckets;
  have_distance = max_distance;
  b = Buckets{};
  b.half = n_buckets / 2;
  b.near = b.half / 2;
  const int wide = b.half - b.near;
  b.n_steps = wide - 1;
  int n = b.near;
  for (int i = 1; i < wide; ++i) {
    Big want;
    for (int t = 0; t < wide; ++t) want.times((uint32_t)(t < i ? max_distance : b.near));
    for (;; ++n) {
      Big have;
      for (int t = 0; t < wide; ++t) have.times((uint32_t)n);
      if (have.at_least(want)) break;
    }
    b.step[i - 1] = n;
  }
  for (int i = b.n_steps; i < kMaxSteps; ++i) b.step[i] = 0x7fffffff;
  return b;
}

int check_attention(int dtype, const void* q, const void* k, const void* v, int64_t ld_t, int64_t ld_h, const void* table, int n_buckets,
                    int max_distance, const int64_t* offsets, int64_t n_seqs, int64_t total, int heads, int d, float scale) {
  NEED(known(dtype), "attention: dtype must be VDB_OP_F32, VDB_OP_BF16 or VDB_OP_F16");
  NEED(n_seqs >= 0 && n_seqs <= kMaxRows && total >= 0 && total <= kMaxRows, "attention: n_seqs and total must be in [0, 2^29]");
  NEED(heads >= 1 && heads <= 1024, "attention: heads must be in [1, 1024]");
  NEED(d >= 1 && d <= VDB_OP_MAX_HEAD_DIM, "attention: head_dim must be in [1, 128]");
  NEED(n_buckets >= 4 && n_buckets <= VDB_OP_MAX_BUCKETS && n_buckets % 2 == 0, "attention: n_buckets must be even and in [4, 128]");
  NEED(max_distance > n_buckets / 4 && max_distance <= VDB_OP_MAX_DISTANCE, "attention: max_distance must be in (n_buckets / 4, 512]");
  NEED(std::isfinite(scale) && scale > 0.f, "attention: scale must be positive and finite");
  NEED((total / 32 + n_seqs + 1) * heads <= kMaxBlocks, "attention: too many sequences, rows and heads for one launch");
  NEED(total == 0 || (q && k && v && table && offsets), "attention: a pointer is NULL");
  NEED(total == 0 || (ld_t >= 0 && ld_h >= 0), "attention: strides must not be negative");
  return VDB_OK;
}

}  // namespace

extern "C" {

int64_t vdb_op_linear_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k) {
  if (!known(dtype) || !widths(m, n, k)) return 0;
  return gemm_workspace_bytes(dtype, false, false, m, n, k);
}

int vdb_op_linear_dev(int device, int dtype, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias, const void* residual,
                      int64_t ldr, void* y, int64_t ldy, void* z, int64_t m, int64_t n, int64_t k, int act, void* workspace,
                      int64_t workspace_bytes, void* stream) {
  NEED(known(dtype), "linear: dtype must be VDB_OP_F32, VDB_OP_BF16 or VDB_OP_F16");
  NEED(widths(m, n, k), "linear: m must be in [0, 2^29], n and k in [1, 2^20]");
  NEED(act >= VDB_ACT_NONE && act <= VDB_ACT_RELU, "linear: unknown activation");
  if (m == 0) return VDB_OK;
  NEED(x && w && y, "linear: a pointer is NULL");
  NEED(ldx >= k && ldw >= k && ldy >= n && (!residual || ldr >= n), "linear: a row stride is smaller than its row");
  NEED(workspace_bytes >= gemm_workspace_bytes(dtype, false, false, m, n, k), "linear: the workspace is too small");
  NEED(workspace || gemm_workspace_bytes(dtype, false, false, m, n, k) == 0, "linear: the workspace is NULL");
  ON_DEVICE("linear");
  GemmArgs a{};
  a.a = x; a.lda = ldx; a.b = w; a.ldb = ldw; a.m = m; a.n = n; a.k = k; a.y = y; a.ldy = ldy; a.bias = bias; a.act = act;
  a.residual = residual; a.ldr = ldr; a.z = z; a.partial = (float*)workspace; a.partial_bytes = workspace_bytes; a.st = (hipStream_t)stream;
  const hipError_t e = launch_gemm(dtype, a);
  return e == hipSuccess ? VDB_OK : hip_fail("linear", e);
}

// scratch of the backward pass: dz, the column sums' parts, and the products' split outputs (one after the other)
static void backward_pieces(int dtype, int64_t m, int64_t n, int64_t k, int act, int64_t* dz, int64_t* cols, int64_t* split) {
  *dz = act == VDB_ACT_NONE ? 0 : pad256(m * n * elem_size(dtype));
  *cols = pad256((int64_t)act_grad_parts(m, n) * n * 4);
  const int64_t s1 = gemm_workspace_bytes(dtype, false, true, m, k, n), s2 = gemm_workspace_bytes(dtype, true, true, n, k, m);
  *split = s1 > s2 ? s1 : s2;
}

int64_t vdb_op_linear_backward_workspace_bytes(int dtype, int64_t m, int64_t n, int64_t k, int act) {
  if (!known(dtype) || !widths(m, n, k)) return 0;
  int64_t dz, cols, split;
  backward_pieces(dtype, m, n, k, act, &dz, &cols, &split);
  return dz + cols + split;
}

int vdb_op_linear_backward_dev(int device, int dtype, const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw,
                               const void* z, void* dx, void* dw, void* db, int64_t m, int64_t n, int64_t k, int act, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  NEED(known(dtype), "linear_backward: dtype must be VDB_OP_F32, VDB_OP_BF16 or VDB_OP_F16");
  NEED(widths(m, n, k), "linear_backward: m must be in [0, 2^29], n and k in [1, 2^20]");
  NEED(act >= VDB_ACT_NONE && act <= VDB_ACT_RELU, "linear_backward: unknown activation");
  NEED(m == 0 || dy, "linear_backward: dy is NULL");
  NEED(m == 0 || ((!dw || x) && (!dx || w)), "linear_backward: x is needed for dw, w for dx");
  NEED(m == 0 || act == VDB_ACT_NONE || z, "linear_backward: z is needed with an activation");
  NEED(lddy >= n && (!dw || ldx >= k) && (!dx || ldw >= k), "linear_backward: a row stride is smaller than its row");
  int64_t dz_b, cols_b, split_b;
  backward_pieces(dtype, m, n, k, act, &dz_b, &cols_b, &split_b);
  NEED(workspace && workspace_bytes >= dz_b + cols_b + split_b, "linear_backward: the workspace is too small");
  ON_DEVICE("linear_backward");
  char* ws = (char*)workspace;
  hipStream_t st = (hipStream_t)stream;
  hipError_t e;
  if (act != VDB_ACT_NONE || db) {
    ActGradArgs g{dy, lddy, z, act, m, n, act != VDB_ACT_NONE ? (void*)ws : nullptr, db, (float*)(ws + dz_b), st};
    if ((e = launch_act_grad(dtype, g)) != hipSuccess) return hip_fail("linear_backward", e);
  }
  const void* dz = act != VDB_ACT_NONE ? (const void*)ws : dy;
  const int64_t lddz = act != VDB_ACT_NONE ? n : lddy;
  GemmArgs a{};
  a.partial = (float*)(ws + dz_b + cols_b); a.partial_bytes = split_b; a.st = st;
  if (dx && m > 0) {
    a.a = dz; a.lda = lddz; a.a_t = false; a.b = w; a.ldb = ldw; a.b_t = true; a.m = m; a.n = k; a.k = n; a.y = dx; a.ldy = k;
    if ((e = launch_gemm(dtype, a)) != hipSuccess) return hip_fail("linear_backward", e);
  }
  if (dw) {
    a.a = dz; a.lda = lddz; a.a_t = true; a.b = x; a.ldb = ldx; a.b_t = true; a.m = n; a.n = k; a.k = m; a.y = dw; a.ldy = k;
    if ((e = launch_gemm(dtype, a)) != hipSuccess) return hip_fail("linear_backward", e);
  }
  return VDB_OK;
}

int vdb_op_attention_dev(int device, int dtype, const void* q, const void* k, const void* v, int64_t ld_t, int64_t ld_h, const void* table,
                         int n_buckets, int max_distance, const int64_t* offsets, int64_t n_seqs, int64_t total, int heads, int head_dim,
                         float scale, void* out, void* rest, float* lse, void* stream) {
  const int rc = check_attention(dtype, q, k, v, ld_t, ld_h, table, n_buckets, max_distance, offsets, n_seqs, total, heads, head_dim, scale);
  if (rc) return rc;
  if (total == 0) return VDB_OK;
  NEED(out, "attention: out is NULL");
  ON_DEVICE("attention");
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.ld_t = ld_t; a.ld_h = ld_h; a.table = table; a.n_buckets = n_buckets; a.bk = make_buckets(n_buckets, max_distance);
  a.offsets = offsets; a.n_seqs = n_seqs; a.total = total; a.heads = heads; a.d = head_dim; a.scale = scale; a.out = out; a.rest = rest; a.lse = lse;
  a.st = (hipStream_t)stream;
  const hipError_t e = launch_attention(dtype, a);
  return e == hipSuccess ? VDB_OK : hip_fail("attention", e);
}

int64_t vdb_op_attention_backward_workspace_bytes(int dtype, int64_t n_seqs, int64_t total, int heads, int head_dim, int n_buckets) {
  if (!known(dtype) || n_seqs < 0 || total < 0 || heads < 1 || n_buckets < 1 || n_seqs > kMaxRows || total > kMaxRows) return 0;
  return attention_backward_workspace(dtype, n_seqs, total, heads, head_dim, n_buckets);
}

int vdb_op_attention_backward_dev(int device, int dtype, const void* q, const void* k, const void* v, int64_t ld_t, int64_t ld_h,
                                  const void* table, int n_buckets, int max_distance, const int64_t* offsets, int64_t n_seqs, int64_t total,
                                  int heads, int head_dim, float scale, const void* out, const void* rest, const float* lse, const void* dout, void* dq, void* dk,
                                  void* dv, int64_t gld_t, int64_t gld_h, void* dtable, void* workspace, int64_t workspace_bytes, void* stream) {
  const int rc = check_attention(dtype, q, k, v, ld_t, ld_h, table, n_buckets, max_distance, offsets, n_seqs, total, heads, head_dim, scale);
  if (rc) return rc;
  NEED(total == 0 || (out && lse && dout && dq && dk && dv), "attention_backward: a pointer is NULL");
  NEED(gld_t >= 0 && gld_h >= 0, "attention_backward: strides must not be negative");
  NEED(workspace && workspace_bytes >= attention_backward_workspace(dtype, n_seqs, total, heads, head_dim, n_buckets),
       "attention_backward: the workspace is too small");
  ON_DEVICE("attention_backward");
  AttnArgs a{};
  a.q = q; a.k = k; a.v = v; a.ld_t = ld_t; a.ld_h = ld_h; a.table = table; a.n_buckets = n_buckets; a.bk = make_buckets(n_buckets, max_distance);
  a.offsets = offsets; a.n_seqs = total ? n_seqs : 0; a.total = total; a.heads = heads; a.d = head_dim; a.scale = scale; a.out = (void*)out; a.rest = (void*)rest; a.lse = (float*)lse;
  a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv; a.gld_t = gld_t; a.gld_h = gld_h; a.dtable = dtable; a.st = (hipStream_t)stream;
  const hipError_t e = launch_attention_backward(dtype, a, (char*)workspace);
  return e == hipSuccess ? VDB_OK : hip_fail("attention_backward", e);
}

int vdb_op_mean_pool_dev(int device, int dtype, const void* hidden, int64_t ld, const int64_t* offsets, int64_t n_seqs, int64_t total,
                         int64_t dim, int normalize, float* y, float* inv_norm, void* stream) {
  NEED(known(dtype), "mean_pool: dtype must be VDB_OP_F32, VDB_OP_BF16 or VDB_OP_F16");
  NEED(n_seqs >= 0 && n_seqs <= kMaxBlocks && total >= 0 && total <= kMaxRows && dim >= 1 && dim <= kMaxWidth,
       "mean_pool: n_seqs must be in [0, 2^24), total in [0, 2^29], dim in [1, 2^20]");
  if (n_seqs == 0) return VDB_OK;
  NEED(offsets && y && (hidden || total == 0), "mean_pool: a pointer is NULL");
  NEED(ld >= dim, "mean_pool: the row stride is smaller than a row");
  ON_DEVICE("mean_pool");
  PoolArgs a{hidden, ld, offsets, n_seqs, total, dim, normalize, y, inv_norm, nullptr, nullptr, (hipStream_t)stream};
  const hipError_t e = launch_mean_pool(dtype, a);
  return e == hipSuccess ? VDB_OK : hip_fail("mean_pool", e);
}

int vdb_op_mean_pool_backward_dev(int device, int dtype, const float* dy, const float* y, const float* inv_norm, const int64_t* offsets,
                                  int64_t n_seqs, int64_t total, int64_t dim, int normalize, void* dhidden, void* stream) {
  NEED(known(dtype), "mean_pool_backward: dtype must be VDB_OP_F32, VDB_OP_BF16 or VDB_OP_F16");
  NEED(n_seqs >= 0 && total >= 0 && total <= kMaxRows && n_seqs <= kMaxBlocks - 1 - total / 32 && dim >= 1 && dim <= kMaxWidth,
       "mean_pool_backward: n_seqs + total / 32 must be below 2^24, dim in [1, 2^20]");
  if (total == 0) return VDB_OK;
  NEED(offsets && dhidden && (n_seqs == 0 || (dy && y && (inv_norm || !normalize))), "mean_pool_backward: a pointer is NULL");
  ON_DEVICE("mean_pool_backward");
  PoolArgs a{nullptr, 0, offsets, n_seqs, total, dim, normalize, (float*)y, (float*)inv_norm, dy, dhidden, (hipStream_t)stream};
  const hipError_t e = launch_mean_pool_backward(dtype, a);
  return e == hipSuccess ? VDB_OK : hip_fail("mean_pool_backward", e);
}

}  // extern "C"
