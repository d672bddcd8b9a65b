// k_attn.hip — launches of the attention operator.
#include <algorithm>
#include "op_attn.h"

namespace vdbk {
namespace {

// Waves per block (32 queries or keys each), by the average length, which is all the host knows: a block that is wider than its
// sequence leaves waves idle, one that is narrower loads the sequence's rows, and looks up its place and its bias, more often.
// Two waves and four, us, 12 heads.  Forward, bf16, heads of 64: 600 texts of 10 to 70 tokens 37 and 51, 64 each 43 and 49, 64 x 384
// 62 and 59, 4095 + 2564 + 1033 174 and 125; fp32, 600 of 40 to 104 232 and 226.  With the backward pass, bf16, heads of 64: 10 to 70
// 215 and 236, 64 each 326 and 296.  Only the 16-bit backward pass of heads of 128, whose tiles fill the LDS with two blocks, gains
// from more of them for longer: 100 x 256 521 and 622, 384 857 and 922, 500 to 1000 3213 and 2985.  One wave was slower everywhere.
int tile_waves(int dtype, int d, bool back, int64_t n_seqs, int64_t total) {
  const int64_t mean = n_seqs ? total / n_seqs : 0;
  return mean < (back && dtype != 0 && d > 64 ? 384 : 64) ? 2 : 4;
}

AttnParams params(const AttnArgs& a, int elem) {
  AttnParams p{};
  p.q = a.q; p.k = a.k; p.v = a.v; p.ld_t = a.ld_t; p.ld_h = a.ld_h; p.table = a.table; p.n_buckets = a.n_buckets;
  p.offsets = a.offsets; p.n_seqs = a.n_seqs; p.total = a.total; p.heads = a.heads; p.d = a.d; p.scale = a.scale;
  p.out = a.out; p.rest = a.rest; p.lse = a.lse; p.dout = a.dout; p.dq = a.dq; p.dk = a.dk; p.dv = a.dv; p.gld_t = a.gld_t; p.gld_h = a.gld_h;
  p.bk = a.bk;
  p.reach = a.bk.n_steps ? a.bk.step[a.bk.n_steps - 1] : a.bk.near;
  const int64_t v = 16 / elem;
  auto al = [](const void* x) { return ((uintptr_t)x & 15) == 0; };
  p.vec = al(a.q) && al(a.k) && al(a.v) && al(a.out) && al(a.rest) && al(a.dout) && al(a.dq) && al(a.dk) && al(a.dv) && a.d % v == 0 && a.ld_t % v == 0 &&
          a.ld_h % v == 0 && a.gld_t % v == 0 && a.gld_h % v == 0 && a.ld_t < ((int64_t)1 << 22);
  return p;
}

// A prime that divides neither length that an XCD's run of n blocks can have
unsigned hop_of(unsigned n) {
  for (unsigned h : {61u, 67u, 71u, 73u, 79u, 83u, 89u, 97u, 101u, 103u, 107u, 109u, 113u, 127u, 131u})
    if ((n >> 3) % h && ((n >> 3) + 1) % h) return h;
  return 1;
}

template <typename T, int DP, int NW>
hipError_t forward(const AttnParams& p, hipStream_t st) {
  const unsigned slots = (unsigned)n_slots(p.total, p.n_seqs, NW * 32), grid = slots * p.heads;
  if (p.vec && p.d == DP && even_scale(p.scale)) {
    attention_kernel<T, DP, NW><<<grid, NW * 64, start_span(p.reach) * sizeof(float), st>>>(p, slots, hop_of(grid));
    return hipGetLastError();
  }
  attention_any_kernel<T, DP, NW><<<grid, NW * 64, (2 * p.reach + 1) * sizeof(float), st>>>(p);
  return hipGetLastError();
}

// Which backward kernels serve.  fp32 heads of 128 stay with the general ones: two gradients and two operands of 128 words a row
// are more than the 512 registers of a lane.
template <typename T> bool tiled(const AttnParams& p) { return p.vec && even_scale(p.scale) && (p.d == 32 || p.d == 64 || (p.d == 128 && sizeof(T) == 2)); }

// Whether the tiled backward kernels take the longest sequences first (attention_order_kernel, one block: the sequences it can count,
// 3 to 8 us).  Without and with, us, 12 heads of 64, bf16: 64 texts of 16 to 384 tokens 121 and 111, 64 x 384 217 and 194, 32 x 64 to
// 128 36 and 32, 2000 + 4000 384 and 331; not for short texts, whose blocks are all alike (256 of 3 to 64 50 and 56, 200 of 30 to
// 60 63 and 68), nor where the blocks are fewer than two a compute unit (8 x 384: 396 blocks, 51 and 55).
bool by_length(int64_t n_seqs, int64_t total, int64_t slots, int heads) {
  return n_seqs > 1 && n_seqs <= kMaxOrdered && total >= 64 * n_seqs && slots <= 8192 && slots * heads >= 512;
}

template <typename T, int DP, int NW>
hipError_t backward(const AttnParams& p, const AttnArgs& a) {
  const int64_t slots = n_slots(p.total, p.n_seqs, NW * 32);
  const unsigned grid = (unsigned)(slots * p.heads);
  const size_t line = (2 * p.reach + 1) * sizeof(float), hist = (size_t)NW * 2 * sums_span(p.reach) * sizeof(float);
  hipError_t e;
  bool done = false;
  if constexpr (sizeof(T) * DP < 512) {
    if (tiled<T>(p)) {
      const size_t start = start_span(p.reach) * sizeof(float);
      if (p.order) {
        attention_order_kernel<<<1, 1024, 0, a.st>>>(p.offsets, (int)p.n_seqs, p.total, NW * 32, (int)slots, (i32x4*)a.order);
        if ((e = hipGetLastError()) != hipSuccess) return e;
      }
      if (a.dtable) attention_dq_kernel<T, DP, NW, true><<<grid, NW * 64, start + hist, a.st>>>(p, (unsigned)slots, hop_of(grid));
      else attention_dq_kernel<T, DP, NW, false><<<grid, NW * 64, start, a.st>>>(p, (unsigned)slots, hop_of(grid));
      if ((e = hipGetLastError()) != hipSuccess) return e;
      attention_dkv_kernel<T, DP, NW><<<grid, NW * 64, start, a.st>>>(p, (unsigned)slots, hop_of(grid));
      done = true;
    }
  }
  if (!done) {
    if (a.dtable) attention_dq_any_kernel<T, DP, NW, true><<<grid, NW * 64, line + hist, a.st>>>(p);
    else attention_dq_any_kernel<T, DP, NW, false><<<grid, NW * 64, line, a.st>>>(p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    attention_dkv_any_kernel<T, DP, NW><<<grid, NW * 64, line, a.st>>>(p);
  }
  if ((e = hipGetLastError()) != hipSuccess || !a.dtable) return e;
  attention_dtable_kernel<T><<<(unsigned)(p.heads * p.n_buckets), 256, 0, a.st>>>(p.part, slots, p.heads, p.n_buckets, (T*)a.dtable);
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t run_dp(const AttnParams& p, const AttnArgs& a, bool back) {
  switch (tile_waves(sizeof(T) == 4 ? 0 : 1, p.d, back, p.n_seqs, p.total)) {
    case 2: return back ? backward<T, DP, 2>(p, a) : forward<T, DP, 2>(p, a.st);
    default: return back ? backward<T, DP, 4>(p, a) : forward<T, DP, 4>(p, a.st);
  }
}

template <typename T>
hipError_t run_t(const AttnArgs& a, bool back) {
  AttnParams p = params(a, sizeof(T));
  p.delta = a.delta; p.from = a.from; p.fix = a.fix; p.part = a.part; p.peak = (const unsigned*)a.gscale; p.order = (const i32x4*)a.order;
  if (back) {
    const unsigned grid = (unsigned)(n_slots(p.total, p.n_seqs, 32) * p.heads);
    if (a.gscale) {
      const long long n = 2ll * p.heads * p.n_seqs;
      if (n) fill_zero_kernel<<<(unsigned)std::min<long long>((n + 255) / 256, 1024), 256, 0, a.st>>>((unsigned*)a.gscale, n);
      attention_delta_kernel<T, true><<<grid, 256, 0, a.st>>>(p, (unsigned*)a.gscale);
    } else if (!tiled<T>(p)) {
      attention_delta_kernel<T, false><<<grid, 256, 0, a.st>>>(p, nullptr);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return p.d <= 32 ? run_dp<T, 32>(p, a, back) : p.d <= 64 ? run_dp<T, 64>(p, a, back) : run_dp<T, 128>(p, a, back);
}

int64_t pad256(int64_t x) { return (x + 255) / 256 * 256; }
}  // namespace

hipError_t launch_attention(int dtype, const AttnArgs& a) {
  return dtype == 0 ? run_t<float>(a, false) : dtype == 1 ? run_t<__bf16>(a, false) : run_t<_Float16>(a, false);
}

int64_t attention_backward_workspace(int dtype, int64_t n_seqs, int64_t total, int heads, int d, int n_buckets) {
  const int64_t slots = n_slots(total, n_seqs, 32 * tile_waves(dtype, d, true, n_seqs, total));
  return 3 * pad256(total * heads * 4) + (dtype == 2 ? pad256(2 * n_seqs * heads * 4) : 0) + pad256(slots * heads * n_buckets * 4) +
         (by_length(n_seqs, total, slots, heads) ? pad256(slots * 16) : 0);
}

hipError_t launch_attention_backward(int dtype, AttnArgs a, char* ws) {
  a.delta = (float*)ws;
  ws += pad256(a.total * a.heads * 4);
  a.from = (float*)ws;
  ws += pad256(a.total * a.heads * 4);
  a.fix = (float*)ws;
  ws += pad256(a.total * a.heads * 4);
  a.gscale = nullptr;
  if (dtype == 2) { a.gscale = (float*)ws; ws += pad256(2 * a.n_seqs * a.heads * 4); }
  a.part = (float*)ws;
  const int64_t slots = n_slots(a.total, a.n_seqs, 32 * tile_waves(dtype, a.d, true, a.n_seqs, a.total));
  a.order = by_length(a.n_seqs, a.total, slots, a.heads) ? ws + pad256(slots * a.heads * a.n_buckets * 4) : nullptr;
  return dtype == 0 ? run_t<float>(a, true) : dtype == 1 ? run_t<__bf16>(a, true) : run_t<_Float16>(a, true);
}

}  // namespace vdbk
