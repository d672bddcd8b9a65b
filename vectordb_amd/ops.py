"""The text encoder's operators on the GPU, as differentiable functions of torch tensors (C ABI: include/vdb_ops.h).

The reference embeds its texts with sentence-transformers' all-mpnet-base-v2 (src/vectordb.py:13-69, src/config.py:36).
These are the operators such an encoder spends its time in; MPNetEmbedder(engine="hip") runs on them:

    linear              act(x W^T + b) + residual
    bucketed_attention  self-attention with a learned relative position bias by buckets
    mean_pool           a text's token rows -> one unit vector

Token rows are packed without padding: row tensors [total, ...] and ``offsets``, int64 [n_texts + 1] on the same GPU, text b
owning rows offsets[b] to offsets[b + 1] (offsets[0] is 0; a text may be empty; rows behind the last text come back as
zeros, and so do their gradients).  The offsets are read on the device: a captured graph may be replayed with others.

float32, bfloat16 and float16, one type per call; sums, softmax and norms are 32-bit.  Everything runs on the current stream of
the tensors' GPU, scratch comes from torch's allocator, nothing waits for the GPU, and results do not depend on timing.  There
is no CPU fallback: tensors elsewhere raise ValueError.  torch.autocast does not reach in here: cast first.  torch.jit.trace and make_fx
would record the outputs' allocation alone: under them the calls raise RuntimeError (torch.compile runs them as they are).  Calls can be captured
into HIP graphs; for a captured backward pass, take leaves of their own inside the capture (t.detach().requires_grad_()) and
torch.autograd.grad, as with any torch function: leaves that an eager graph holds as well accumulate on another stream."""
from __future__ import annotations

import functools
from typing import Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _capi

__all__ = ["linear", "bucketed_attention", "mean_pool", "ACTIVATIONS"]

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
#: names `linear` takes for its activation
ACTIVATIONS = {"none": 0, "gelu": 1, "gelu_tanh": 2, "relu": 3}


_lib = None


def _library():
    global _lib
    if _lib is None:
        _lib = _capi.load_library()
    return _lib


def _chk(rc: int) -> None:
    if rc != 0:
        _capi.check(_library(), None, rc)


#: the current stream's handle without building a Stream object: a call on one text is over in a few microseconds
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda device: torch.cuda.current_stream(device).cuda_stream)


@functools.lru_cache(maxsize=4096)
def _linear_scratch(dt: int, m: int, n: int, k: int) -> int:
    return _library().vdb_op_linear_workspace_bytes(dt, m, n, k)


def _scratch(n: int, like: torch.Tensor) -> Optional[torch.Tensor]:
    return torch.empty(n, dtype=torch.uint8, device=like.device) if n else None


def _ptr(t: Optional[torch.Tensor]):
    """An optional tensor's address.  One without memory (a freed storage, a wrapper around other tensors) is not an absent one."""
    if t is None:
        return None
    p = t.data_ptr()
    if not p and t.numel():
        raise ValueError(f"a tensor of shape {tuple(t.shape)} has no memory of its own")
    return p


_is_tracing, _modes, _key_included = torch._C._is_tracing, torch._C._len_torch_dispatch_stack, torch._C._dispatch_tls_is_dispatch_key_included
_PRE_DISPATCH = torch._C.DispatchKey.PreDispatch


def _refuse_tracing() -> None:
    """Tracers see torch's own operators only: what a kernel writes would be missing from the trace."""
    tracing = _is_tracing()
    if not tracing and (_modes() or _key_included(_PRE_DISPATCH)):
        from torch.fx.experimental.proxy_tensor import get_proxy_mode
        tracing = get_proxy_mode() is not None
    if tracing:
        raise RuntimeError("vectordb_amd.ops cannot be traced: torch.jit.trace and make_fx would record the output's allocation without the kernel that writes it")


def _first(t, name: str) -> int:
    """Check a call's leading tensor; -> the C ABI's number of its type."""
    _refuse_tracing()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor; got {type(t).__name__}")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU (there is no CPU fallback); got {t.device}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16; got {t.dtype}")
    return _DTYPES[t.dtype]


def _whole(t: torch.Tensor) -> torch.Tensor:
    """The tensor with its values in memory: a lazily negated view (x.conj().imag) holds them with the other sign."""
    return t.resolve_neg() if t.is_neg() else t


def _like(t, name: str, ref: torch.Tensor, shape) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor; got {type(t).__name__}")
    if t.device != ref.device or t.dtype != ref.dtype:
        raise ValueError(f"{name} must be {ref.dtype} on {ref.device}; got {t.dtype} on {t.device}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {tuple(shape)}; got {tuple(t.shape)}")


def _check_offsets(offsets, ref: torch.Tensor) -> torch.Tensor:
    if not isinstance(offsets, torch.Tensor):
        raise TypeError(f"offsets must be a torch.Tensor; got {type(offsets).__name__}")
    if offsets.device != ref.device or offsets.dtype != torch.int64 or offsets.dim() != 1 or offsets.shape[0] < 1:
        raise ValueError(f"offsets must be int64 [n_texts + 1] on {ref.device}; got {offsets.dtype} {tuple(offsets.shape)} on {offsets.device}")
    return offsets.contiguous()


def _rows(t: torch.Tensor) -> torch.Tensor:
    """A matrix whose rows are dense and do not overlap: itself, or a copy."""
    t = _whole(t)
    if t.is_contiguous():
        return t
    if t.stride(1) == 1 or t.shape[1] == 1:
        if t.stride(0) >= t.shape[1] or t.shape[0] <= 1:
            return t
    return t.contiguous()


def _ld(t: torch.Tensor) -> int:
    return max(t.stride(0), t.shape[1])


def _wants_grad(*tensors) -> bool:
    if getattr(forward_ad, "_current_level", -1) >= 0:      # dual numbers: the autograd function refuses them, a plain call would drop them
        return True
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- linear ----------------------------------------------------------------------------------------------------------

def _linear_forward(x, weight, bias, residual, act: int, keep_z: bool):
    lib = _library()
    dt = _DTYPES[x.dtype]
    m, k = x.shape
    n = weight.shape[0]
    y = torch.empty((m, n), dtype=x.dtype, device=x.device)
    z = torch.empty_like(y) if keep_z else None
    size = _linear_scratch(dt, m, n, k)
    ws = _scratch(size, x)
    _chk(lib.vdb_op_linear_dev(x.device.index, dt, x.data_ptr(), _ld(x), weight.data_ptr(), _ld(weight), _ptr(bias),
                               _ptr(residual), 0 if residual is None else _ld(residual), y.data_ptr(), n, _ptr(z), m, n, k, act,
                               _ptr(ws), size, _raw_stream(x.device.index)))
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        y, z = _linear_forward(x, weight, bias, residual, act, act != 0)
        ctx.act = act
        ctx.save_for_backward(x, weight, z)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dy = _rows(dy)
        dx = dw = db = None
        if need_x or need_w or need_b:
            lib = _library()
            dt = _DTYPES[x.dtype]
            (m, k), n = x.shape, weight.shape[0]
            dx = torch.empty((m, k), dtype=x.dtype, device=x.device) if need_x else None
            dw = torch.empty((n, k), dtype=x.dtype, device=x.device) if need_w else None
            db = torch.empty((n,), dtype=x.dtype, device=x.device) if need_b else None
            size = lib.vdb_op_linear_backward_workspace_bytes(dt, m, n, k, ctx.act)
            ws = _scratch(size, x)
            _chk(lib.vdb_op_linear_backward_dev(x.device.index, dt, dy.data_ptr(), _ld(dy), x.data_ptr(), _ld(x), weight.data_ptr(),
                                                _ld(weight), _ptr(z), _ptr(dx), _ptr(dw), _ptr(db), m, n, k, ctx.act, _ptr(ws), size,
                                                _raw_stream(x.device.index)))
        return dx, dw, db, dy if need_r else None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """act(x weight^T + bias) + residual, in one kernel, differentiable in x, weight, bias and residual.

    x [..., k]; weight [n, k]; bias [n]; residual [..., n]; all of x's type and on x's GPU.  activation: "none", "gelu" (by
    the error function), "gelu_tanh" or "relu".  Rows may be strided; a tensor whose last dimension is not dense is copied.
    With an activation and a gradient wanted, the sum before the activation is kept in x's type, and so is its gradient
    before the products of the backward pass."""
    _first(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"x must have shape [..., k] with k >= 1; got {tuple(x.shape)}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(ACTIVATIONS)}; got {activation!r}")
    k = x.shape[-1]
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2 or weight.shape[0] < 1:
        raise ValueError("weight must be a tensor of shape [n, k] with n >= 1")
    n = weight.shape[0]
    _like(weight, "weight", x, (n, k))
    lead = tuple(x.shape[:-1])
    if bias is not None:
        _like(bias, "bias", x, (n,))
    if residual is not None:
        _like(residual, "residual", x, (*lead, n))
    flat = x.dim() == 2
    x2 = _rows(x if flat else x.reshape(-1, k))
    w2 = _rows(weight)
    b2 = None if bias is None else _whole(bias).contiguous()
    r2 = None if residual is None else _rows(residual if flat else residual.reshape(-1, n))
    act = ACTIVATIONS[activation]
    if _wants_grad(x, weight, bias, residual):
        y = _Linear.apply(x2, w2, b2, r2, act)
    else:
        y = _linear_forward(x2, w2, b2, r2, act, False)[0]
    return y if flat else y.reshape(*lead, n)


# ---- attention ---------------------------------------------------------------------------------------------------------

def _attention_args(qkv, table, offsets, scale, max_distance):
    total, _, heads, d = qkv.shape
    base, step = qkv.data_ptr(), qkv.stride(1) * qkv.element_size()
    # a single row's stride says nothing
    ld_t = qkv.stride(0) if total > 1 else 3 * heads * d
    ld_h = qkv.stride(2) if heads > 1 else d
    return (qkv.device.index, _DTYPES[qkv.dtype], base, base + step, base + 2 * step, ld_t, ld_h, table.data_ptr(), table.shape[0], max_distance,
            offsets.data_ptr(), offsets.shape[0] - 1, total, heads, d, scale)


def _attention_forward(qkv, table, offsets, scale, max_distance, keep: bool):
    lib = _library()
    total, _, heads, d = qkv.shape
    out = torch.empty((total, heads, d), dtype=qkv.dtype, device=qkv.device)
    lse = torch.empty((heads, total), dtype=torch.float32, device=qkv.device) if keep else None
    rest = torch.empty_like(out) if keep and qkv.dtype != torch.float32 else None
    _chk(lib.vdb_op_attention_dev(*_attention_args(qkv, table, offsets, scale, max_distance), out.data_ptr(), _ptr(rest), _ptr(lse), _raw_stream(qkv.device.index)))
    return out, rest, lse


class _BucketedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, table, offsets, scale, max_distance):
        out, rest, lse = _attention_forward(qkv, table, offsets, scale, max_distance, True)
        ctx.scale, ctx.max_distance = scale, max_distance
        ctx.save_for_backward(qkv, table, offsets, out, rest, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        qkv, table, offsets, out, rest, lse = ctx.saved_tensors
        lib = _library()
        total, _, heads, d = qkv.shape
        dout = _whole(dout).contiguous()
        dqkv = torch.empty((total, 3, heads, d), dtype=qkv.dtype, device=qkv.device)
        dtable = torch.empty_like(table) if ctx.needs_input_grad[1] else None
        size = lib.vdb_op_attention_backward_workspace_bytes(_DTYPES[qkv.dtype], offsets.shape[0] - 1, total, heads, d, table.shape[0])
        ws = _scratch(size, qkv)
        base, step = dqkv.data_ptr(), heads * d * dqkv.element_size()
        _chk(lib.vdb_op_attention_backward_dev(*_attention_args(qkv, table, offsets, ctx.scale, ctx.max_distance), out.data_ptr(), _ptr(rest), lse.data_ptr(),
                                               dout.data_ptr(), base, base + step, base + 2 * step, 3 * heads * d, d, _ptr(dtable),
                                               _ptr(ws), size, _raw_stream(qkv.device.index)))
        return dqkv if ctx.needs_input_grad[0] else None, dtable, None, None, None


def bucketed_attention(qkv: torch.Tensor, table: torch.Tensor, offsets: torch.Tensor, scale: Optional[float] = None,
                       max_distance: int = 128) -> torch.Tensor:
    """Self-attention within each text: out_i = sum_j softmax_j(scale q_i.k_j + table[bucket(j - i), head]) v_j, [total, heads, d].

    qkv [total, 3, heads, d], d <= 128 (tokens, the three and heads may be strided); table [n_buckets, heads], n_buckets even, 4 to
    128; both of one type.  scale: default d ** -0.5.  Buckets: the lower half for keys at or before the query, the upper half
    for keys behind it; in each, a quarter of n_buckets for the nearest distances one by one, the others growing by equal ratios
    up to max_distance (at most 512), beyond which the last holds.  Differentiable in qkv and table; only bucket sums of the
    scores' gradient leave the kernel, never a [length, length] matrix."""
    _first(qkv, "qkv")
    if qkv.dim() != 4 or qkv.shape[1] != 3 or qkv.shape[2] < 1 or not 1 <= qkv.shape[3] <= 128:
        raise ValueError(f"qkv must have shape [total, 3, heads, d] with d from 1 to 128; got {tuple(qkv.shape)}")
    total, _, heads, d = qkv.shape
    if not isinstance(table, torch.Tensor) or table.dim() != 2:
        raise ValueError("table must be a tensor of shape [n_buckets, heads]")
    _like(table, "table", qkv, (table.shape[0], heads))
    offsets = _check_offsets(offsets, qkv)
    scale = float(d) ** -0.5 if scale is None else float(scale)
    if qkv.stride(3) != 1 and d > 1 or min(qkv.stride()) < 0 or (heads > 1 and qkv.stride(2) < d):
        qkv = qkv.contiguous()
    qkv, table = _whole(qkv), _whole(table).contiguous()
    if _wants_grad(qkv, table):
        return _BucketedAttention.apply(qkv, table, offsets, scale, int(max_distance))
    return _attention_forward(qkv, table, offsets, scale, int(max_distance), False)[0]


# ---- pooling -----------------------------------------------------------------------------------------------------------

def _pool_forward(hidden, offsets, normalize: bool, keep: bool):
    lib = _library()
    total, dim = hidden.shape
    n = offsets.shape[0] - 1
    y = torch.empty((n, dim), dtype=torch.float32, device=hidden.device)
    inv = torch.empty((n,), dtype=torch.float32, device=hidden.device) if keep and normalize else None
    _chk(lib.vdb_op_mean_pool_dev(hidden.device.index, _DTYPES[hidden.dtype], hidden.data_ptr(), _ld(hidden), offsets.data_ptr(), n, total, dim,
                                  int(normalize), y.data_ptr(), _ptr(inv), _raw_stream(hidden.device.index)))
    return y, inv


class _MeanPool(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, offsets, normalize):
        y, inv = _pool_forward(hidden, offsets, normalize, True)
        ctx.normalize, ctx.total, ctx.dtype = normalize, hidden.shape[0], hidden.dtype
        ctx.save_for_backward(y, inv, offsets)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        y, inv, offsets = ctx.saved_tensors
        n, dim = y.shape
        dy = _whole(dy).contiguous()
        dh = torch.empty((ctx.total, dim), dtype=ctx.dtype, device=y.device)
        _chk(_library().vdb_op_mean_pool_backward_dev(y.device.index, _DTYPES[ctx.dtype], dy.data_ptr(), y.data_ptr(), _ptr(inv), offsets.data_ptr(), n,
                                                      ctx.total, dim, int(ctx.normalize), dh.data_ptr(), _raw_stream(y.device.index)))
        return dh, None, None


def mean_pool(hidden: torch.Tensor, offsets: torch.Tensor, normalize: bool = True) -> torch.Tensor:
    """float32 [n_texts, dim]: the mean of each text's rows of hidden [total, dim], divided by its 2-norm (at least 1e-12) unless
    normalize is false.  An empty text gives zeros.  Differentiable in hidden.  The result can go into the store as it is
    (Collection.add takes it in place)."""
    _first(hidden, "hidden")
    if hidden.dim() != 2 or hidden.shape[1] < 1:
        raise ValueError(f"hidden must have shape [total, dim] with dim >= 1; got {tuple(hidden.shape)}")
    offsets = _check_offsets(offsets, hidden)
    h = _rows(hidden)
    if _wants_grad(hidden):
        return _MeanPool.apply(h, offsets, bool(normalize))
    return _pool_forward(h, offsets, bool(normalize), False)[0]
