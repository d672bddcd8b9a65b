"""Plain 64-bit forms of the encoder operators with element-wise error bounds, for tests/test_gpu_ops.py.

Each function returns pairs (exact value, bound).  The bounds are derived, not tuned: u is half a step of the type that a
value is rounded to (torch.finfo(t).eps / 2), E = 2^-24 that of the 32-bit sums, and a sum of n products is off by at most
(n + 2) E sum |a b|.  Roundings to the 16-bit type inside the operators (the kept sum before an activation, dz, p, ds) count u
each; nothing else is rounded to 16 bits."""
import functools
import math

import torch

E = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half the distance between the type's smallest values: a rounding there is absolute."""
    return 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -126


def act(z, name):
    """value, slope, bound of |slope'|"""
    if name == "gelu":
        cdf, pdf = torch.special.ndtr(z), torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        return z * (1 + th) / 2, (1 + th) / 2 + z * (1 - th * th) / 2 * c * (1 + 3 * 0.044715 * z * z)
    if name == "relu":
        return z.clamp(min=0), (z > 0).double()
    return z, torch.ones_like(z)


def linear(x, w, b, name, r, dy=None):
    t = x.dtype
    u = half_step(t)
    x, w = x.double(), w.double()
    m, k = x.shape
    z = x @ w.t() + (0 if b is None else b.double())
    zb = (k + 4) * E * (x.abs() @ w.abs().t() + (0 if b is None else b.double().abs()))
    y, slope = act(z, name)
    # |slope| <= 1.13; the 32-bit evaluation of an activation is off by a few steps of |z|
    yb = 1.13 * zb + (0 if name == "none" else 16 * E * z.abs())
    if r is not None:
        y = y + r.double()
        yb = yb + E * y.abs()
    yb = yb + u * (y.abs() + yb) + tiny(t)
    if dy is None:
        return [(y, yb)]
    g = dy.double()
    dz = g * slope
    # slope' is at most 0.8 (gelu), 0.81 (its tanh form); z is kept rounded (the step of relu keeps its side: a sum does not round across 0)
    zerr = zb + (u * z.abs() + tiny(t) if name != "none" else 0)
    curved = name in ("gelu", "gelu_tanh")
    d32 = g.abs() * ((0.81 * zerr if curved else 0) + (24 * E * (1 + z.abs()) if curved else 0)) + E * dz.abs()
    dzb = d32 + (u * dz.abs() + tiny(t) if name != "none" else 0)
    dx, dw, db = dz @ w, dz.t() @ x, dz.sum(0)
    n = w.shape[0]
    dxb = dzb @ w.abs() + (n + 4) * E * (dz.abs() @ w.abs())
    dwb = dzb.t() @ x.abs() + (m + 4) * E * (dz.abs().t() @ x.abs())
    dbb = d32.sum(0) + (m + 4) * E * dz.abs().sum(0)
    return [(y, yb)] + [(v, e + u * (v.abs() + e) + tiny(t)) for v, e in ((dx, dxb), (dw, dwb), (db, dbb))]


def bucket(e, n_buckets, max_distance):
    half = n_buckets // 2
    near = half // 2
    n = abs(e)
    low = n if n < near else near + sum(n ** (half - near) >= near ** (half - near - i) * max_distance ** i for i in range(1, half - near))
    return low + (half if e > 0 else 0)


@functools.lru_cache(maxsize=64)
def buckets_of(n, n_buckets, max_distance):
    """[n, n] buckets of key - query."""
    line = torch.tensor([bucket(e, n_buckets, max_distance) for e in range(-n, n + 1)])
    place = torch.arange(n)
    return line[place[None, :] - place[:, None] + n]


def attention(qkv, table, ends, scale, max_distance, dout=None):
    """ends: the host list of offsets.  [(out, bound)] and, with dout, (dqkv, bound), (dtable, bound)."""
    t = qkv.dtype
    u = half_step(t)
    p16 = 0.0 if t == torch.float32 else u
    x, tab = qkv.double(), table.double()
    total, _, heads, d = x.shape
    out, outb = torch.zeros(total, heads, d, dtype=torch.float64), torch.zeros(total, heads, d, dtype=torch.float64)
    dx, dxb = torch.zeros_like(x), torch.zeros_like(x)
    dt, dtb = torch.zeros_like(tab), torch.zeros_like(tab)
    for lo, hi in zip(ends, ends[1:]):
        n = hi - lo
        if n <= 0:
            continue
        which = buckets_of(n, tab.shape[0], max_distance)
        for h in range(heads):
            q, k, v = (x[lo:hi, i, h] for i in range(3))
            s = scale * (q @ k.t()) + tab[:, h][which]
            p = torch.softmax(s, 1)
            # absolute error of a score, in the exponent (base 2 and back: a few more steps of its size)
            mag = scale * (q.abs() @ k.abs().t())
            finite = torch.where(p > 0, s, torch.zeros_like(s)).abs()      # a score whose p is 0 has no error to pass on
            es = ((d + 6) * E * mag + 8 * E * finite + 8 * E * finite.max(1, keepdim=True).values).max(1, keepdim=True).values
            ep = 2 * es + (n + 16) * E                                   # relative error of p in 32 bits
            o = p @ v
            ob = (ep + p16 + (n + 4) * E) * (p @ v.abs())
            kept = ob + p16 * u * o.abs() + (2.0 ** -25 if t == torch.float16 else 0)      # out and the rest of its rounding, rounded too
            ob = ob + u * (o.abs() + ob) + tiny(t)
            out[lo:hi, h], outb[lo:hi, h] = o, ob
            if dout is None:
                continue
            g = dout[lo:hi, h].double()
            dp = g @ v.t()
            delta = (g * o).sum(1, keepdim=True)
            eb = (d + 4) * E * (g.abs() @ v.abs().t()) + (g.abs() * kept).sum(1, keepdim=True) + (d + 4) * E * (g * o).abs().sum(1, keepdim=True)
            ds = p * (dp - delta)
            d32 = p * (eb + (ep + 2 * E) * ((dp - delta).abs() + eb))
            # one product of p and ds rounded, with the 16-bit type's own floor: fp16 lifts ds by a power of two, whose floor is
            # 2^-25 of at most 2 d max|dout| max|v| / 2^14
            floor = 0.0 if t != torch.float16 else 2.0 ** -25 * 4 * d * float(g.abs().max() * v.abs().max()) / 2 ** 14
            dsb = d32 + p16 * (ds.abs() + d32) + floor
            pb = p * (ep + p16) + (0 if t != torch.float16 else 2.0 ** -25)
            acc = (n + 4) * E
            for i, (val, err) in enumerate(((scale * ds @ k, scale * (dsb @ k.abs() + acc * (ds.abs() @ k.abs()))),
                                            (scale * ds.t() @ q, scale * (dsb.t() @ q.abs() + acc * (ds.abs().t() @ q.abs()))),
                                            (p.t() @ g, pb.t() @ g.abs() + acc * (p.t() @ g.abs())))):
                dx[lo:hi, i, h], dxb[lo:hi, i, h] = val, err + u * (val.abs() + err) + tiny(t)
            flat = which.reshape(-1)
            dt[:, h].index_add_(0, flat, ds.reshape(-1))
            dtb[:, h].index_add_(0, flat, (d32 + (n + 8) * E * ds.abs()).reshape(-1))
    if dout is None:
        return [(out, outb)]
    return [(out, outb), (dx, dxb), (dt, dtb + u * (dt.abs() + dtb) + tiny(t))]


def mean_pool(hidden, ends, normalize, dy=None):
    t = hidden.dtype
    u = half_step(t)
    x = hidden.double()
    b, dim = len(ends) - 1, x.shape[1]
    y, yb = torch.zeros(b, dim, dtype=torch.float64), torch.zeros(b, dim, dtype=torch.float64)
    dx, dxb = torch.zeros_like(x), torch.zeros_like(x)
    for i, (lo, hi) in enumerate(zip(ends, ends[1:])):
        if hi <= lo:
            continue
        n = hi - lo
        mean = x[lo:hi].mean(0)
        mb = (n + 4) * E * x[lo:hi].abs().mean(0)
        inv, invb = 1.0, 0.0
        if normalize:
            size = float(torch.linalg.vector_norm(mean))
            inv = 1 / max(size, 1e-12)
            # relative error of the norm: its sum of squares and the mean's own error
            invb = (dim + 8) * E + float(torch.linalg.vector_norm(mb)) * inv
        y[i] = mean * inv
        yb[i] = mb * inv + (invb + 4 * E) * y[i].abs() + 2.0 ** -126
        if dy is not None:
            g = dy[i].double()
            dot, project = float(y[i] @ g), normalize and inv < 1e12
            val = (g - (y[i] * dot if project else 0)) * inv / n
            err = ((yb[i] * abs(dot) + y[i].abs() * (float(yb[i] @ g.abs()) + (dim + 4) * E * float((y[i] * g).abs().sum())) if project else 0)
                   + 4 * E * (g.abs() + y[i].abs() * abs(dot))) * inv / n + (invb + 4 * E) * val.abs()
            dx[lo:hi], dxb[lo:hi] = val, err + u * (val.abs() + err) + tiny(t)
    return [(y, yb)] if dy is None else [(y, yb), (dx, dxb)]
