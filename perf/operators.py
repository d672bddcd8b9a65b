"""What is measured of the text encoder's operators (vectordb_amd.ops): the cases, their inputs, the plain forms
and the definitions in 64 bits.

Three operators carry the embedding model behind the embed_fn seam, on token rows packed without padding:

  linear              y = act(x W^T + b) + r, and the gradients of x, W, b and r
  bucketed_attention  softmax(scale q k^T + bias) v over each sequence, the bias learned per head and per bucket of
                      the distance between key and query, and the gradients of q, k, v and the table
  mean_pool           the mean over a sequence's rows, scaled to unit length, and the rows' gradient

`own` is False: run() computes the plain form.  True: run() calls vectordb_amd.ops."""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}
BUCKETS, DISTANCE = 32, 128


def listed():
    return [
        # one product description asked for: the fused query/key/value projection of a 768-wide encoder, latency counts
        dict(name="linear one text bf16", op="linear", dtype="bf16", m=14, n=2304, k=768, act="none", residual=False, train=False),
        # an odd number of packed tokens through the widening layer of a 384-wide encoder
        dict(name="linear ragged gelu f16", op="linear", dtype="f16", m=1999, n=1536, k=384, act="gelu", residual=False, train=False),
        # the embedder's default precision: attention output projection with the residual, 64 texts of 96 tokens
        dict(name="linear residual f32", op="linear", dtype="f32", m=6144, n=768, k=768, act="none", residual=True, train=False),
        # a catalogue being indexed: 128 texts at the embedder's greatest length
        dict(name="linear full batch bf16", op="linear", dtype="bf16", m=49152, n=2304, k=768, act="none", residual=False, train=False),
        # fine-tuning: widening layer, forward and all gradients
        dict(name="linear train gelu bf16", op="linear", dtype="bf16", m=8192, n=1536, k=768, act="gelu", residual=False, train=True),
        # one product description
        dict(name="attention one text bf16", op="attention", dtype="bf16", b=1, lo=14, hi=14, spare=0, h=12, d=64, train=False),
        # a batch of short descriptions, ragged, in a buffer larger than they are
        dict(name="attention ragged f16", op="attention", dtype="f16", b=512, lo=3, hi=64, spare=61, h=12, d=32, train=False),
        # the default precision at the embedder's greatest length
        dict(name="attention full f32", op="attention", dtype="f32", b=16, lo=384, hi=384, spare=0, h=12, d=64, train=False),
        # whole documents, of odd lengths
        dict(name="attention long bf16", op="attention", dtype="bf16", b=3, lo=1033, hi=4095, spare=0, h=12, d=64, train=False),
        # fine-tuning on ragged texts: forward and all gradients
        dict(name="attention train bf16", op="attention", dtype="bf16", b=64, lo=16, hi=384, spare=0, h=12, d=64, train=True),
        # one product description's embedding
        dict(name="pool one text f32", op="pool", dtype="f32", b=1, lo=14, hi=14, spare=0, dim=768, train=False),
        # fine-tuning: embeddings of a ragged batch and the gradient of their token rows
        dict(name="pool train bf16", op="pool", dtype="bf16", b=1024, lo=3, hi=128, spare=0, dim=768, train=True),
    ]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "attention", "attention", "pool"])
    dtype, train = rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.4
    if op == "linear":
        while True:
            m, n, k = _spread(rng, 1, 49152), _spread(rng, 16, 2304), _spread(rng, 16, 2304)
            if rng.random() < 0.7:                       # most layers are whole multiples of eight wide, not all
                n, k = -(-n // 8) * 8, -(-k // 8) * 8
            if m * n * k * (3 if train else 1) <= 4e10:
                break
        # relu's slope has a step at 0, and which side a 32-bit sum next to it falls on is the summing order's, not the operator's
        acts = ["none", "gelu", "gelu_tanh"] + (["relu"] if not (train and dtype == "f32") else [])
        return dict(op=op, dtype=dtype, m=m, n=n, k=k, act=rng.choice(acts),
                    residual=rng.random() < 0.5, train=train)
    if op == "attention":
        while True:
            b, hi, h, d = _spread(rng, 1, 512), _spread(rng, 1, 4095), rng.choice([1, 4, 6, 12, 16]), rng.choice([8, 24, 32, 64, 64, 80, 128])
            if b * h * hi * hi <= (1e8 if train else 4e8):
                break
        return dict(op=op, dtype=dtype, b=b, lo=rng.randint(0, hi), hi=hi, spare=rng.choice([0, 0, 5, 130]), h=h, d=d, train=train)
    while True:
        b, hi, dim = _spread(rng, 1, 2048), _spread(rng, 1, 512), _spread(rng, 8, 1500)
        if b * hi * dim <= 1.1e8:
            break
    return dict(op=op, dtype=dtype, b=b, lo=rng.randint(0, hi), hi=hi, spare=rng.choice([0, 0, 7]), dim=dim, train=train)


def _lengths(case):
    """Lengths spread evenly from hi down to lo; prepare() puts them in an order of its own."""
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(1, b - 1) for i in range(b)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, train = DTYPES[case["dtype"]], case["train"]

    def normal(*shape, scale=1.0, grad=train):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dt).requires_grad_(grad)

    s = dict(op=case["op"], train=train)
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        s.update(x=normal(m, k), weight=normal(n, k, scale=k ** -0.5), bias=normal(n, scale=0.1), activation=case["act"],
                 residual=normal(m, n) if case["residual"] else None, dy=normal(m, n, grad=False) if train else None)
        return s
    lengths = torch.tensor(_lengths(case))[torch.randperm(case["b"], generator=torch.Generator().manual_seed(seed))]
    offsets = torch.zeros(case["b"] + 1, dtype=torch.int64)
    offsets[1:] = lengths.cumsum(0)
    t = int(offsets[-1]) + case["spare"]
    s.update(offsets=offsets.cuda(), longest=case["hi"])
    if case["op"] == "attention":
        h, d = case["h"], case["d"]
        # as the fused projection leaves them: one row a token, the three side by side
        qkv = normal(t, 3, h, d)
        s.update(qkv=qkv, table=normal(BUCKETS, h), dy=normal(t, h, d, grad=False) if train else None)
    else:
        s.update(hidden=normal(t, case["dim"]), dy=torch.randn(case["b"], case["dim"], generator=g, device="cuda") if train else None)
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------

def _padded_rows(offsets, longest, total):
    """[b, longest] row numbers of the packed tokens; a place behind a sequence's end holds `total`."""
    place = torch.arange(longest, device=offsets.device)
    rows = offsets[:-1, None] + place
    return torch.where(rows < offsets[1:, None], rows, total)


def _plain_act(z, name):
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    return torch.clamp(z, min=0) if name == "relu" else z


def _plain_linear(x, weight, bias, activation, residual):
    y = _plain_act(x.float() @ weight.float().t() + bias.float(), activation)
    if residual is not None:
        y = y + residual.float()
    return y.to(x.dtype)


def _thresholds():
    """Smallest distance of each bucket on the logarithmic half, found with whole numbers."""
    half = BUCKETS // 2
    near = half // 2
    wide = half - near
    return near, [next(n for n in range(near, DISTANCE + 1) if n ** wide >= near ** (wide - i) * DISTANCE ** i) for i in range(1, wide)]


def _padded(x, rows):
    """The packed tokens x as [b, longest, ...], zeros behind each sequence's end."""
    x = torch.cat([x.float(), x.new_zeros(1, *x.shape[1:], dtype=torch.float32)])
    return x.index_select(0, rows.reshape(-1)).reshape(*rows.shape, *x.shape[1:])


def _plain_attention(qkv, table, offsets, longest):
    total, _, heads, d = qkv.shape
    dev = qkv.device
    rows = _padded_rows(offsets, longest, total)
    there = rows < total
    q, k, v = _padded(qkv, rows).permute(2, 0, 3, 1, 4)
    near, steps = _thresholds()
    distance = torch.arange(-longest + 1, longest, device=dev)          # key place - query place
    n = distance.abs()
    bucket = torch.where(n < near, n, near + sum((n >= step).long() for step in steps)) + (BUCKETS // 2) * (distance > 0)
    line = table.float()[bucket].t()                                     # [heads, 2 longest - 1]
    bias = line.unfold(1, longest, 1).flip(1)                            # [heads, query, key]
    s = q @ k.transpose(2, 3).contiguous() * d ** -0.5 + bias
    s = s.masked_fill(~there[:, None, None, :], torch.finfo(torch.float32).min)
    e = torch.exp(s - s.detach().amax(3, keepdim=True)) * there[:, None, None, :]
    o = (e @ v) / e.sum(3, keepdim=True).clamp(min=1e-30)
    out = torch.zeros(total + 1, heads, d, device=dev).index_put((rows.reshape(-1),), o.transpose(1, 2).reshape(-1, heads, d))
    return out[:total].to(qkv.dtype)


def _plain_pool(hidden, offsets, longest):
    total = hidden.shape[0]
    rows = _padded_rows(offsets, longest, total)
    mean = _padded(hidden, rows).sum(1) / (offsets[1:] - offsets[:-1]).clamp(min=1)[:, None]
    return mean / mean.square().sum(1, keepdim=True).sqrt().clamp(min=1e-12)


def run(s):
    if s["op"] == "linear":
        args = s["x"], s["weight"], s["bias"], s["activation"], s["residual"]
        leaves = [t for t in (s["x"], s["weight"], s["bias"], s["residual"]) if t is not None]
        if own:
            from vectordb_amd import ops
            y = ops.linear(*args)
        else:
            y = _plain_linear(*args)
    elif s["op"] == "attention":
        leaves = [s["qkv"], s["table"]]
        if own:
            from vectordb_amd import ops
            y = ops.bucketed_attention(s["qkv"], s["table"], s["offsets"], max_distance=DISTANCE)
        else:
            y = _plain_attention(s["qkv"], s["table"], s["offsets"], s["longest"])
    else:
        leaves = [s["hidden"]]
        if own:
            from vectordb_amd import ops
            y = ops.mean_pool(s["hidden"], s["offsets"])
        else:
            y = _plain_pool(s["hidden"], s["offsets"], s["longest"])
    if not s["train"]:
        return [y]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


# ---- what a pass cannot do without -------------------------------------------------------------------------------

def work(case):
    size, train = BYTES[case["dtype"]], case["train"]
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        values = m * k + n * k + n + m * n * (2 if case["residual"] else 1)
        if train:                                          # dy in; dx, dW, db and dr out
            values += m * n + m * k + n * k + n + (m * n if case["residual"] else 0)
        return {"bytes": values * size, "flops": 2.0 * m * n * k * (3 if train else 1)}
    lengths = _lengths(case)
    tokens = sum(lengths)
    if case["op"] == "attention":
        squares = sum(n * n for n in lengths)
        # q k^T and p v; with the gradients also dp, dv, dq and dk
        return {"bytes": (tokens + case["spare"]) * case["h"] * case["d"] * size * (8 if train else 4), "flops": squares * case["h"] * case["d"] * (12.0 if train else 4.0)}
    rows = (tokens + case["spare"]) * case["dim"] * size * (2 if train else 1)
    return {"bytes": rows + case["b"] * case["dim"] * 4 * (2 if train else 1), "flops": tokens * case["dim"] * (3.0 if train else 1.0)}


# ---- the definitions, in 64 bits ---------------------------------------------------------------------------------

def _exact_act(z, name):
    """act(z) and its derivative."""
    if name == "gelu":
        cdf = torch.special.ndtr(z)
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (z + 0.044715 * z ** 3))
        return z * (1 + th) / 2, (1 + th) / 2 + z * (1 - th * th) / 2 * c * (1 + 3 * 0.044715 * z * z)
    if name == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).double()
    return z, torch.ones_like(z)


def _exact_bucket(distance):
    """Bucket of key place - query place: the near half one by one, then steps that grow to DISTANCE by equal ratios."""
    half = BUCKETS // 2
    near = half // 2
    n = abs(distance)
    low = n
    if n >= near:
        low = near
        while low < half - 1 and n ** (half - near) >= near ** (half - 1 - low) * DISTANCE ** (low + 1 - near):
            low += 1
    return low + (half if distance > 0 else 0)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        dy = None if s.get("dy") is None else s["dy"].double()
        if case["op"] == "linear":
            x, w, b = (s[n].detach().double() for n in ("x", "weight", "bias"))
            y, slope = _exact_act(torch.addmm(b, x, w.t()), case["act"])
            r = s["residual"]
            y = y if r is None else y + r.detach().double()
            if not case["train"]:
                return [y]
            dz = dy * slope
            return [y, dz @ w, dz.t() @ x, dz.sum(0)] + ([] if r is None else [dy])
        ends = s["offsets"].tolist()
        if case["op"] == "pool":
            x = s["hidden"].detach().double()
            y = torch.zeros(case["b"], case["dim"], dtype=torch.float64, device="cuda")
            dx = torch.zeros_like(x)
            for i, (lo, hi) in enumerate(zip(ends, ends[1:])):
                if lo < hi:
                    mean = x[lo:hi].mean(0)
                    size = torch.linalg.vector_norm(mean)
                    y[i] = mean / size
                    if dy is not None:
                        dx[lo:hi] = (dy[i] - y[i] * (y[i] @ dy[i])) / (size * (hi - lo))
            return [y, dx] if case["train"] else [y]
        qkv, table = s["qkv"].detach().double(), s["table"].detach().double()
        out, dqkv, dtable = torch.zeros_like(qkv[:, 0]), torch.zeros_like(qkv), torch.zeros_like(table)
        scale, longest = case["d"] ** -0.5, case["hi"]
        bucket = torch.tensor([_exact_bucket(e) for e in range(-longest, longest + 1)], device="cuda")
        for lo, hi in zip(ends, ends[1:]):
            place = torch.arange(hi - lo, device="cuda")
            which = bucket[place[None, :] - place[:, None] + longest]
            for h in range(case["h"] if lo < hi else 0):
                q, k, v = (qkv[lo:hi, i, h] for i in range(3))
                p = torch.softmax(scale * (q @ k.t()) + table[:, h][which], 1)
                out[lo:hi, h] = p @ v
                if dy is not None:
                    g = dy[lo:hi, h]
                    ds = p * (g @ v.t() - (g * out[lo:hi, h]).sum(1, keepdim=True))
                    dqkv[lo:hi, 0, h], dqkv[lo:hi, 1, h], dqkv[lo:hi, 2, h] = scale * ds @ k, scale * ds.t() @ q, p.t() @ g
                    # the bucket's sum, taken along the diagonals of equal distance
                    line = torch.zeros(2 * longest + 1, dtype=torch.float64, device="cuda")
                    n = hi - lo
                    skew = torch.nn.functional.pad(ds.flip(0), (0, n)).reshape(-1)[: n * (2 * n - 1)].reshape(n, 2 * n - 1)
                    line[longest - n + 1: longest + n] = skew.sum(0)
                    dtable[:, h].index_add_(0, bucket, line)
        return [out, dqkv, dtable] if case["train"] else [out]
