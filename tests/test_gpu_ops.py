"""GPU suite of the encoder operators (vectordb_amd.ops) against 64-bit plain forms with derived bounds (ops_reference.py)."""
import math

import pytest

torch = pytest.importorskip("torch")

import ops_reference as ref  # noqa: E402

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
TYPES = list(DT)


@pytest.fixture(scope="module", autouse=True)
def _native(hip_lib):
    yield


@pytest.fixture(scope="module")
def ops():
    from vectordb_amd import ops as o
    return o


def rnd(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g) * scale).to(dtype)


def hold(got, want, what=""):
    """|got - exact| <= bound everywhere."""
    for i, (t, (exact, bound)) in enumerate(zip(got, want)):
        t = t.detach().to(exact.device).double()
        assert t.shape == exact.shape, (what, i, t.shape, exact.shape)
        assert torch.isfinite(t).all(), (what, i, "not finite")
        off = (t - exact).abs()
        worst = torch.where(off == 0, off, off / bound).max().item() if t.numel() else 0.0      # 0 of a bound of 0 holds
        assert worst <= 1.0, f"{what} output {i}: {worst:.3g} times its bound"


def offsets_of(lengths, device="cuda"):
    return torch.tensor([0, *torch.tensor(lengths, dtype=torch.int64).cumsum(0).tolist()], dtype=torch.int64, device=device)


# ---- linear -------------------------------------------------------------------------------------------------------------

LINEAR = [  # m, n, k
    (1, 1, 1), (1, 768, 768), (2, 5, 7), (3, 64, 32), (14, 2304, 768), (16, 48, 64), (17, 16, 136), (31, 33, 65), (48, 384, 96), (64, 64, 64),
    (65, 129, 72), (100, 768, 384), (127, 250, 8), (128, 128, 128), (129, 260, 1000), (257, 96, 40), (300, 1, 300), (333, 513, 257), (512, 512, 64), (1000, 24, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", LINEAR)
def test_linear_forward(ops, dtype, m, n, k):
    g = torch.Generator().manual_seed(m * 7 + n * 3 + k)
    names = ["none", "gelu", "gelu_tanh", "relu"]
    x, w, b, r = rnd(g, m, k, dtype=DT[dtype]), rnd(g, n, k, dtype=DT[dtype], scale=k ** -0.5), rnd(g, n, dtype=DT[dtype]), rnd(g, m, n, dtype=DT[dtype])
    for i, name in enumerate(names):
        bias, res = (b if (m + i) % 3 else None), (r if (n + i) % 2 else None)
        y = ops.linear(x.cuda(), w.cuda(), None if bias is None else bias.cuda(), name, None if res is None else res.cuda())
        assert y.dtype == DT[dtype]
        hold([y], ref.linear(x, w, bias, name, res), f"{name} {dtype}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", ["none", "gelu", "gelu_tanh", "relu"])
@pytest.mark.parametrize("m,n,k", [(1, 3, 5), (14, 64, 96), (33, 40, 24), (130, 136, 200), (257, 384, 64), (700, 72, 8), (1024, 128, 128), (2100, 33, 31), (4096, 64, 64)])
def test_linear_gradients(ops, dtype, name, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    x, w, b, r = rnd(g, m, k, dtype=DT[dtype]), rnd(g, n, k, dtype=DT[dtype], scale=k ** -0.5), rnd(g, n, dtype=DT[dtype]), rnd(g, m, n, dtype=DT[dtype])
    dy = rnd(g, m, n, dtype=DT[dtype])
    if name == "relu":      # keep the sums off the step
        z = x.double() @ w.double().t() + b.double()
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    leaves = [t.cuda().requires_grad_() for t in (x, w, b, r)]
    y = ops.linear(leaves[0], leaves[1], leaves[2], name, leaves[3])
    grads = torch.autograd.grad(y, leaves, dy.cuda())
    assert torch.equal(grads[3].cpu(), dy)
    hold([y, *grads[:3]], ref.linear(x, w, b, name, r, dy), f"{name} {dtype}")
    # a gradient asked for alone is the same
    for i in range(3):
        only = [t.detach().requires_grad_(j == i) for j, t in enumerate(leaves)]
        one, = torch.autograd.grad(ops.linear(only[0], only[1], only[2], name, only[3]), [only[i]], dy.cuda())
        assert torch.equal(one, grads[i])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,name", [(1000, 776, 776, "none"), (2049, 1400, 72, "gelu"), (8200, 4104, 72, "none"), (8200, 4104, 136, "gelu_tanh"), (2100, 1409, 200, "relu"),
                                        (16385, 2056, 64, "gelu"), (5000, 40, 1000, "none"),
                                        (500, 768, 1032, "gelu"), (1001, 768, 2312, "relu")])
def test_linear_forward_large(ops, dtype, m, n, k, name):
    """Sizes that take each of the tiled kernels, with ragged edges in all three dimensions (64-bit form on the GPU)."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w = (torch.randn(*s, generator=g, device="cuda").to(DT[dtype]) for s in ((m, k), (n, k)))
    b, r = (torch.randn(*s, generator=g, device="cuda").to(DT[dtype]) for s in ((n,), (m, n)))
    w = w * k ** -0.5
    hold([ops.linear(x, w, b, name, r)], ref.linear(x, w, b, name, r), dtype)
    hold([ops.linear(x, w)], ref.linear(x, w, None, "none", None), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,name", [(8192, 512, 384, "gelu"), (6001, 264, 776, "none"), (20000, 136, 136, "gelu_tanh"), (4096, 1408, 1416, "none"), (3000, 33, 520, "gelu")])
def test_linear_gradients_large(ops, dtype, m, n, k, name):
    """Long contractions that are split over blocks and joined, and their ragged ends."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w, b, dy = (torch.randn(*s, generator=g, device="cuda").to(DT[dtype]) for s in ((m, k), (n, k), (n,), (m, n)))
    w = w * k ** -0.5
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.linear(x, w, b, name)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        hold([y, *grads], ref.linear(x, w, b, name, None, dy), dtype)
    again = torch.autograd.grad(ops.linear(x, w, b, name), leaves, dy)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("m,n,k,name", [(1999, 636, 644, "gelu"), (1537, 1024, 1020, "relu"), (6100, 768, 72, "none")])
def test_linear_tiles_that_spread_evenly(ops, m, n, k, name):
    """fp32 products whose 64 x 64 tiles leave some compute units one more than others: the tiles of 96 rows, with ragged edges."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w, b, r, dy = (torch.randn(*s, generator=g, device="cuda") for s in ((m, k), (n, k), (n,), (m, n), (m, n)))
    w = w * k ** -0.5
    if name == "relu":      # keep the sums off the step
        z = x.double() @ w.double().t() + b.double()
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.linear(x, w, b, name, r)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        hold([y, *grads], ref.linear(x, w, b, name, r, dy))


def test_linear_layouts_strides_and_alignment(ops):
    g = torch.Generator().manual_seed(5)
    for dtype in TYPES:
        t = DT[dtype]
        big = rnd(g, 70, 3, 96, dtype=t)
        w, b = rnd(g, 50, 96, dtype=t, scale=0.1), rnd(g, 50, dtype=t)
        x = big[:, 1]                                            # rows 288 apart
        hold([ops.linear(big.cuda()[:, 1], w.cuda(), b.cuda())], ref.linear(x, w, b, "none", None), "strided rows")
        flat = rnd(g, 70 * 96 + 1, dtype=t)
        odd = flat[1:].view(70, 96)                              # rows off 16-byte borders
        hold([ops.linear(flat.cuda()[1:].view(70, 96), w.cuda(), b.cuda(), "gelu")], ref.linear(odd, w, b, "gelu", None), "unaligned rows")
        wide = rnd(g, 50, 97, dtype=t)
        hold([ops.linear(x.contiguous().cuda(), wide.cuda()[:, 1:])], ref.linear(x, wide[:, 1:], None, "none", None), "unaligned weight")
        xt = rnd(g, 96, 70, dtype=t)
        hold([ops.linear(xt.cuda().t(), w.cuda())], ref.linear(xt.t(), w, None, "none", None), "transposed input")
        row = rnd(g, 96, dtype=t)
        hold([ops.linear(row.cuda().expand(9, 96), w.cuda())], ref.linear(row.expand(9, 96), w, None, "none", None), "one row, nine times")
        assert ops.linear(row.cuda(), w.cuda()).shape == (50,) and ops.linear(big.cuda(), w.cuda()).shape == (70, 3, 50)
        res = rnd(g, 70, 100, dtype=t)
        hold([ops.linear(x.cuda(), w.cuda(), residual=res.cuda()[:, 50:])], ref.linear(x, w, None, "none", res[:, 50:]), "strided residual")
        # gradients through strided and expanded operands and a gradient with strides of its own
        lx, lw = big.cuda().requires_grad_(), wide.cuda().requires_grad_()
        y = ops.linear(lx[:, 1], lw[:, 1:], activation="gelu")
        dyt = rnd(g, 50, 70, dtype=t)
        dx, dw = torch.autograd.grad(y, [lx, lw], dyt.cuda().t())
        want = ref.linear(x, wide[:, 1:], None, "gelu", None, dyt.t())
        hold([y, dx[:, 1], dw[:, 1:]], want[:3], "strided gradients")
        assert not dx[:, 0].any() and not dx[:, 2].any() and not dw[:, 0].any()
        lb = b.cuda().requires_grad_()
        db, = torch.autograd.grad(ops.linear(x.cuda(), w.cuda(), lb).sum(), [lb])
        assert torch.equal(db.cpu().float(), torch.full((50,), 70.0))


def test_linear_without_rows(ops):
    for dtype in TYPES:
        x = torch.zeros(0, 40, dtype=DT[dtype], device="cuda", requires_grad=True)
        w = torch.ones(24, 40, dtype=DT[dtype], device="cuda", requires_grad=True)
        b = torch.ones(24, dtype=DT[dtype], device="cuda", requires_grad=True)
        for name in ("none", "gelu"):
            y = ops.linear(x, w, b, name)
            dx, dw, db = torch.autograd.grad(y, [x, w, b], torch.zeros_like(y))
            assert y.shape == (0, 24) and dx.shape == x.shape and not dw.any() and not db.any()


def test_linear_far_values(ops):
    """Activations at the ends of the line, and infinities and NaN that stay in their rows."""
    for dtype in TYPES:
        t = DT[dtype]
        big = 6e4 if dtype == "f16" else 1e18
        z = torch.tensor([0.0, -0.0, 1e-4, -1e-4, 5.0, -5.0, 12.0, -12.0, big, -big], dtype=t)
        w = torch.ones(1, 1, dtype=t)
        for name in ("gelu", "gelu_tanh", "relu"):
            hold([ops.linear(z[:, None].cuda(), w.cuda(), None, name)], ref.linear(z[:, None], w, None, name, None), name)
            x = z[:, None].cuda().requires_grad_()
            dx, = torch.autograd.grad(ops.linear(x, w.cuda(), None, name), [x], torch.ones(10, 1, dtype=t, device="cuda"))
            hold([dx[2:]], [tuple(v[2:] for v in ref.linear(z[:, None], w, None, name, None, torch.ones(10, 1, dtype=t))[1])], name)
        x = torch.ones(40, 64, dtype=t)
        x[3, 5], x[20, 1] = math.inf, math.nan
        y = ops.linear(x.cuda(), torch.ones(32, 64, dtype=t).cuda()).cpu()
        assert torch.isinf(y[3]).all() and torch.isnan(y[20]).all()
        keep = [i for i in range(40) if i not in (3, 20)]
        assert (y[keep].float() == 64).all()


# ---- attention ------------------------------------------------------------------------------------------------------------

SEQS = {
    "one token": [1], "a text": [14], "a tile": [32], "one over": [33], "ragged": [3, 0, 1, 64, 17, 31, 0, 40], "two tiles over": [129, 65],
    "empty ends": [0, 0, 9, 0], "long": [300, 7], "many": [5, 2, 9, 1, 30, 4] * 6,
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("name", list(SEQS))
@pytest.mark.parametrize("heads,d", [(3, 64), (2, 32), (1, 128), (2, 8), (1, 24), (2, 5), (1, 80)])
def test_attention_forward_and_gradients(ops, dtype, name, heads, d):
    lengths = SEQS[name]
    t = DT[dtype]
    g = torch.Generator().manual_seed(sum(lengths) + heads + d)
    spare = 5 if name in ("ragged", "many") else 0
    total = sum(lengths) + spare
    qkv, table, dout = rnd(g, total, 3, heads, d, dtype=t), rnd(g, 32, heads, dtype=t), rnd(g, total, heads, d, dtype=t)
    qkv[total - spare:] = math.nan                       # rows behind the last text are not looked at
    off = offsets_of(lengths)
    want = ref.attention(qkv, table, off.tolist(), d ** -0.5, 128, dout)
    lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off)
    assert torch.equal(out.detach(), ops.bucketed_attention(lq.detach(), lt.detach(), off))
    grads = torch.autograd.grad(out, [lq, lt], dout.cuda())
    hold([out, *grads], want, f"{name} {dtype}")
    again = torch.autograd.grad(ops.bucketed_attention(lq, lt, off), [lq, lt], dout.cuda())
    assert all(torch.equal(a, b) for a, b in zip(grads, again))      # nothing depends on timing
    one, = torch.autograd.grad(ops.bucketed_attention(lq, lt.detach(), off), [lq], dout.cuda())
    assert torch.equal(one, grads[0])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128, 96])
@pytest.mark.parametrize("lengths", [[63], [64], [65, 62], [127, 0, 64], [383], [384], [700, 389]], ids=str)
def test_attention_average_lengths(ops, dtype, d, lengths):
    """Both sides of the average lengths at which the width of a block changes."""
    t, heads = DT[dtype], 2
    g = torch.Generator().manual_seed(sum(lengths) + d)
    total = sum(lengths)
    qkv, table, dout = rnd(g, total, 3, heads, d, dtype=t), rnd(g, 32, heads, dtype=t), rnd(g, total, heads, d, dtype=t)
    off = offsets_of(lengths)
    want = ref.attention(qkv, table, off.tolist(), d ** -0.5, 128, dout)
    lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off)
    hold([out, *torch.autograd.grad(out, [lq, lt], dout.cuda())], want, f"{lengths} {dtype}")


BATCHES = {
    "mixed": ([200, 0, 1, 384, 64, 65, 127, 128, 129, 300, 33, 0, 90, 90, 17, 250, 5, 160] * 2, 77),
    "alike": ([128] * 20, 0),
    "most that are ordered": ([64 + (i * 37) % 9 for i in range(255)] + [0], 3),
    "one more": ([64 + (i * 37) % 9 for i in range(257)], 0),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("name", list(BATCHES))
def test_attention_gradients_of_many_blocks(ops, dtype, d, name):
    """Batches large enough that the backward pass takes the longest texts first."""
    lengths, spare = BATCHES[name]
    t, heads = DT[dtype], 18 if len(lengths) < 100 else 3
    g = torch.Generator(device="cuda").manual_seed(len(lengths) + d)
    total = sum(lengths) + spare
    qkv, dout = (torch.randn(total, *s, heads, d, generator=g, device="cuda").to(t) for s in ((3,), ()))
    table = torch.randn(32, heads, generator=g, device="cuda").to(t)
    qkv[total - spare:] = math.nan
    dout[total - spare:] = math.nan
    off = offsets_of(lengths)
    lq, lt = qkv.requires_grad_(), table.requires_grad_()
    out = ops.bucketed_attention(lq, lt, off)
    grads = torch.autograd.grad(out, [lq, lt], dout, retain_graph=True)
    with torch.no_grad():
        want = ref.attention(qkv.cpu(), table.cpu(), off.tolist(), d ** -0.5, 128, dout.cpu())
    hold([out, *grads], want, f"{name} {dtype}")
    again = torch.autograd.grad(out, [lq, lt], dout)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))


def test_attention_order_with_offsets_of_any_content(ops):
    """Lists that are no offsets at all, at a size where the longest text goes first: nothing leaves its buffers, and the next call is right."""
    heads, d, n, total = 18, 32, 40, 5000
    g = torch.Generator(device="cuda").manual_seed(2)
    qkv = torch.randn(total, 3, heads, d, generator=g, device="cuda").bfloat16().requires_grad_()
    table = torch.randn(32, heads, generator=g, device="cuda").bfloat16().requires_grad_()
    dout = torch.randn(total, heads, d, generator=g, device="cuda").bfloat16()
    good = offsets_of([total // n] * n)
    want = torch.autograd.grad(ops.bucketed_attention(qkv, table, good), [qkv, table], dout)
    for off in ([0, total] * (n // 2) + [total], list(range(n + 1))[::-1], [-2 ** 62] * (n + 1), [2 ** 62] * (n + 1), [0] * (n + 1),
                [0] + [total] * n, [total - 1] * n + [3]):
        bad = torch.tensor(off, dtype=torch.int64, device="cuda")
        torch.autograd.grad(ops.bucketed_attention(qkv, table, bad), [qkv, table], dout)
        got = torch.autograd.grad(ops.bucketed_attention(qkv, table, good), [qkv, table], dout)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_buckets,max_distance", [(4, 2), (4, 512), (6, 9), (32, 128), (32, 9), (32, 512), (64, 100), (128, 33), (128, 512)])
def test_attention_buckets(ops, dtype, n_buckets, max_distance):
    t = DT[dtype]
    g = torch.Generator().manual_seed(n_buckets + max_distance)
    lengths = [150, 40]
    qkv, table, dout = rnd(g, 190, 3, 2, 16, dtype=t), rnd(g, n_buckets, 2, dtype=t, scale=2.0), rnd(g, 190, 2, 16, dtype=t)
    off = offsets_of(lengths)
    want = ref.attention(qkv, table, off.tolist(), 0.3, max_distance, dout)
    lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off, scale=0.3, max_distance=max_distance)
    hold([out, *torch.autograd.grad(out, [lq, lt], dout.cuda())], want, f"{n_buckets} {max_distance}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [32, 64, 128])
def test_attention_widest_buckets(ops, dtype, d):
    """The largest table and distance with the widest heads: the most LDS a block can ask for."""
    t = DT[dtype]
    g = torch.Generator().manual_seed(d)
    qkv, table, dout = rnd(g, 300, 3, 1, d, dtype=t), rnd(g, 128, 1, dtype=t), rnd(g, 300, 1, d, dtype=t)
    off = offsets_of([260, 40])
    want = ref.attention(qkv, table, off.tolist(), d ** -0.5, 512, dout)
    lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off, max_distance=512)
    hold([out, *torch.autograd.grad(out, [lq, lt], dout.cuda())], want, dtype)


def test_what_is_refused(ops):
    """Arguments that do not fit together raise before any launch."""
    x, w = torch.zeros(4, 8, device="cuda"), torch.zeros(6, 8, device="cuda")
    off = torch.zeros(2, dtype=torch.int64, device="cuda")
    for args, kw, text in (((x, w.half()), {}, "weight"), ((x, w[:, :4]), {}, "weight"), ((x, w[0]), {}, "weight"), ((x, w, x), {}, "bias"),
                           ((x, w, torch.zeros(6)), {}, "bias"), ((x, w), dict(residual=x), "residual"), ((x, w), dict(activation="tanh"), "activation"),
                           ((x.double(), w.double()), {}, "float32"), ((x.cpu(), w), {}, "GPU"), ((x[:, :0], w[:, :0]), {}, "k >= 1")):
        with pytest.raises(ValueError, match=text):
            ops.linear(*args, **kw)
    with pytest.raises(TypeError):
        ops.linear(x, w, bias=1.0)
    q, t = torch.zeros(5, 3, 2, 16, device="cuda"), torch.zeros(32, 2, device="cuda")
    for args, kw, text in (((q[:, :2], t, off), {}, "qkv"), ((torch.zeros(5, 3, 2, 136, device="cuda"), t, off), {}, "qkv"), ((q, t[:, :1], off), {}, "table"),
                           ((q, t.bfloat16(), off), {}, "table"), ((q, t[0], off), {}, "table"), ((q, t, off.int()), {}, "offsets"),
                           ((q, t, off.cpu()), {}, "offsets"), ((q, t, off[:0]), {}, "offsets"), ((q, t, off[None]), {}, "offsets")):
        with pytest.raises(ValueError, match=text):
            ops.bucketed_attention(*args, **kw)
    from vectordb_amd import VdbError
    for kw, text in ((dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(max_distance=8), "max_distance"), (dict(max_distance=513), "max_distance")):
        with pytest.raises(VdbError, match=text):
            ops.bucketed_attention(q, t, off, **kw)
    for n in (2, 33, 130):
        with pytest.raises(VdbError, match="n_buckets"):
            ops.bucketed_attention(q, torch.zeros(n, 2, device="cuda"), off)
    for args, text in (((x[0], off), "hidden"), ((x, off.int()), "offsets"), ((x, off.cpu()), "offsets"), ((x.to(torch.int32), off), "float32")):
        with pytest.raises(ValueError, match=text):
            ops.mean_pool(*args)
    # a second derivative is refused, not wrong
    lx = x.clone().requires_grad_()
    first, = torch.autograd.grad(ops.linear(lx, w, activation="gelu").sum(), [lx], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), [lx])
    # an operand changed between the two passes is noticed
    lw = w.clone().requires_grad_()
    y = ops.linear(lx, lw, activation="gelu")
    with torch.no_grad():
        lw.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_against_differences(ops, dtype):
    """The gradients along a direction against central differences of the 64-bit form."""
    t = DT[dtype]
    g = torch.Generator().manual_seed(9)
    qkv, table, dout = rnd(g, 50, 3, 2, 16, dtype=t), rnd(g, 32, 2, dtype=t), rnd(g, 50, 2, 16, dtype=t)
    off = offsets_of([33, 17])
    lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    grads = torch.autograd.grad(ops.bucketed_attention(lq, lt, off), [lq, lt], dout.cuda())
    bounds = ref.attention(qkv, table, off.tolist(), 0.25, 128, dout)[1:]

    def value(a, b):
        return (ref.attention(a, b, off.tolist(), 0.25, 128)[0][0] * dout.double()).sum().item()

    for which in (0, 1):
        base = [qkv.double(), table.double()]
        step = torch.randn(base[which].shape, generator=g, dtype=torch.float64)
        h = 1e-4
        ends = []
        for sign in (1, -1):
            moved = list(base)
            moved[which] = base[which] + sign * h * step
            ends.append(value(*moved))
        diff = (ends[0] - ends[1]) / (2 * h)
        along = (grads[which].cpu().double() * step).sum().item()
        # the bounds of the gradient's elements, and h^2 times a third derivative of order 1 a token
        assert abs(along - diff) <= (bounds[which][1] * step.abs()).sum().item() + 50 * h


def test_attention_strides_and_alignment(ops):
    g = torch.Generator().manual_seed(2)
    off = offsets_of([20, 45])
    for dtype in TYPES:
        t = DT[dtype]
        table = rnd(g, 32, 4, dtype=t)
        for make in (lambda z: z[:, :, ::2],                                            # every second head
                     lambda z: z[:, :, :4, 8:24],                                       # part of each head
                     lambda z: z[:, :, :4, 1:14],                                       # off 16-byte borders, odd width
                     lambda z: z.flip(0)[:, :, :4, :16],                                # a copy (flip makes one)
                     lambda z: z[..., :24].transpose(2, 3)[:, :, :16, :4].transpose(2, 3)):
            whole = rnd(g, 65, 3, 8, 32, dtype=t)
            view, dev = make(whole), make(whole.cuda())
            heads, d = view.shape[2:]
            leaf = whole.cuda().requires_grad_()
            dout = rnd(g, 65, heads, d, dtype=t)
            want = ref.attention(view, table, off.tolist(), d ** -0.5, 128, dout)
            assert torch.equal(ops.bucketed_attention(dev, table.cuda(), off), ops.bucketed_attention(dev.contiguous(), table.cuda(), off)) or d % 8
            out = ops.bucketed_attention(make(leaf), table.cuda(), off)
            grad, = torch.autograd.grad(out, [leaf], dout.cuda())
            hold([out, make(grad)], want[:2], dtype)
        whole = rnd(g, 65, 3, 4, 16, dtype=t).cuda()
        turned = whole.transpose(2, 3).contiguous().transpose(2, 3)                      # last dimension not dense
        assert torch.equal(ops.bucketed_attention(turned, table.cuda(), off), ops.bucketed_attention(whole, table.cuda(), off))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_forbidden_distances(ops, dtype):
    """A bias of -inf forbids its distances; of the type's lowest value too, unless nothing else is there."""
    t = DT[dtype]
    g = torch.Generator().manual_seed(4)
    qkv, dout = rnd(g, 90, 3, 2, 16, dtype=t), rnd(g, 90, 2, 16, dtype=t)
    off = offsets_of([70, 1, 19])
    table = rnd(g, 32, 2, dtype=t)
    for low in (-math.inf, torch.finfo(t).min):
        one = table.clone()
        one[16:] = low                                   # no key behind the query
        want = ref.attention(qkv, one, off.tolist(), 0.25, 128, dout)
        lq, lt = qkv.cuda().requires_grad_(), one.cuda().requires_grad_()
        out = ops.bucketed_attention(lq, lt, off)
        hold([out, *torch.autograd.grad(out, [lq, lt], dout.cuda())], want, "causal")
    flat = torch.full((32, 2), torch.finfo(t).min, dtype=t)
    if dtype != "f16":                                   # fp16's lowest leaves room for the scores in 32 bits
        out = ops.bucketed_attention(qkv.cuda(), flat.cuda(), off).cpu().double()
        v = qkv[:, 2].double()
        for lo, hi in ((0, 70), (70, 71), (71, 90)):     # the scores vanish beside it: an even average
            mean = v[lo:hi].mean(0, keepdim=True)
            bound = (ref.half_step(t) * 3 + 200 * ref.E) * v[lo:hi].abs().mean(0, keepdim=True)
            assert ((out[lo:hi] - mean).abs() <= bound).all()
    none = torch.full((32, 2), -math.inf, dtype=t)       # nothing is left of any row: zeros, and no gradient
    lq, lt = qkv.cuda().requires_grad_(), none.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off)
    grads = torch.autograd.grad(out, [lq, lt], dout.cuda())
    assert not out.any() and not grads[0].any() and not grads[1].any()


def test_attention_keeps_texts_apart(ops):
    """What one text holds, NaN and infinities too, does not reach another."""
    g = torch.Generator().manual_seed(8)
    lengths = [31, 40, 2, 33, 64]
    off = offsets_of(lengths)
    ends = off.tolist()
    for dtype in TYPES:
        t = DT[dtype]
        qkv, table, dout = rnd(g, 170, 3, 2, 32, dtype=t).cuda(), rnd(g, 32, 2, dtype=t).cuda(), rnd(g, 170, 2, 32, dtype=t).cuda()
        dirty = qkv.clone()
        dirty[ends[1]:ends[2]] = math.nan
        dirty[ends[3]:ends[4]] = math.inf
        outs = []
        for x in (qkv, dirty):
            leaf = x.clone().requires_grad_()
            out = ops.bucketed_attention(leaf, table, off)
            grad, = torch.autograd.grad(out, [leaf], dout)
            outs.append((out.detach(), grad))
        for b in (0, 2, 4):
            for clean, other in zip(*outs):
                assert torch.equal(clean[ends[b]:ends[b + 1]], other[ends[b]:ends[b + 1]])


def test_attention_large_values(ops):
    """Scores far beyond an exponential's range, and gradients far below one."""
    g = torch.Generator().manual_seed(12)
    off = offsets_of([100, 40])
    for dtype in TYPES:
        t = DT[dtype]
        qkv, table, dout = rnd(g, 140, 3, 2, 64, dtype=t), rnd(g, 32, 2, dtype=t), rnd(g, 140, 2, 64, dtype=t, scale=1e-4)
        qkv[:, :2] *= 6
        want = ref.attention(qkv, table, off.tolist(), 0.125, 128, dout)
        lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
        out = ops.bucketed_attention(lq, lt, off)
        hold([out, *torch.autograd.grad(out, [lq, lt], dout.cuda())], want, dtype)


def test_attention_without_rows(ops):
    for dtype in TYPES:
        for n in (0, 3):
            qkv = torch.zeros(0, 3, 2, 16, dtype=DT[dtype], device="cuda", requires_grad=True)
            table = torch.ones(32, 2, dtype=DT[dtype], device="cuda", requires_grad=True)
            out = ops.bucketed_attention(qkv, table, torch.zeros(n + 1, dtype=torch.int64, device="cuda"))
            dq, dt = torch.autograd.grad(out, [qkv, table], torch.zeros_like(out))
            assert out.shape == (0, 2, 16) and dq.shape == qkv.shape and not dt.any()
        # rows, but no text
        qkv = torch.full((7, 3, 2, 16), math.nan, dtype=DT[dtype], device="cuda", requires_grad=True)
        out = ops.bucketed_attention(qkv, table, torch.zeros(1, dtype=torch.int64, device="cuda"))
        dq, dt = torch.autograd.grad(out, [qkv, table], torch.ones_like(out))
        assert not out.any() and not dq.any() and not dt.any()


def test_offsets_of_any_content_stay_in_bounds(ops):
    """Offsets outside the rows are clamped: what lies inside is right, the rest is zeros."""
    g = torch.Generator().manual_seed(3)
    qkv, table = rnd(g, 60, 3, 2, 32).cuda(), rnd(g, 32, 2).cuda()
    good = ops.bucketed_attention(qkv, table, torch.tensor([0, 20, 60], device="cuda"))
    assert torch.equal(ops.bucketed_attention(qkv, table, torch.tensor([-9, 20, 1 << 40], device="cuda")), good)
    assert torch.equal(ops.bucketed_attention(qkv, table, torch.tensor([7, 20, 60], device="cuda")), good)   # the first is 0
    h = rnd(g, 60, 40).cuda()
    assert torch.equal(ops.mean_pool(h, torch.tensor([5, 20, 1 << 40], device="cuda")), ops.mean_pool(h, torch.tensor([0, 20, 60], device="cuda")))
    down = ops.mean_pool(h, torch.tensor([0, 50, 20, 60], device="cuda"))                 # descending: empty, no harm
    assert not down[1].any()


# ---- pooling ---------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dim", [1, 7, 64, 384, 768, 1001, 2500])
def test_mean_pool(ops, dtype, normalize, dim):
    t = DT[dtype]
    g = torch.Generator().manual_seed(dim)
    for lengths, spare in (([1], 0), ([14], 0), ([0, 5, 64, 0, 33, 1], 9), ([400, 3], 0), ([2] * 70, 1)):
        total = sum(lengths) + spare
        x, dy = rnd(g, total, dim, dtype=t), rnd(g, len(lengths), dim)
        x[total - spare:] = math.nan
        off = offsets_of(lengths)
        want = ref.mean_pool(x, off.tolist(), normalize, dy)
        leaf = x.cuda().requires_grad_()
        y = ops.mean_pool(leaf, off, normalize)
        assert y.dtype == torch.float32 and torch.equal(y.detach(), ops.mean_pool(leaf.detach(), off, normalize))
        hold([y, *torch.autograd.grad(y, [leaf], dy.cuda())], want, f"{lengths[:3]}")
    wide = rnd(g, 30, dim + 3, dtype=t)                        # strided, unaligned rows
    off = offsets_of([11, 19])
    leaf = wide.cuda().requires_grad_()
    dy = rnd(g, 2, dim)
    y = ops.mean_pool(leaf[:, 2:2 + dim], off, normalize)
    grad, = torch.autograd.grad(y, [leaf], dy.cuda())
    hold([y, grad[:, 2:2 + dim]], ref.mean_pool(wide[:, 2:2 + dim], off.tolist(), normalize, dy), "strided")


def test_mean_pool_of_nothing(ops):
    """A zero mean stays zero, and its gradient is dy over the smallest norm, as the clamp says."""
    x = torch.zeros(6, 16, device="cuda", requires_grad=True)
    dy = torch.full((2, 16), 1e-13, device="cuda")
    y = ops.mean_pool(x, offsets_of([2, 4]))
    grad, = torch.autograd.grad(y, [x], dy)
    assert not y.any() and torch.allclose(grad, torch.tensor([0.05] * 2 + [0.025] * 4, device="cuda")[:, None].expand(6, 16), rtol=1e-5, atol=0)
    assert ops.mean_pool(torch.zeros(0, 8, device="cuda"), torch.zeros(1, dtype=torch.int64, device="cuda")).shape == (0, 8)
    assert not ops.mean_pool(torch.zeros(0, 8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")).any()


# ---- together, streams and graphs ----------------------------------------------------------------------------------------------

def _layer(ops, x, p, off):
    qkv = ops.linear(x, p["wqkv"], p["bqkv"]).view(-1, 3, 4, 16)
    ctx = ops.bucketed_attention(qkv, p["table"], off).reshape(-1, 64)
    x = torch.nn.functional.layer_norm(ops.linear(ctx, p["wo"], p["bo"], residual=x), (64,))
    return torch.nn.functional.layer_norm(ops.linear(ops.linear(x, p["w1"], p["b1"], "gelu"), p["w2"], p["b2"], residual=x), (64,))


def _plain_layer(x, p, off, ends):
    n = x.shape[0]
    qkv = (x @ p["wqkv"].t() + p["bqkv"]).view(-1, 3, 4, 16)
    ctx = []
    for lo, hi in zip(ends, ends[1:]):
        which = ref.buckets_of(hi - lo, 32, 128)
        q, k, v = qkv[lo:hi].permute(1, 2, 0, 3)
        s = 0.25 * (q @ k.transpose(1, 2)) + p["table"].t()[:, which]
        ctx.append((torch.softmax(s, -1) @ v).transpose(0, 1).reshape(hi - lo, 64))
    ctx = torch.cat(ctx)
    assert ctx.shape[0] == n
    x = torch.nn.functional.layer_norm(ctx @ p["wo"].t() + p["bo"] + x, (64,))
    return torch.nn.functional.layer_norm(torch.nn.functional.gelu(x @ p["w1"].t() + p["b1"]) @ p["w2"].t() + p["b2"] + x, (64,))


def _layer_params(g, dtype):
    shapes = dict(wqkv=(192, 64), bqkv=(192,), wo=(64, 64), bo=(64,), w1=(128, 64), b1=(128,), w2=(64, 128), b2=(64,), table=(32, 4))
    return {n: rnd(g, *s, dtype=dtype, scale=0.125) for n, s in shapes.items()}


@pytest.mark.parametrize("dtype", TYPES)
def test_an_encoder_layer_forward_and_backward(ops, dtype):
    """The operators in the order a model uses them: two layers, pooling, all gradients."""
    t = DT[dtype]
    g = torch.Generator().manual_seed(77)
    off = offsets_of([9, 30, 1, 45])
    ends = off.tolist()
    x, ps, dy = rnd(g, ends[-1], 64, dtype=t), [_layer_params(g, t) for _ in range(2)], rnd(g, 4, 64)
    lx = x.cuda().requires_grad_()
    lps = [{n: v.cuda().requires_grad_() for n, v in p.items()} for p in ps]
    h = lx
    for p in lps:
        h = _layer(ops, h, p, off)
    y = ops.mean_pool(h, off)
    got = torch.autograd.grad(y, [lx, *(v for p in lps for v in p.values())], dy.cuda())
    ex = x.double().requires_grad_()
    eps = [{n: v.double().requires_grad_() for n, v in p.items()} for p in ps]
    h = ex
    for p in eps:
        h = _plain_layer(h, p, off, ends)
    m = torch.stack([h[a:b].mean(0) for a, b in zip(ends, ends[1:])])
    m = m / m.norm(dim=1, keepdim=True)
    want = torch.autograd.grad(m, [ex, *(v for p in eps for v in p.values())], dy.double())
    # about ten roundings of u in a row, each followed by a layer of gain near one: in the 2-norm well under 16 u (32 bits: the
    # sums of up to 192 products add their own, at most 200 E each)
    u = ref.half_step(t)
    tol = 40 * u if dtype != "f32" else 16 * 200 * ref.E
    for a, b in zip([y, *got], [m, *want]):
        a, b = a.detach().cpu().double(), b.detach()
        assert (a - b).norm() <= tol * b.norm(), ((a - b).norm() / b.norm()).item()


def test_other_streams_and_two_calls_at_once(ops):
    g = torch.Generator().manual_seed(6)
    off = offsets_of([50, 300, 20])
    p = {n: v.cuda() for n, v in _layer_params(g, torch.bfloat16).items()}
    xs = [rnd(g, 370, 64, dtype=torch.bfloat16).cuda() for _ in range(4)]
    want = [_layer(ops, x, p, off) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, s in zip(xs, streams):
        with torch.cuda.stream(s):
            got.append(_layer(ops, x, p, off))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # split contractions' scratch: two weight gradients side by side
    x, dy = rnd(g, 4096, 64, dtype=torch.bfloat16).cuda(), rnd(g, 4096, 64, dtype=torch.bfloat16).cuda()
    ws = [rnd(g, 64, 64, dtype=torch.bfloat16).cuda().requires_grad_() for _ in range(4)]
    want = [torch.autograd.grad(ops.linear(x * i, w), [w], dy)[0] for i, w in enumerate(ws)]
    torch.cuda.synchronize()
    got = []
    for i, (w, s) in enumerate(zip(ws, streams)):
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(ops.linear(x * i, w), [w], dy)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_forward_mode_derivatives_are_refused(ops):
    """A tangent is never dropped without a word."""
    from torch.autograd import forward_ad
    x, w, off = torch.ones(5, 8, device="cuda"), torch.ones(4, 8, device="cuda"), offsets_of([2, 3])
    q, table = torch.ones(5, 3, 1, 8, device="cuda"), torch.ones(32, 1, device="cuda")
    with forward_ad.dual_level():
        for call in (lambda: ops.linear(forward_ad.make_dual(x, x), w), lambda: ops.linear(x, forward_ad.make_dual(w, w), activation="gelu"),
                     lambda: ops.bucketed_attention(forward_ad.make_dual(q, q), table, off), lambda: ops.mean_pool(forward_ad.make_dual(x, x), off)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(ops.linear(x, w), torch.full((5, 4), 8.0, device="cuda"))
    assert torch.equal(ops.linear(x, w), torch.full((5, 4), 8.0, device="cuda"))


def test_captured_and_replayed(ops):
    """A whole layer and the pooling in one HIP graph, replayed with other rows and other offsets in between eager calls."""
    g = torch.Generator().manual_seed(10)
    for dtype in TYPES:
        t = DT[dtype]
        p = {n: v.cuda() for n, v in _layer_params(g, t).items()}
        x = rnd(g, 200, 64, dtype=t).cuda()
        off = offsets_of([50, 60, 90])

        def step():
            return ops.mean_pool(_layer(ops, x, p, off), off)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step()
        for lengths in ([50, 60, 90], [1, 0, 199], [0, 0, 0], [70, 70, 10], [200, 0, 0]):
            x.copy_(rnd(g, 200, 64, dtype=t).cuda())
            off.copy_(offsets_of(lengths))
            eager = step().clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager), (dtype, lengths)


def test_gradients_captured_and_replayed(ops):
    """Forward and backward in one graph (leaves of its own), two graphs in turn: scratch is each graph's own."""
    g = torch.Generator().manual_seed(14)
    off = offsets_of([33, 100, 67])
    graphs = []
    for seed in range(2):
        x, table = rnd(g, 200, 192, dtype=torch.bfloat16).cuda(), rnd(g, 32, 4, dtype=torch.bfloat16).cuda()
        w = rnd(g, 64, 64, dtype=torch.bfloat16, scale=0.125).cuda()
        dy = rnd(g, 3, 64).cuda()

        def step(x=x, table=table, w=w, dy=dy):
            leaves = [x.detach().requires_grad_(), table.detach().requires_grad_(), w.detach().requires_grad_()]
            ctx = ops.bucketed_attention(leaves[0].view(-1, 3, 4, 16), leaves[1], off).reshape(-1, 64)
            y = ops.mean_pool(ops.linear(ctx, leaves[2], activation="gelu"), off)
            return [y.detach(), *torch.autograd.grad(y, leaves, dy)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs, step, x))
    for turn in range(4):
        for graph, outs, step, x in graphs:
            x.copy_(rnd(g, 200, 192, dtype=torch.bfloat16).cuda())
            eager = [v.clone() for v in step()]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


def test_rows_beyond_32_bits(ops):
    """Element offsets past 2^31: the last rows of a large tensor, strided so that little of it is touched."""
    big = torch.zeros(2 ** 31 + 4096, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    step = 2 ** 31 // 64
    x = big.as_strided((65, 32), (step, 1))
    rows = rnd(g, 65, 32, dtype=torch.bfloat16)
    x.copy_(rows.cuda())
    w = rnd(g, 24, 32, dtype=torch.bfloat16)
    hold([ops.linear(x, w.cuda())], ref.linear(rows, w, None, "none", None), "linear")
    hold([ops.mean_pool(x, offsets_of([3, 62]))], ref.mean_pool(rows, [0, 3, 65], True), "pool")
    q = big.as_strided((65, 3, 2, 16), (step, 32, 16, 1))
    vals = rnd(g, 65, 3, 2, 16, dtype=torch.bfloat16)
    q.copy_(vals.cuda())
    table = rnd(g, 32, 2, dtype=torch.bfloat16)
    hold([ops.bucketed_attention(q, table.cuda(), offsets_of([3, 62]))], ref.attention(vals, table, [0, 3, 65], 0.25, 128), "attention")
