"""GPU suite of the encoder operators at their edges: values beyond a type's range, infinities and NaN where the definition keeps them
to themselves, probabilities below fp16's normal range, and the tiled kernels on other streams and in graphs."""
import math

import pytest

torch = pytest.importorskip("torch")

import ops_reference as ref  # noqa: E402
from test_gpu_ops import DT, TYPES, hold, offsets_of, rnd  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _native(hip_lib):
    yield


@pytest.fixture(scope="module")
def ops():
    from vectordb_amd import ops as o
    return o


@pytest.mark.parametrize("name", ["gelu", "gelu_tanh", "relu"])
def test_activation_gradients_of_sums_beyond_fp16(ops, name):
    """The sum before the activation is kept in fp16: below -65504 as -inf, whose slope is 0 and above as +inf, whose slope is 1."""
    x = torch.tensor([[-300.0], [300.0], [1.0], [-1.0]], dtype=torch.float16)
    for rows in (4, 300):                            # a few rows, and a tile
        xs = x.repeat(rows // 4, 1)
        w = torch.full((48, 1), 300.0, dtype=torch.float16)
        lx, lw = xs.cuda().requires_grad_(), w.cuda().requires_grad_()
        b = torch.zeros(48, dtype=torch.float16, device="cuda", requires_grad=True)
        y = ops.linear(lx, lw, b, name)
        dx, dw, db = (t.cpu() for t in torch.autograd.grad(y, [lx, lw, b], torch.ones_like(y)))
        slope = torch.tensor([0.0, 1.0, 1.0, 0.0]).repeat(rows // 4)     # at 300 and -300 the slopes are 1 and 0 to the last bit, too
        y = y.detach().cpu()
        assert (y[0::4] == 0).all() and (y[1::4] == math.inf).all() and (y[2::4] == 300).all() and (y[3::4] == 0).all()
        assert torch.equal(dx[:, 0].float(), slope * 48 * 300)
        assert torch.equal(dw[:, 0].float(), (slope * xs[:, 0].float()).sum().half().float().expand(48))
        assert torch.equal(db.float(), slope.sum().expand(48))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("lengths", [[14], [33, 70, 5], [129, 64, 257], [31] * 40], ids=["one", "ragged", "tiles", "many"])
def test_attention_infinite_values(ops, dtype, d, lengths):
    """An infinity in a text's v reaches the column it stands in, as p > 0 times it, and no other; so does one in dout's rows for dv.
    The last row of a text is where a kernel that repeats it behind the text's end would meet it again."""
    t, heads = DT[dtype], 2
    g = torch.Generator().manual_seed(sum(lengths) + d)
    off = offsets_of(lengths)
    ends = off.tolist()
    total = ends[-1]
    qkv, table, dout = rnd(g, total, 3, heads, d, dtype=t, scale=0.5), rnd(g, 32, heads, dtype=t, scale=0.5), rnd(g, total, heads, d, dtype=t)
    last = [e - 1 for e in ends[1:]]
    zero, inf = qkv.clone(), qkv.clone()
    for x, a, b in ((zero, 0.0, 0.0), (inf, math.inf, -math.inf)):
        x[last, 2, :, 0], x[last, 2, :, 1] = a, b
    want, got = (ops.bucketed_attention(x.cuda(), table.cuda(), off).cpu() for x in (zero, inf))
    assert (got[..., 0] == math.inf).all() and (got[..., 1] == -math.inf).all()
    assert torch.equal(got[..., 2:], want[..., 2:])
    gz, gi = dout.clone(), dout.clone()
    gz[last, :, 0], gi[last, :, 0] = 0.0, math.inf
    grads = []
    for do in (gz, gi):
        leaf = qkv.cuda().requires_grad_()
        dq, = torch.autograd.grad(ops.bucketed_attention(leaf, table.cuda(), off), [leaf], do.cuda())
        grads.append(dq[:, 2].cpu())
    assert (grads[1][..., 0] == math.inf).all()
    assert torch.equal(grads[1][..., 1:], grads[0][..., 1:])


@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_attention_probabilities_below_fp16s_normal_range(ops, d):
    """One key holds nearly all of a row's weight, 4000 others 2^-16 of it each: together 6 %.  In fp16 2^-16 is a subnormal, off by at
    most 2^-25, 2^-9 of it."""
    n = 4001
    qkv = torch.zeros(n, 3, 1, d, dtype=torch.float16)
    qkv[:, 0, 0, 0] = 8
    qkv[7, 1, 0, 0] = 16 * math.log(2) / 8 * math.sqrt(d)
    qkv[:, 2] = 1
    qkv[7, 2] = 0
    small = math.exp(-8 * float(qkv[7, 1, 0, 0]) / math.sqrt(d))
    part = (n - 1) * small / (1 + (n - 1) * small)
    out = ops.bucketed_attention(qkv.cuda(), torch.zeros(32, 1, dtype=torch.float16, device="cuda"), offsets_of([n])).cpu().double()
    # the score, of size 11, is off by (d + 6) E 11; the sum's terms by 2^-9; the rounded output by half a step
    assert ((out - part).abs() <= part * (2.0 ** -9 + 11 * (d + 20) * ref.E + n * ref.E + ref.half_step(torch.float16))).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_mean_pool_keeps_nan(ops, dtype):
    """A NaN in a text's rows makes its norm NaN: the whole vector, and the whole gradient.  The other texts' do not change."""
    t = DT[dtype]
    for dim in (40, 37, 768):
        g = torch.Generator().manual_seed(dim)
        for count in (4, 600):                        # both widths of a block
            off = offsets_of([5, 9, 2, 6] * (count // 4))
            ends = off.tolist()
            x, dy = rnd(g, ends[-1], dim, dtype=t), rnd(g, count, dim)
            bad = x.clone()
            bad[ends[1] + 3, 11] = math.nan
            outs = []
            for h in (x, bad):
                leaf = h.cuda().requires_grad_()
                y = ops.mean_pool(leaf, off)
                dh, = torch.autograd.grad(y, [leaf], dy.cuda())
                outs.append((y.detach().cpu(), dh.cpu()))
            (y0, d0), (y1, d1) = outs
            assert torch.isnan(y1[1]).all() and torch.isnan(d1[ends[1]:ends[2]]).all()
            keep = [i for i in range(count) if i != 1]
            rows = [i for i in range(ends[-1]) if not ends[1] <= i < ends[2]]
            assert torch.equal(y1[keep], y0[keep]) and torch.equal(d1[rows], d0[rows])
            plain = ops.mean_pool(bad.cuda(), off, normalize=False).cpu()
            assert torch.isnan(plain[1]).sum() == 1 and torch.isnan(plain).sum() == 1


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("scale", [2e-38, 1e-30, 1e-18, 1e18, 1e30, 1e38])
def test_attention_scales_far_from_one(ops, dtype, d, scale):
    """With q = 0 (or a scale so small that q.k vanishes) the scores are the bias alone, whatever the scale."""
    t, lengths = DT[dtype], [50, 17]
    g = torch.Generator().manual_seed(d)
    qkv, table, dout = rnd(g, 67, 3, 2, d, dtype=t), rnd(g, 32, 2, dtype=t, scale=20.0), rnd(g, 67, 2, d, dtype=t)
    qkv[:, 0] = 0 if scale > 1 else 0.5
    qkv[:, 1] *= 0.125
    off = offsets_of(lengths)
    want = ref.attention(qkv, table, off.tolist(), scale, 128, dout)
    lq, lt = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off, scale=scale)
    grads = torch.autograd.grad(out, [lq, lt], dout.cuda())
    # biases of up to 80 take probabilities below 2^-126, where they are 0: ds is off by 2^-126 |dp - delta| at each of a bucket's places
    # (at most 50^2 + 17^2 of them), dv by 2^-126 |dout| at each of a key's (at most 50)
    most = float(dout.abs().max())
    far_ds, far_dv = 2.0 ** -126 * 2800 * 2 * d * most * float(qkv[:, 2].abs().max()), 2.0 ** -126 * 50 * most
    hold([out, grads[1]], [want[0], (want[2][0], want[2][1] + far_ds)], f"{scale} {dtype}")
    hold([grads[0][:, 2]], [(want[1][0][:, 2], want[1][1][:, 2] + far_dv)], f"dv {scale} {dtype}")


def test_lazily_negated_views(ops):
    """x.conj().imag and torch._neg_view hold their values with the other sign in memory."""
    g = torch.Generator().manual_seed(1)

    def both(*shape):
        z = torch.randn(*shape, dtype=torch.complex64, generator=g).cuda().conj().imag
        n = torch._neg_view(torch.randn(*shape, generator=g).cuda())
        assert z.is_neg() and n.is_neg()
        return z, n
    off, one = offsets_of([3, 4]), torch.ones(1, 1, device="cuda")
    for x, w, b, r, q, t, do, dy, dm in zip(both(7, 1), both(1, 1), both(1), both(7, 1), both(7, 3, 1, 8), both(32, 1), both(7, 1, 8), both(7, 1), both(2, 1)):
        plain = [v.clone().resolve_neg() for v in (x, w, b, r, q, t, do, dy, dm)]
        outs = []
        for x, w, b, r, q, t, do, dy, dm in ((x, w, b, r, q, t, do, dy, dm), plain):
            leaf = [v.detach().clone().resolve_neg().requires_grad_() for v in (x, q)]
            outs.append([ops.linear(x, w, b, "gelu", r), ops.bucketed_attention(q, t, off), ops.mean_pool(x, off, normalize=False),
                         *torch.autograd.grad(ops.linear(leaf[0], one, None, "gelu"), [leaf[0]], dy),
                         *torch.autograd.grad(ops.bucketed_attention(leaf[1], plain[5], off), [leaf[1]], do),
                         *torch.autograd.grad(ops.mean_pool(leaf[0], off, normalize=False), [leaf[0]], dm)])
        assert all(torch.equal(p, q) for p, q in zip(*outs))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_attention_nan_and_infinity_in_the_table(ops, dtype, d, value):
    """A bias of NaN or +inf makes every row NaN that meets its bucket (inf - inf), forward and back, and no other row or head."""
    t = DT[dtype]
    g = torch.Generator().manual_seed(d)
    off = offsets_of([200, 1, 9])
    qkv, table, dout = rnd(g, 210, 3, 2, d, dtype=t), rnd(g, 32, 2, dtype=t), rnd(g, 210, 2, d, dtype=t)

    def both(tab):
        leaf = qkv.cuda().requires_grad_()
        out = ops.bucketed_attention(leaf, tab.cuda(), off)
        dq, = torch.autograd.grad(out, [leaf], dout.cuda())
        return out.detach().cpu(), dq[:, 0].cpu()
    clean = both(table)
    for bucket in (3, 15, 31):                       # at the diagonal, and both ends of the line
        bad = table.clone()
        bad[bucket, 1] = value
        for got, want in zip(both(bad), clean):
            assert torch.equal(got[:, 0], want[:, 0])
            for lo, hi in ((0, 200), (200, 201), (201, 210)):
                meets = (ref.buckets_of(hi - lo, 32, 128) == bucket).any(1)
                assert torch.isnan(got[lo:hi][meets, 1]).all()
                assert torch.equal(got[lo:hi][~meets], want[lo:hi][~meets])


@pytest.mark.parametrize("dtype,low", [("f32", torch.finfo(torch.float32).min), ("bf16", torch.finfo(torch.bfloat16).min), ("f32", -1e30), ("bf16", -1e11),
                                       ("f32", 2e38), ("f16", -math.inf)])
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("lengths", [[300, 1, 19, 70], [40] * 9], ids=["long", "short"])
def test_attention_rows_of_one_great_bias(ops, dtype, low, d, lengths):
    """Where every bias of a row is the same great number, the scores vanish beside it: p = 1 / length, forward and back.  (fp16's lowest value leaves
    room for the scores in 32 bits; -inf leaves nothing of a row.)  The head beside it has ordinary biases."""
    t, heads = DT[dtype], 2
    g = torch.Generator().manual_seed(sum(lengths) + d)
    total = sum(lengths)
    qkv, table, dout = rnd(g, total, 3, heads, d, dtype=t), rnd(g, 32, heads, dtype=t), rnd(g, total, heads, d, dtype=t)
    off = offsets_of(lengths)
    great = table.clone()
    great[:, 1] = low
    lq, lt = qkv.cuda().requires_grad_(), great.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, lt, off)
    dqkv, dtable = torch.autograd.grad(out, [lq, lt], dout.cuda())
    # without q, or without k, the scores are 0 and so is what an even bias changes
    flat = table.clone()
    flat[:, 1] = 0
    wants = []
    for which in (0, 1):
        x = qkv.clone()
        x[:, which, 1] = 0
        wants.append(ref.attention(x, flat, off.tolist(), d ** -0.5, 128, dout))
    (o, g0, dt), g1 = wants[0], wants[1][1]
    if low == -math.inf:
        assert not out[:, 1].any() and not dqkv[:, :, 1].any() and not dtable[:, 1].any()
        pick = slice(0, 1)
    else:
        pick = slice(0, 2)
    hold([out[:, pick], dtable[:, pick]], [tuple(v[:, pick] for v in o), tuple(v[:, pick] for v in dt)], f"{dtype} {low}")
    for i, w in ((0, g0), (1, g1), (2, g0)):         # dq holds k and no q, dk q and no k
        for h in range(pick.stop):
            if h == 0 or i != 1 or w is g1:
                hold([dqkv[:, i, h]], [tuple(v[:, i, h] for v in w)], f"{dtype} {low} gradient {i} head {h}")


@pytest.mark.parametrize("dtype,low", [("f32", torch.finfo(torch.float32).min), ("bf16", -1e9), ("bf16", torch.finfo(torch.bfloat16).min)])
@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_attention_one_row_left_to_great_biases(ops, dtype, low, d):
    """Keys strictly before the query, by great negative biases: the first row of a text has none and takes all keys evenly, beside rows
    that have some."""
    t, n = DT[dtype], 150
    g = torch.Generator().manual_seed(d)
    qkv, table, dout = rnd(g, n, 3, 1, d, dtype=t), rnd(g, 32, 1, dtype=t), rnd(g, n, 1, d, dtype=t)
    table[0], table[16:] = low, low
    lq = qkv.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, table.cuda(), offsets_of([n]))
    dqkv, = torch.autograd.grad(out, [lq], dout.cuda())
    q, k, v = qkv[:, :, 0].double().unbind(1)
    s = d ** -0.5 * (q @ k.t()) + table[:, 0].double()[ref.buckets_of(n, 32, 128)]
    s[0] = 0
    p, go = torch.softmax(s, 1), dout[:, 0].double()
    # scores of size 5 are off by (d + 20) E 5 in the exponent; p, rounded to 16 bits, by u; the sums by (n + d) E; the result by u
    u = ref.half_step(t)
    rel = (2 * u if dtype != "f32" else u) + (n + 12 * (d + 20)) * ref.E
    hold([out[:, 0], dqkv[:, 2, 0]], [(p @ v, rel * (p @ v.abs()) + 2.0 ** -126), (p.t() @ go, rel * (p.t() @ go.abs()) + 2.0 ** -120)], f"{dtype} {low}")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("size", [1e4, 1e9, 1e15])
def test_attention_great_scores(ops, dtype, d, size):
    """Scores of 1e8 to 1e31: each row is the value of its greatest score, to the bit (where no other comes within the sums' rounding)."""
    t, n = DT[dtype], 150
    g = torch.Generator().manual_seed(d)
    qkv, table, dout = rnd(g, n, 3, 1, d, dtype=t), rnd(g, 32, 1, dtype=t), rnd(g, n, 1, d, dtype=t)
    qkv[:, :2] *= size
    q, k, v = qkv[:, :, 0].double().unbind(1)
    s = q @ k.t()
    top = s.topk(2, 1)
    clear = top.values[:, 0] - top.values[:, 1] > 2 * (d + 6) * ref.E * (q.abs() @ k.abs().t()).max(1).values + 1e3
    assert clear.sum() > n * 3 // 4
    lq = qkv.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, table.cuda(), offsets_of([n]))
    assert torch.isfinite(out).all() and torch.equal(out.detach().cpu()[clear, 0], qkv[top.indices[clear, 0], 2, 0])
    dqkv, = torch.autograd.grad(out, [lq], dout.cuda())
    assert torch.isfinite(dqkv).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_relu_lets_no_infinity_back(ops, dtype):
    """Where relu's sum is not positive its gradient is 0, whatever arrives there."""
    t = DT[dtype]
    for m, n, k in ((5, 3, 4), (300, 136, 40)):
        g = torch.Generator().manual_seed(m)
        x, w = rnd(g, m, k, dtype=t), rnd(g, n, k, dtype=t)
        z = x.double() @ w.double().t()
        dy = rnd(g, m, n, dtype=t)
        clean, dirty = dy.masked_fill(z < -0.1, 0.0), dy.masked_fill(z < -0.1, math.inf)
        dirty[z < -1] = math.nan
        b = torch.zeros(n, dtype=t)
        grads = []
        for d in (clean, dirty):
            leaves = [v.cuda().requires_grad_() for v in (x, w, b)]
            grads.append(torch.autograd.grad(ops.linear(leaves[0], leaves[1], leaves[2], "relu"), leaves, d.cuda()))
        assert all(torch.equal(p, q) for p, q in zip(*grads))


@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("small", [1.37 * 2.0 ** -18, 1.37 * 2.0 ** -23, 1.37 * 2.0 ** -26])
def test_attention_small_probabilities_keep_their_bits_in_fp16(ops, d, small):
    """Beside a key that holds nearly all of a row's weight, probabilities of 2^-18 to 2^-26: forward and in v's gradient as close as an fp16
    rounding of a normal number."""
    n, u = 500, ref.half_step(torch.float16)
    qkv = torch.zeros(n, 3, 1, d, dtype=torch.float16)
    qkv[:, 0, 0, 0] = 8
    qkv[7, 1, 0, 0] = -math.log(small) / 8 * math.sqrt(d)
    qkv[:, 2] = 2.0 ** 14
    qkv[7, 2] = 0
    dout = torch.zeros(n, 1, d, dtype=torch.float16)
    dout[0] = 2.0 ** 14
    small = math.exp(-8 * float(qkv[7, 1, 0, 0]) / math.sqrt(d))        # of the key as it is rounded
    p = small / (1 + (n - 1) * small)
    leaf = qkv.cuda().requires_grad_()
    out = ops.bucketed_attention(leaf, torch.zeros(32, 1, dtype=torch.float16, device="cuda"), offsets_of([n]))
    dv = torch.autograd.grad(out, [leaf], dout.cuda())[0][:, 2].cpu().double()
    keep = [i for i in range(n) if i != 7]
    # scores of size s are off by (d + 20) E s in the exponent; p by u (2^-29 of the greatest is the last normal one), the results by u or, as subnormals, 2^-25
    rel = 2 * u + 20 * (d + 20) * ref.E + n * ref.E
    part = (n - 1) * p * 2.0 ** 14
    assert ((out.detach().cpu().double() - part).abs() <= rel * part + 2.0 ** -25).all()
    assert ((dv[keep] - p * 2.0 ** 14).abs() <= rel * p * 2.0 ** 14 + 2.0 ** -25).all()


def test_an_error_is_reported_once(ops, hip_lib):
    """A call refused by the runtime leaves nothing behind for the next call, or for torch's next kernel."""
    x, w = torch.ones(5, 8, device="cuda"), torch.ones(3, 8, device="cuda")
    want, out = ops.linear(x, w), torch.empty(5, 3, device="cuda")
    off = offsets_of([5])
    for call in (lambda: hip_lib.vdb_op_linear_dev(99, 0, x.data_ptr(), 8, w.data_ptr(), 8, None, None, 0, out.data_ptr(), 3, None, 5, 3, 8, 0, None, 0, None),
                 lambda: hip_lib.vdb_op_mean_pool_dev(99, 0, x.data_ptr(), 8, off.data_ptr(), 1, 5, 8, 1, out.data_ptr(), None, None)):
        assert call() == -2 and b"device" in hip_lib.vdb_last_error(None)
        assert torch.equal(ops.linear(x, w), want)
        assert call() == -2
        assert (torch.ones(4, device="cuda") + 1).sum().item() == 8


def test_a_stores_failed_reservation_is_reported_once(ops, hip_lib):
    """Rows that no GPU holds are refused by the allocator, and the operators' and torch's next calls do not hear of it."""
    from vectordb_amd import VdbError
    from vectordb_amd.index import FlatIndex
    x, w = torch.ones(5, 8, device="cuda"), torch.ones(3, 8, device="cuda")
    want = ops.linear(x, w)
    idx = FlatIndex(4096)
    for _ in range(2):
        with pytest.raises(VdbError):
            idx.reserve(2 ** 31 - 4096)              # 35 TB
        assert torch.equal(ops.linear(x, w), want)
        with pytest.raises(VdbError):
            idx.reserve(2 ** 31 - 4096)
        assert (torch.ones(4, device="cuda") + 1).sum().item() == 8


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 64])
def test_attention_of_broadcast_inputs(ops, dtype, d):
    """One bias column for all heads, one head, one row or one of q, k and v for all: the same outputs as from copies, and the copies' gradients
    summed."""
    t, n, heads = DT[dtype], 70, 4
    g = torch.Generator().manual_seed(d)
    off = offsets_of([50, 20])
    dout = rnd(g, n, heads, d, dtype=t).cuda()
    shapes = {"heads": (n, 3, 1, d), "rows": (1, 3, heads, d), "the three": (n, 1, heads, d)}
    column = rnd(g, 32, 1, dtype=t).cuda()
    for name, shape in shapes.items():
        small = rnd(g, *shape, dtype=t).cuda()
        one, col = small.clone().requires_grad_(), column.clone().requires_grad_()
        out = ops.bucketed_attention(one.expand(n, 3, heads, d), col.expand(32, heads), off)
        got = torch.autograd.grad(out, [one, col], dout)
        full, table = small.expand(n, 3, heads, d).contiguous().requires_grad_(), column.expand(32, heads).contiguous().requires_grad_()
        want = ops.bucketed_attention(full, table, off)
        assert torch.equal(out, want), name
        whole = torch.autograd.grad(want, [full, table], dout)
        dims = [i for i, s in enumerate(shape) if s == 1]
        for a, b, axes in ((got[0], whole[0], dims), (got[1], whole[1], [1])):
            exact = b.double().sum(axes, keepdim=True)
            # autograd's sum over the copies, rounded to the type at each of at most n steps
            assert ((a.double() - exact).abs() <= 2 * n * ref.half_step(t) * b.double().abs().sum(axes, keepdim=True) + 1e-30).all(), name


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_attention_great_scores_beside_greater_biases(ops, dtype, d):
    """Biases of 1e12 and scores of 1e10: steps of 1e5 in 32 bits, which different orders of the same sums do not share.  Forward and in v's
    gradient a row is still its greatest score's alone."""
    t, n = DT[dtype], 150
    g = torch.Generator().manual_seed(d)
    qkv, dout = rnd(g, n, 3, 1, d, dtype=t), rnd(g, n, 1, d, dtype=t)
    qkv[:, :2] *= 1e5
    table = torch.full((32, 1), 1e12).to(t)
    q, k, v = qkv[:, :, 0].double().unbind(1)
    s = d ** -0.5 * (q @ k.t())
    top = s.topk(2, 1)
    clear = top.values[:, 0] - top.values[:, 1] > 16 * 1e12 * ref.E * (d + 4)      # d roundings of sums of 1e12, and both sides' few more
    assert clear.sum() > n // 2
    dout[~clear] = 0
    lq = qkv.cuda().requires_grad_()
    out = ops.bucketed_attention(lq, table.cuda(), offsets_of([n]))
    dqkv, = torch.autograd.grad(out, [lq], dout.cuda())
    assert torch.isfinite(out).all() and torch.isfinite(dqkv).all()
    best = top.indices[:, 0]
    assert torch.equal(out.detach().cpu()[clear, 0], qkv[best[clear], 2, 0])
    want = torch.zeros(n, d, dtype=torch.float64).index_add_(0, best, dout[:, 0].double())
    size = torch.zeros(n, d, dtype=torch.float64).index_add_(0, best, dout[:, 0].double().abs())
    hold([dqkv[:, 2, 0]], [(want, (n + 16) * ref.E * size + ref.half_step(t) * want.abs() + 2.0 ** -120)], dtype)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_attention_rows_sum_to_one_beside_great_biases(ops, dtype, d):
    """Biases of -1e20 and scores of 1e14: in 32 bits some of a row's greatest scores are one number, and share the row.  Whatever p is there,
    with v = 1 an output is 1, and each row hands all of its gradient on to v."""
    t, n = DT[dtype], 52
    ones = torch.ones(n, 1, d, dtype=t)
    for seed in range(40):
        g = torch.Generator().manual_seed(seed)
        qkv = rnd(g, n, 3, 1, d, dtype=t)
        qkv[:, :2] *= 1e8
        qkv[:, 2] = 1
        lq = qkv.cuda().requires_grad_()
        out = ops.bucketed_attention(lq, torch.full((32, 1), -1e20, dtype=t, device="cuda"), offsets_of([n]), scale=1e-3)
        dqkv, = torch.autograd.grad(out, [lq], ones.cuda())
        # halves, thirds and the like, rounded to the type; sums of 52 rows
        u = ref.half_step(t)
        assert ((out.detach().float() - 1).abs() <= 4 * u + 64 * ref.E).all()
        assert ((dqkv[:, 2].double().sum(0) - n).abs() <= n * (4 * u + 64 * ref.E)).all()
        assert torch.isfinite(dqkv).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_attention_scores_are_the_same_numbers_forward_and_back(ops, dtype, d):
    """Texts of one token, whose score is a small difference of a great bias and a great product: p is 1 both ways only where both passes make
    that difference in the same order."""
    t, n = DT[dtype], 64
    scale, bias = (1e-3, -1e4) if dtype != "f16" else (1.0, -1e4)
    g = torch.Generator().manual_seed(d)
    qkv, dout = rnd(g, n, 3, 1, d, dtype=t), rnd(g, n, 1, d, dtype=t)
    qkv[:, 0] = (1e4 / scale / d) ** 0.5                      # q.k close to 1e4 / scale
    qkv[:, 1] = (qkv[:, 0].double() * (1 + 0.05 * torch.randn(n, 1, d, generator=g).double())).to(t)
    leaf = qkv.cuda().requires_grad_()
    out = ops.bucketed_attention(leaf, torch.full((32, 1), bias, dtype=t, device="cuda"), offsets_of([1] * n), scale=scale)
    dqkv, = torch.autograd.grad(out, [leaf], dout.cuda())
    s = (scale * (qkv[:, 0, 0].double() * qkv[:, 1, 0].double()).sum(1) + float(torch.tensor(bias, dtype=t))).abs().max()
    # lse is rounded (E |s| log2(e) ln 2 in p), p to the type, the result to the type
    rel = 2 * float(s) * ref.E + 8 * ref.E + 2 * ref.half_step(t)
    # p is not 1 to the last bit in fp32 (the score's product is exact inside the exponent, its maximum rounded): out = (p v) (1 / p), three
    # roundings of E and their products
    v = qkv[:, 2, 0].double()
    assert ((out.detach().cpu()[:, 0].double() - v).abs() <= 4 * ref.E * v.abs()).all()
    assert ((dqkv[:, 2].cpu().double() - dout.double()).abs() <= rel * dout.double().abs() + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 32, 64, 128])
def test_attention_rows_left_nothing_are_zeros_whatever_v_holds(ops, dtype, d):
    """All of a head's distances forbidden: zeros, and no gradient, beside infinities and NaN in v."""
    t, lengths = DT[dtype], [1, 70, 33]
    g = torch.Generator().manual_seed(d)
    off = offsets_of(lengths)
    qkv, table, dout = rnd(g, 104, 3, 2, d, dtype=t), rnd(g, 32, 2, dtype=t), rnd(g, 104, 2, d, dtype=t)
    table[:, 1] = -math.inf
    qkv[0, 2, 1, 3], qkv[50, 2, 1, 5], qkv[103, 2, 1, 0] = math.inf, math.nan, -math.inf
    leaf, tab = qkv.cuda().requires_grad_(), table.cuda().requires_grad_()
    out = ops.bucketed_attention(leaf, tab, off)
    dqkv, dtable = torch.autograd.grad(out, [leaf, tab], dout.cuda())
    assert not out[:, 1].any() and not dqkv[:, :, 1].any() and not dtable[:, 1].any()
    assert torch.isfinite(out[:, 0]).all() and torch.isfinite(dqkv[:, :, 0]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [24, 32, 64, 128])
@pytest.mark.parametrize("value", [math.nan, math.inf])
def test_attention_gradients_know_no_bucket_that_the_text_does_not_meet(ops, dtype, d, value):
    """NaN or +inf in the buckets of distances from 8 on: texts of at most 8 tokens have the gradients that they have without."""
    t, lengths = DT[dtype], [1, 8, 5, 1, 7]
    g = torch.Generator().manual_seed(d)
    off = offsets_of(lengths)
    qkv, table, dout = rnd(g, 22, 3, 2, d, dtype=t).cuda(), rnd(g, 32, 2, dtype=t).cuda(), rnd(g, 22, 2, d, dtype=t).cuda()
    bad = table.clone()
    bad[8:16], bad[24:] = value, value
    grads = []
    for tab in (table, bad):
        leaf, tab = qkv.clone().requires_grad_(), tab.clone().requires_grad_()
        out = ops.bucketed_attention(leaf, tab, off)
        grads.append([out.detach(), *torch.autograd.grad(out, [leaf, tab], dout)])
    assert all(torch.equal(a, b) for a, b in zip(*grads))
