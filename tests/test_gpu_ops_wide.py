"""GPU suite of the encoder operators' tiled kernels where the smaller tests take the general ones: heads of 64 and persistent tiles on other
streams and in captured graphs, the largest tiles with a kept sum, the embedding engine at its model's head width."""
import pytest

torch = pytest.importorskip("torch")

import ops_reference as ref  # noqa: E402
from test_gpu_ops import DT, TYPES, hold, offsets_of, rnd  # noqa: E402

pytestmark = pytest.mark.gpu
HEADS, D = 4, 64
WIDE = HEADS * D
#: 80 texts, 8000 rows: the tiled attention kernels, the longest first in the backward pass
LENGTHS = [20 + (i * 61) % 161 for i in range(80)]
ROWS = 8100


@pytest.fixture(scope="module", autouse=True)
def _native(hip_lib):
    yield


@pytest.fixture(scope="module")
def ops():
    from vectordb_amd import ops as o
    return o


def params(g, dtype):
    shapes = dict(wqkv=(3 * WIDE, WIDE), bqkv=(3 * WIDE,), wo=(WIDE, WIDE), bo=(WIDE,), w1=(2304, WIDE), b1=(2304,), w2=(WIDE, 2304), b2=(WIDE,), table=(32, HEADS))
    return {n: rnd(g, *s, dtype=dtype, scale=s[-1] ** -0.5).cuda() for n, s in shapes.items()}


def layer(ops, x, p, off):
    qkv = ops.linear(x, p["wqkv"], p["bqkv"]).view(-1, 3, HEADS, D)
    ctx = ops.bucketed_attention(qkv, p["table"], off).reshape(-1, WIDE)
    x = torch.nn.functional.layer_norm(ops.linear(ctx, p["wo"], p["bo"], residual=x), (WIDE,))
    up = ops.linear(x, p["w1"], p["b1"], "gelu")        # 16 bits: 64 x 18 tiles of 128 x 128 on 512 blocks
    return torch.nn.functional.layer_norm(ops.linear(up, p["w2"], p["b2"], residual=x), (WIDE,))


def gradients(ops, x, p, off, dy):
    """Leaves of its own, every operator's backward pass."""
    leaves = {n: v.detach().requires_grad_() for n, v in dict(p, x=x).items()}
    qkv = ops.linear(leaves["x"], leaves["wqkv"], leaves["bqkv"]).view(-1, 3, HEADS, D)
    ctx = ops.bucketed_attention(qkv, leaves["table"], off).reshape(-1, WIDE)
    h = ops.linear(ops.linear(ctx, leaves["w1"], leaves["b1"], "gelu"), leaves["w2"], leaves["b2"], residual=leaves["x"])
    y = ops.mean_pool(h, off)
    wanted = [v for n, v in leaves.items() if n not in ("wo", "bo")]
    return [y.detach(), *torch.autograd.grad(y, wanted, dy)]


def shifted(by):
    """As many texts of other lengths, as many rows or fewer."""
    return [max(0, n - by * (1 + i % 3)) for i, n in enumerate(LENGTHS)]


def test_the_batch_is_what_it_should_be():
    assert sum(LENGTHS) <= ROWS and sum(LENGTHS) >= 64 * len(LENGTHS)
    assert (ROWS // 128 + len(LENGTHS) + 1) * HEADS >= 512       # blocks enough for the longest to go first


@pytest.mark.parametrize("dtype", TYPES)
def test_tiled_kernels_on_other_streams(ops, dtype):
    t = DT[dtype]
    g = torch.Generator().manual_seed(6)
    p = params(g, t)
    xs = [rnd(g, ROWS, WIDE, dtype=t).cuda() for _ in range(4)]
    offs = [offsets_of(shifted(i)) for i in range(4)]
    dy = rnd(g, len(LENGTHS), WIDE).cuda()
    want = [[layer(ops, x, p, off), *gradients(ops, x, p, off, dy)] for x, off in zip(xs, offs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, off, s in zip(xs, offs, streams):
        with torch.cuda.stream(s):
            got.append([layer(ops, x, p, off), *gradients(ops, x, p, off, dy)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for one, other in zip(got, want) for a, b in zip(one, other))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_largest_tiles_on_other_streams_and_in_a_graph(ops, dtype):
    """33 x 16 tiles of 256 x 256 on 256 blocks."""
    t = DT[dtype]
    g = torch.Generator(device="cuda").manual_seed(7)
    w, b = torch.randn(4096, 64, generator=g, device="cuda").to(t) / 8, torch.randn(4096, generator=g, device="cuda").to(t)
    xs = [torch.randn(8400, 64, generator=g, device="cuda").to(t) for _ in range(3)]
    want = [ops.linear(x, w, b, "relu") for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in xs], []
    for x, s in zip(xs, streams):
        with torch.cuda.stream(s):
            got.append(ops.linear(x, w, b, "relu"))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.linear(x, w, b, "relu")
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i])


@pytest.mark.parametrize("dtype", TYPES)
def test_tiled_kernels_captured_and_replayed(ops, dtype):
    """A layer with pooling, and all gradients, in two graphs replayed in turn with other rows and offsets between eager calls."""
    t = DT[dtype]
    g = torch.Generator().manual_seed(10)
    p = params(g, t)
    x, dy, off = rnd(g, ROWS, WIDE, dtype=t).cuda(), rnd(g, len(LENGTHS), WIDE).cuda(), offsets_of(LENGTHS)
    steps = [lambda: [ops.mean_pool(layer(ops, x, p, off), off)], lambda: gradients(ops, x, p, off, dy)]
    graphs = []
    for step in steps:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs, step))
    for turn, lengths in enumerate((LENGTHS, shifted(3), [0] * len(LENGTHS), shifted(7), [ROWS] + [0] * (len(LENGTHS) - 1))):
        x.copy_(rnd(g, ROWS, WIDE, dtype=t).cuda())
        off.copy_(offsets_of(lengths))
        for graph, outs, step in graphs:
            eager = [v.clone() for v in step()]
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, eager)), turn


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["gelu", "relu"])
def test_largest_tiles_keep_their_sum(ops, dtype, name):
    """33 x 17 ragged tiles of 256 x 256 with a gradient wanted: the second pass over a tile's outputs that writes the sum before the
    activation, past the L2s."""
    m, n, k = 8200, 4104, 72
    g = torch.Generator(device="cuda").manual_seed(m)
    x, w, b, dy = (torch.randn(*s, generator=g, device="cuda").to(DT[dtype]) for s in ((m, k), (n, k), (n,), (m, n)))
    w = w * k ** -0.5
    if name == "relu":      # keep the sums off the step
        z = x.double() @ w.double().t() + b.double()
        dy = torch.where(z.abs() < 1e-4, torch.zeros_like(dy), dy)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    y = ops.linear(x, w, b, name)
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        assert torch.equal(y, ops.linear(x, w, b, name))
        hold([y, *grads], ref.linear(x, w, b, name, None, dy), dtype)


def test_engine_at_its_models_head_width(tmp_path):
    """MPNetEmbedder(engine="hip") with four heads of 64 against transformers' own passes: vectors, and every parameter's gradient."""
    pytest.importorskip("transformers")
    from test_embedder_engine import TEXTS
    from test_embedders import _write_tiny_mpnet
    from vectordb_amd.embedders import MPNetEmbedder
    d = _write_tiny_mpnet(str(tmp_path), hidden=WIDE)
    want = MPNetEmbedder(d, device="cuda:0", batch_size=3).embed_device(TEXTS)
    hip = MPNetEmbedder(d, device="cuda:0", batch_size=3, engine="hip")
    got = hip.embed_device(TEXTS)
    # two layers of 32-bit sums of up to 256 products on each side, unit vectors of 256 values
    assert float((got - want).abs().max()) < 2e-6
    for amp, tol in (("bf16", 1e-2), ("fp16", 2e-3)):
        low = MPNetEmbedder(d, device="cuda:0", autocast=amp, engine="hip").embed_device(TEXTS)
        assert float((low - want).abs().max()) < tol
    dy = torch.randn(len(TEXTS), WIDE, generator=torch.Generator().manual_seed(1)).cuda()
    named = {n: p for n, p in hip.model.named_parameters() if not n.startswith("pooler")}
    ours = dict(zip(named, torch.autograd.grad(hip.encode(TEXTS), list(named.values()), dy)))
    enc = hip.tok(TEXTS, padding=True, truncation=True, max_length=384, return_tensors="pt").to("cuda")
    h = hip.model(**enc).last_hidden_state
    mask = enc["attention_mask"].unsqueeze(-1).float()
    theirs = dict(zip(named, torch.autograd.grad(torch.nn.functional.normalize((h * mask).sum(1) / mask.sum(1), dim=1), list(named.values()), dy)))
    # six products a layer, forward and back, of at most 256 terms: 6 * 258 E = 9e-5 of their sums of absolute values
    for n in named:
        if n.endswith("k.bias"):        # a shift of all keys changes no softmax: the gradient is 0 up to rounding
            assert float(ours[n].norm()) < 1e-4 * float(theirs[n.replace("k.bias", "q.bias")].norm()) + 1e-5
        else:
            assert float((ours[n] - theirs[n]).norm()) <= 1e-4 * float(theirs[n].norm()), n


def test_engine_inside_autocast(tmp_path):
    """A caller's autocast region changes nothing: the engine casts by itself."""
    pytest.importorskip("transformers")
    from test_embedder_engine import TEXTS
    from test_embedders import _write_tiny_mpnet
    from vectordb_amd.embedders import MPNetEmbedder
    d = _write_tiny_mpnet(str(tmp_path), hidden=WIDE)
    for amp in (None, "bf16", "fp16"):
        hip = MPNetEmbedder(d, device="cuda:0", engine="hip", autocast=amp)
        want = hip.embed_device(TEXTS)
        for inside in (torch.bfloat16, torch.float16):
            with torch.autocast("cuda", dtype=inside):
                assert torch.equal(hip.embed_device(TEXTS), want)
                assert torch.equal(hip.encode(TEXTS[:3]).detach(), hip.embed_device(TEXTS[:3]))
