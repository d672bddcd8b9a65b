"""MPNetEncoder without a GPU: its weights, positions and buckets, on plain forms of the operators (ops_plain.py)."""
import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

import ops_plain  # noqa: E402

TOKENS = [[0, 5, 6, 2], [0, 7, 2], [0, 9, 8, 7, 6, 5, 11, 12, 13, 14, 15, 2]]


@pytest.fixture(autouse=True)
def _plain(monkeypatch):
    from vectordb_amd import encoder
    monkeypatch.setattr(encoder, "ops", ops_plain)


def model_of(hidden=32, **kw):
    from transformers import MPNetConfig, MPNetModel
    torch.manual_seed(1)
    return MPNetModel(MPNetConfig(**{**dict(vocab_size=20, hidden_size=hidden, num_hidden_layers=2, num_attention_heads=4, intermediate_size=48,
                                            max_position_embeddings=40), **kw})).eval()


def encoder_of(model, dtype=torch.float32):
    from vectordb_amd.encoder import MPNetEncoder
    return MPNetEncoder(model, dtype)


def vectors(enc, grad=False):
    with torch.set_grad_enabled(grad):
        return enc.encode(*enc.pack(TOKENS, "cpu"))


def models_own(model):
    """The model's own forward pass, one text at a time."""
    out = []
    with torch.no_grad():
        for t in TOKENS:
            h = model(input_ids=torch.tensor([t]), attention_mask=torch.ones(1, len(t), dtype=torch.long)).last_hidden_state[0]
            out.append(torch.nn.functional.normalize(h.mean(0), dim=0))
    return torch.stack(out)


def test_gives_the_models_vectors():
    model = model_of()
    enc = encoder_of(model)
    # unit vectors after two layers of 32-bit sums of up to 48 products
    assert float((vectors(enc) - models_own(model)).abs().max()) < 2e-6
    assert torch.equal(vectors(enc), vectors(enc, grad=True).detach())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("own", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layers", [0, 1, 3])
def test_numbers_of_layers_and_types_of_models(dtype, own, layers):
    """With and without gradients the same, whatever type the model's parameters have; no layers at all, too."""
    model = model_of(num_hidden_layers=layers).to(own)
    enc = encoder_of(model, dtype)
    got = vectors(enc)
    assert got.dtype == torch.float32 and torch.equal(got, vectors(enc, grad=True).detach())
    # 16-bit layers: three roundings of half a step a product, unit vectors of 32 values after at most three layers
    wide = vectors(encoder_of(model.float()))
    assert float((got - wide).abs().max()) < (2e-6 if dtype == torch.float32 else 0.05)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("how", ["sgd", "fused adamw", "replaced parameters", "data", "inference tensors", "another model's weights"])
def test_every_change_of_the_weights_shows(dtype, how):
    """Whatever changes the parameters, the next call without gradients computes with what they hold then: fused optimisers and writes
    through .data count no version, and a new parameter may come to lie where the old one was."""
    model = model_of()
    if how == "inference tensors":
        with torch.inference_mode():
            for p in list(model.parameters()):
                p.data = p.detach().clone()
    enc = encoder_of(model, dtype)
    params = list(model.encoder.parameters())
    first = vectors(enc)
    for turn in range(3):
        if how in ("sgd", "fused adamw"):
            for p in params:
                p.grad = torch.sin(torch.arange(p.numel()).float() + turn).view_as(p)
            (torch.optim.SGD(params, lr=0.3) if how == "sgd" else torch.optim.AdamW(params, lr=0.3, fused=True)).step()
        elif how == "replaced parameters":
            for layer in model.encoder.layer:
                for lin in (layer.attention.attn.q, layer.attention.attn.v, layer.output.dense):
                    for _ in range(2):
                        lin.weight = torch.nn.Parameter(torch.cos(torch.arange(lin.weight.numel()).float() * (turn + 2)).view_as(lin.weight))
        elif how == "data":
            for p in params:
                p.data += 0.3 * torch.sin(torch.arange(p.numel()).float() + turn).view_as(p)
        elif how == "inference tensors":
            with torch.inference_mode():
                for p in params:
                    p.add_(0.3 * torch.sin(torch.arange(p.numel()).float() + turn).view_as(p))
        else:
            model.load_state_dict(model_of(initializer_range=0.5 + turn).state_dict())
        now = vectors(enc)
        assert not torch.equal(now, first)
        assert torch.equal(now, vectors(encoder_of(model, dtype)))
        first = now


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_what_runs_between_the_layers_is_32_bits(dtype):
    """Layers whose products are all 0 leave embeddings, sums and normalisations: nothing there is rounded to 16 bits.  (Four
    normalisations with gains of order one in 32 bits on both sides; one rounding to 16 bits would be 1e-4 and more.)"""
    model = model_of()
    g = torch.Generator().manual_seed(3)
    with torch.no_grad():
        for n, p in model.named_parameters():
            if "LayerNorm" in n:
                p.normal_(generator=g)
            elif n.startswith("encoder.layer"):
                p.zero_()
    enc = encoder_of(model, dtype)
    want = models_own(model)
    assert float((vectors(enc) - want).abs().max()) < 2e-6
    assert float((vectors(enc, grad=True) - want).abs().max()) < 2e-6


@pytest.mark.parametrize("pad", [0, 1, 3])
def test_positions_count_as_the_models_whatever_its_pad_token(pad):
    """The model numbers positions by a padding index of its own, not by the configuration's pad token."""
    model = model_of(pad_token_id=pad)
    assert float((vectors(encoder_of(model)) - models_own(model)).abs().max()) < 2e-6


def test_buckets_are_the_models_whatever_its_table():
    """The model looks up 32 buckets: the first rows of a larger table, whose others have no gradient.  A smaller one is refused."""
    model = model_of(relative_attention_num_buckets=64)
    with torch.no_grad():
        model.encoder.relative_attention_bias.weight.normal_(generator=torch.Generator().manual_seed(5))
    enc = encoder_of(model)
    assert float((vectors(enc) - models_own(model)).abs().max()) < 2e-6
    vectors(enc, grad=True).sum().backward()
    grad = model.encoder.relative_attention_bias.weight.grad
    assert grad[:32].any() and not grad[32:].any()
    with pytest.raises(ValueError, match="16 buckets"):
        encoder_of(model_of(relative_attention_num_buckets=16))


def test_layers_that_are_no_plain_products_are_refused():
    """An adapter around a layer computes more than its weight says; a parametrised layer's weight is what it computes."""
    class Adapted(torch.nn.Linear):
        def forward(self, x):
            return super().forward(x) + 1.0

    class Doubled(torch.nn.Module):
        def forward(self, w):
            return 2 * w
    model = model_of()
    enc = encoder_of(model)
    q = model.encoder.layer[1].attention.attn.q
    model.encoder.layer[1].attention.attn.q = Adapted(q.in_features, q.out_features)
    for grad in (False, True):
        with pytest.raises(ValueError, match="Adapted"):
            vectors(enc, grad)
    model.encoder.layer[1].attention.attn.q = q
    before = vectors(enc)
    torch.nn.utils.parametrize.register_parametrization(model.encoder.layer[0].output.dense, "weight", Doubled())
    assert not torch.equal(vectors(enc), before) and float((vectors(enc) - models_own(model)).abs().max()) < 2e-6
    from transformers import BertConfig, BertModel
    with pytest.raises(ValueError, match="BertModel"):
        encoder_of(BertModel(BertConfig(vocab_size=20, hidden_size=16, num_hidden_layers=1, num_attention_heads=2, intermediate_size=16)))


def test_nothing_is_kept_between_calls():
    """No tensor outlives a call, so no later call on another stream, and no captured graph, can meet one that is unwritten or freed."""
    enc = encoder_of(model_of(), torch.bfloat16)
    before = {id(t) for t in _tensors(enc)}
    vectors(enc)
    assert {id(t) for t in _tensors(enc)} == before


def _tensors(x, seen=None):
    seen = set() if seen is None else seen
    if id(x) in seen:
        return
    seen.add(id(x))
    if isinstance(x, torch.Tensor):
        yield x
    elif isinstance(x, dict):
        for v in x.values():
            yield from _tensors(v, seen)
    elif isinstance(x, (list, tuple, set)):
        for v in x:
            yield from _tensors(v, seen)
    elif hasattr(x, "__dict__"):
        yield from _tensors(vars(x), seen)
