"""MPNetEmbedder(engine="hip"): the embedding model on the framework's operators against transformers' own forward and backward
pass, from a tiny randomly initialised checkpoint that the test writes."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

import ops_reference as ref  # noqa: E402
from test_embedders import VOCAB, _write_tiny_mpnet  # noqa: E402

TEXTS = ["beef ribeye boneless", "ground chuck roll 80 20", "pork", "lamb steaks bone in", "beef <pad> pork", "",
         " ".join(VOCAB[5:17] * 3), "beef ribeye boneless"]


def test_bucketing_is_the_models():
    """The rule the operators use gives the model's own bucket for every distance."""
    from transformers import MPNetConfig, MPNetModel
    enc = MPNetModel(MPNetConfig(vocab_size=8, hidden_size=8, num_hidden_layers=1, num_attention_heads=1, intermediate_size=8,
                                 max_position_embeddings=16)).encoder
    place = torch.arange(-600, 601)
    assert enc.relative_position_bucket(place, num_buckets=32).tolist() == [ref.bucket(int(e), 32, 128) for e in place]


def test_engine_arguments(tmp_path, monkeypatch):
    from vectordb_amd.embedders import MPNetEmbedder, resolve_embedder
    d = _write_tiny_mpnet(str(tmp_path), hidden=32)
    with pytest.raises(ValueError, match="engine"):
        MPNetEmbedder(d, device="cpu", engine="cuda")
    with pytest.raises(ValueError, match="GPU"):
        MPNetEmbedder(d, device="cpu", engine="hip")
    with pytest.raises(ValueError, match="engine='hip'"):
        MPNetEmbedder(d, device="cpu").encode(["beef"])
    monkeypatch.delenv("VECTORDB_EMBED_ENGINE", raising=False)
    assert isinstance(resolve_embedder(d), MPNetEmbedder)


def test_packing_counts_positions_as_the_model_does(tmp_path):
    from vectordb_amd.embedders import MPNetEmbedder
    from vectordb_amd.encoder import MPNetEncoder
    emb = MPNetEmbedder(_write_tiny_mpnet(str(tmp_path), hidden=32), device="cpu")
    enc = MPNetEncoder(emb.model)
    ids, places, offsets = enc.pack([[0, 5, 6, 2], [], [0, 1, 7, 2]], "cpu")
    assert ids.tolist() == [0, 5, 6, 2, 0, 1, 7, 2] and offsets.tolist() == [0, 4, 4, 8]
    assert places.tolist() == [2, 3, 4, 5, 2, 1, 3, 4]          # a pad token inside a text takes the pad position
    enc.pack([[0] * 62], "cpu")
    with pytest.raises(ValueError, match="62 positions"):
        enc.pack([[0] * 63], "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("hidden", [32, 64])
def test_hip_engine_gives_the_models_vectors(tmp_path, hip_lib, hidden):
    from vectordb_amd.embedders import MPNetEmbedder
    d = _write_tiny_mpnet(str(tmp_path), hidden=hidden)
    plain = MPNetEmbedder(d, device="cuda:0", batch_size=3)
    want = plain.embed_device(TEXTS)
    hip = MPNetEmbedder(d, device="cuda:0", batch_size=3, engine="hip")
    got = hip.embed_device(TEXTS)
    assert got.dtype == torch.float32 and not got.requires_grad
    # two layers of 32-bit sums of up to 64 products on each side, unit vectors
    assert float((got - want).abs().max()) < 2e-6
    assert torch.equal(hip.embed_device(TEXTS), got)
    assert torch.equal(got[0], got[7]) and np.array_equal(np.stack(hip(TEXTS[:1]))[0], hip.embed_device(TEXTS[:1])[0].cpu().numpy())
    assert hip.embed_device([]).shape == (0, hidden) and hip.encode([]).shape == (0, hidden)
    for amp, tol in (("bf16", 1e-2), ("fp16", 2e-3)):
        low = MPNetEmbedder(d, device="cuda:0", autocast=amp, engine="hip").embed_device(TEXTS)
        assert low.dtype == torch.float32 and float((low - want).abs().max()) < tol
        assert torch.allclose(low.norm(dim=1), torch.ones(len(TEXTS), device="cuda"), atol=1e-6)


@pytest.mark.gpu
def test_hip_engine_gradients_are_the_models(tmp_path, hip_lib):
    """encode() is differentiable: every parameter's gradient against transformers' backward pass (eval mode, 32 bits)."""
    from vectordb_amd.embedders import MPNetEmbedder
    d = _write_tiny_mpnet(str(tmp_path), hidden=64)
    hip = MPNetEmbedder(d, device="cuda:0", engine="hip")
    dy = torch.randn(len(TEXTS), 64, generator=torch.Generator().manual_seed(1)).cuda()
    params = {n: p for n, p in hip.model.named_parameters() if not n.startswith("pooler")}
    got = dict(zip(params, torch.autograd.grad(hip.encode(TEXTS), list(params.values()), dy)))
    enc = hip.tok(TEXTS, padding=True, truncation=True, max_length=384, return_tensors="pt").to("cuda")
    h = hip.model(**enc).last_hidden_state
    mask = enc["attention_mask"].unsqueeze(-1).float()
    y = torch.nn.functional.normalize((h * mask).sum(1) / mask.sum(1), dim=1)
    want = dict(zip(params, torch.autograd.grad(y, list(params.values()), dy)))
    for n in params:
        if n.endswith("k.bias"):        # a shift of all keys changes no softmax: the gradient is 0 up to rounding
            assert float(got[n].norm()) < 1e-5 * float(want[n.replace("k.bias", "q.bias")].norm()) + 1e-5
            continue
        assert float((got[n] - want[n]).norm()) <= 2e-5 * float(want[n].norm()), n


@pytest.mark.gpu
def test_hip_engine_sees_changed_weights(tmp_path, hip_lib):
    """A step of an optimiser, or another checkpoint loaded over the model, shows in the next vectors."""
    from vectordb_amd.embedders import MPNetEmbedder
    d = _write_tiny_mpnet(str(tmp_path), hidden=64)
    for amp in (None, "bf16"):
        hip = MPNetEmbedder(d, device="cuda:0", engine="hip", autocast=amp)
        before = hip.embed_device(TEXTS)
        opt = torch.optim.SGD(hip.model.parameters(), lr=0.5)
        (1 - (hip.encode(TEXTS[:1]) * hip.encode(TEXTS[1:2])).sum()).backward()
        opt.step()
        after = hip.embed_device(TEXTS)
        assert not torch.equal(before, after)
        fresh = MPNetEmbedder(d, device="cuda:0", engine="hip", autocast=amp)
        fresh.model.load_state_dict(hip.model.state_dict())
        assert torch.equal(fresh.embed_device(TEXTS), after)
        fresh.model.encoder.layer[0].output.dense.bias.data.add_(1.0)       # a write that leaves no trace: only once asked
        fresh.refresh()
        assert not torch.equal(fresh.embed_device(TEXTS), after)


@pytest.mark.gpu
def test_product_vector_db_on_the_hip_engine(tmp_path, hip_lib, monkeypatch):
    """Add and query through the reference's own calls with the engine named by the environment."""
    import pandas as pd
    from vectordb_amd.embedders import SentenceTransformerEmbeddingFunction
    from vectordb_amd.vectordb import ProductVectorDB
    monkeypatch.setenv("VECTORDB_MODEL_DIR", _write_tiny_mpnet(str(tmp_path), hidden=64))
    monkeypatch.setenv("VECTORDB_EMBED_ENGINE", "hip")
    assert SentenceTransformerEmbeddingFunction(model_name="all-mpnet-base-v2")._hip is not None
    assert SentenceTransformerEmbeddingFunction(model_name="all-mpnet-base-v2", engine="transformers")._hip is None
    words = VOCAB[5:17]
    texts = sorted({f"{a} {b} {c}" for a in words for b in words[:5] for c in words[7:]})[:100]
    db = ProductVectorDB(persist_directory=str(tmp_path / "s"), usda_lookup_map={})
    db.add_products_to_db(pd.DataFrame({"product_description": texts, "product_code": [str(i) for i in range(len(texts))]}), recreate=True)
    assert db.collection.count() == len(texts)
    for q in texts[::17]:
        assert db.get_similar_products(q, n_results=3).iloc[0]["product_description"] == q
