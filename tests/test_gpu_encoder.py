"""MPNetEncoder on the GPU at the model's own head width (64): other streams, captured graphs, changed weights."""
import pytest

torch = pytest.importorskip("torch")
transformers = pytest.importorskip("transformers")

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module", autouse=True)
def _native(hip_lib):
    yield


def model_of(hidden=256, layers=2):
    from transformers import MPNetConfig, MPNetModel
    torch.manual_seed(1)
    return MPNetModel(MPNetConfig(vocab_size=100, hidden_size=hidden, num_hidden_layers=layers, num_attention_heads=hidden // 64,
                                  intermediate_size=2 * hidden, max_position_embeddings=300)).cuda().eval()


def encoder_of(model, dtype=torch.float32):
    from vectordb_amd.encoder import MPNetEncoder
    return MPNetEncoder(model, dtype)


def batch(enc, lengths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return enc.pack([[0, *torch.randint(5, 100, (n - 2,), generator=g).tolist(), 2] for n in lengths], "cuda")


def change(model, turn):
    """A fused optimiser's step, which counts no version."""
    params = list(model.encoder.parameters())
    for p in params:
        p.grad = torch.sin(torch.arange(p.numel(), device="cuda").float() + turn).view_as(p)
    torch.optim.AdamW(params, lr=0.05, fused=True).step()


@pytest.mark.parametrize("dtype", DTYPES)
def test_changed_weights_on_other_streams(dtype):
    """Calls on four streams right behind a change of the weights, each of its own batch, against calls one after the other."""
    model = model_of()
    enc = encoder_of(model, dtype)
    streams = [torch.cuda.Stream() for _ in range(4)]
    batches = [batch(enc, [70 + i, 5, 200 - i, 33], i) for i in range(4)]
    with torch.no_grad():
        first = enc.encode(*batches[0])
        for turn in range(3):
            change(model, turn)
            changed = torch.cuda.Event()
            changed.record()
            got = []
            for s, b in zip(streams, batches):
                s.wait_event(changed)
                with torch.cuda.stream(s):
                    got.append(enc.encode(*b))
            torch.cuda.synchronize()
            fresh = encoder_of(model, dtype)
            want = [fresh.encode(*b) for b in batches]
            assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
            assert not torch.equal(got[0], first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_captured_encoder_follows_the_weights(dtype):
    """A graph captured around encode() - the first call of its encoder, too - holds no memory that a later call or change frees, and
    computes with the weights of the time of each replay.  Eager calls between replays are not disturbed."""
    model = model_of()
    warm = encoder_of(model, dtype)
    lengths = [40, 130, 7, 64]
    ids, places, offsets = batch(warm, lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.no_grad(), torch.cuda.stream(side):
        warm.encode(ids, places, offsets)
    torch.cuda.current_stream().wait_stream(side)
    enc = encoder_of(model, dtype)
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = enc.encode(ids, places, offsets)
    with torch.no_grad():
        eager = enc.encode(ids, places, offsets)      # before any replay
        assert torch.equal(eager, encoder_of(model, dtype).encode(ids, places, offsets))
        for turn in range(4):
            for a, b in zip((ids, places, offsets), batch(enc, lengths, turn)):
                a.copy_(b)
            change(model, turn)
            eager = enc.encode(ids, places, offsets)
            junk = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(8)]       # what was freed is written over
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, eager), turn
            del junk
