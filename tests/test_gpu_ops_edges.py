"""GPU suite of the encoder operators at their edges: values beyond a type's range, infinities and NaN where the definition keeps them
to themselves, probabilities below fp16's normal range, and the tiled kernels on other streams and in graphs."""
import math

import pytest

torch = pytest.importorskip("torch")

import ops_reference as ref  # noqa: E402
from test_gpu_ops import DT, TYPES, offsets_of, rnd  # noqa: E402

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
