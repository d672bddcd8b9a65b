"""CPU suite of the encoder operators' boundary: the header and the binding agree, and bad calls are refused before any launch."""
import ctypes as C
import os
import re

import pytest

torch = pytest.importorskip("torch")

import ops_reference as ref  # noqa: E402
from vectordb_amd import _capi, ops  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_header_binding_and_library_agree(hip_lib):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "vdb_ops.h")).read(), flags=re.S)
    names = sorted(set(re.findall(r"\b(vdb_op_[a-z_0-9]+)\s*\(", text)))
    assert names == sorted(_capi.OP_SYMBOLS)
    for n in names:
        assert hasattr(hip_lib, n)


def _refused(lib, rc, text):
    assert rc == -1 and text in lib.vdb_last_error(None).decode(), lib.vdb_last_error(None)


P = 4096     # an address nothing reads: every call here is refused before a launch


def test_linear_refusals(hip_lib):
    def call(dtype=1, x=P, ldx=8, w=P, ldw=8, r=None, ldr=0, y=P, ldy=8, m=4, n=8, k=8, act=0, ws=None, size=0):
        return hip_lib.vdb_op_linear_dev(0, dtype, x, ldx, w, ldw, None, r, ldr, y, ldy, None, m, n, k, act, ws, size, None)
    _refused(hip_lib, call(dtype=3), "dtype")
    _refused(hip_lib, call(dtype=-1), "dtype")
    _refused(hip_lib, call(m=-1), "m must be")
    _refused(hip_lib, call(n=0), "n and k")
    _refused(hip_lib, call(k=0), "n and k")
    _refused(hip_lib, call(m=1 << 40), "m must be")
    _refused(hip_lib, call(act=4), "activation")
    _refused(hip_lib, call(act=-1), "activation")
    for name in ("x", "w", "y"):
        _refused(hip_lib, call(**{name: None}), "NULL")
    for name in ("ldx", "ldw", "ldy"):
        _refused(hip_lib, call(**{name: 7}), "stride")
    _refused(hip_lib, call(r=P, ldr=7), "stride")
    assert call(m=0, x=None, w=None, y=None) == 0            # nothing to do is done
    for dtype in range(3):                                   # sizes that leave nothing to do have a workspace too
        for sizes in ((0, 1, 1), (0, 24, 40), (1, 1, 1), (1 << 30, 1 << 20, 1)):
            assert hip_lib.vdb_op_linear_workspace_bytes(dtype, *sizes) >= 0
            assert hip_lib.vdb_op_linear_backward_workspace_bytes(dtype, *sizes, 1) >= 0
    k = 1 << 16
    need = hip_lib.vdb_op_linear_workspace_bytes(0, 100, 100, k)
    if need:
        _refused(hip_lib, call(dtype=0, m=100, n=100, k=k, ldx=k, ldw=k, ldy=100, ws=P, size=need - 1), "workspace")
        _refused(hip_lib, call(dtype=0, m=100, n=100, k=k, ldx=k, ldw=k, ldy=100, ws=None, size=need), "workspace")


def test_linear_backward_refusals(hip_lib):
    need = hip_lib.vdb_op_linear_backward_workspace_bytes(1, 4, 8, 8, 1)
    assert need > 0

    def call(dtype=1, dy=P, lddy=8, x=P, ldx=8, w=P, ldw=8, z=P, dx=P, dw=P, m=4, n=8, k=8, act=1, ws=P, size=need):
        return hip_lib.vdb_op_linear_backward_dev(0, dtype, dy, lddy, x, ldx, w, ldw, z, dx, dw, None, m, n, k, act, ws, size, None)
    _refused(hip_lib, call(dtype=9), "dtype")
    _refused(hip_lib, call(act=9), "activation")
    _refused(hip_lib, call(dy=None), "NULL")
    _refused(hip_lib, call(x=None), "x is needed")
    _refused(hip_lib, call(w=None), "x is needed")
    _refused(hip_lib, call(z=None), "z is needed")
    _refused(hip_lib, call(lddy=3), "stride")
    _refused(hip_lib, call(ldx=3), "stride")
    _refused(hip_lib, call(size=need - 1), "workspace")
    _refused(hip_lib, call(ws=None), "workspace")


def test_attention_refusals(hip_lib):
    def call(dtype=1, q=P, table=P, nb=32, dist=128, off=P, seqs=2, total=10, heads=2, d=16, scale=0.25, out=P, ld_t=96):
        return hip_lib.vdb_op_attention_dev(0, dtype, q, P, P, ld_t, 16, table, nb, dist, off, seqs, total, heads, d, scale, out, None, None, None)
    _refused(hip_lib, call(dtype=5), "dtype")
    for name, bad in (("q", None), ("table", None), ("off", None), ("out", None)):
        _refused(hip_lib, call(**{name: bad}), "NULL")
    for nb in (0, 2, 3, 33, 130):
        _refused(hip_lib, call(nb=nb), "n_buckets")
    for dist in (0, 8, 513, -1):
        _refused(hip_lib, call(dist=dist), "max_distance")
    for heads in (0, -1, 1025):
        _refused(hip_lib, call(heads=heads), "heads")
    for d in (0, 129):
        _refused(hip_lib, call(d=d), "head_dim")
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        _refused(hip_lib, call(scale=scale), "scale")
    _refused(hip_lib, call(total=-1), "total")
    _refused(hip_lib, call(seqs=-1), "n_seqs")
    _refused(hip_lib, call(ld_t=-1), "stride")
    _refused(hip_lib, call(seqs=1 << 29, heads=1024), "too many")
    assert call(total=0, q=None, table=None, off=None, out=None) == 0
    rc = hip_lib.vdb_op_attention_backward_dev(0, 1, P, P, P, 96, 16, P, 32, 128, P, 2, 10, 2, 16, 0.25, P, None, P, P, P, P, P, 96, 16, P, P, 1, None)
    _refused(hip_lib, rc, "workspace")
    rc = hip_lib.vdb_op_attention_backward_dev(0, 1, P, P, P, 96, 16, P, 32, 128, P, 2, 10, 2, 16, 0.25, P, None, None, P, P, P, P, 96, 16, P, P, 1 << 30, None)
    _refused(hip_lib, rc, "NULL")


def test_pool_refusals(hip_lib):
    def call(dtype=0, h=P, ld=8, off=P, seqs=2, total=10, dim=8, y=P):
        return hip_lib.vdb_op_mean_pool_dev(0, dtype, h, ld, off, seqs, total, dim, 1, y, None, None)
    _refused(hip_lib, call(dtype=4), "dtype")
    _refused(hip_lib, call(dim=0), "dim")
    _refused(hip_lib, call(ld=7), "stride")
    for name in ("h", "off", "y"):
        _refused(hip_lib, call(**{name: None}), "NULL")
    assert call(seqs=0) == 0
    rc = hip_lib.vdb_op_mean_pool_backward_dev(0, 0, P, P, None, P, 2, 10, 8, 1, P, None)
    _refused(hip_lib, rc, "NULL")


def test_sizes_beyond_one_launch_are_refused(hip_lib):
    """A launch has fewer than 2^32 threads along a dimension: what would need more is refused before it, not by it."""
    _refused(hip_lib, hip_lib.vdb_op_linear_dev(0, 1, P, 1, P, 1, None, None, 0, P, 1, None, 2 ** 30, 1, 1, 0, None, 0, None), "m must be")
    _refused(hip_lib, hip_lib.vdb_op_mean_pool_dev(0, 0, P, 8, P, 2 ** 24, 10, 8, 1, P, None, None), "n_seqs")
    _refused(hip_lib, hip_lib.vdb_op_mean_pool_backward_dev(0, 0, P, P, P, P, 2 ** 23, 2 ** 28, 8, 1, P, None), "n_seqs")
    _refused(hip_lib, hip_lib.vdb_op_attention_dev(0, 1, P, P, P, 96, 16, P, 32, 128, P, 2 ** 23, 10, 2, 16, 0.25, P, None, None, None), "too many")


def test_a_library_without_the_operators_loads(tmp_path):
    """VECTORDB_AMD_LIB may name an older build: the store's symbols are what it needs."""
    import ctypes
    bare = ctypes.CDLL(None)
    assert not hasattr(bare, _capi.OP_SYMBOLS[0]) and _capi._declare_ops(bare) is bare


def test_no_gpu_means_loud_failure(hip_lib):
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    assert hip_lib.vdb_op_linear_dev(0, 1, P, 8, P, 8, None, None, 0, P, 8, None, 4, 8, 8, 0, None, 0, None) == -2
    assert hip_lib.vdb_op_mean_pool_dev(0, 0, P, 8, P, 2, 10, 8, 1, P, None, None) == -2
    assert b"mean_pool" in hip_lib.vdb_last_error(None)


def test_python_refuses_what_is_not_on_a_gpu():
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear(x, w)
    with pytest.raises(ValueError, match="GPU"):
        ops.bucketed_attention(torch.zeros(3, 3, 2, 8), torch.zeros(32, 2), torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="GPU"):
        ops.mean_pool(x, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.linear([1.0], w)
    with pytest.raises(TypeError, match="torch.Tensor"):
        ops.mean_pool(None, torch.zeros(2, dtype=torch.int64))


def test_bucket_rule():
    """The reference form's own check: near distances one by one, equal ratios behind them, the last bucket from there on."""
    got = [ref.bucket(-n, 32, 128) for n in range(200)]
    assert got[:8] == list(range(8)) and got[8] == 8 and got[127] == got[199] == 15 and got == sorted(got)
    assert got.index(10) == 16 and got.index(12) == 32 and got.index(14) == 64      # 8 * 16^(2/8), 16^(4/8), 16^(6/8): whole numbers
    assert [ref.bucket(n, 32, 128) for n in range(1, 200)] == [b + 16 for b in got[1:]]


def test_tracers_are_refused():
    """A trace would hold the outputs' allocation alone and return whatever the memory held."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.flop_counter import FlopCounterMode
    x, w, off = torch.zeros(3, 4), torch.zeros(5, 4), torch.tensor([0, 3])
    q, table = torch.zeros(3, 3, 2, 8), torch.zeros(32, 2)
    calls = ((lambda a: ops.linear(a, w), x), (lambda a: ops.bucketed_attention(a, table, off), q), (lambda a: ops.mean_pool(a, off), x))
    for call, arg in calls:
        with pytest.raises(RuntimeError, match="traced"):
            torch.jit.trace(call, (arg,))
        for kw in (dict(), dict(tracing_mode="fake"), dict(pre_dispatch=True)):
            with pytest.raises(RuntimeError, match="traced"):
                make_fx(call, **kw)(arg)
        for _ in range(2):                       # nothing of it lasts, and a mode that traces nothing refuses nothing (but the CPU is refused)
            with pytest.raises(ValueError, match="GPU"):
                call(arg)
        with FlopCounterMode(display=False), pytest.raises(ValueError, match="GPU"):
            call(arg)


def test_an_optional_tensor_without_memory_is_not_an_absent_one():
    """A bias whose storage was freed has a null address, which the C ABI takes for none."""
    t = torch.ones(3)
    assert ops._ptr(None) is None and ops._ptr(t) == t.data_ptr() and not ops._ptr(torch.ones(0))
    t.untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="no memory"):
        ops._ptr(t)
