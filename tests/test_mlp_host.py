"""The norm and gated MLP without a GPU: the oracle against differences of its own forward pass, the C entry
points' checks of arguments, and the Python layer's refusals."""

import ctypes

import numpy as np
import pytest
import torch

from flicker_amd import _lib, autograd, mlp, norm
from oracle import mlp as M

BF16, F16, F32 = 0, 1, 2
OK, INVALID, ALIGN, UNSUPPORTED, SCRATCH = 0, -1, -2, -3, -4


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.fail("libflicker_hip.so is not built (python -m flicker_amd.build)")
    return _lib.lib()


def _difference(f, at, along, h=1e-5):
    """Central difference of f at `at` along `along`: off by O(h^2) and by 1e-16 |f| / h."""
    return (f(at + h * along) - f(at - h * along)) / (2 * h)


@pytest.mark.parametrize("seed", [0, 1])
def test_oracle_gradients_are_the_forward_pass_differences(seed):
    r = np.random.RandomState(seed)
    x, dy, d = r.randn(3, 7, 10) + 0.4, r.randn(3, 7, 10), r.randn(3, 7, 10)
    factor, offset = 1 + 0.3 * r.randn(3, 1, 10), r.randn(3, 1, 10)
    dx, dn, db = M.layer_norm_grads(dy, x, factor)
    loss = lambda x, f, o: float((M.layer_norm(x, f, o) * dy).sum())  # noqa: E731
    df, do = r.randn(3, 1, 10), r.randn(3, 1, 10)
    # second and third derivatives are of order ten here: h^2 of them, 1e-9
    assert abs((dx * d).sum() - _difference(lambda v: loss(v, factor, offset), x, d)) < 1e-6
    assert abs((dn.sum(1, keepdims=True) * df).sum() - _difference(lambda v: loss(x, v, offset), factor, df)) < 1e-6
    assert abs((db.sum(1, keepdims=True) * do).sum() - _difference(lambda v: loss(x, factor, v), offset, do)) < 1e-6
    gu, dh, e = 2 * r.randn(5, 12), r.randn(5, 6), r.randn(5, 12)
    assert abs((M.swiglu_grads(dh, gu) * e).sum() - _difference(lambda v: float((M.swiglu(v) * dh).sum()), gu, e)) < 1e-6
    ops = [r.randn(4, 6), r.randn(6, 16), r.randn(8, 6)]
    dy = r.randn(4, 6)
    for i, grad in enumerate(M.gated_mlp_grads(dy, *ops)):
        along = r.randn(*ops[i].shape)
        got = _difference(lambda v: float((M.gated_mlp(*ops[:i], v, *ops[i + 1:]) * dy).sum()), ops[i], along)
        assert abs((grad * along).sum() - got) < 1e-5


def test_oracle_sigmoid_at_the_ends():
    gu = np.array([[-1e4, -800.0, 0.0, 800.0, 1e4, 1.0, 2.0, 3.0, 4.0, 5.0]])
    with np.errstate(all="raise", under="ignore"):
        assert np.array_equal(M.swiglu(gu), [[-0.0, -0.0, 0.0, 3200.0, 5e4]])
        assert np.array_equal(M.swiglu_grads(np.ones((1, 5)), gu)[0, 5:], [0.0, 0.0, 0.0, 800.0, 1e4])


P16 = 4096   # any address: the checks come before the launch


def _norm(lib, **k):
    a = dict(x=P16, xb=0, xr=64, dtype=BF16, factor=P16, offset=P16, params=BF16, pstride=64, add=1, eps=1e-6, batch=0,
             length=4, width=64, y=P16, yb=0, yr=64)
    a.update(k)
    return lib.flk_layer_norm(*a.values(), None)


def test_layer_norm_checks(lib):
    assert _norm(lib) == OK and _norm(lib, batch=2, length=0, x=None, y=None) == OK
    assert _norm(lib, dtype=3) == INVALID and _norm(lib, dtype=-1) == INVALID and _norm(lib, params=5) == INVALID
    assert _norm(lib, width=0) == INVALID and _norm(lib, batch=-1) == INVALID and _norm(lib, length=-1) == INVALID
    assert _norm(lib, eps=-1.0) == INVALID and _norm(lib, eps=float("nan")) == INVALID
    assert _norm(lib, pstride=32) == INVALID
    assert _norm(lib, batch=65536, length=65536) == INVALID
    assert _norm(lib, width=16385, pstride=0) == UNSUPPORTED
    assert _norm(lib, batch=1, x=None) == INVALID and _norm(lib, batch=1, y=None) == INVALID
    assert _norm(lib, batch=1, x=P16 + 1) == ALIGN and _norm(lib, batch=1, dtype=F32, params=F32, y=P16 + 2) == ALIGN
    assert _norm(lib, batch=1, params=F32, factor=P16 + 2) == ALIGN
    assert _norm(lib, batch=1, dtype=F32, params=BF16) == UNSUPPORTED
    assert _norm(lib, batch=1, dtype=BF16, params=F16) == UNSUPPORTED


def _norm_backward(lib, **k):
    a = dict(dy=P16, gb=0, gr=64, x=P16, xb=0, xr=64, dtype=BF16, factor=P16, params=BF16, pstride=64, add=1, eps=1e-6,
             batch=0, length=4, width=64, dx=P16, ob=0, orow=64, dfactor=P16, doffset=P16, ws=P16, nbytes=1 << 30)
    a.update(k)
    return lib.flk_layer_norm_backward(*a.values(), None)


def test_layer_norm_backward_checks(lib):
    assert _norm_backward(lib) == OK
    assert _norm_backward(lib, batch=1, dy=None) == INVALID
    assert _norm_backward(lib, batch=1, dy=P16 + 1) == ALIGN and _norm_backward(lib, batch=1, doffset=P16 + 1) == ALIGN
    size = ctypes.c_int64(-1)
    assert lib.flk_layer_norm_backward_plan(2, 4, 64, 0, ctypes.byref(size)) == OK and size.value >= 2 * 2 * 64 * 4
    need = size.value
    assert _norm_backward(lib, batch=2, nbytes=need - 1) == SCRATCH and _norm_backward(lib, batch=2, ws=None) == SCRATCH
    assert _norm_backward(lib, batch=2, ws=P16 + 4) == ALIGN
    assert _norm_backward(lib, batch=1 << 23, length=1) == INVALID   # more groups than one launch takes
    assert lib.flk_layer_norm_backward_plan(0, 4, 64, 0, ctypes.byref(size)) == OK and size.value == 0
    assert lib.flk_layer_norm_backward_plan(1, 4, 0, 0, ctypes.byref(size)) == INVALID
    assert lib.flk_layer_norm_backward_plan(1, 4, 8, 0, None) == INVALID


def test_norm_batch_limits(lib):
    """Each side of the limit on parameter rows, before anything is launched: the plan and the launch agree, and
    no product of batch and width is in the way."""
    most = 1 << 22
    size = ctypes.c_int64(-1)
    for batch, width, status in ((65535, 4096, OK), (65536, 4096, OK), (65537, 4096, OK), (most, 64, OK), (most, 16384, OK),
                                 (most + 1, 64, INVALID)):
        assert lib.flk_layer_norm_backward_plan(batch, 1, width, 0, ctypes.byref(size)) == status
        assert status != OK or size.value >= batch * 2 * width * 4
        # a workspace of no bytes is the last thing that is refused
        assert _norm_backward(lib, batch=batch, length=1, width=width, pstride=width, nbytes=0) == (SCRATCH if status == OK else status)
    assert _norm(lib, batch=most + 1, length=1) == INVALID
    assert _norm(lib, batch=most, length=0) == OK
    # one row of parameters for all entries: no limit but the rows'
    assert lib.flk_layer_norm_backward_plan(most + 1, 1, 64, 1, ctypes.byref(size)) == OK
    assert _norm_backward(lib, batch=most + 1, length=1, pstride=0, nbytes=0) == SCRATCH


def test_swiglu_checks(lib):
    def call(dtype=BF16, batch=0, length=3, hidden=5, gu=P16, h=P16):
        return lib.flk_swiglu(gu, 0, 10, dtype, batch, length, hidden, h, 0, 5, None)

    def back(dtype=BF16, batch=0, length=3, hidden=5, dh=P16, gu=P16, dgu=P16):
        return lib.flk_swiglu_backward(dh, 0, 5, gu, 0, 10, dtype, batch, length, hidden, dgu, 0, 10, None)

    for f in (call, back):
        assert f() == OK and f(dtype=3) == INVALID and f(hidden=0) == INVALID and f(batch=-1) == INVALID
        assert f(length=-1) == INVALID and f(hidden=2 ** 31 - 1) == INVALID
        assert f(batch=1, gu=None) == INVALID and f(batch=1, gu=P16 + 1) == ALIGN and f(batch=1, dtype=F32, gu=P16 + 2) == ALIGN
    assert call(batch=1, h=None) == INVALID and back(batch=1, dh=None) == INVALID and back(batch=1, dgu=P16 + 1) == ALIGN


def test_mlp_checks(lib):
    def gate(x=P16, xr=64, w=P16, wr=256, dtype=BF16, m=0, width=64, hidden=128, h=P16, hr=128, gu=P16, ws=P16):
        return lib.flk_mlp_gate(x, xr, w, wr, dtype, m, width, hidden, h, hr, gu, ws, 1 << 40, None)

    def back(x=P16, xr=64, w=P16, wr=64, gu=P16, dtype=BF16, m=0, width=64, hidden=128, h=P16, hr=256, ws=P16):
        return lib.flk_mlp_gate_backward(x, xr, w, wr, gu, dtype, m, width, hidden, h, hr, ws, 1 << 40, None)

    def mm(x=P16, xr=64, at=0, w=P16, wr=128, bt=0, dtype=BF16, rows=0, cols=128, inner=64, h=P16, hr=128):
        return lib.flk_mlp_matmul(x, xr, at, w, wr, bt, dtype, rows, cols, inner, h, hr, P16, 1 << 40, None)

    for f in (gate, back):
        assert f() == OK and f(dtype=F32) == INVALID and f(m=-1) == INVALID and f(width=-8) == INVALID
        assert f(xr=56) == INVALID and f(wr=56) == INVALID and f(hr=120) == INVALID
        assert f(m=1, x=None) == INVALID and f(m=1, w=None) == INVALID and f(m=1, h=None) == INVALID
        assert f(m=1, width=0) == INVALID and f(m=2 ** 31 - 1) == INVALID
        assert f(m=1, width=60) == UNSUPPORTED and f(m=1, hidden=100) == UNSUPPORTED
        assert f(m=1, xr=68) == ALIGN and f(m=1, wr=260) == ALIGN and f(m=1, hr=260) == ALIGN
        assert f(m=1, x=P16 + 8) == ALIGN and f(m=1, w=P16 + 8) == ALIGN and f(m=1, h=P16 + 8) == ALIGN
        assert f(m=1, gu=P16 + 8) == ALIGN
    assert back(m=1, gu=None) == INVALID
    assert mm() == OK and mm(rows=-1) == INVALID and mm(dtype=F32) == INVALID and mm(at=1, bt=1, wr=64) == UNSUPPORTED
    assert mm(xr=56) == INVALID and mm(wr=120) == INVALID and mm(hr=120) == INVALID
    assert mm(rows=1, inner=0) == INVALID and mm(rows=1, x=None) == INVALID
    assert mm(rows=1, inner=60) == UNSUPPORTED and mm(rows=1, cols=124) == UNSUPPORTED
    assert mm(at=1, rows=60, xr=64) == UNSUPPORTED
    assert mm(rows=1, xr=(1 << 22) + 8) == INVALID and mm(rows=1, wr=(1 << 22) + 8) == INVALID
    assert gate(m=1, wr=(1 << 22) + 8) == INVALID and back(m=1, xr=(1 << 22) + 8) == INVALID
    assert mm(rows=1, xr=68) == ALIGN and mm(rows=1, w=P16 + 8) == ALIGN
    size = ctypes.c_int64(-1)
    for product in range(5):
        assert lib.flk_mlp_plan(product, 1, 4096, 1024, ctypes.byref(size)) == OK and size.value >= 0
    assert lib.flk_mlp_plan(5, 1, 8, 8, ctypes.byref(size)) == INVALID
    assert lib.flk_mlp_plan(0, -1, 8, 8, ctypes.byref(size)) == INVALID and lib.flk_mlp_plan(0, 1, 8, 8, None) == INVALID


def test_mlp_tile_limits(lib):
    """Products past 2^22 tiles of 256 x 256 are refused by the plan and by the launch, and no smaller ones: where
    smaller tiles would be too many for one launch, larger ones are taken."""
    size = ctypes.c_int64(-1)
    most = 256 << 22
    for product in range(4):
        assert lib.flk_mlp_plan(product, most, 8, 8, ctypes.byref(size)) == OK and size.value == 0
        assert lib.flk_mlp_plan(product, most + 1, 8, 8, ctypes.byref(size)) == INVALID
    gate = lambda m: lib.flk_mlp_gate(P16, 8, P16, 16, BF16, m, 8, 8, P16, 8, None, None, 0, None)  # noqa: E731
    back = lambda m: lib.flk_mlp_gate_backward(P16, 8, P16, 8, P16, BF16, m, 8, 8, P16, 16, None, 0, None)  # noqa: E731
    for f in (gate, back):
        assert f(most + 1) == INVALID


def test_tiles_of_the_tested_sizes(lib):
    """The GPU tests' sizes reach every tile of every product, so that a change of the costs that choose between them
    does not leave one untested."""
    from tests.test_gpu_mlp import TILES
    reached = set()
    for product, tile, rows, cols, inners in TILES:
        for inner in inners:
            assert lib.flk_mlp_kernel(product, rows, cols, inner).decode() == tile, (product, rows, cols, inner)
        reached.add((product, tile))
    names = {"256x256", "192x256", "128x128 x2", "128x128 x2 split", "128x128 deep", "128x128 deep split", "128x32 split"}
    assert reached == {(p, n) for p in range(5) for n in names} - {(mlp._MATMUL_AT, "128x32 split")}
    for bad in ((5, 1, 8, 8), (-1, 1, 8, 8), (0, 0, 8, 8), (0, 1, 0, 8), (0, 1, 8, 0), (0, -1, 8, 8), (0, 2 ** 30 + 1, 8, 8)):
        assert lib.flk_mlp_kernel(*bad) == b""


def test_operand_layouts_of_the_products(lib, monkeypatch):
    """Rows further apart than the products address, or off 16 bytes, are copied; others are read in place."""
    monkeypatch.setattr(mlp, "_on_gpu", lambda name, t: None)
    most = 1 << 22
    memory = torch.zeros(2 * most + 64, dtype=torch.bfloat16)
    for row, offset, taken in ((most, 0, True), (most + 8, 0, False), (64, 0, True), (68, 0, False), (64, 4, False)):
        t = memory[offset:].as_strided((2, 64), (row, 1))
        t[1, 63] = 3.0
        m = mlp._matrix("x", t)
        assert torch.equal(m, t) and m.stride(1) == 1 and (m.data_ptr() == t.data_ptr()) == taken
        assert lib.flk_mlp_matmul(P16, m.stride(0), 0, P16, 8, 0, BF16, 0, 8, 64, P16, 8, None, 0, None) == OK
    first = torch.zeros(3, most // 64 + 1, 64, dtype=torch.bfloat16)[:, 0]   # each image's first token
    assert mlp._matrix("x", first).stride(0) == 64


def _owners(t, hidden, chunk):
    """Address -> the lanes of t's elements there; a lane takes `chunk` columns of a row, of both halves of a wide one."""
    found = {}
    for b, r, c in np.ndindex(*t.shape):
        at = t.data_ptr() + t.element_size() * (b * t.stride(0) + r * t.stride(1) + c * t.stride(2))
        found.setdefault(at, set()).add((b, r, c % hidden // chunk))
    return found


def test_overlapping_outputs_are_refused():
    """Random views of one small buffer, element by element: an output is accepted where no lane writes what another
    reads, and refused only where it shares memory."""
    r = np.random.RandomState(0)
    memory = torch.zeros(2000)
    accepted, refused, in_place = 0, 0, set()
    for _ in range(3000):
        kind, hidden = r.choice(["norm", "swiglu", "dh"]), int(r.choice([3, 8, 16, 20]))
        columns = {"norm": (0,), "swiglu": (0, hidden), "dh": (0, -hidden)}[kind]
        shape = (int(r.randint(1, 4)), int(r.randint(1, 4)))
        row = int(r.choice([hidden, 2 * hidden, 2 * hidden + 5, 50]))
        strides = (int(r.choice([0, row * shape[1], row * shape[1] + 7, 200])), int(r.choice([row, row, 2 * hidden])), 1)
        t = memory[40 + int(r.randint(0, 60)):].as_strided((*shape, hidden * (1 + (kind == "swiglu"))), strides)
        if r.rand() < 0.5:
            strides = (row * shape[1], row, 1)
        start = t.storage_offset() + int(r.choice([*columns, r.randint(-40, 60), r.randint(-40, 300)]))
        out = memory[start:].as_strided((*shape, hidden * (1 + (kind == "dh"))), strides)
        if not norm._rows_apart(out):
            continue
        chunk = hidden if kind == "norm" else 8   # a norm's rows are read whole before they are written
        written, read = _owners(out, hidden, chunk), _owners(t, hidden, chunk)
        shared = written.keys() & read.keys()
        try:
            norm._refuse_overlap("t", out, t, columns)
        except ValueError as error:
            assert shared and "shares memory with t" in str(error)
            refused += 1
            continue
        assert all(read[at] == written[at] and len(read[at]) == 1 for at in shared), (kind, out.stride(), start, t.stride(), t.storage_offset())
        accepted += not shared
        if shared:
            in_place.add((kind, out.data_ptr() == t.data_ptr()))
    assert accepted > 300 and refused > 300 and len(in_place) == 5, (accepted, refused, in_place)


def test_python_refuses_host_tensors_and_bad_calls():
    x = torch.zeros(2, 3, 16, dtype=torch.bfloat16)
    for call in (lambda: norm.layer_norm(x), lambda: norm.modulate(x, x[:, 0], x[:, 0]), lambda: mlp.swiglu(x),
                 lambda: norm.layer_norm_backward(x, x), lambda: mlp.swiglu_backward(x[..., :8], x),
                 lambda: mlp.gated_mlp(x, torch.zeros(16, 32), torch.zeros(16, 16)),
                 lambda: autograd.layer_norm(x), lambda: autograd.swiglu(x)):
        with pytest.raises(ValueError, match="GPU only"):
            call()
    with pytest.raises(TypeError, match="torch.Tensor"):
        norm.layer_norm([1.0, 2.0])


def test_autograd_refuses_a_captured_backward_pass(monkeypatch):
    """A backward pass of an eager forward pass, under capture: refused before it computes anything."""
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="explicit"):
        autograd._Swiglu.backward(None, None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="first derivatives only"):
        autograd._Swiglu.backward(None, None)


def test_autograd_refuses_forward_mode(monkeypatch):
    """An operand with a tangent, with and without recorded gradients beside it: no result without its tangent."""
    import torch.autograd.forward_ad as fwd
    monkeypatch.setattr(autograd._norm, "layer_norm", lambda x, w, b, eps: x * 2)
    monkeypatch.setattr(autograd._norm, "modulate", lambda x, shift, scale, eps: x * 2)
    monkeypatch.setattr(autograd._mlp, "swiglu", lambda gu: gu[..., :4] * 2)
    monkeypatch.setattr(autograd._mlp, "gated_mlp", lambda x, w_in, w_out, keep=False:
                        (x * 2, mlp.Kept(x[:, :1], x[:, :1])) if keep else x * 2)
    x, w_in, w_out = torch.randn(3, 8), torch.randn(8, 16), torch.randn(8, 8)
    assert torch.equal(autograd.gated_mlp(x, w_in, w_out), x * 2)
    assert not autograd.gated_mlp(x, w_in, w_out).requires_grad
    assert autograd.gated_mlp(x, w_in.requires_grad_(), w_out).requires_grad
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: autograd.layer_norm(dual), lambda: autograd.modulate(dual, x, x), lambda: autograd.swiglu(dual),
                     lambda: autograd.gated_mlp(dual, w_in, w_out), lambda: autograd.gated_mlp(dual, w_in.detach(), w_out),
                     lambda: autograd.gated_mlp(x, w_in.detach(), fwd.make_dual(w_out, torch.ones_like(w_out)))):
            with pytest.raises(NotImplementedError):
                call()
