"""Attention and its neighbours without a GPU: the oracle against differences of its own forward pass, the C entry points'
checks of arguments, and the Python layer's refusals."""

import ctypes

import numpy as np
import pytest
import torch

from flicker_amd import _lib, attention, autograd, kernels, norm
from oracle import attention as O

OK, INVALID, ALIGN, UNSUPPORTED, SCRATCH = 0, -1, -2, -3, -4
BF16, F16, F32 = 0, 1, 2
P = 4096   # any aligned address: the checks come before the launch


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.fail("libflicker_hip.so is not built (python -m flicker_amd.build)")
    return _lib.lib()


@pytest.mark.parametrize("masked", [False, True])
def test_oracle_gradients_are_the_forward_pass_differences(masked):
    r = np.random.RandomState(3)
    q, k, v, do = r.randn(5, 8), r.randn(7, 8), r.randn(7, 8), r.randn(5, 8)
    keep = np.array([1, 0, 1, 1, 0, 1, 1], bool) if masked else None
    ops = [q, k, v]
    for i, grad in enumerate(O.attention_grads(do, q, k, v, keep)):
        along, h = r.randn(*ops[i].shape), 1e-5

        def loss(t):
            return float((O.attention(*ops[:i], t, *ops[i + 1:], keep) * do).sum())
        got = (loss(ops[i] + h * along) - loss(ops[i] - h * along)) / (2 * h)
        assert abs((grad * along).sum() - got) < 1e-6


def test_oracle_leaves_masked_keys_out():
    r = np.random.RandomState(4)
    q, k, v, do = r.randn(3, 8), r.randn(6, 8), r.randn(6, 8), r.randn(3, 8)
    keep = np.array([1, 1, 0, 1, 0, 1], bool)
    k[~keep], v[~keep] = np.nan, np.inf
    assert np.allclose(O.attention(q, k, v, keep), O.attention(q, k[keep], v[keep]))
    dq, dk, dv = O.attention_grads(do, q, k, v, keep)
    assert not dk[~keep].any() and not dv[~keep].any()
    none = np.zeros(6, bool)
    assert not O.attention(q, k, v, none).any() and np.isneginf(O.probabilities(q, k, none)[2]).all()


def _strides(*s):
    return (ctypes.c_int64 * 3)(*s)


def _bytes(lib, b, h, kv, nq, nk, masked, backward):
    size = ctypes.c_int64(-1)
    assert lib.flk_attention_plan(b, h, kv, nq, nk, masked, backward, ctypes.byref(size)) == OK
    return size.value


def test_plan(lib):
    size = ctypes.c_int64(0)
    plan = lib.flk_attention_plan
    for bad in ((-1, 2, 2, 4, 4), (1, 0, 1, 4, 4), (1, 3, 2, 4, 4), (1, 2, 0, 4, 4), (1, 2, 2, -4, 4), (1, 2, 2, 4, -4),
                (1, 1, 1, 2 ** 29, 4), (1, 1, 1, 4, 2 ** 29), (64, 64, 64, 2 ** 20, 4), (2 ** 21, 1, 1, 1, 1)):
        assert plan(*bad, 0, 0, ctypes.byref(size)) == INVALID, bad
    assert plan(1, 2, 2, 4, 4, 0, 0, None) == INVALID
    assert _bytes(lib, 0, 2, 2, 4, 4, 1, 1) == 0 and _bytes(lib, 1, 2, 2, 0, 4, 1, 1) == 0
    assert _bytes(lib, 1, 24, 24, 512, 64, 0, 0) == 0               # nothing to cut, no mask
    assert _bytes(lib, 1, 24, 24, 512, 64, 1, 0) == 0               # nor a mask that needs room
    assert _bytes(lib, 1, 24, 24, 512, 2049, 1, 0) > 0
    assert _bytes(lib, 1, 24, 24, 1, 4608, 0, 0) > 0                # cut along the keys
    for b, h, kv, nq, nk in ((1, 24, 24, 4608, 4608), (3, 12, 4, 987, 1203), (2, 6, 1, 1, 2 ** 20), (1, 1, 1, 2 ** 20, 1)):
        for masked in (0, 1):
            for backward in (0, 1):
                n = _bytes(lib, b, h, kv, nq, nk, masked, backward)
                assert 0 <= n < 2 ** 32 and n % 16 == 0


def _forward(lib, **kw):
    a = dict(q=P, qs=_strides(0, 1280, 128), k=P, ks=_strides(0, 1280, 128), v=P, vs=_strides(0, 1280, 128), dtype=BF16, mask=None,
             mb=0, b=1, h=2, kv=2, nq=10, nk=10, d=128, o=P, os=_strides(0, 128, 256), low=None, lse=None, ws=None, nb=0, st=None)
    a.update(kw)
    return lib.flk_attention(*a.values())


def test_forward_validation(lib):
    assert _forward(lib, b=0) == OK and _forward(lib, nq=0) == OK
    for kw in (dict(dtype=F32), dict(dtype=7), dict(h=3), dict(nq=-1), dict(nk=2 ** 29), dict(q=None), dict(k=None), dict(v=None),
               dict(o=None), dict(qs=None), dict(ks=_strides(0, 0, 2 ** 25 + 8)), dict(vs=_strides(0, 0, -128))):
        assert _forward(lib, **kw) == INVALID, kw
    assert _forward(lib, d=64) == UNSUPPORTED
    assert _forward(lib, low=P) == INVALID and _forward(lib, lse=P) == INVALID
    for kw in (dict(q=P + 8), dict(k=P + 2), dict(o=P + 4), dict(low=P + 8, lse=P), dict(low=P, lse=P + 2), dict(qs=_strides(0, 1280, 132)),
               dict(os=_strides(4, 128, 256))):
        assert _forward(lib, **kw) == ALIGN, kw
    assert _forward(lib, mask=P, nk=2049) == SCRATCH
    need = _bytes(lib, 1, 2, 2, 10, 2049, 1, 0)
    assert _forward(lib, mask=P, nk=2049, ws=P, nb=need - 1) == SCRATCH
    assert _forward(lib, mask=P, nk=2049, ws=P + 16, nb=need) == ALIGN


def _backward(lib, **kw):
    s = _strides(0, 1280, 128)
    a = dict(do=P, dos=_strides(0, 128, 256), q=P, qs=s, k=P, ks=s, v=P, vs=s, o=P, os=_strides(0, 128, 256), low=P, lse=P,
             dtype=BF16, mask=None, mb=0, b=1, h=2, kv=2, nq=10, nk=10, d=128, dq=P, dqs=s, dk=P, dks=s, dv=P, dvs=s, ws=P,
             nb=1 << 20, st=None)
    a.update(kw)
    return lib.flk_attention_backward(*a.values())


def test_backward_validation(lib):
    for kw in (dict(b=0), dict(nq=0), dict(nk=0)):
        assert _backward(lib, **kw) == OK
    for name in ("do", "q", "k", "v", "o", "dq", "dk", "dv"):
        assert _backward(lib, **{name: None}) == INVALID and _backward(lib, **{name: P + 8}) == ALIGN, name
        assert _backward(lib, **{name + "s": None}) == INVALID, name
        assert _backward(lib, **{name + "s": _strides(0, 4, 128)}) == ALIGN, name
    for kw in (dict(low=None), dict(lse=None), dict(dtype=F32), dict(kv=3)):
        assert _backward(lib, **kw) == INVALID, kw
    assert _backward(lib, low=P + 8) == ALIGN and _backward(lib, lse=P + 1) == ALIGN and _backward(lib, d=256) == UNSUPPORTED
    need = _bytes(lib, 1, 2, 2, 10, 10, 0, 1)
    assert need > 0 and _backward(lib, nb=need - 1) == SCRATCH and _backward(lib, ws=None) == SCRATCH
    assert _backward(lib, ws=P + 16) == ALIGN


def test_qk_prep_backward_validation(lib):
    size = ctypes.c_int64(0)
    plan = lib.flk_qk_prep_backward_plan
    for bad in ((-1, 4, 2), (1, -1, 2), (1, 4, 0), (1, 2 ** 31 - 1, 1), (2 ** 20, 2 ** 20, 24)):
        assert plan(*bad, ctypes.byref(size)) == INVALID, bad
    assert plan(1, 100, 3, ctypes.byref(size)) == OK and size.value > 0
    s = _strides(0, 1280, 128)

    def call(**kw):
        a = dict(dq=P, dqs=s, dk=P, dks=s, dv=P, dvs=s, qkv=P, qb=0, qr=1152, cos=P, sin=P, tr=128, qsc=P, ksc=P, f32=0, gain=1.0,
                 b=1, n=10, h=3, d=128, out=P, ob=0, orow=1152, dqsc=P, dksc=P, ws=P, nb=1 << 22, st=None)
        a.update(kw)
        return lib.flk_qk_prep_backward(*a.values())
    assert call(b=0) == OK and call(n=0) == OK and call(d=64) == UNSUPPORTED
    for name in ("dq", "dk", "dv", "qkv", "cos", "sin", "qsc", "ksc", "out"):
        assert call(**{name: None}) == INVALID and call(**{name: P + 8}) == ALIGN, name
    for kw in (dict(dqsc=None), dict(dksc=None), dict(tr=64), dict(h=0), dict(dqs=None)):
        assert call(**kw) == INVALID, kw
    for kw in (dict(qr=1156), dict(orow=1156), dict(tr=130), dict(dks=_strides(0, 1280, 130)), dict(dqsc=P + 1), dict(f32=1, dksc=P + 2),
               dict(ws=P + 8)):
        assert call(**kw) == ALIGN, kw
    assert call(ws=None) == SCRATCH and call(nb=4) == SCRATCH


def test_residual_norm_validation(lib):
    def forward(**kw):
        a = dict(x=P, xb=64, xr=64, br=P, bb=64, brr=64, dtype=BF16, gate=P, f=P, o=P, pd=BF16, ps=64, one=1, eps=1e-6, b=1, n=3,
                 w=64, r=P, rb=64, rr=64, y=P, yb=64, yr=64, st=None)
        a.update(kw)
        return lib.flk_residual_norm(*a.values())
    assert forward(b=0) == OK and forward(n=0) == OK
    for kw in (dict(x=None), dict(br=None), dict(r=None), dict(y=None), dict(gate=None), dict(dtype=5), dict(pd=5), dict(w=0),
               dict(eps=float("nan")), dict(ps=32)):
        assert forward(**kw) == INVALID, kw
    assert forward(w=16385, ps=16385) == UNSUPPORTED and forward(pd=F16) == UNSUPPORTED
    for kw in (dict(br=P + 1), dict(gate=P + 1), dict(r=P + 1)):
        assert forward(**kw) == ALIGN, kw
    size, half = ctypes.c_int64(0), ctypes.c_int64(0)
    assert lib.flk_residual_norm_backward_plan(2, 9, 64, 0, ctypes.byref(size)) == OK
    assert lib.flk_layer_norm_backward_plan(2, 9, 64, 0, ctypes.byref(half)) == OK and size.value * 2 == half.value * 3
    assert lib.flk_residual_norm_backward_plan(2, 9, 0, 0, ctypes.byref(size)) == INVALID

    def backward(**kw):
        rows = {n + s: v for n in ("dr", "dy", "x", "br") for s, v in (("", P), ("b", 64), ("r", 64))}
        a = dict(rows, dtype=BF16, gate=P, f=P, pd=BF16, ps=64, one=1, eps=1e-6, b=1, n=3, w=64, dx=P, dxb=64, dxr=64, db=P, dbb=64,
                 dbr=64, dg=P, df=P, do=P, ws=P, nb=1 << 20, st=None)
        a.update(kw)
        return lib.flk_residual_norm_backward(*a.values())
    assert backward(n=0) == OK
    for name in ("dr", "dy", "x", "br", "dx", "db", "gate"):
        assert backward(**{name: None}) == INVALID and backward(**{name: P + 1}) == ALIGN, name
    assert backward(nb=4) == SCRATCH and backward(ws=None) == SCRATCH and backward(ws=P + 8) == ALIGN
    assert backward(dg=P + 1) == ALIGN


def test_python_refuses_host_tensors():
    q = torch.zeros(1, 2, 4, 128, dtype=torch.bfloat16)
    x, row = torch.zeros(1, 4, 64), torch.zeros(1, 64)
    qkv, scale = torch.zeros(1, 4, 768, dtype=torch.bfloat16), torch.ones(128)
    freqs = kernels.Freqs(torch.zeros(4, 128), torch.zeros(4, 128), 1.0)
    kept = attention.Kept(torch.zeros(1, 4, 256), torch.zeros(1, 4, 256), torch.zeros(1, 2, 4))
    for call in (lambda: attention.attention(q, q, q), lambda: attention.attention_backward(kept.o, q, q, q, kept),
                 lambda: autograd.attention(q, q, q), lambda: norm.residual_modulate(x, x, row, row, row),
                 lambda: norm.residual_modulate_backward(x, x, x, x, row, row, row),
                 lambda: autograd.residual_modulate(x, x, row, row, row),
                 lambda: kernels.qk_prep_backward(q, q, q, qkv, scale, scale, freqs, 2),
                 lambda: autograd.qk_prep(qkv, scale, scale, freqs, 2)):
        with pytest.raises(ValueError, match="GPU only"):
            call()
    with pytest.raises(TypeError, match="torch.Tensor"):
        attention.attention(None, q, q)


@pytest.mark.parametrize("name", ["_ResidualModulate", "_QkPrep", "_Attention"])
def test_autograd_refuses_capture_and_second_derivatives(monkeypatch, name):
    fn = getattr(autograd, name)
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with torch.no_grad(), pytest.raises(RuntimeError, match="explicit"):
        fn.backward(None, None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    with torch.enable_grad(), pytest.raises(RuntimeError, match="first derivatives only"):
        fn.backward(None, None)


def test_autograd_refuses_forward_mode(monkeypatch):
    import torch.autograd.forward_ad as fwd
    monkeypatch.setattr(autograd._attention, "attention", lambda q, k, v, key_mask=None, keep=False:
                        (q * 2, attention.Kept(q * 2, q, q)) if keep else q * 2)
    monkeypatch.setattr(autograd._norm, "residual_modulate", lambda x, b, g, s, c, eps: (x * 2, x * 3))
    x = torch.randn(3, 4)
    assert torch.equal(autograd.attention(x, x, x), x * 2)
    assert autograd.attention(x, x.clone().requires_grad_(), x).requires_grad
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for call in (lambda: autograd.attention(dual, x, x), lambda: autograd.residual_modulate(x, dual, x, x, x)):
            with pytest.raises(NotImplementedError):
                call()


def test_sizes_whose_products_pass_64_bits(lib):
    """Sizes that each are in range are refused by their product, also where it wraps around to nothing."""
    size = ctypes.c_int64(0)
    for heads in (2 ** 24, 2 ** 30):
        assert lib.flk_attention_plan(2 ** 20, heads, heads, 2 ** 28, 2 ** 28, 0, 1, ctypes.byref(size)) == INVALID
        assert lib.flk_attention_plan(2 ** 20, heads, 1, 2 ** 28, 1, 0, 1, ctypes.byref(size)) == INVALID
    for batch, length, heads in ((2 ** 30, 2 ** 30, 2 ** 20), (2 ** 30, 2 ** 28, 2 ** 10)):
        assert lib.flk_qk_prep_backward_plan(batch, length, heads, ctypes.byref(size)) == INVALID
