"""norm.layer_norm / modulate and mlp.swiglu with their gradients on the GPU against the float64 oracle.

Tolerances.  An output of type t is rounded once: half a step, eps(t) / 2 of its value (and half the smallest
subnormal).  What the float32 arithmetic before it adds, in units of u = 2^-24:
  * a row's mean: at most 128 additions deep (64 a lane, then the lanes), so off by 130 u mean|x|; the
    centred value, its square mean and 1 / sqrt are off by 140 u of their own on top.  n = (x - m) q is off by
    dn = 300 u (|n| + q mean|x|).
  * y = n a + c: |a| dn + 4 u (|n a| + |c|).
  * dx = q (t - mean t - n mean(t n)): the two means are off by 130 u of their absolute values' means, and by what dn
    makes of the second; q by 300 u of itself.
  * a parameter's gradient over R rows: additions at most R + 64 deep, so (R + 64) u sum|dy n| + sum |dy| dn.
  * the gate: exp(-|g|) is off by (|g| + 4) u, the sigmoid and one minus it by as much of their own value plus
    4 u; products add 4 u.  Where exp(-|g|) < 2^-126 it may be zero: 2^-126 |g u|.
"""

import numpy as np
import pytest
import torch

from flicker_amd import autograd, mlp, norm
from oracle import mlp as M

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -150}


def _f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def _close(label, got, want, extra):
    assert got.shape == tuple(want.shape), (label, got.shape, want.shape)
    tol = torch.finfo(got.dtype).eps / 2 * (np.abs(want) + extra) + extra + TINY[got.dtype]
    over = np.abs(_f64(got) - want) - tol
    assert np.isfinite(_f64(got)).all() and over.max(initial=-1.0) <= 0, \
        f"{label}: {np.argwhere(over > 0)[:5].tolist()} of {int((over > 0).sum())}, worst {over.max():.3g} over {tol.flat[over.argmax()]:.3g}"


def _stream(seed, batch, length, width, dtype, device):
    """A residual stream: tokens off zero and of different size, a few large channels."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(batch, length, width, generator=g) * torch.exp(0.5 * torch.randn(batch, length, 1, generator=g))
    x = x + torch.randn(batch, length, 1, generator=g)
    x[..., ::97] *= 10.0
    return x.to(dtype).to(device), g


def _mean_abs(x):
    return np.abs(x).mean(-1, keepdims=True)


def _norm_case(x, factor, offset, dy, over, eps=norm.EPS):
    """(y, its tolerance), (dx, ...), (dfactor, ...), (doffset, ...) of float64 operands."""
    n, rstd = M._stats(x, eps)
    dn = 300 * U * (np.abs(n) + rstd * _mean_abs(x))
    y = n * factor + offset
    y_tol = np.abs(factor) * dn + 4 * U * (np.abs(n * factor) + np.abs(offset))
    dx, dyn, dyo = M.layer_norm_grads(dy, x, factor, eps)
    t = np.abs(dy * factor)
    tn_off = 130 * U * (t * np.abs(n)).mean(-1, keepdims=True) + (t * dn).mean(-1, keepdims=True)
    mtn = np.abs((dy * factor * n).mean(-1, keepdims=True))
    dx_tol = rstd * (8 * U * t + 130 * U * t.mean(-1, keepdims=True) + np.abs(n) * tn_off + dn * mtn
                     + 300 * U * (t + t.mean(-1, keepdims=True) + np.abs(n) * mtn))
    rows = np.prod([x.shape[i] for i in over])
    da_tol = (rows + 64) * U * np.abs(dyn).sum(over) + (np.abs(dy) * dn).sum(over)
    return (y, y_tol), (dx, dx_tol), (dyn.sum(over), da_tol), (dyo.sum(over), (rows + 64) * U * np.abs(dyo).sum(over))


WIDTHS = [1, 2, 7, 8, 64, 511, 513, 1000, 1536, 2049, 24 * 128, 4096, 5001, 8200, 16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("dtype,params", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
def test_modulate(device, width, dtype, params):
    batch, length = 2, 11
    print(f"modulate width={width} {dtype}/{params}", flush=True)
    x, g = _stream(width, batch, length, width, TYPES[dtype], device)
    shift, scale = (torch.randn(batch, 1, width, generator=g).to(TYPES[params]).to(device) for _ in range(2))
    dy = torch.randn(batch, length, width, generator=g).to(TYPES[dtype]).to(device)
    y, dx, da, dc = _norm_case(_f64(x), 1 + _f64(scale), _f64(shift), _f64(dy), (1,))
    _close("y", norm.modulate(x, shift, scale), *y)
    got_dx, dshift, dscale = norm.modulate_backward(dy, x, shift, scale)
    _close("dx", got_dx, *dx)
    assert dshift.dtype == shift.dtype and dscale.dtype == scale.dtype
    _close("dscale", dscale.view(batch, width), *da)
    _close("dshift", dshift.view(batch, width), *dc)
    assert dshift.shape == shift.shape and dscale.shape == scale.shape


@pytest.mark.parametrize("batch,length", [(1, 1), (1, 2), (3, 1), (1, 257), (2, 700), (5, 1031)])
@pytest.mark.parametrize("width,dtype", [(96, "bf16"), (1111, "fp32"), (4000, "fp16")])
def test_layer_norm_rows(device, batch, length, width, dtype):
    print(f"layer_norm batch={batch} length={length} width={width} {dtype}", flush=True)
    x, g = _stream(3, batch, length, width, TYPES[dtype], device)
    weight = (1 + 0.2 * torch.randn(width, generator=g)).to(TYPES[dtype]).to(device)
    bias = torch.randn(width, generator=g).to(TYPES[dtype]).to(device)
    dy = torch.randn(batch, length, width, generator=g).to(TYPES[dtype]).to(device)
    y, dx, da, dc = _norm_case(_f64(x), _f64(weight), _f64(bias), _f64(dy), (0, 1))
    _close("y", norm.layer_norm(x, weight, bias), *y)
    grads = norm.layer_norm_backward(dy, x, weight, bias)
    for label, got, want in zip(("dx", "dweight", "dbias"), grads, (dx, da, dc)):
        _close(label, got, *want)
    again = norm.layer_norm_backward(dy, x, weight, bias)
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "the sums' order does not depend on timing"


@pytest.mark.parametrize("length,width", [(700000, 7), (50001, 100), (333, 16001)])
def test_large_float32_outputs(device, length, width):
    """Float32 outputs past 18 MB are stored through the caches, by kernels of their own for narrow, ordinary and wide rows."""
    assert 4 * length * width > 18 << 20
    print(f"layer_norm length={length} width={width} float32", flush=True)
    x, g = _stream(width, 1, length, width, torch.float32, device)
    weight, bias = ((1 + 0.2 * torch.randn(width, generator=g)).to(device) for _ in range(2))
    dy = torch.randn(x.shape, generator=g).to(device)
    y, dx, da, dc = _norm_case(_f64(x), _f64(weight), _f64(bias), _f64(dy), (0, 1))
    _close("y", norm.layer_norm(x, weight, bias), *y)
    for label, got, want in zip(("dx", "dweight", "dbias"), norm.layer_norm_backward(dy, x, weight, bias), (dx, da, dc)):
        _close(label, got, *want)


def test_many_rows(device):
    """Enough rows that every block of the backward pass walks many, with as many batch entries as rows too."""
    x, g = _stream(5, 4, 9000, 40, torch.bfloat16, device)
    dy = torch.randn(x.shape, generator=g).to(torch.bfloat16).to(device)
    one = torch.ones(40, dtype=torch.bfloat16, device=device)
    _, dx, da, dc = _norm_case(_f64(x), 1.0, 0.0, _f64(dy), (0, 1))
    grads = norm.layer_norm_backward(dy, x, one, one)
    for label, got, want in zip(("dx", "dweight", "dbias"), grads, (dx, da, dc)):
        _close(label, got, *want)
    xs, gs = x.view(-1, 3, 40), dy.view(-1, 3, 40)
    zero = torch.zeros(xs.shape[0], 40, device=device)
    _, dx, da, dc = _norm_case(_f64(xs), 1.0, 0.0, _f64(gs), (1,))
    for label, got, want in zip(("dx", "dshift", "dscale"), norm.modulate_backward(gs, xs, zero, zero), (dx, dc, da)):
        _close(label, got, *want)


def test_more_parameter_rows_than_one_launch_takes(device):
    """Per-token modulation of many tokens: every entry's outputs are those of a call on fewer entries."""
    batch, width, part = 65536 + 3, 4096, 16384
    g = torch.Generator(device).manual_seed(12)
    x, dy, shift, scale = (torch.randn(batch, 1, width, generator=g, device=device, dtype=torch.bfloat16) for _ in range(4))
    print(f"modulate batch={batch} width={width}", flush=True)
    y = norm.modulate(x, shift, scale)
    print(f"modulate_backward batch={batch} width={width}", flush=True)
    grads = norm.modulate_backward(dy, x, shift, scale)
    assert torch.equal(grads[1], dy)   # a sum of one row
    for at in range(0, batch, part):
        s = slice(at, at + part)
        assert torch.equal(y[s], norm.modulate(x[s], shift[s], scale[s]))
        for got, want in zip(grads, norm.modulate_backward(dy[s], x[s], shift[s], scale[s])):
            assert torch.equal(got[s], want)


def test_most_batch_entries(device):
    """2^22 entries with blocks of 576 threads, more work-items than one launch takes, of one row and no parameters."""
    from flicker_amd import _lib
    batch, width = 1 << 22, 4104
    x = torch.randn(1, width, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(device)
    want = norm.layer_norm(x)
    y = torch.zeros(batch, width, dtype=torch.bfloat16, device=device)
    print(f"flk_layer_norm batch={batch} width={width}", flush=True)
    _lib.run("flk_layer_norm", (x, y), x.data_ptr(), 0, width, 0, None, None, 0, width, 0, 1e-6, batch, 1, width, y.data_ptr(),
             width, width, _lib.stream_of(x))
    assert all(bool((part == want).all()) for part in y.split(1 << 18))


def test_optional_parameters(device):
    x, g = _stream(7, 2, 5, 72, torch.float32, device)
    w, b = torch.randn(72, generator=g).to(device), torch.randn(72, generator=g).to(device)
    dy = torch.randn(x.shape, generator=g).to(device)
    for weight, bias in ((None, None), (w, None), (None, b)):
        y, dx, da, dc = _norm_case(_f64(x), 1.0 if weight is None else _f64(w), 0.0 if bias is None else _f64(b), _f64(dy), (0, 1))
        _close("y", norm.layer_norm(x, weight, bias), *y)
        got = norm.layer_norm_backward(dy, x, weight, bias)
        _close("dx", got[0], *dx)
        for value, given, want in zip(got[1:], (weight, bias), (da, dc)):
            assert (value is None) == (given is None)
            if given is not None:
                _close("parameter", value, *want)


def test_eps_and_constant_rows(device):
    """A row of one value has no variance: n = 0 exactly where the mean is exact, and 1 / sqrt(eps) scales dx."""
    x = torch.full((1, 3, 64), 3.0, dtype=torch.bfloat16, device=device)
    w, b = torch.full((64,), 2.0, device=device), torch.full((64,), -1.5, device=device)
    assert torch.equal(norm.layer_norm(x, w, b), torch.full_like(x, -1.5))
    g = torch.Generator().manual_seed(0)
    dy = torch.randn(1, 3, 64, generator=g).to(torch.bfloat16).to(device)
    for eps in (1e-6, 0.25):
        _, dx, da, dc = _norm_case(_f64(x), 2.0, 0.0, _f64(dy), (0, 1), eps)
        for label, got, want in zip(("dx", "dw", "db"), norm.layer_norm_backward(dy, x, w, b, eps=eps), (dx, da, dc)):
            _close(label, got, *want)


@pytest.mark.parametrize("width", [64, 1024, 16384])
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_small_variance_without_eps(device, width, dtype):
    """Rows of +-2^-66, whose squares and variance are float32 subnormals (2^-132, exact): n is exactly +-1, and
    with dy = n / 2 + 1 (+ 1 on the first half) every mean that dx takes is a sum of few powers of two."""
    sign = torch.ones(width, device=device)
    sign[1::2] = -1.0
    x = (sign * 2.0 ** -66).to(TYPES[dtype]).repeat(3, 1)
    assert torch.equal(norm.layer_norm(x, eps=0.0), sign.to(x.dtype).repeat(3, 1))
    dy = (sign / 2 + 1).repeat(3, 1)
    dy[:, :width // 2] += 1.0
    dy = dy.to(x.dtype)
    one = torch.ones(width, dtype=x.dtype, device=device)
    dx, dw, db = norm.layer_norm_backward(dy, x, one, one, eps=0.0)
    half = torch.full((3, width), -0.5, device=device)   # dy - mean dy - n mean(dy n)
    half[:, :width // 2] = 0.5
    assert torch.equal(dx, (half * 2.0 ** 66).to(x.dtype))
    assert torch.equal(dw, (3 * dy[0].float() * sign).to(x.dtype)) and torch.equal(db, (3 * dy[0].float()).to(x.dtype))


def test_not_finite_values_stay_in_their_rows(device):
    x = torch.randn(1, 6, 80, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(device)
    clean = norm.layer_norm(x)
    bad = x.clone()
    bad[0, 2, 5], bad[0, 4, 79] = float("nan"), float("inf")
    got = norm.layer_norm(bad)
    assert got[0, [2, 4]].isnan().all() and torch.equal(got[0, [0, 1, 3, 5]], clean[0, [0, 1, 3, 5]])


def test_views_are_read_and_written_in_place(device):
    """One stream of a joint sequence in, columns of a wider buffer out: rows beside them stay as they were."""
    joint, g = _stream(9, 2, 30, 136, torch.bfloat16, device)
    shift, scale = (torch.randn(2, 136, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    x = joint[:, 11:]
    want = norm.modulate(x.contiguous(), shift, scale)
    assert torch.equal(norm.modulate(x, shift, scale), want)
    wide = torch.full((2, 25, 150), 7.0, dtype=torch.bfloat16, device=device)
    assert norm.modulate(x, shift, scale, out=wide[:, 3:22, 9:145]).data_ptr() == wide[:, 3:22, 9:145].data_ptr()
    assert torch.equal(wide[:, 3:22, 9:145], want)
    wide[:, 3:22, 9:145] = 7.0
    assert (wide == 7.0).all()
    turned = torch.empty(19, 2, 136, dtype=torch.bfloat16, device=device).transpose(0, 1)   # rows of two images in turns
    assert torch.equal(norm.modulate(x, shift, scale, out=turned), want)
    same = x.clone()
    assert torch.equal(norm.modulate(same, shift, scale, out=same), want)
    for got, w in zip(norm.modulate_backward(x * 0.5, x, shift, scale),
                      norm.modulate_backward((x * 0.5).contiguous(), x.contiguous(), shift, scale)):
        assert torch.equal(got, w)
    # an odd element offset, a transposed and an expanded operand
    flat = joint.reshape(-1)[1:1 + 7 * 135].view(7, 135)
    assert torch.equal(norm.layer_norm(flat), norm.layer_norm(flat.clone()))
    assert torch.equal(norm.layer_norm(joint.transpose(1, 2)), norm.layer_norm(joint.transpose(1, 2).contiguous()))
    one = joint[:1].expand(3, -1, -1)
    assert torch.equal(norm.layer_norm(one)[2], norm.layer_norm(joint[:1])[0])
    assert torch.equal(norm.layer_norm(joint[0, 0]), norm.layer_norm(joint)[0, 0])


def test_empty(device):
    x = torch.empty(2, 0, 24, dtype=torch.bfloat16, device=device)
    p = torch.ones(2, 24, dtype=torch.bfloat16, device=device)
    assert norm.modulate(x, p, p).shape == x.shape
    dx, dshift, dscale = norm.modulate_backward(x, x, p, p)
    assert dx.shape == x.shape and not dshift.any() and not dscale.any() and dscale.shape == p.shape
    gu = torch.empty(0, 6, device=device)
    assert mlp.swiglu(gu).shape == (0, 3) and mlp.swiglu_backward(gu[:, :3], gu).shape == (0, 6)


def test_norm_refusals(device):
    x = torch.zeros(2, 3, 16, dtype=torch.bfloat16, device=device)
    p = torch.zeros(16, dtype=torch.bfloat16, device=device)
    with pytest.raises(TypeError, match="float16 or float32"):
        norm.layer_norm(x.double())
    with pytest.raises(TypeError, match="or float32"):
        norm.layer_norm(x, p.half())
    with pytest.raises(TypeError, match="share one dtype"):
        norm.layer_norm(x, p, p.float())
    with pytest.raises(ValueError, match="weight must be"):
        norm.layer_norm(x, p[:8])
    with pytest.raises(ValueError, match="shift must be"):
        norm.modulate(x, p, p)
    with pytest.raises(TypeError, match="both"):
        norm.modulate(x, None, torch.zeros(2, 16, device=device))
    with pytest.raises(ValueError, match=r"\(B, L, width\)"):
        norm.modulate(x[0], p, p)
    with pytest.raises(ValueError, match="width"):
        norm.layer_norm(x[0, 0, 0])
    with pytest.raises(ValueError, match="dy must be"):
        norm.layer_norm_backward(x[:1], x)
    with pytest.raises(ValueError, match="out must be"):
        norm.layer_norm(x, out=x.float())
    with pytest.raises(ValueError, match="do not overlap"):
        norm.layer_norm(x, out=x[:, :1].expand(2, 3, 16))
    with pytest.raises(ValueError, match="do not overlap"):
        norm.layer_norm(x, out=torch.zeros(2, 16, 3, dtype=torch.bfloat16, device=device).transpose(1, 2))
    from flicker_amd._lib import HipKernelError
    with pytest.raises(HipKernelError):
        norm.layer_norm(x, eps=-1.0)
    with pytest.raises(HipKernelError, match="unsupported"):
        norm.layer_norm(torch.zeros(1, 16392, device=device))


def _gate_case(gu, dh):
    half = gu.shape[-1] // 2
    g, u = gu[..., :half], gu[..., half:]
    rel = 2 * U * (np.abs(g) + 16)
    s, rest, low = M._sigmoid(g), M._sigmoid(-g), 2.0 ** -126 * np.abs(g)
    h = M.swiglu(gu)
    dgu = M.swiglu_grads(dh, gu)
    dg_tol = np.abs(dh * u) * (s * (1 + np.abs(g) * rest) * rel + low * (1 + np.abs(g)))
    return (h, np.abs(h) * rel + low * np.abs(u)), (dgu, np.concatenate((dg_tol, np.abs(dh * g) * (s * rel + 2.0 ** -126)), -1))


@pytest.mark.parametrize("shape", [(1, 1, 1), (1, 1, 8), (3, 5, 7), (2, 33, 129), (1, 4, 9216), (2, 700, 40), (7, 1000)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_swiglu(device, shape, dtype):
    print(f"swiglu {shape} {dtype}", flush=True)
    g = torch.Generator().manual_seed(sum(shape))
    *rows, hidden = shape
    gu = (4 * torch.randn(*rows, 2 * hidden, generator=g)).to(TYPES[dtype]).to(device)
    dh = torch.randn(*shape, generator=g).to(TYPES[dtype]).to(device)
    h, dgu = _gate_case(_f64(gu), _f64(dh))
    _close("h", mlp.swiglu(gu), *h)
    _close("dgu", mlp.swiglu_backward(dh, gu), *dgu)


def test_swiglu_far_from_zero(device):
    """Gates where exp overflows or vanishes: silu(g) is 0 or g, its slope 0 or 1."""
    g = torch.tensor([-3e38, -1e4, -104.0, -88.0, -87.0, -30.0, -17.0, -1.278, -1e-30, 0.0, 1e-30, 17.0, 88.0, 104.0, 1e4, 1e30])
    gu = torch.stack((g, torch.full_like(g, 1.5)), 0).reshape(1, -1).to(device)
    dh = torch.full((1, 16), 0.75, device=device)
    h, dgu = _gate_case(_f64(gu), _f64(dh))
    _close("h", mlp.swiglu(gu), *h)
    _close("dgu", mlp.swiglu_backward(dh, gu), *dgu)


def test_swiglu_in_place_of_a_single_block(device):
    """The mlp columns of linear1's output in, the columns beside the attention's output in linear2's input out."""
    g = torch.Generator().manual_seed(2)
    hidden, width = 48, 40
    linear1 = torch.randn(2, 9, 3 * width + 2 * hidden, generator=g).to(torch.bfloat16).to(device)
    linear2 = torch.full((2, 9, width + hidden), 3.0, dtype=torch.bfloat16, device=device)
    gu = linear1[..., 3 * width:]
    mlp.swiglu(gu, out=linear2[..., width:])
    assert (linear2[..., :width] == 3.0).all()
    assert torch.equal(linear2[..., width:], mlp.swiglu(gu.contiguous()))
    dh, dlinear1 = linear2[..., width:] * 0.5, torch.zeros_like(linear1)
    mlp.swiglu_backward(dh, gu, out=dlinear1[..., 3 * width:])
    assert not dlinear1[..., :3 * width].any()
    want = mlp.swiglu_backward(dh.contiguous(), gu.contiguous())
    assert torch.equal(dlinear1[..., 3 * width:], want)
    own = gu.contiguous()
    assert torch.equal(mlp.swiglu_backward(dh, own, out=own), want)
    with pytest.raises(ValueError, match="2 \\* hidden"):
        mlp.swiglu(linear1[..., :7])
    with pytest.raises(ValueError, match="dh must be"):
        mlp.swiglu_backward(gu, gu)


def test_outputs_over_their_operands(device):
    """In place where each lane writes what it has read, beside the operands in one buffer, and refused otherwise."""
    wide = torch.randn(2, 5, 200, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(device)
    for at in (20, 60):   # silu(g) u over g, over u
        w = wide.clone()
        want = mlp.swiglu(w[..., 20:100].contiguous())
        assert torch.equal(mlp.swiglu(w[..., 20:100], out=w[..., at:at + 40]), want)
        w = wide.clone()
        out, dh = w[..., 20:100], w[..., at:at + 40]   # the gradient where dh was
        gu = wide[..., 100:180]
        want = mlp.swiglu_backward(dh.contiguous(), gu)
        assert torch.equal(mlp.swiglu_backward(dh, gu, out=out), want)
    w = wide.clone()
    want = norm.layer_norm(w[..., 20:100].contiguous())
    assert torch.equal(norm.layer_norm(w[..., 20:100], out=w[..., 100:180]), want)
    assert torch.equal(w[..., 20:100], wide[..., 20:100])
    for call in (lambda: mlp.swiglu(w[..., 20:100], out=w[..., 21:61]), lambda: mlp.swiglu(w[..., 20:100], out=w[..., 10:50]),
                 lambda: mlp.swiglu(w[:, :4, 20:100], out=w[:, 1:, 20:60]),
                 lambda: mlp.swiglu_backward(wide[..., 100:140], w[..., 20:100], out=w[..., 21:101]),
                 lambda: mlp.swiglu_backward(w[..., 70:110], wide[..., 20:100], out=w[..., 20:100]),
                 lambda: norm.layer_norm(w[..., 20:100], out=w[..., 21:101]), lambda: norm.layer_norm(w[:, :4], out=w[:, 1:]),
                 lambda: norm.layer_norm(wide, w[0, 0], out=w)):
        with pytest.raises(ValueError, match="shares memory"):
            call()
    # rows of parameters that are not dense are copied before anything is written
    want = norm.modulate(wide, wide[:, 0].clone(), wide[:, 1].clone())
    w = wide.clone()
    assert torch.equal(norm.modulate(w, w[:, 0], w[:, 1], out=w), want)
    x, w_in = wide[0, :, :64].contiguous(), wide[..., :160].reshape(10, 160)[:8].repeat(8, 1)
    w_out = torch.zeros(80 * 64, dtype=torch.bfloat16, device=device)
    with pytest.raises(ValueError, match="shares memory"):
        mlp.gated_mlp(x, w_in, w_out.view(80, 64), out=w_out[:5 * 64].view(5, 64))


def test_autograd_matches_the_explicit_calls(device):
    x, g = _stream(4, 2, 9, 56, torch.bfloat16, device)
    x.requires_grad_()
    shift, scale = (torch.randn(2, 1, 56, generator=g).to(device).requires_grad_() for _ in range(2))
    dy = torch.randn(x.shape, generator=g).to(torch.bfloat16).to(device)
    y = autograd.modulate(x, shift, scale)
    y.backward(dy)
    for got, want in zip((x.grad, shift.grad, scale.grad), norm.modulate_backward(dy, x, shift, scale)):
        assert torch.equal(got, want)
    w = torch.ones(56, device=device, requires_grad=True)
    autograd.layer_norm(x.detach(), w).float().square().sum().backward()
    assert w.grad is not None
    gu = torch.randn(3, 20, generator=g).to(device).requires_grad_()
    autograd.swiglu(gu).sum().backward()   # an expanded incoming gradient
    assert torch.equal(gu.grad, mlp.swiglu_backward(torch.ones(3, 10, device=device), gu.detach()))
    with torch.no_grad():
        assert not autograd.swiglu(gu).requires_grad
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(autograd.swiglu(gu).sum(), gu, create_graph=True)


# The steps are h = 2^-5 and 2 h = 2^-4; the docstring's 1/8 is no step of this test.
def test_gradients_are_the_forward_pass_differences(device):
    """A float32 norm and gate moved along a direction.  The central difference with h = 1/8 is off by
    h^2 / 6 times the third derivative along it, which the differences with h and 2 h show: their
    difference is three times the error of the first, and so bounds it."""
    x, g = _stream(6, 1, 4, 200, torch.float32, device)
    dy, d = torch.randn(x.shape, generator=g).to(device), torch.randn(x.shape, generator=g).to(device)
    for f, grad in ((lambda v: norm.layer_norm(v), norm.layer_norm_backward(dy, x)[0]),
                    (lambda v: mlp.swiglu(v), mlp.swiglu_backward(dy[..., :100].contiguous(), x))):
        out = f(x)
        weight = dy[..., :out.shape[-1]].double()
        slope = lambda h: float(((f(x + h * d).double() - f(x - h * d).double()) * weight).sum()) / (2 * h)  # noqa: E731
        near, far = slope(2.0 ** -5), slope(2.0 ** -4)
        noise = 300 * U * float((out.double().abs() * weight.abs()).sum()) * 2 ** 5
        assert abs(float((grad.double() * d.double()).sum()) - near) <= abs(far - near) + noise


def test_offsets_past_32_bits(device):
    """The last rows of tensors of more than 2^31 elements are those of a call on them alone."""
    width, rows = 8192, 2 ** 18 + 700
    part, g = _stream(8, 1, 700, width, torch.bfloat16, device)
    x = torch.zeros(1, rows, width, dtype=torch.bfloat16, device=device)
    x[:, -700:] = part
    shift, scale = (torch.randn(1, width, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    assert torch.equal(norm.modulate(x, shift, scale)[:, -700:], norm.modulate(part, shift, scale))
    dx, dshift, dscale = norm.modulate_backward(x, x, shift, scale)
    want = norm.modulate_backward(part, part, shift, scale)
    assert torch.equal(dx[:, -700:], want[0]) and not dx[:, :-700].any()
    # the other rows add zeros to the sums, in another order of float32 additions: 1e-4 of the terms' absolute sum
    n = M._stats(_f64(part), norm.EPS)[0]
    for got, exact, terms in ((dshift, want[1], np.abs(_f64(part))), (dscale, want[2], np.abs(_f64(part) * n))):
        off = np.abs(_f64(got) - _f64(exact))[0]
        assert (off <= 2.0 ** -7 * np.abs(_f64(exact))[0] + 1e-4 * terms[0].sum(0)).all()
    h = mlp.swiglu(x)
    assert torch.equal(h[:, -700:], mlp.swiglu(part)) and not h[:, :-700].any()
    dgu = mlp.swiglu_backward(h, x)
    assert torch.equal(dgu[:, -700:], mlp.swiglu_backward(mlp.swiglu(part), part)) and not dgu[:, :-700].any()


class Declines:
    """A native call path that takes no call."""

    def __getattr__(self, name):
        return lambda *_: None


@pytest.mark.parametrize("dtype,params", [("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp32")])
@pytest.mark.parametrize("width", [1, 96, 1003])
def test_native_path_equals_the_python_path(device, monkeypatch, dtype, params, width):
    """Plain calls take the native path, and have the Python path's values, shapes and types."""
    x, g = _stream(width, 2, 9, width, TYPES[dtype], device)
    wide = torch.randn(2, 9, 5 + 2 * width, generator=g).to(TYPES[dtype]).to(device)
    dy = torch.randn(2, 9, width, generator=g).to(TYPES[dtype]).to(device)
    rows = [torch.randn(2, 1, width, generator=g).to(TYPES[params]).to(device) for _ in range(2)]
    w, b = rows[0][0, 0], rows[1][1, 0]
    calls = {
        "modulate": lambda: norm.modulate(x, *rows),
        "modulate_backward": lambda: norm.modulate_backward(dy, x, *rows),
        "layer_norm": lambda: norm.layer_norm(x[0], w, None),
        "layer_norm_backward": lambda: norm.layer_norm_backward(dy, x, None, b),
        "swiglu": lambda: mlp.swiglu(wide[..., 5:]),
        "swiglu_backward": lambda: mlp.swiglu_backward(dy, wide[..., 5:]),
    }
    taken = {
        "modulate": norm._native.modulate(x, *rows, 1e-6), "layer_norm": norm._native.layer_norm(x[0], w, None, 1e-6),
        "modulate_backward": norm._native.modulate_backward(dy, x, *rows, 1e-6),
        "layer_norm_backward": norm._native.layer_norm_backward(dy, x, None, b, 1e-6),
        "swiglu": norm._native.swiglu(wide[..., 5:]), "swiglu_backward": norm._native.swiglu_backward(dy, wide[..., 5:]),
    }
    assert all(v is not None for v in taken.values()), [k for k, v in taken.items() if v is None]
    got = {k: f() for k, f in calls.items()}
    monkeypatch.setattr(norm, "_native", Declines())
    monkeypatch.setattr(mlp, "_native", Declines())
    for k, f in calls.items():
        for a, c, e in zip(*(v if isinstance(v, tuple) else (v,) for v in (got[k], f(), taken[k])), strict=True):
            if c is None:
                assert a is None and e is None
                continue
            for t in (a, e):
                assert t.shape == c.shape and t.dtype == c.dtype and torch.equal(t, c), k
    assert norm._native.modulate(x, *rows) is None
