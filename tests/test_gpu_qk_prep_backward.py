"""kernels.qk_prep_backward on the GPU against the formulas in float64.

Tolerances, u = 2^-24: inv is off by 12 u of itself (a sum of 128 squares, 16 lanes and 8 terms deep, a root and
a quotient), n = x inv by 14 u; dy, two products of |c|, |s| <= 1, by 6 u (|dr_j| + |dr_j'|) of its pair.  A scale's
gradient over R rows: (R + 64) u sum|dy n| and the rows' own errors.  dx = inv (dn - n mean(dn n)): the mean is off by
40 u mean|dn n| and dy's error, the rest by 40 u of each term.  v's section is exact.
"""

import numpy as np
import pytest
import torch

from flicker_amd import kernels, rope
from tests.test_gpu_norm import _close, _f64

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
D = 128


def make(seed, batch, length, heads, device, params=torch.bfloat16, total=None):
    g = torch.Generator().manual_seed(seed)
    total = total or length
    grads = [torch.randn(batch, heads, total, D, generator=g).to(torch.bfloat16).to(device) for _ in range(3)]
    size = torch.exp(torch.randn(3 * heads, 1, generator=g)).expand(-1, D).reshape(-1)
    qkv = (torch.randn(batch, length, 3 * heads * D, generator=g) * size).to(torch.bfloat16).to(device)
    scales = [(1 + 0.3 * torch.randn(D, generator=g)).to(params).to(device) for _ in range(2)]
    ids = torch.from_numpy(np.stack([np.zeros(length), np.arange(length) // 7, np.arange(length) % 7, np.arange(length)], -1))
    return grads, qkv, scales, rope.rope_lanes(ids.float().to(device), D ** -0.5)


def expected(grads, qkv, scales, freqs, heads, offset):
    """(dqkv, its tolerance), (dq_scale, ...), (dk_scale, ...)."""
    batch, length, _ = qkv.shape
    x = _f64(qkv).reshape(batch, length, 3, heads, D)
    cos, sin = (_f64(t)[:, None] for t in freqs[:2])

    def turned(a, back):   # swaps each pair
        return np.stack((back[..., 1::2], back[..., 0::2]), -1).reshape(a.shape)
    sections, offs, outs = [], [], []
    for i, (grad, scale, gain) in enumerate(zip(grads, scales, (freqs.q_gain, 1.0))):
        dr = np.float64(np.float32(gain)) * _f64(grad)[:, :, offset:offset + length].transpose(0, 2, 1, 3)
        dy = cos * dr + turned(dr, sin * dr)
        dy_off = 6 * U * (np.abs(dr) + turned(dr, np.abs(dr)))
        s = _f64(scale)
        inv = 1 / np.sqrt((x[:, :, i] ** 2).mean(-1, keepdims=True) + 1e-6)
        n = x[:, :, i] * inv
        dn = dy * s
        mean = (dn * n).mean(-1, keepdims=True)
        mean_off = 40 * U * np.abs(dn * n).mean(-1, keepdims=True) + (np.abs(s) * dy_off * np.abs(n)).mean(-1, keepdims=True)
        sections.append(inv * (dn - n * mean))
        offs.append(inv * (np.abs(s) * dy_off + np.abs(n) * mean_off + 40 * U * (np.abs(dn) + np.abs(n * mean))))
        rows = batch * length * heads
        size = np.abs(dy * n).sum((0, 1, 2))
        outs.append(((dy * n).sum((0, 1, 2)), (rows + 64) * U * size + (dy_off * np.abs(n)).sum((0, 1, 2)) + 14 * U * size))
    dv = _f64(grads[2])[:, :, offset:offset + length].transpose(0, 2, 1, 3)
    shape = qkv.shape
    return [(np.stack((*sections, dv), 2).reshape(shape), np.stack((*offs, 0 * dv), 2).reshape(shape)), *outs]


def check(grads, qkv, scales, freqs, heads, offset=0, **kw):
    got = kernels.qk_prep_backward(*grads, qkv, *scales, freqs, heads, offset=offset, **kw)
    for name, t, (want, tol) in zip(("dqkv", "dq_scale", "dk_scale"), got, expected(grads, qkv, scales, freqs, heads, offset)):
        _close(name, t, want, tol)
    return got


@pytest.mark.parametrize("params", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,length,heads", [(1, 1, 1), (2, 7, 3), (1, 64, 2), (3, 65, 5), (1, 333, 24), (2, 512, 6)])
def test_sizes(device, batch, length, heads, params):
    print(f"qk_prep_backward batch={batch} length={length} heads={heads} {params}", flush=True)
    check(*make(length, batch, length, heads, device, params), heads)


@pytest.mark.parametrize("length,offset,total", [(50, 0, 130), (80, 50, 130), (1, 129, 130)])
def test_rows_of_a_joint_sequence(device, length, offset, total):
    check(*make(offset, 2, length, 4, device, total=total), 4, offset)


def test_many_blocks(device):
    """More blocks of tokens than the launch has blocks: each walks several."""
    check(*make(1, 1, 2999, 12, device), 12)


def test_views(device):
    """Token-major gradients, a projection and a result inside wider rows."""
    heads = 3
    grads, qkv, scales, freqs = make(2, 2, 70, heads, device)
    grads = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in grads]
    wide = torch.full((2, 70, 3 * heads * D + 256), float("nan"), dtype=qkv.dtype, device=device)
    wide[..., 128:128 + qkv.shape[2]] = qkv
    out = torch.zeros_like(wide)
    check(grads, wide[..., 128:128 + qkv.shape[2]], scales, freqs, heads, out=out[..., 64:64 + qkv.shape[2]])
    assert not out[..., :64].any() and not out[..., 64 + qkv.shape[2]:].any()


def test_position_ids(device):
    """Lanes from position ids: the tables' gradients bit for bit."""
    heads, length = 2, 90
    grads, qkv, scales, _ = make(3, 1, length, heads, device)
    ids = torch.randint(0, 60, (length, 4), generator=torch.Generator().manual_seed(0)).float().to(device)
    a = kernels.qk_prep_backward(*grads, qkv, *scales, rope.rope_lanes(ids, 0.25), heads)
    b = kernels.qk_prep_backward(*grads, qkv, *scales, rope.position_ids(ids, 0.25), heads)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_against_differences(device):
    """The projection's gradient against differences of qk_prep itself, whose bf16 steps bound how near they are."""
    heads, length = 2, 64
    grads, qkv, scales, freqs = make(4, 1, length, heads, device)
    got, _, _ = kernels.qk_prep_backward(*grads, qkv, *scales, freqs, heads)
    way = torch.randn(qkv.shape, generator=torch.Generator().manual_seed(1)).to(device) * qkv.float().abs().mean(
        (0, 1), keepdim=True)
    step = 0.25
    ends = [(qkv.float() + s * way).to(torch.bfloat16) for s in (-step, step)]
    outs = [kernels.qk_prep(e, *scales, freqs, heads) for e in ends]
    moved = ends[1].double() - ends[0].double()
    slope = sum(float(((b.double() - a.double()) * g.double()).sum()) for a, b, g in zip(*outs, grads))
    want = float((moved * got.double()).sum())
    # two ends of 3 roundings each, of values that add up with random signs: their root sum of squares, six times over;
    # the norm's curvature over +-step of each row's size
    noise = 6 * 2.0 ** -8 * 6 ** 0.5 * sum(float((b.double() * g.double()).norm()) for (_, b, g) in zip(*outs, grads))
    size = sum(float((b.double() * g.double()).norm()) for (_, b, g) in zip(*outs, grads))
    assert abs(slope - want) <= noise + 6 * step ** 2 * size


def test_empty(device):
    grads, qkv, scales, freqs = make(5, 1, 4, 1, device)
    none = qkv[:, :0]
    got = kernels.qk_prep_backward(*grads, none, *scales, kernels.Freqs(freqs.cos[:0], freqs.sin[:0], 1.0), 1)
    assert got[0].shape == none.shape and not got[1].any() and not got[2].any()


def test_captured_and_replayed(device):
    heads = 6
    grads, qkv, scales, freqs = make(6, 1, 200, heads, device)

    def step():
        return kernels.qk_prep_backward(*grads, qkv, *scales, freqs, heads)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        qkv.add_(0.5)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_refusals(device):
    grads, qkv, scales, freqs = make(7, 1, 8, 2, device)
    dq, dk, dv = grads
    with pytest.raises(TypeError, match="dk must be bfloat16"):
        kernels.qk_prep_backward(dq, dk.float(), dv, qkv, *scales, freqs, 2)
    with pytest.raises(ValueError, match="of one shape"):
        kernels.qk_prep_backward(dq, dk[:, :, :7], dv, qkv, *scales, freqs, 2)
    with pytest.raises(ValueError, match="exceeds"):
        kernels.qk_prep_backward(dq, dk, dv, qkv, *scales, freqs, 2, offset=1)
    with pytest.raises(ValueError, match="out must be"):
        kernels.qk_prep_backward(dq, dk, dv, qkv, *scales, freqs, 2, out=torch.empty_like(qkv)[:, :4])
    with pytest.raises(ValueError, match="head_dim"):
        kernels.qk_prep_backward(dq, dk, dv, qkv, *scales, freqs, 4)
