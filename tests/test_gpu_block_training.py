"""The operators of a block's attention half run together under autograd, as a program that fine-tunes it does.

The reference is the same block in float64 from torch's elementary operations.  Its bf16 form rounds an activation about
a dozen times on the way to the output and as often on the way back, each time by at most e = 2^-8 of itself; the
norms, the softmax and the products between pass a relative error on with a gain near one.  Norms of differences are
held to 24 e of the result's norm (rounding errors of random sign, a third of e each, come to a tenth of that).
"""

import math

import pytest
import torch

from flicker_amd import autograd, kernels, modules, rope

pytestmark = pytest.mark.gpu
E = 2.0 ** -8
HEADS, D = 2, 128
WIDTH, HIDDEN, TEXT, GRID = HEADS * D, 320, 40, 8


def _params(g, device):
    def randn(*shape, s=1.0):
        return (s * torch.randn(*shape, generator=g)).to(torch.bfloat16).to(device).requires_grad_()
    names = {"qkv": (WIDTH, 3 * WIDTH, WIDTH ** -0.5), "proj": (WIDTH, WIDTH, WIDTH ** -0.5),
             "w_in": (WIDTH, 2 * HIDDEN, WIDTH ** -0.5), "w_out": (HIDDEN, WIDTH, HIDDEN ** -0.5)}
    p = {n: randn(a, b, s=s) for n, (a, b, s) in names.items()}
    for n in ("shift1", "scale1", "gate1", "shift2", "scale2", "gate2"):
        p[n] = randn(2, 1, WIDTH, s=0.3)
    for n in ("q_scale", "k_scale"):
        p[n] = (1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(device).requires_grad_()
    return p


def _block(x, p, freqs, keep):
    h = autograd.modulate(x, p["shift1"], p["scale1"])
    q, k, v = autograd.qk_prep(h @ p["qkv"], p["q_scale"], p["k_scale"], freqs, HEADS)
    a = autograd.attention(q, k, v, key_mask=keep)
    r, y = autograd.residual_modulate(x, a @ p["proj"], p["gate1"], p["shift2"], p["scale2"])
    return r + p["gate2"] * autograd.gated_mlp(y, p["w_in"], p["w_out"])


def _norm64(x):
    var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
    return (x - mean) * torch.rsqrt(var + 1e-6)


def _block64(x, p, freqs, keep):
    h = (1 + p["scale1"]) * _norm64(x) + p["shift1"]
    q, k, v = (h @ p["qkv"]).unflatten(-1, (3, HEADS, D)).permute(2, 0, 3, 1, 4)
    out = []
    for t, scale, gain in ((q, p["q_scale"], freqs.q_gain), (k, p["k_scale"], 1.0)):
        t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * scale
        swapped = torch.stack((t[..., 1::2], t[..., 0::2]), -1).flatten(-2)
        out.append(gain * (freqs.cos.double() * t + freqs.sin.double() * swapped))
    s = torch.where(keep[:, None, None], out[0] @ out[1].transpose(-1, -2), -math.inf)
    a = (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(2)
    r = x + p["gate1"] * (a @ p["proj"])
    y = (1 + p["scale2"]) * _norm64(r) + p["shift2"]
    g, u = (y @ p["w_in"]).chunk(2, -1)
    return r + p["gate2"] * ((torch.nn.functional.silu(g) * u) @ p["w_out"])


def test_a_block_trains(device):
    g = torch.Generator().manual_seed(0)
    p = _params(g, device)
    length = TEXT + GRID * GRID
    x = torch.randn(2, length, WIDTH, generator=g).to(torch.bfloat16).to(device).requires_grad_()
    freqs = rope.rope_lanes(rope.sequence_ids(TEXT, GRID, GRID), 1 / math.sqrt(D), device=device)
    keep = torch.ones(2, length, dtype=torch.bool, device=device)
    keep[0, 11:TEXT] = False
    dy = torch.randn(x.shape, generator=g).to(torch.bfloat16).to(device)
    y = _block(x, p, freqs, keep)
    y.backward(dy)
    leaves = {n: t.detach().double().requires_grad_() for n, t in {**p, "x": x}.items()}
    want = _block64(leaves["x"], leaves, freqs, keep)
    want.backward(dy.double())
    for name, got, ref in (("y", y, want), *((n, t.grad, leaves[n].grad) for n, t in {**p, "x": x}.items())):
        off = float((got.detach().double() - ref.detach()).norm() / ref.detach().norm())
        print(f"{name} {off:.2e}", flush=True)
        assert got.shape == ref.shape and off <= 24 * E, (name, off)


def test_joint_streams(device):
    """A double block's attention: two projections prepared into one joint sequence, whose gradients each stream
    takes its rows of, against one projection of the joint sequence."""
    g = torch.Generator().manual_seed(1)
    parts = [torch.randn(2, n, 3 * WIDTH, generator=g).to(torch.bfloat16).to(device) for n in (64, 128)]
    scales = [(1 + 0.2 * torch.randn(D, generator=g)).to(torch.bfloat16).to(device) for _ in range(2)]
    freqs = rope.rope_lanes(rope.sequence_ids(64, 8, 16), 1 / math.sqrt(D), device=device)
    joint = tuple(torch.empty(2, HEADS, 192, D, dtype=torch.bfloat16, device=device) for _ in range(3))
    for part, at in zip(parts, (0, 64)):
        f = modules._slice(freqs, at, at + part.shape[1])
        kernels.qk_prep(part, *scales, f, HEADS, out=joint, out_offset=at)
    from flicker_amd import attention
    do = torch.randn(2, 192, WIDTH, generator=g).to(torch.bfloat16).to(device)
    o, kept = attention.attention(*joint, keep=True)
    grads = attention.attention_backward(do, *joint, kept)
    whole = torch.cat(parts, 1)
    want, *_ = kernels.qk_prep_backward(*grads, whole, *scales, freqs, HEADS)
    for part, at in zip(parts, (0, 64)):
        end = at + part.shape[1]
        got, *_ = kernels.qk_prep_backward(*grads, part, *scales, modules._slice(freqs, at, end), HEADS, offset=at)
        assert torch.equal(got, want[:, at:end])


def test_autograd_matches_the_explicit_calls(device):
    from flicker_amd import attention, norm
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(1, h, 50, D, generator=g).to(torch.bfloat16).to(device).requires_grad_() for h in (4, 2, 2))
    o = autograd.attention(q, k, v)
    o.sum().backward()       # an expanded incoming gradient
    _, kept = attention.attention(q, k, v, keep=True)
    want = attention.attention_backward(torch.ones_like(o), q, k, v, kept)
    assert all(torch.equal(t.grad, w) for t, w in zip((q, k, v), want))
    x, b = (torch.randn(2, 9, 64, generator=g).to(device).requires_grad_() for _ in range(2))
    rows = [torch.randn(2, 64, generator=g).to(device).requires_grad_() for _ in range(3)]
    r, y = autograd.residual_modulate(x, b, *rows)
    y.square().sum().backward()      # r is not used: its gradient is zeros
    want = norm.residual_modulate_backward(torch.zeros_like(x), 2 * y.detach(), x, b, *rows)
    assert all(torch.equal(t.grad, w) for t, w in zip((x, b, *rows), want))
    with torch.no_grad():
        assert not autograd.attention(q, k, v).requires_grad
    assert not autograd.attention(q.detach(), k.detach(), v.detach()).requires_grad
    with pytest.raises(RuntimeError, match="first derivatives only"):
        torch.autograd.grad(autograd.attention(q, k, v).float().sum(), q, create_graph=True)


def test_broadcast_keys(device):
    """Keys and values that a batch shares by broadcasting: their gradients sum over it."""
    g = torch.Generator().manual_seed(3)
    q = torch.randn(3, 2, 30, D, generator=g).to(torch.float16).to(device)
    k, v = (torch.randn(1, 2, 40, D, generator=g).to(torch.float16).to(device).requires_grad_() for _ in range(2))
    do = torch.randn(3, 30, 2 * D, generator=g).to(torch.float16).to(device)
    autograd.attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1)).backward(do)
    ke, ve = (t.detach().expand(3, -1, -1, -1).contiguous().requires_grad_() for t in (k, v))
    autograd.attention(q, ke, ve).backward(do)
    assert torch.equal(k.grad, ke.grad.sum(0, keepdim=True)) and torch.equal(v.grad, ve.grad.sum(0, keepdim=True))


def test_capture_with_gradients_is_refused(device):
    q = torch.randn(1, 1, 32, D, device=device, dtype=torch.bfloat16, requires_grad=True)
    autograd.attention(q, q, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="explicit"):
            autograd.attention(q, q, q)
        with torch.no_grad():
            out = autograd.attention(q, q, q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, autograd.attention(q, q, q))
