"""A double block under autograd: text and image keep weights of their own and attend to each other, so q, k and v of both are
concatenated and each takes its rows of the result.  Against the same block in float64 from torch's elementary operations, with
test_gpu_block_training's tolerance: the joint sequence adds no rounding to a stream's."""

import math

import pytest
import torch

from flicker_amd import autograd, modules, rope
from tests.test_gpu_block_training import D, E, HEADS, WIDTH, _norm64, _params

pytestmark = pytest.mark.gpu
LENGTHS = (40, 72)   # text, image of 8 x 9


def _block(xs, ps, freqs, keep):
    parts, at = [], 0
    for x, p in zip(xs, ps):
        h = autograd.modulate(x, p["shift1"], p["scale1"])
        rows = modules._slice(freqs, at, at + x.shape[1])
        parts.append(autograd.qk_prep(h @ p["qkv"], p["q_scale"], p["k_scale"], rows, HEADS))
        at += x.shape[1]
    a = autograd.attention(*(torch.cat(t, 2) for t in zip(*parts)), key_mask=keep)
    out = []
    for x, p, part in zip(xs, ps, a.split([x.shape[1] for x in xs], 1)):
        r, y = autograd.residual_modulate(x, part @ p["proj"], p["gate1"], p["shift2"], p["scale2"])
        out.append(r + p["gate2"] * autograd.gated_mlp(y, p["w_in"], p["w_out"]))
    return out


def _block64(xs, ps, freqs, keep):
    parts, at = [], 0
    for x, p in zip(xs, ps):
        h = (1 + p["scale1"]) * _norm64(x) + p["shift1"]
        q, k, v = (h @ p["qkv"]).unflatten(-1, (3, HEADS, D)).permute(2, 0, 3, 1, 4)
        cos, sin = (t[at:at + x.shape[1]].double() for t in (freqs.cos, freqs.sin))
        turned = []
        for t, scale, gain in ((q, p["q_scale"], freqs.q_gain), (k, p["k_scale"], 1.0)):
            t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + 1e-6) * scale
            swapped = torch.stack((t[..., 1::2], t[..., 0::2]), -1).flatten(-2)
            turned.append(gain * (cos * t + sin * swapped))
        parts.append((*turned, v))
        at += x.shape[1]
    q, k, v = (torch.cat(t, 2) for t in zip(*parts))
    s = torch.where(keep[:, None, None], q @ k.transpose(-1, -2), -math.inf)
    a = (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(2)
    out = []
    for x, p, part in zip(xs, ps, a.split([x.shape[1] for x in xs], 1)):
        r = x + p["gate1"] * (part @ p["proj"])
        g, u = (((1 + p["scale2"]) * _norm64(r) + p["shift2"]) @ p["w_in"]).chunk(2, -1)
        out.append(r + p["gate2"] * ((torch.nn.functional.silu(g) * u) @ p["w_out"]))
    return out


def test_a_double_block_trains(device):
    g = torch.Generator().manual_seed(4)
    ps = [_params(g, device) for _ in LENGTHS]
    xs = [torch.randn(2, n, WIDTH, generator=g).to(torch.bfloat16).to(device).requires_grad_() for n in LENGTHS]
    freqs = rope.rope_lanes(rope.sequence_ids(LENGTHS[0], 8, 9), 1 / math.sqrt(D), device=device)
    keep = torch.ones(2, sum(LENGTHS), dtype=torch.bool, device=device)
    keep[1, 23:LENGTHS[0]] = False
    dys = [torch.randn(x.shape, generator=g).to(torch.bfloat16).to(device) for x in xs]
    ys = _block(xs, ps, freqs, keep)
    torch.autograd.backward(ys, dys)
    leaves = [{n: t.detach().double().requires_grad_() for n, t in {**p, "x": x}.items()} for p, x in zip(ps, xs)]
    wants = _block64([p["x"] for p in leaves], leaves, freqs, keep)
    torch.autograd.backward(wants, [dy.double() for dy in dys])
    for i, (p, x) in enumerate(zip(ps, xs)):
        for name, got, ref in (("y", ys[i], wants[i]), *((n, t.grad, leaves[i][n].grad) for n, t in {**p, "x": x}.items())):
            off = float((got.detach().double() - ref.detach()).norm() / ref.detach().norm())
            print(f"stream {i} {name} {off:.2e}", flush=True)
            assert got.shape == ref.shape and off <= 24 * E, (i, name, off)
