"""Shapes that attention's plan gives to each form of its forward pass, for the host test that holds them to it and the GPU
tests that run them; and the float64 form of a whole call with tolerances, on the GPU."""

from __future__ import annotations

import torch

from tests.test_gpu_attention import D, FLUSH, TINY, U

# name: (batch, heads, kv_heads, queries, keys), (rows of a block, whole blocks, cut blocks, pieces of a cut one)
FORMS = {
    "192": ((1, 24, 24, 370, 405), (192, 48, 0, 1)),             # 13 units: the unrolled loop and what follows it
    "192 cut": ((1, 24, 24, 190, 2000), (192, 0, 24, 7)),        # pieces of 9 units
    "192 shared": ((2, 16, 4, 300, 330), (192, 64, 0, 1)),
    "256": ((1, 172, 172, 300, 411), (256, 344, 0, 1)),
    "256 cut": ((1, 12, 12, 250, 4600), (256, 0, 12, 12)),       # of 12
    "256 both": ((1, 260, 260, 50, 640), (256, 256, 4, 5)),
    "256 shared": ((3, 90, 45, 120, 350), (256, 270, 0, 1)),
    "256 long": ((1, 64, 64, 1000, 2500), (256, 256, 0, 1)),     # a masked list past the 64 units that a wave holds
    "16": ((1, 4, 2, 60, 300), (16, 16, 0, 1)),
    "16 cut": ((1, 8, 8, 3, 4000), (16, 0, 8, 16)),
}


def expected(q, k, v, do, keep):
    """[(o, tol), (lse, tol), (dq, tol), (dk, tol), (dv, tol)] as test_gpu_attention.expected, in torch's float64 on the
    operands' device, a key head at a time."""
    e, t0 = torch.finfo(q.dtype).eps / 2, TINY[q.dtype]
    (batch, heads, queries, _), (_, kv_heads, keys, _) = q.shape, k.shape
    group = heads // kv_heads

    def zeros(*shape):
        return torch.zeros(shape, dtype=torch.float64, device=q.device), torch.zeros(shape, dtype=torch.float64, device=q.device)
    o, lse = zeros(batch, queries, heads, D), zeros(batch, heads, queries)
    dq, dk, dv = zeros(*q.shape), zeros(*k.shape), zeros(*v.shape)
    lse[0].fill_(-torch.inf)
    do = do.view(batch, queries, heads, D).transpose(1, 2)
    for b in range(batch):
        on = torch.ones(keys, dtype=torch.bool, device=q.device) if keep is None else keep[b]
        if not on.any():
            continue
        for h in range(heads):
            hk = h // group
            qh, gh = q[b, h].double(), do[b, h].double()
            kh, vh = (torch.where(on[:, None], t[b, hk].double(), 0.0) for t in (k, v))
            aq, ak, av, ag = qh.abs(), kh.abs(), vh.abs(), gh.abs()
            s = torch.where(on, qh @ kh.T.contiguous(), -torch.inf)
            ls = torch.logsumexp(s, -1)
            p = torch.exp(s - ls[:, None])
            oh = p @ vh
            dp = gh @ vh.T.contiguous()
            delta = (gh * oh).sum(-1, keepdim=True)
            ds = p * (dp - delta)
            size = torch.where(on, aq @ ak.T.contiguous(), 0.0).amax(-1)
            big = torch.where(on, s.abs(), 0.0).amax(-1)
            r = (2 * 130 * U * size + 8 * U * (big + ls.abs()) + (64 + keys + 64) * U)[:, None]
            o_off = (2 * e + 2 * r + (keys + 64) * U) * (p @ av) + t0 * av.sum(0)
            delta_off = (ag * (o_off + (e * e + 130 * U) * oh.abs())).sum(-1, keepdim=True)
            spread = (dp - delta).abs()
            a_ds = p * spread
            ds_off = (e + r + 4 * U) * a_ds + p * (130 * U * (ag @ av.T.contiguous()) + delta_off) + (t0 + FLUSH * spread) * on
            p_off = p * (e + r) + (t0 + FLUSH) * on
            for (want, tol), a, c in (((o[0][b, :, h], o[1][b, :, h]), oh, o_off), ((lse[0][b, h], lse[1][b, h]), ls, r[:, 0])):
                want.copy_(a)
                tol.copy_(c)
            dq[0][b, h], dk[0][b, hk] = ds @ kh, dk[0][b, hk] + ds.T.contiguous() @ qh
            dv[0][b, hk] += p.T.contiguous() @ gh
            dq[1][b, h] = ds_off @ ak + (keys + 64) * U * (a_ds @ ak)
            dk[1][b, hk] += ds_off.T.contiguous() @ aq + (queries * heads + 64) * U * (a_ds.T.contiguous() @ aq)
            dv[1][b, hk] += p_off.T.contiguous() @ ag + (queries * heads + 64) * U * (p.T.contiguous() @ ag)
    flat = (batch, queries, heads * D)
    return [tuple(t.reshape(flat) for t in o), lse, dq, dk, dv]


def close(label, got, want, extra):
    """test_gpu_attention's _close on the device."""
    tol = torch.finfo(got.dtype).eps / 2 * (want.abs() + extra) + extra + TINY.get(got.dtype, 0.0)
    g = got.double()
    over = torch.where(g == want, -1.0, (g - want).abs() - tol)
    assert got.shape == want.shape and not g.isnan().any(), (label, int(g.isnan().sum()))
    worst = over.argmax()
    assert over.max() <= 0, f"{label}: {int((over > 0).sum())} of {over.numel()}, worst {float(over.max()):.3g} over {float(tol.flatten()[worst]):.3g}"


def check(label, call, want):
    """What ``call`` = (o, kept, dq, dk, dv) gives against expected()'s."""
    o, kept, *grads = call
    close(f"{label}: o", o, *want[0])
    lse, (lse_want, lse_off) = kept.lse.double(), want[1]
    assert torch.equal(lse.isneginf(), lse_want.isneginf()), label
    fin = lse_want.isfinite()
    assert ((lse[fin] - lse_want[fin]).abs() <= lse_off[fin] + 2 * U * lse_want[fin].abs()).all(), label
    for name, got, (w, extra) in zip(("dq", "dk", "dv"), grads, want[2:]):
        close(f"{label}: {name}", got, w, extra)
