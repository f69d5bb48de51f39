"""attention.attention and attention_backward on the GPU against the float64 oracle.

Tolerances, with u = 2^-24, e = finfo(t).eps / 2 of the operands' type and t0 its smallest rounding (half the smallest
subnormal; float16's P and dS reach it).  Per row of one head:
  * S: sums of 128 products, off by 130 u sum|q k|; scaled, subtracted and exponentiated, P is off by
    r = 2 max_j (130 u sum|q k|) + 8 u (max|S| + |lse|) + 64 u of itself (twice: its own S, and lse's), plus the
    additions of a row's sum, at most keys + 64 deep: (keys + 64) u.
  * o: P is rounded (e of itself, t0 at most: P's largest is at least 1) and divided by the sum of the rounded, so off by
    (2 e + 2 r) sum P|v| + t0 sum|v|, the products' sums by (keys + 64) u sum P|v|; then rounded to its type.
  * lse is off by r.
  * delta: sum_d |g| times what o is off by before its last rounding, which low holds to e^2, and 130 u sum|g o|.
  * dS = P (dP - delta): off by (e + r + 4 u)|dS| + P (130 u sum|g v| + delta's) + t0.
  * dq, dk: those times |k|, |q|, summed, and (terms + 64) u sum|dS k|; dv: sum of (P (e + r) + t0)|g| likewise.
Masked keys hold infinities and NaN.
"""

import numpy as np
import pytest
import torch

from flicker_amd import attention as A
from oracle import attention as O

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TINY = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
D = 128


def _f64(t):
    return t.detach().to("cpu", torch.float64).numpy()


def _close(label, got, want, extra):
    assert got.shape == tuple(want.shape), (label, got.shape, want.shape)
    tol = torch.finfo(got.dtype).eps / 2 * (np.abs(want) + extra) + extra + TINY.get(got.dtype, 0.0)
    g = _f64(got)
    over = np.where(g == want, -1.0, np.abs(g - want) - tol)
    assert not np.isnan(g).any() and over.max(initial=-1.0) <= 0, \
        f"{label}: {np.argwhere(over > 0)[:5].tolist()} of {int((over > 0).sum())}, worst {over.max():.3g} over {tol.flat[over.argmax()]:.3g}"


def make(seed, batch, heads, kv_heads, queries, keys, dtype, mask=None, layout="heads", scale=1.0, device="cuda"):
    """q, k, v, do and the key mask; masked keys hold what must not be read."""
    g = torch.Generator().manual_seed(seed)

    def randn(h, length, s=1.0):
        t = (s * torch.randn(batch, length, h, D, generator=g)).to(TYPES[dtype])
        return t.transpose(1, 2) if layout == "tokens" else t.transpose(1, 2).contiguous()
    q, k, v = randn(heads, queries, scale * D ** -0.5), randn(kv_heads, keys), randn(kv_heads, keys)
    keep = None
    if mask is not None:
        keep = torch.rand(batch, keys, generator=g) < 0.6
        if mask == "middle":      # a run of padding, longer than a tile where there is room
            keep[:] = True
            for b in range(batch):
                keep[b, keys // 5:keys // 5 + keys // 2 + b] = False
        elif mask == "first":
            keep[:] = False
            keep[:, 0] = True
        elif mask == "last":
            keep[:] = False
            keep[:, -1] = True
        elif mask == "none":
            keep[:] = False
        if mask == "empty":
            keep[-1] = False
        for t, junk in ((k, float("nan")), (v, float("inf"))):
            t[~keep[:, None, :].expand(batch, kv_heads, keys)] = junk
        k[:, :, ::2][~keep[:, None, ::2].expand(k[:, :, ::2].shape[:3])] = float("-inf")
    do = torch.randn(batch, queries, heads * D, generator=g).to(TYPES[dtype])
    q, k, v, do = (t.to(device) for t in (q, k, v, do))
    return q, k, v, do, None if keep is None else keep.to(device)


def expected(q, k, v, do, keep):
    """[(o, tol), (lse, tol), (dq, tol), (dk, tol), (dv, tol)] of the whole call, tolerances without the last rounding."""
    dtype = q.dtype
    e, t0 = torch.finfo(dtype).eps / 2, TINY[dtype]
    q, k, v, do = (_f64(t) for t in (q, k, v, do))
    keep = None if keep is None else keep.cpu().numpy()
    (batch, heads, queries, _), (_, kv_heads, keys, _) = q.shape, k.shape
    g4 = do.reshape(batch, queries, heads, D).transpose(0, 2, 1, 3)
    o, lse = np.zeros((batch, queries, heads, D)), np.zeros((batch, heads, queries))
    dq, dk, dv = np.zeros(q.shape), np.zeros(k.shape), np.zeros(v.shape)
    tols = [np.zeros(t.shape) for t in (o, lse, dq, dk, dv)]
    for b in range(batch):
        on = np.ones(keys, bool) if keep is None else keep[b]
        for h in range(heads):
            hk = h // (heads // kv_heads)
            qh, kh, vh, gh = q[b, h], np.where(on[:, None], k[b, hk], 0.0), np.where(on[:, None], v[b, hk], 0.0), g4[b, h]
            s, p, ls = O.probabilities(qh, kh, on)
            o[b, :, h], lse[b, h] = p @ vh, ls
            for out, grad in zip((dq[b, h], dk[b, hk], dv[b, hk]), O.attention_grads(gh, qh, kh, vh, on)):
                out += grad
            if not on.any():
                continue
            aq, ak, av, ag = (np.abs(t) for t in (qh, kh, vh, gh))
            size = np.where(on, aq @ ak.T, 0.0).max(-1)
            big = np.where(on, np.abs(qh @ kh.T), 0.0).max(-1)
            r = (2 * 130 * U * size + 8 * U * (big + np.abs(ls)) + (64 + keys + 64) * U)[:, None]
            o_off = (2 * e + 2 * r + (keys + 64) * U) * (p @ av) + t0 * av.sum(0)
            tols[0][b, :, h], tols[1][b, h] = o_off, r[:, 0]
            delta_off = (ag * (o_off + (e * e + 130 * U) * np.abs(o[b, :, h]))).sum(-1, keepdims=True)
            dp = gh @ vh.T
            ds = np.abs(p * (dp - (gh * o[b, :, h]).sum(-1, keepdims=True)))
            ds_off = (e + r + 4 * U) * ds + p * (130 * U * (ag @ av.T) + delta_off) + t0 * on
            p_off = p * (e + r) + t0 * on
            tols[2][b, h] += ds_off @ ak + (keys + 64) * U * (ds @ ak)
            tols[3][b, hk] += ds_off.T @ aq + (queries * heads + 64) * U * (ds.T @ aq)
            tols[4][b, hk] += p_off.T @ ag + (queries * heads + 64) * U * (p.T @ ag)
    flat = (batch, queries, heads * D)
    return list(zip((o.reshape(flat), lse, dq, dk, dv), (tols[0].reshape(flat), *tols[1:])))


def check(*args, **kw):
    print("attention", args, kw, flush=True)
    q, k, v, do, keep = make(*args, **kw)
    want = expected(q, k, v, do, keep)
    o = A.attention(q, k, v, key_mask=keep)
    _close("o", o, *want[0])
    o2, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    assert torch.equal(o2, o) and kept.o is o2
    lse_want, lse_off = want[1]
    lse = _f64(kept.lse)
    assert (np.isneginf(lse) == np.isneginf(lse_want)).all()
    fin = np.isfinite(lse_want)
    assert (np.abs(lse[fin] - lse_want[fin]) <= lse_off[fin] + 2 * U * np.abs(lse_want[fin])).all()
    grads = A.attention_backward(do, q, k, v, kept, key_mask=keep)
    for name, got, (w, extra) in zip(("dq", "dk", "dv"), grads, want[2:]):
        _close(name, got, w, extra)
    if keep is not None:
        off = ~keep[:, None, :, None]
        assert not (grads[1] * off).any() and not (grads[2] * off).any()
    return q, k, v, do, keep, o, grads


LENGTHS = [(1, 1), (1, 2), (2, 1), (1, 300), (16, 16), (17, 31), (32, 33), (33, 32), (63, 65), (64, 64), (65, 63),
           (127, 129), (128, 128), (129, 127), (200, 257), (257, 200), (1, 1000), (300, 1), (511, 513)]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("queries,keys", LENGTHS)
def test_lengths(device, queries, keys, dtype):
    check(queries * 1000 + keys, 1, 2, 2, queries, keys, dtype)


@pytest.mark.parametrize("mask", ["random", "middle", "first", "last", "none", "empty"])
@pytest.mark.parametrize("queries,keys", [(1, 1), (5, 70), (70, 64), (100, 130), (129, 333), (1, 700)])
def test_masks(device, queries, keys, mask):
    check(keys, 2, 2, 1, queries, keys, "bf16", mask)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (6, 2), (3, 3), (5, 1)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_heads_and_layouts(device, heads, kv_heads, layout):
    check(heads, 2, heads, kv_heads, 77, 141, "fp16", "random", layout)


@pytest.mark.parametrize("scale", [0.0, 4.0, 30.0])
def test_logit_sizes(device, scale):
    """Logits that are all equal, and ones far past exp's range without a running maximum."""
    check(7, 1, 2, 2, 90, 150, "bf16", "middle", scale=scale)


@pytest.mark.parametrize("queries,keys", [(700, 900), (1030, 517)])
def test_longer(device, queries, keys):
    check(3, 1, 1, 1, queries, keys, "bf16", "middle")


@pytest.mark.parametrize("heads,kv_heads,queries,keys,mask", [
    (2, 2, 3, 5000, None), (2, 1, 40, 3000, "middle"), (3, 3, 260, 2100, "random"), (1, 1, 1500, 100, None),
    (4, 1, 900, 70, "random"), (6, 2, 33, 1999, "empty")])
def test_cut_blocks(device, heads, kv_heads, queries, keys, mask):
    """Too few blocks for the GPU: each is cut along the units it walks, and the partial sums are added."""
    check(keys, 2, heads, kv_heads, queries, keys, "bf16", mask)


@pytest.mark.parametrize("queries,keys", [(270, 1500), (1500, 200)])
def test_whole_and_cut_blocks(device, queries, keys):
    """A few blocks more than the GPU's CUs: those are cut, the others are not."""
    check(keys, 2, 66, 66, queries, keys, "fp16", "middle" if keys == 200 else None)
