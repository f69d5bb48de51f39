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
    In the gradients a P below float32's smallest normal number, z = 2^-126, is zero: exp2 gives no subnormals.  P is off by
    z more, dS by z |dP - delta|.  (z is far below every other term unless all P of a key are about as small.)
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
FLUSH = 2.0 ** -126
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
            spread = np.abs(dp - (gh * o[b, :, h]).sum(-1, keepdims=True))
            ds = p * spread
            ds_off = (e + r + 4 * U) * ds + p * (130 * U * (ag @ av.T) + delta_off) + (t0 + FLUSH * spread) * on
            p_off = p * (e + r) + (t0 + FLUSH) * on
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


def test_repeats_bit_for_bit(device):
    """Sums are in a fixed order: two calls give the same bits, cut blocks and shared heads among them."""
    for args in ((1, 6, 2, 300, 2100), (2, 4, 1, 900, 500)):
        q, k, v, do, keep = make(5, *args, "bf16", "random")
        one, two = ((o, *A.attention_backward(do, q, k, v, kept, key_mask=keep))
                    for o, kept in (A.attention(q, k, v, key_mask=keep, keep=True) for _ in range(2)))
        assert all(torch.equal(a, b) for a, b in zip(one, two))


def test_strided_operands(device):
    """Columns of a wider projection, a row stride that is not 16 bytes (copied), keys and values shared by the batch, and
    a mask that is a view."""
    q, k, v, do, keep = make(11, 2, 3, 3, 70, 70, "bf16", "random")
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    want = A.attention_backward(do, q, k, v, kept, key_mask=keep)
    wide = torch.full((2, 70, 3 * 3 * D + 24), float("nan"), dtype=q.dtype, device=device)
    views = []
    for i, t in enumerate((q, k, v)):
        view = wide[..., i * 3 * D:(i + 1) * 3 * D]
        view.copy_(t.transpose(1, 2).reshape(2, 70, 3 * D))
        views.append(view.view(2, 70, 3, D).transpose(1, 2))
    masks = torch.ones(2, 3, 90, dtype=torch.bool, device=device)
    masks[:, 1, :70] = keep
    got, kept2 = A.attention(*views, key_mask=masks[:, 1, :70], keep=True)
    assert torch.equal(got, o)
    assert all(torch.equal(a, b) for a, b in zip(A.attention_backward(do, *views, kept2, key_mask=masks[:, 1, :70]), want))
    odd = torch.empty(2, 3, 70, D + 3, dtype=q.dtype, device=device)[..., :D].copy_(q)
    assert torch.equal(A.attention(odd, k, v, key_mask=keep), o)
    far = torch.zeros(70, 2 ** 25 + 8, dtype=q.dtype, device=device)[:, :D].view(1, 1, 70, D).copy_(q[:1, :1])   # copied
    assert torch.equal(A.attention(far, k[:1, :1], v[:1, :1], key_mask=keep[:1]),
                       A.attention(q[:1, :1], k[:1, :1], v[:1, :1], key_mask=keep[:1]))
    every = do.repeat(1, 1, 2)[..., ::2]
    assert all(torch.equal(a, b) for a, b in zip(A.attention_backward(every, q, k, v, kept, key_mask=keep),
                                                 A.attention_backward(every.contiguous(), q, k, v, kept, key_mask=keep)))
    shared = A.attention(q, k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1), key_mask=keep[:1].expand(2, -1))
    assert torch.equal(shared[1], A.attention(q[1:], k[:1], v[:1], key_mask=keep[:1])[0])


def test_out(device):
    """A result inside wider rows, whose other columns and rows stay as they were; an overlap is refused."""
    q, k, v, do, _ = make(12, 2, 2, 2, 45, 60, "fp16")
    buffer = torch.full((2, 50, 2 * D + 64), 7.0, dtype=q.dtype, device=device)
    out = buffer[:, :45, 32:32 + 2 * D]
    got, kept = A.attention(q, k, v, out=out, keep=True)
    want, plain = A.attention(q, k, v, keep=True)
    assert got is out and torch.equal(out, want)
    assert (buffer[:, 45:] == 7).all() and (buffer[..., :32] == 7).all() and (buffer[..., 32 + 2 * D:] == 7).all()
    assert all(torch.equal(a, b) for a, b in zip(A.attention_backward(do, q, k, v, kept),
                                                 A.attention_backward(do, q, k, v, plain)))
    with pytest.raises(ValueError, match="shares memory with q"):
        A.attention(q, k, v, out=q.view(-1)[:2 * 45 * 2 * D].view(2, 45, 2 * D))
    with pytest.raises(ValueError, match="do not overlap"):
        A.attention(q, k, v, out=buffer[:1, :45, :2 * D].expand(2, -1, -1))
    with pytest.raises(ValueError, match="out must be"):
        A.attention(q, k, v, out=buffer[:, :45, :2 * D - 8])


def test_empty(device):
    q, k, v, do, _ = make(13, 2, 2, 1, 5, 7, "bf16")
    none = k[:, :, :0]
    o, kept = A.attention(q, none, none, keep=True)
    assert not o.any() and torch.isneginf(kept.lse).all()
    dq, dk, dv = A.attention_backward(do, q, none, none, kept)
    assert not dq.any() and dk.shape == none.shape
    assert not A.attention(q, none, none, key_mask=torch.ones(2, 0, dtype=torch.bool, device=device)).any()
    o, kept = A.attention(q[:, :, :0], k, v, keep=True)
    dq, dk, dv = A.attention_backward(do[:, :0], q[:, :, :0], k, v, kept)
    assert o.shape == (2, 0, 2 * D) and not dk.any() and not dv.any()
    assert A.attention(q[:0], k[:0], v[:0]).shape == (0, 5, 2 * D)


def test_captured_and_replayed(device):
    """Masks are read when a graph is replayed, not when it is captured; two graphs replayed in turn do not disturb each
    other."""
    cases = [make(14, 2, 4, 2, 200, 300, "bf16", "random"), make(15, 1, 2, 2, 33, 2000, "bf16", "middle")]

    def step(q, k, v, do, keep):
        o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
        return o, *A.attention_backward(do, q, k, v, kept, key_mask=keep)
    graphs = []
    for case in cases:
        step(*case)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*case)
        graphs.append((graph, out))
    for i in range(3):
        wants = []
        for q, k, v, do, keep in cases:
            q.mul_(1.25)
            k.nan_to_num_(0.0, 0.0, 0.0)
            v.nan_to_num_(0.0, 0.0, 0.0)
            keep.copy_(torch.rand(keep.shape, generator=torch.Generator().manual_seed(i)).to(device) < 0.5)
            wants.append(step(q, k, v, do, keep))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, wants):
            assert all(torch.equal(a, b) for a, b in zip(out, want)), i


def test_two_streams_at_once(device):
    cases = [make(16 + i, 1, 3, 3, 400, 900, "bf16", "middle") for i in range(2)]

    def step(q, k, v, do, keep):
        o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
        return o, *A.attention_backward(do, q, k, v, kept, key_mask=keep)
    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(4):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(step(*c))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(a, b) for o in outs for a, b in zip(o, w))


def test_offsets_past_32_bits(device):
    """A cache of more than 2^31 elements whose last units alone are kept, and rows 2^21 elements apart."""
    keys = 2 ** 24 + 2 ** 10
    q, part_k, part_v, do, _ = make(18, 1, 1, 1, 40, 96, "bf16")
    k, v = (torch.zeros(1, 1, keys, D, dtype=q.dtype, device=device) for _ in range(2))
    k[:, :, -96:], v[:, :, -96:] = part_k, part_v
    keep = torch.zeros(1, keys, dtype=torch.bool, device=device)
    keep[:, -96:] = True
    want = expected(q, part_k, part_v, do, None)
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    _close("o", o, *want[0])
    dq, dk, dv = A.attention_backward(do, q, k, v, kept, key_mask=keep)
    _close("dq", dq, *want[2])
    _close("dk", dk[:, :, -96:], *want[3])
    _close("dv", dv[:, :, -96:], *want[4])
    assert not dk[:, :, :-96].any() and not dv[:, :, :-96].any()
    del k, v, dk, dv
    rows = torch.zeros(1100, 2 ** 21, dtype=q.dtype, device=device)
    q, k, v, do, _ = make(19, 1, 1, 1, 1090, 1100, "bf16")
    far = rows[:, :D].view(1, 1, 1100, D)
    far.copy_(k)
    assert torch.equal(A.attention(q, far, v), A.attention(q, k, v))


def test_refusals(device):
    q, k, v, do, keep = make(20, 2, 4, 2, 9, 11, "bf16", "random")
    o, kept = A.attention(q, k, v, keep=True)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        A.attention(q.float(), k.float(), v.float())
    with pytest.raises(TypeError, match="like q"):
        A.attention(q, k.half(), v)
    with pytest.raises(ValueError, match="of one shape"):
        A.attention(q, k, v[:, :, :10])
    with pytest.raises(ValueError, match="share"):
        A.attention(q[:, :3], k, v)
    with pytest.raises(ValueError, match="head_dim 64"):
        A.attention(q[..., :64], k[..., :64], v[..., :64])
    with pytest.raises(ValueError, match=r"\(B, H, L, D\)"):
        A.attention(q[0], k, v)
    with pytest.raises(TypeError, match="must be bool"):
        A.attention(q, k, v, key_mask=keep.float())
    with pytest.raises(ValueError, match="key_mask must be"):
        A.attention(q, k, v, key_mask=keep[:, :10])
    with pytest.raises(ValueError, match="GPU only"):
        A.attention(q, k.cpu(), v)
    with pytest.raises(ValueError, match="do must be"):
        A.attention_backward(do[:, :8], q, k, v, kept)
    with pytest.raises(ValueError, match="kept.lse"):
        A.attention_backward(do, q, k, v, kept._replace(lse=kept.lse[:, :3]))
    with pytest.raises(ValueError, match="kept.low"):
        A.attention_backward(do, q, k, v, kept._replace(low=kept.low.float()))


@pytest.mark.parametrize("heads,kv_heads", [(50, 50), (100, 50)])
def test_long_cuts_of_the_queries(device, heads, kv_heads):
    """dk and dv in cuts of two dozen units and more: each adds the units of its own range and no others."""
    check(21, 2, heads, kv_heads, 1500 * kv_heads // heads, 100, "bf16")


def test_cuts_that_begin_near_a_head_s_end(device):
    """Four query heads of ten units a key head, in cuts of 14, 13 and 13: the last begins three units before a head ends."""
    check(22, 1, 280, 70, 320, 100, "bf16")


@pytest.mark.parametrize("heads,kv_heads,queries", [(2, 2, 1), (16, 1, 1), (17, 1, 1), (6, 2, 5), (6, 2, 6), (2, 2, 16), (32, 2, 1)])
@pytest.mark.parametrize("keys,mask", [(31, None), (129, "random"), (2000, "middle"), (4133, None)])
def test_few_rows(device, heads, kv_heads, queries, keys, mask):
    """A key head's rows, at most 16 or just past it, in blocks of their own and cut along the keys."""
    check(heads * keys, 2, heads, kv_heads, queries, keys, "bf16", mask)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("scale", [0.0, 4.0, 30.0])
def test_few_rows_logit_sizes(device, scale, dtype):
    check(11, 3, 8, 2, 2, 700, dtype, "random", scale=scale)


def test_few_rows_of_many_entries(device):
    """Enough entries that none is cut, each with more units than a wave fetches at once."""
    g = torch.Generator("cuda").manual_seed(0)
    batch, keys = 520, 8333
    q = (torch.randn(batch, 1, 1, D, generator=g, device=device) * D ** -0.5).bfloat16()
    k, v = (torch.randn(1, 1, keys, D, generator=g, device=device).bfloat16().expand(batch, -1, -1, -1) for _ in range(2))
    keep = torch.rand(batch, keys, generator=g, device=device) < 0.5
    keep[:5] = True
    keep[5] = False
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    s = (q[:, 0, 0].double() @ k[0, 0].double().T).masked_fill(~keep, -torch.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep, torch.exp(s - lse[:, None]), 0.0)
    want, size = p @ v[0, 0].double(), p @ v[0, 0].double().abs()
    r = 400 * U * q[:, 0, 0].double().abs() @ k[0, 0].double().abs().T.amax(1, keepdim=True) + 2 * (keys + 64) * U
    tol = (2 * 2.0 ** -8 + 2 * r) * size + 2.0 ** -8 * want.abs()
    assert ((o[:, 0].double() - want).abs() <= tol * 1.01).all()
    assert torch.isneginf(kept.lse[5]).all() and not o[5].any()
    rest = torch.arange(batch, device=device) != 5
    assert ((kept.lse[rest, 0, 0].double() - lse[rest]).abs() <= r[rest, 0] + 2 * U * lse[rest].abs()).all()
    assert torch.equal(o, A.attention(q, k, v, key_mask=keep))


def test_few_rows_leave_the_rest(device):
    """Strided outputs and operands of a cache longer than its keys: what lies behind them is neither read nor written."""
    g = torch.Generator("cuda").manual_seed(1)
    cache = torch.randn(2, 2, 900, 2, D, generator=g, device=device).half()
    cache[:, :, 500:] = float("nan")
    k, v = cache[:, :, :500, 0], cache[:, :, :500, 1]
    q = (torch.randn(2, 4, 2, D, generator=g, device=device) * D ** -0.5).half()
    wide = torch.full((2, 5, 4 * D + 64), 7.0, dtype=torch.float16, device=device)
    out = A.attention(q, k, v, out=wide[:, 2:4, 32:32 + 4 * D])
    want = A.attention(q, k.contiguous(), v.contiguous())
    assert torch.equal(out, want) and torch.isfinite(out).all()
    wide[:, 2:4, 32:32 + 4 * D] = 7.0
    assert (wide == 7.0).all()


@pytest.mark.parametrize("mask", ["random", "middle", "last", "empty"])
@pytest.mark.parametrize("queries,keys", [(1, 2047), (3, 2048), (2, 2049), (40, 2048), (40, 2080)])
def test_masks_of_64_units_and_more(device, queries, keys, mask):
    """Up to 64 units each wave finds the live ones itself; past them a launch does."""
    check(keys, 2, 2, 1, queries, keys, "bf16", mask)


@pytest.mark.parametrize("keys", [67, 2300])
def test_mask_views(device, keys):
    """Rows of a wider mask that start at any byte, one row for every entry, and bytes that are not 1."""
    q, k, v, _, keep = make(3, 3, 2, 2, 20, keys, "bf16", "random")
    want = A.attention(q, k, v, key_mask=keep)
    wide = torch.zeros(3, keys + 9, dtype=torch.bool, device=device)
    wide[:, 5:5 + keys] = keep
    assert torch.equal(want, A.attention(q, k, v, key_mask=wide[:, 5:5 + keys]))
    assert torch.equal(want, A.attention(q, k, v, key_mask=(keep.to(torch.uint8) * 128).view(torch.bool)))
    row = keep[:1].expand(3, -1)
    k, v = (torch.where(row[:, None, :, None], torch.randn_like(t), t.new_tensor(float("nan"))) for t in (k, v))
    assert torch.equal(A.attention(q, k, v, key_mask=row), A.attention(q, k, v, key_mask=row.contiguous()))


@pytest.mark.parametrize("queries,keys,mask,dtype", [
    (33, 1, None, "bf16"), (33, 31, None, "fp16"), (47, 64, "random", "bf16"), (63, 129, "middle", "fp16"), (40, 97, "none", "bf16"),
    (40, 97, "first", "bf16"), (65, 66, "empty", "fp16"), (34, 300, "random", "bf16"), (257, 33, "last", "bf16")])
def test_many_heads(device, queries, keys, mask, dtype):
    """Short sequences of enough heads that blocks of 256 queries take them, not blocks of 16."""
    check(queries, 64, 8, 8, queries, keys, dtype, mask)


@pytest.mark.parametrize("batch,queries", [(2, 5), (64, 33)])
@pytest.mark.parametrize("size,scale", [(2.0 ** -80, 1.0), (2.0 ** 100, 1.0), (2.0 ** -80, 30.0)])
def test_sizes_of_values(device, batch, queries, size, scale):
    """Values far from 1 in either direction: bfloat16 has float32's range, and sums of P v keep it."""
    q, k, v, do, keep = make(9, batch, 8, 8, queries, 100, "bf16", "random", scale=scale)
    v = torch.where(keep[:, None, :, None], v * size, v)
    want = expected(q, k, v, do, keep)
    _close("o", A.attention(q, k, v, key_mask=keep), *want[0])
