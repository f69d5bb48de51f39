"""attention and its gradients where values are far from what a norm leaves: logits up to the type's and float32's ends,
infinities and NaN in operands that are not masked.  Each in every form of the forward pass (attention_forms.FORMS)."""

import pytest
import torch

from flicker_amd import attention as A
from tests.attention_forms import FORMS, expected
from tests.test_gpu_attention import D, TINY, TYPES, U, make

pytestmark = pytest.mark.gpu
SHORT = ["16", "16 cut", "192", "192 cut", "256", "256 cut", "256 both", "256 shared"]


def exact_logits(seed, form, dtype, q_size, k_size, masked, negative, device):
    """q rows of one value +-q_size, k of whole numbers times k_size: logits that float32 holds exactly, in each row one largest
    that is far above the others.  (q, k, v, do, keep, index (B, H, Lq) of the largest's key, its logit)."""
    batch, heads, kv_heads, queries, keys = FORMS[form][0]
    g = torch.Generator().manual_seed(seed)
    n = torch.randint(-99, -1 if negative else 100, (batch, kv_heads, keys, D), generator=g).double()
    keep = torch.rand(batch, keys, generator=g) < 0.7 if masked else torch.ones(batch, keys, dtype=torch.bool)
    keep[:, keys // 2:keys // 2 + 2] = True
    high, low = torch.empty(batch, kv_heads, D, dtype=torch.long), torch.empty(batch, kv_heads, D, dtype=torch.long)
    for b in range(batch):
        on = keep[b].nonzero().flatten()
        for h in range(kv_heads):
            for i, (to, value) in enumerate(((low, -100.0), (high, -1.0 if negative else 100.0))):   # of different keys
                to[b, h] = on[i::2][torch.randint(len(on) // 2, (D,), generator=g)]
                n[b, h].scatter_(0, to[b, h][None], value)
    n[~keep[:, None, :].expand(batch, kv_heads, keys)] = 127.0
    column = torch.arange(queries) % D
    sign = torch.ones(batch, heads, queries) if negative else torch.randint(0, 2, (batch, heads, queries), generator=g) * 2.0 - 1
    q = torch.zeros(batch, heads, queries, D, dtype=torch.float64)
    q[:, :, torch.arange(queries), column] = sign.double() * q_size
    group = heads // kv_heads
    high, low = (t.repeat_interleave(group, 1)[:, :, column] for t in (high, low))
    index = torch.where(sign > 0, high, low)
    top = sign * q_size * k_size * n.repeat_interleave(group, 1)[torch.arange(batch)[:, None, None], torch.arange(heads)[:, None], index,
                                                                column]
    t = TYPES[dtype]
    v = torch.randn(batch, kv_heads, keys, D, generator=g).to(t)
    do = torch.randn(batch, queries, heads * D, generator=g).to(t)
    return [x.to(device) for x in (q.to(t), (n * k_size).to(t), v, do, keep, index, top)]


SIZES = [("fp16", 2.0 ** 6, 2.0 ** 6), ("fp16", 2.0 ** 15, 2.0 ** 9), ("bf16", 2.0 ** 10, 2.0 ** 15), ("bf16", 2.0 ** 40, 2.0 ** 56),
         ("bf16", 2.0 ** 60, 2.0 ** 60)]


@pytest.mark.parametrize("form", SHORT)
@pytest.mark.parametrize("negative", [False, True])
@pytest.mark.parametrize("dtype,q_size,k_size", SIZES)
def test_far_logits(device, form, dtype, q_size, k_size, negative):
    """The logits' differences are all of q_size * k_size >= 2^12 and more, so the largest's P is 1 and the others' 0: o is that
    key's v, exactly; lse its logit, off by a rounding and 2^-20 of a logarithm; dv the sums of do, off by their additions, at
    most queries * group + 64 deep, and by P's error, 8 u |lse|, where |lse| is less than 2^23 (past it lse is that logit).  dS is
    what dP and delta leave of each other: 2 * 130 u sum|do v| and, from o's rounding being held to e^2, sum|do o| e^2."""
    print(f"far logits {form} {dtype} {q_size} {k_size} {negative}", flush=True)
    masked = form != "192"
    q, k, v, do, keep, index, top = exact_logits(1, form, dtype, q_size, k_size, masked, negative, device)
    mask = keep if masked else None
    (batch, heads, queries, _), (_, kv_heads, keys, _) = q.shape, k.shape
    group = heads // kv_heads
    o, kept = A.attention(q, k, v, key_mask=mask, keep=True)
    pick = index[..., None].expand(-1, -1, -1, D)
    want = v.repeat_interleave(group, 1).gather(2, pick).transpose(1, 2).reshape(o.shape)
    assert torch.equal(o, want) and torch.equal(A.attention(q, k, v, key_mask=mask), want)
    assert ((kept.lse.double() - top).abs() <= 2 * U * top.abs() + 2.0 ** -20).all()
    dq, dk, dv = A.attention_backward(do, q, k, v, kept, key_mask=mask)
    g4 = do.view(batch, queries, heads, D).transpose(1, 2).double()
    sums, sizes = (torch.zeros(batch, heads, keys, D, dtype=torch.float64, device=device).scatter_add_(2, pick, t).view(
        batch, kv_heads, group, keys, D).sum(2) for t in (g4, g4.abs()))
    e = torch.finfo(q.dtype).eps / 2
    p_off = 8 * U * min(float(top.abs().max()), 2.0 ** 23)
    p_off = p_off + e if p_off > 0 else e
    off = (p_off + (queries * group + 64) * U) * sizes
    tiny = 2.0 ** -25 if dtype == "fp16" else 0.0
    assert ((dv.double() - sums).abs() <= e * (sums.abs() + off) + off + tiny).all()
    o4 = want.view(batch, queries, heads, D).transpose(1, 2).double()
    ds = ((260 * U + e * e) * (1 + p_off) * (g4.abs() * o4.abs()).sum(-1, keepdim=True))
    size = k.double().abs().repeat_interleave(group, 1).gather(2, pick)
    # what lies below float16's range in dS is dropped or kept, off by 2^-25 at most
    assert (dq.double().abs() <= (ds + tiny) * (1 + e) * size + tiny).all()
    assert torch.isfinite(dq).all() and torch.isfinite(dk).all()


def _plain(q, k, v, do):
    """(o, lse, dq, dk, dv) in float64 from the formulas; no mask."""
    (batch, heads, queries, _), kv_heads = q.shape, k.shape[1]
    group = heads // kv_heads
    g = do.view(batch, queries, heads, D).transpose(1, 2).double().contiguous()
    q, k, v = q.double(), *(t.double().repeat_interleave(group, 1) for t in (k, v))
    s = q @ k.transpose(2, 3).contiguous()
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p = p / total
    o = p @ v
    ds = p * (g @ v.transpose(2, 3).contiguous() - (g * o).sum(-1, keepdim=True))
    shared = (batch, kv_heads, group, *k.shape[2:])
    dk, dv = (t.transpose(2, 3).contiguous() @ x for t, x in ((ds, q), (p, g)))
    return o.transpose(1, 2).flatten(2), (top + total.log())[..., 0], ds @ k, dk.view(shared).sum(2), dv.view(shared).sum(2)


@pytest.mark.parametrize("form", ["16", "16 cut", "192", "192 cut", "256 shared"])
@pytest.mark.parametrize("which,value", [("q", "nan"), ("q", "inf"), ("k", "nan"), ("k", "inf"), ("k", "-inf"), ("v", "nan"), ("v", "inf"),
                                         ("v", "-inf"), ("do", "nan"), ("do", "inf")])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_not_finite(device, form, which, value, dtype):
    """One value that is not finite reaches every result that the formulas give it to, and no other: those stay within
    the tolerance of the call without it."""
    print(f"not finite {form} {which} {value} {dtype}", flush=True)
    ops = dict(zip(("q", "k", "v", "do", "keep"), make(3, *FORMS[form][0], dtype)))
    clean = _plain(ops["q"], ops["k"], ops["v"], ops["do"])
    tols = expected(*ops.values())
    t = ops[which]
    ops[which] = t = t.clone()
    at = (0, t.shape[1] // 2, t.shape[2] // 3) if t.dim() == 3 else (0, t.shape[1] - 1, t.shape[2] // 2, 77)
    t[at] = float(value)
    want = _plain(ops["q"], ops["k"], ops["v"], ops["do"])
    o, kept = A.attention(ops["q"], ops["k"], ops["v"], keep=True)
    assert torch.equal(o.nan_to_num(1e4), A.attention(ops["q"], ops["k"], ops["v"]).nan_to_num(1e4))
    got = (o, kept.lse, *A.attention_backward(ops["do"], ops["q"], ops["k"], ops["v"], kept))
    assert not all(w.isfinite().all() for w in want)
    for name, g, w, c, (_, off) in zip(("o", "lse", "dq", "dk", "dv"), got, want, clean, tols):
        finite = w.isfinite()
        assert torch.equal(g.isfinite(), finite), (name, int((g.isfinite() & ~finite).sum()), int((~g.isfinite() & finite).sum()))
        same = finite & (w == c)
        e = torch.finfo(g.dtype).eps / 2
        off = e * (c.abs() + off) + off + TINY.get(g.dtype, 2 * U)
        assert ((g.double() - c).abs() <= off)[same].all(), name


@pytest.mark.parametrize("form", ["16", "192", "256 shared"])
def test_every_logit_minus_infinity(device, form):
    """A row with nothing to weigh is one without keys; the others of its block are not touched."""
    q, k, v, _, _ = make(4, *FORMS[form][0], "bf16")
    k[..., 0] = float("-inf")
    q[..., 0] = 0.5
    q[:, :, 1::2] = float("nan")
    o, kept = A.attention(q, k, v, keep=True)
    o = o.unflatten(2, (q.shape[1], D))
    assert not o[:, ::2].any() and o[:, 1::2].isnan().all()
    assert kept.lse[:, :, ::2].isneginf().all() and kept.lse[:, :, 1::2].isnan().all()


@pytest.mark.parametrize("form", SHORT)
@pytest.mark.parametrize("dtype,size", [("fp16", 2.0 ** 10), ("bf16", 2.0 ** 10), ("bf16", 2.0 ** 50)])
def test_far_logits_of_many_terms(device, form, dtype, size):
    """Logits of 128 unequal terms each, whose roundings are far more than 1: forwards and backwards form the same ones, so that
    P of a row's largest is 1 where the next is far below, off by no more than lse's rounding at 2^-1 of its unit."""
    print(f"far logits of many terms {form} {dtype} {size}", flush=True)
    batch, heads, kv_heads, queries, keys = FORMS[form][0]
    group = heads // kv_heads
    q, k, v, do, _ = make(6, *FORMS[form][0], dtype, scale=D ** 0.5)
    q, k = q * size, k * size
    s = q.double() @ k.double().repeat_interleave(group, 1).transpose(2, 3).contiguous()
    (first, second), at = s.topk(2, -1).values.unbind(-1), s.argmax(-1)
    clear = first - second > 200 + 4 * 130 * U * (q.double().abs().sum(-1) * k.double().abs().amax())
    assert clear.float().mean() > 0.9
    o, kept = A.attention(q, k, v, keep=True)
    pick = at[..., None].expand(-1, -1, -1, D)
    want = v.repeat_interleave(group, 1).gather(2, pick)
    got = o.unflatten(2, (heads, D)).transpose(1, 2)
    assert torch.equal(got[clear], want[clear])
    do = torch.where(clear.transpose(1, 2)[..., None], do.unflatten(2, (heads, D)), 0.0).flatten(2)
    dq, dk, dv = A.attention_backward(do, q, k, v, kept)
    g4 = do.view(batch, queries, heads, D).transpose(1, 2).double()
    sums, sizes = (torch.zeros(batch, heads, keys, D, dtype=torch.float64, device=device).scatter_add_(2, pick, t).view(
        batch, kv_heads, group, keys, D).sum(2) for t in (g4, g4.abs()))
    e = torch.finfo(q.dtype).eps / 2
    off = (queries * group + 64) * U * sizes
    assert ((dv.double() - sums).abs() <= e * (sums.abs() + off) + off + (2.0 ** -25 if dtype == "fp16" else 0.0)).all()
    assert not dq.isnan().any() and not dk.isnan().any()
