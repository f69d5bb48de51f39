"""float16 attention where P and dS leave float16's range or its full precision: gradients of every size, long rows.

P and dS are rounded to 11 bits of themselves, with no regard to their size: e = 2^-11 of each at most, and independently.  An
output's error is then a sum of independent terms, none above e |dS_ij k_jd| (P's own error r, as in test_gpu_attention, adds to
e), and over a row of 128 or more outputs its norm stays within 4 times the norm of their standard deviations'
bounds, sqrt(sum_j ((e + r) dS_ij k_jd)^2).  delta is off by o's error, of which P's rounding leaves sqrt(sum_j (2 e P_ij v_jd)^2) a
value and Kept.low e^2 of it, times do, and reaches dq as delta's error times sum_j P_ij k_j, dk as its sum over rows.  Last, each
output is rounded to float16: e of itself and 2^-25 at most.
"""

import pytest
import torch

from flicker_amd import attention as A
from tests.attention_forms import FORMS
from tests.test_gpu_attention import D, U, make

pytestmark = pytest.mark.gpu
E = 2.0 ** -11


def bounds(q, k, v, do, keep):
    """[(dq, dev), (dk, dev), (dv, dev)]: float64 gradients, and what each value's deviation is at most."""
    (batch, heads, queries, _), (_, kv_heads, keys, _) = q.shape, k.shape
    group = heads // kv_heads
    out = [(torch.zeros(t.shape, dtype=torch.float64, device=q.device), torch.zeros(t.shape, dtype=torch.float64, device=q.device))
           for t in (q, k, v)]
    do = do.view(batch, queries, heads, D).transpose(1, 2)
    for b in range(batch):
        on = torch.ones(keys, dtype=torch.bool, device=q.device) if keep is None else keep[b]
        for h in range(heads):
            hk = h // group
            qh, gh = q[b, h].double(), do[b, h].double()
            kh, vh = (torch.where(on[:, None], t[b, hk].double(), 0.0) for t in (k, v))
            s = torch.where(on, qh @ kh.T.contiguous(), -torch.inf)
            p = torch.softmax(s, -1)
            o = p @ vh
            dp = gh @ vh.T.contiguous() - (gh * o).sum(-1, keepdim=True)
            ds = p * dp
            size = torch.where(on, qh.abs() @ kh.abs().T.contiguous(), 0.0).amax(-1)
            r = (260 * U * size + 16 * U * torch.where(on, s.abs(), 0.0).amax(-1) + (keys + 128) * U)[:, None]
            off = E + r
            delta2 = (gh ** 2 * ((2 * off * p) ** 2 @ vh ** 2 + (E * E * o) ** 2)).sum(-1, keepdim=True)
            # dP: 130 products' roundings
            dp2 = (130 * U) ** 2 * (gh ** 2 @ (vh ** 2).T.contiguous())
            ds2 = (off * ds) ** 2 + p ** 2 * dp2
            p2 = (off * p) ** 2
            out[0][0][b, h] = ds @ kh
            out[0][1][b, h] = ds2 @ kh ** 2 + delta2 * (p @ kh) ** 2
            out[1][0][b, hk] += ds.T.contiguous() @ qh
            out[1][1][b, hk] += ds2.T.contiguous() @ qh ** 2 + (p ** 2 * delta2).T.contiguous() @ qh ** 2
            out[2][0][b, hk] += p.T.contiguous() @ gh
            out[2][1][b, hk] += p2.T.contiguous() @ gh ** 2
    return [(w, d.sqrt()) for w, d in out]


def within(label, got, want, dev, dims):
    """The norm over ``dims`` of the difference against 4 times the deviations' and the last rounding's."""
    diff = (got.double() - want)
    off = (4 * torch.linalg.vector_norm(dev, dim=dims) + E * torch.linalg.vector_norm(want, dim=dims)
           + 2.0 ** -25 * (got.numel() / max(1, want.sum(dims).numel())) ** 0.5)
    err = torch.linalg.vector_norm(diff, dim=dims)
    worst = (err / off).max()
    print(f"  {label} {float(worst):.3f} of its bound, {float(diff.norm() / want.norm()):.2e} of the norm", flush=True)
    assert torch.isfinite(got).all() and worst <= 1, (label, float(worst))


# what the gradients' sizes and the operands' are multiplied by; q k stays, so that dq, or dk, is within float16's range
@pytest.mark.parametrize("of_do", [-14, -10, -7, 0, 8])
@pytest.mark.parametrize("of_k", [7, -7])
@pytest.mark.parametrize("form", ["192", "192 cut", "192 shared", "256 cut"])
def test_sizes_of_gradients(device, form, of_do, of_k):
    print(f"gradients {form} 2^{of_do} 2^{of_k}", flush=True)
    q, k, v, do, keep = make(1, *FORMS[form][0], "fp16", "random" if form == "192 shared" else None)
    q, k, do = (t * 2.0 ** s for t, s in ((q, -of_k), (k, of_k), (do, of_do)))
    if keep is not None:
        k, v = (torch.where(keep[:, None, :, None], t, float("nan")) for t in (k, v))
    want = bounds(q, k, v, do, keep)
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    grads = A.attention_backward(do, q, k, v, kept, key_mask=keep)
    for name, got, (w, dev) in zip(("dq", "dk", "dv"), grads, want):
        if w.abs().max() < 60000:
            within(name, got, w, dev, (2, 3))


@pytest.mark.parametrize("form", ["192", "192 shared"])
def test_rows_of_different_sizes(device, form):
    """Each row of dq is as precise as its own gradient allows."""
    q, k, v, do, _ = make(2, *FORMS[form][0], "fp16")
    sizes = 2.0 ** -(torch.arange(do.shape[1], device=device) % 14).to(do.dtype)
    do = do * sizes[:, None]
    q, k = q / 128, k * 128
    (dq, dev), *_ = bounds(q, k, v, do, None)
    o, kept = A.attention(q, k, v, keep=True)
    within("dq", A.attention_backward(do, q, k, v, kept)[0], dq, dev, (3,))


def test_large_products(device):
    """dS past 65504, from a few keys of large values: dq is within range through small keys, dk through small queries."""
    for of_k in (-10, 6):
        q, k, v, do, _ = make(3, 1, 24, 24, 370, 9, "fp16")
        q, k, v, do = q * 2.0 ** -of_k, k * 2.0 ** of_k, v * 2.0 ** 7, do * 2.0 ** 9
        want = bounds(q, k, v, do, None)
        o, kept = A.attention(q, k, v, keep=True)
        grads = A.attention_backward(do, q, k, v, kept)
        i = 0 if of_k < 0 else 1
        assert want[i][0].abs().max() < 60000
        within("dq" if of_k < 0 else "dk", grads[i], *want[i], (2, 3))


@pytest.mark.parametrize("keys", [3000, 20000])
def test_long_rows(device, keys):
    """P about 2^-14 and far below: dv of each key is as precise as its own P."""
    q, k, v, do, _ = make(4, 1, 2, 2, 300, keys, "fp16", scale=2.0)
    do = do * 2.0 ** 6
    want = bounds(q, k, v, do, None)
    o, kept = A.attention(q, k, v, keep=True)
    grads = A.attention_backward(do, q, k, v, kept)
    for name, got, (w, dev), dims in zip(("dq", "dk", "dv"), grads, want, ((3,), (2, 3), (3,))):
        within(name, got, w, dev, dims)


def test_zero_gradients_and_values(device):
    q, k, v, do, _ = make(5, *FORMS["192"][0], "fp16")
    o, kept = A.attention(q, k, v, keep=True)
    assert not any(t.any() for t in A.attention_backward(do * 0, q, k, v, kept))
    o, kept = A.attention(q, k, v * 0, keep=True)
    dq, dk, dv = A.attention_backward(do, q, k, v * 0, kept)
    assert not dq.any() and not dk.any() and dv.any()


@pytest.mark.parametrize("form", ["16", "16 cut", "192", "192 cut", "256", "256 both", "256 cut"])
def test_many_small_weights(device, form):
    """All keys but one at 2^-25.4 of the largest P, and o theirs alone.  P 2^8 is a subnormal of float16 there, off by 2^-25 at
    most, which is 2^-33 of the largest P; the sum that divides o is 1 and at most 2e-4 more."""
    batch, heads, kv_heads, queries, keys = FORMS[form][0]
    q, k, v = (torch.zeros(batch, h, n, D, dtype=torch.float16, device=device)
               for h, n in ((heads, queries), (kv_heads, keys), (kv_heads, keys)))
    q[..., 5] = 1.0
    k[..., 5] = -17.625
    v[:] = 64.0
    for h in range(kv_heads):                       # the largest in another unit of each head
        k[:, h, (37 * h) % keys, 5] = 0.0
        v[:, h, (37 * h) % keys] = 0.0
    p = torch.exp(torch.tensor(-17.625, dtype=torch.float64))
    want = float(64 * (keys - 1) * p / (1 + (keys - 1) * p))
    o, kept = A.attention(q, k, v, keep=True)
    off = 64 * (keys - 1) * 2.0 ** -33 + 2 * E * want + 64 * U * keys * want
    assert ((o.double() - want).abs() <= off + E * want + 2.0 ** -25).all(), (float(o.min()), float(o.max()), want)
    assert torch.equal(o, A.attention(q, k, v))
    total = float(torch.log1p((keys - 1) * p))
    assert ((kept.lse.double() - total).abs() <= 64 * U * 18).all()


@pytest.mark.parametrize("queries,keys,masked", [(16, 16896, False), (40, 9000, True), (3000, 20, False), (1, 5000, True)])
def test_long_and_short(device, queries, keys, masked):
    """Pieces of long walks each find their own powers of two, by the units of their lists."""
    q, k, v, do, keep = make(6, 2, 3, 1, queries, keys, "fp16", "random" if masked else None)
    sizes = 2.0 ** -(torch.arange(keys, device=device) // 500 % 10).to(v.dtype)     # values that differ along the keys
    v = torch.where(torch.isfinite(v), v * sizes[:, None], v)
    q, k, do = q / 64, k * 64, do * 2.0 ** -10
    (dq, dev), (dk, dk_dev), (dv, dv_dev) = bounds(q, k, v, do, keep)
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    got = A.attention_backward(do, q, k, v, kept, key_mask=keep)
    within("dq", got[0], dq, dev, (2, 3))
    q, k, do = q * 2 ** 12, k / 2 ** 12, do * 2.0 ** 10
    want = bounds(q, k, v, do, keep)
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    for name, g, (w, d) in zip(("dk", "dv"), A.attention_backward(do, q, k, v, kept, key_mask=keep)[1:], want[1:]):
        within(name, g, w, d, (2, 3))
