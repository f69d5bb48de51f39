"""Each form of attention's forward pass against float64: blocks of 192 and of 256 queries, whole, cut and both at once, with
enough units for their unrolled loops, and blocks of 16 rows with more units than a wave fetches at once.  The plan decides the
form; tests/test_attention_plan_host.py holds these shapes to theirs.  Tolerances are test_gpu_attention's."""

import pytest
import torch

from flicker_amd import _lib
from flicker_amd import attention as A
from tests.attention_forms import FORMS, check, close, expected
from tests.test_gpu_attention import D, U, make

pytestmark = pytest.mark.gpu


def step(q, k, v, do, keep):
    o, kept = A.attention(q, k, v, key_mask=keep, keep=True)
    return o, kept, *A.attention_backward(do, q, k, v, kept, key_mask=keep)


def bits(out):
    o, kept, *grads = out
    return [o, kept.low, kept.lse, *grads]


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mask", [None, "random", "middle"])
@pytest.mark.parametrize("form", [f for f in FORMS if f != "256 long"])
def test_forms(device, form, mask, dtype):
    """With and without what the gradients need, the same o; its gradients; the same bits a second time."""
    print(f"form {form} {mask} {dtype}", flush=True)
    ops = make(7, *FORMS[form][0], dtype, mask)
    out = step(*ops)
    check(form, out, expected(*ops))
    assert torch.equal(A.attention(*ops[:3], key_mask=ops[4]), out[0])
    assert all(torch.equal(a, b) for a, b in zip(bits(out), bits(step(*ops))))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("mask", [None, "random"])
def test_long_lists(device, mask, dtype):
    """Whole blocks of 256 queries that walk 79 units."""
    ops = make(8, *FORMS["256 long"][0], dtype, mask)
    check("256 long", step(*ops), expected(*ops))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("form", ["192", "192 cut", "256", "256 both", "256 shared"])
@pytest.mark.parametrize("scale,mask", [(0.0, None), (8.0, "random"), (30.0, None)])
def test_logit_sizes(device, form, scale, mask, dtype):
    """Logits whose running maximum has to rise after the first unit, in most rows more than once."""
    print(f"form {form} scale {scale} {dtype}", flush=True)
    ops = make(9, *FORMS[form][0], dtype, mask, scale=scale)
    check(form, step(*ops), expected(*ops))


def test_empty_entries(device):
    for form in ("192", "256 shared", "192 shared"):
        batch, *rest = FORMS[form][0]
        ops = make(10, max(batch, 2), *rest, "bf16", "empty")
        check(form, step(*ops), expected(*ops))


@pytest.mark.parametrize("names", [("192 cut", "256 cut"), ("256 both", "192")])
def test_captured_and_replayed(device, names):
    """Two graphs, replayed in turn with eager calls between them."""
    cases = [make(11 + i, *FORMS[n][0], "bf16", "random") for i, n in enumerate(names)]
    graphs = []
    for case in cases:
        step(*case)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*case)
        graphs.append((graph, out))
    for i in range(3):
        for q, *_ in cases:
            q.mul_(1.25)
        wants = [bits(step(*case)) for case in cases]
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (_, out), want in zip(graphs, wants):
            assert all(torch.equal(a, b) for a, b in zip(bits(out), want)), i


def test_two_streams_at_once(device):
    cases = [make(13 + i, *FORMS[n][0], "bf16", "middle") for i, n in enumerate(("192 cut", "256 cut"))]
    wants = [bits(step(*c)) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(4):
        for outs, stream, case in zip(got, streams, cases):
            with torch.cuda.stream(stream):
                outs.append(bits(step(*case)))
    torch.cuda.synchronize()
    for outs, want in zip(got, wants):
        assert all(torch.equal(a, b) for out in outs for a, b in zip(out, want))


@pytest.mark.parametrize("form", ["192", "256 shared"])
def test_strided_operands(device, form):
    """Columns of one projection and a result inside wider rows."""
    batch, heads, kv_heads, queries, keys = FORMS[form][0]
    q, k, v, _, keep = make(15, batch, heads, kv_heads, queries, keys, "bf16", "random")
    want = A.attention(q, k, v, key_mask=keep)
    views = []
    for t in (q, k, v):
        b, h, n, _ = t.shape
        wide = torch.full((b, n, h * D + 64), float("nan"), dtype=t.dtype, device=device)
        view = wide[..., 32:32 + h * D].view(b, n, h, D).transpose(1, 2)
        view.copy_(t)
        views.append(view)
    buffer = torch.full((batch, queries + 3, heads * D + 64), 7.0, dtype=q.dtype, device=device)
    out = A.attention(*views, key_mask=keep, out=buffer[:, 2:-1, 32:-32])
    assert torch.equal(out, want)
    buffer[:, 2:-1, 32:-32] = 7.0
    assert (buffer == 7.0).all()


# (batch, heads, keys) of blocks of 16 rows whose waves walk more than 64 units each
LONG_ROWS = [(513, 16, 8400), (1, 16, 2 ** 20 - 77)]


@pytest.mark.parametrize("batch,heads,keys", LONG_ROWS)
@pytest.mark.parametrize("masked", [False, True])
def test_few_rows_of_long_lists(device, batch, heads, keys, masked):
    """One query of 16 heads that share a key head, whole and cut: a wave fetches its list of live units 64 at a time."""
    g = torch.Generator("cuda").manual_seed(batch)
    q = (torch.randn(batch, heads, 1, D, generator=g, device=device) * D ** -0.5).bfloat16()
    k, v = (torch.randn(1, 1, keys, D, generator=g, device=device).bfloat16().expand(batch, -1, -1, -1) for _ in range(2))
    keep = None
    if masked:
        keep = torch.rand(batch, keys, generator=g, device=device) < 0.5
        keep[:3] = True
    o = A.attention(q, k, v, key_mask=keep)
    for b in range(0, batch, 37):
        on = slice(None) if keep is None else keep[b]
        kb, vb = k[0, 0][on].double(), v[0, 0][on].double()
        s = q[b, :, 0].double() @ kb.T.contiguous()
        lse = torch.logsumexp(s, -1, keepdim=True)
        p = torch.exp(s - lse)
        size = (q[b, :, 0].double().abs() @ kb.abs().T.contiguous()).amax(-1, keepdim=True)
        r = 2 * 130 * U * size + 8 * U * (s.abs().amax(-1, keepdim=True) + lse.abs()) + (keys + 128) * U
        off = (2 * 2.0 ** -8 + 2 * r + (keys + 64) * U) * (p @ vb.abs())
        close(f"entry {b}", o[b, 0].view(heads, D), p @ vb, off)


def test_most_heads(device):
    """As many heads as a call takes, one query and one key each: the gradients' blocks of queries and of keys together are
    more work-items than a launch counts.  P = 1: o is v and dv do; dS is what 2 * 130 roundings leave of dP - delta."""
    g = torch.Generator("cuda").manual_seed(0)
    batch, heads = 2 ** 20, 4
    q, k, v, do = (torch.randn(batch, heads, 1, D, generator=g, device=device, dtype=torch.bfloat16) for _ in range(4))
    q *= D ** -0.5
    o, kept = A.attention(q, k, v, keep=True)
    assert torch.equal(o.view(v.shape), v)
    dq, dk, dv = A.attention_backward(do.view(batch, 1, heads * D), q, k, v, kept)
    assert torch.equal(dv, do)
    for first in range(0, batch, 2 ** 17):
        part = slice(first, first + 2 ** 17)
        off = 260 * U * (do[part].float() * v[part].float()).abs().sum(-1, keepdim=True) * 1.01
        for grad, by in ((dq, k), (dk, q)):
            assert (grad[part].float().abs() <= off * by[part].float().abs()).all()
    del o, kept, dq, dk, dv
    with pytest.raises(_lib.HipKernelError, match="flk_attention_plan"):
        A.attention(torch.empty(batch, heads + 1, 1, D, dtype=torch.bfloat16, device=device), *[torch.empty(
            batch, heads + 1, 1, D, dtype=torch.bfloat16, device=device)] * 2)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("sizes,mask", [((1, 1, 1, 2 ** 20 + 5, 3), None), ((1, 2, 1, 1, 2 ** 21 + 3), "random"), ((1, 1, 1, 70000, 40), "random"),
                                        ((700, 3, 3, 2, 2), "random"), ((1, 64, 1, 33, 77), "middle")])
def test_long_sides(device, sizes, mask, dtype):
    """One side of a million rows beside a few; many entries of two; 64 heads on one."""
    print(f"sides {sizes} {mask} {dtype}", flush=True)
    ops = make(17, *sizes, dtype, mask)
    check(str(sizes), step(*ops), expected(*ops))
