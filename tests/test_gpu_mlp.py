"""The gated MLP's matrix products on the GPU.

The products are checked with small whole numbers: every partial sum is exact in float32 (below 2^24), so the
result is the exact product rounded once, whatever the order -- a missing, doubled or misplaced term shows as
a different value.  The gate's g and u come out unrounded and must be exact; h and the gate's gradients
follow from them within the gate's own error (tests/test_gpu_norm.py) and one rounding.

The whole operator on real values, against float64: h is rounded to the operands' type between the products,
half a step, e = eps / 2, of each of its terms, and y's terms move by e |h| |w|; backwards dgu is rounded
likewise.  float32 sums of n terms add n u of the terms' absolute sum, u = 2^-24, at most.
"""

import numpy as np
import pytest
import torch

from flicker_amd import _lib, autograd, mlp, modules, norm
from oracle import mlp as M
from tests.test_gpu_norm import TINY, Declines, _close, _f64, _gate_case

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
BOTH = [torch.bfloat16, torch.float16]


def _whole(seed, shape, dtype, device, top=4):
    """Whole numbers in [-top, top]."""
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-top, top + 1, shape, generator=g).to(dtype).to(device)


def _rounded(exact, dtype):
    """float64 whole numbers (below 2^24, so float32 holds them) rounded once."""
    return torch.from_numpy(exact).to(torch.float32).to(dtype)


# rows, cols, inner: one of everything, edges of the 128-wide tiles and either side of them, ragged, long inner axes (larger
# tiles: TILES)
SIZES = [(1, 8, 8), (1, 512, 1000), (3, 64, 96), (16, 128, 64), (17, 136, 72), (33, 8, 2048), (64, 72, 40), (100, 256, 256),
         (129, 248, 136), (255, 264, 200), (257, 512, 64), (300, 1024, 328), (512, 520, 72), (1000, 776, 1160)]


@pytest.mark.parametrize("rows,cols,inner", SIZES)
@pytest.mark.parametrize("dtype", BOTH)
def test_products_are_exact_on_whole_numbers(device, rows, cols, inner, dtype):
    top = 4
    assert top * top * inner < 2 ** 24
    a, b = _whole(1, (rows, inner), dtype, device), _whole(2, (inner, cols), dtype, device)
    want = _rounded(_f64(a) @ _f64(b), dtype)
    for a_t, b_t in ((False, False), (False, True)):
        print(f"matmul rows={rows} cols={cols} inner={inner} {dtype} a_t={a_t} b_t={b_t}", flush=True)
        out = torch.full((rows, cols), 77.0, dtype=dtype, device=device)
        mlp._matmul(a, b.t().contiguous() if b_t else b, out, b_t=b_t)
        assert torch.equal(out.cpu(), want), f"a_t={a_t} b_t={b_t}: {int((out.cpu() != want).sum())} differ"
    # the tokens' axis inside: `inner` tokens may be any number, the others are widths
    tokens = rows
    x, y = _whole(3, (tokens, inner), dtype, device), _whole(4, (tokens, cols), dtype, device)
    print(f"matmul transposed a: tokens={tokens} {inner} x {cols} {dtype}", flush=True)
    out = torch.full((inner, cols), 77.0, dtype=dtype, device=device)
    mlp._matmul(x, y, out, a_t=True)
    want = _rounded(_f64(x).T @ _f64(y), dtype)
    assert torch.equal(out.cpu(), want), f"{int((out.cpu() != want).sum())} differ"


@pytest.mark.parametrize("dtype", BOTH)
def test_products_of_strided_operands(device, dtype):
    """Rows inside wider buffers, none of whose other values are read or written."""
    rows, cols, inner = 150, 88, 104
    wide = torch.full((rows, 3, 128), float("nan"), dtype=dtype, device=device)
    a = wide[:, 1, 8:8 + inner]
    a.copy_(_whole(1, (rows, inner), dtype, device))
    wb = torch.full((inner + 2, 200), float("nan"), dtype=dtype, device=device)
    b = wb[1:-1, 16:16 + cols]
    b.copy_(_whole(2, (inner, cols), dtype, device))
    big = torch.full((rows + 2, cols + 16), 5.0, dtype=dtype, device=device)
    mlp._matmul(a, b, big[1:-1, 8:-8])
    assert torch.equal(big[1:-1, 8:-8].cpu(), _rounded(_f64(a) @ _f64(b), dtype))
    big[1:-1, 8:-8] = 5.0
    assert (big == 5.0).all()


@pytest.mark.parametrize("m,width,hidden", [(1, 8, 8), (1, 1024, 136), (2, 64, 64), (9, 72, 200), (16, 512, 96), (31, 136, 1032),
                                            (64, 64, 128), (130, 264, 72), (257, 96, 392), (600, 328, 520)])
@pytest.mark.parametrize("dtype", BOTH)
def test_gate_products(device, m, width, hidden, dtype):
    """flk_mlp_gate and flk_mlp_gate_backward on whole numbers scaled to keep the gate's argument small."""
    print(f"gate m={m} width={width} hidden={hidden} {dtype}", flush=True)
    x, w = _whole(1, (m, width), dtype, device, 3), _whole(2, (width, 2 * hidden), dtype, device, 1) * 2.0 ** -6
    gu = torch.full((m, 2 * hidden), 77.0, device=device)
    want = _f64(x) @ _f64(w)
    for kept in (gu, None):
        h = torch.full((m, hidden), 77.0, dtype=dtype, device=device)
        ws, nbytes = mlp._workspace(mlp._GATE, m, hidden, width, device)
        _lib.run("flk_mlp_gate", (x, w, h, kept, ws), x.data_ptr(), width, w.data_ptr(), 2 * hidden, mlp._dtype("x", x), m,
                 width, hidden, h.data_ptr(), hidden, _lib.ptr(kept), _lib.ptr(ws), nbytes, _lib.stream_of(x))
        _close("h", h, *_gate_case(want, np.zeros((m, hidden)))[0])
    assert np.array_equal(_f64(gu), want)
    dy, w_out = _whole(3, (m, width), dtype, device, 3), _whole(4, (hidden, width), dtype, device, 2) * 2.0 ** -6
    dgu = torch.full((m, 2 * hidden), 77.0, dtype=dtype, device=device)
    ws, nbytes = mlp._workspace(mlp._GATE_BACKWARD, m, hidden, width, device)
    _lib.run("flk_mlp_gate_backward", (dy, w_out, gu, dgu, ws), dy.data_ptr(), width, w_out.data_ptr(), width, gu.data_ptr(),
             mlp._dtype("x", x), m, width, hidden, dgu.data_ptr(), 2 * hidden, _lib.ptr(ws), nbytes, _lib.stream_of(x))
    _close("dgu", dgu, *_gate_case(want, _f64(dy) @ _f64(w_out).T)[1])


def _operands(seed, m, width, hidden, dtype, device):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(m, width, generator=g).to(dtype).to(device) for _ in range(2))
    w_in = (width ** -0.5 * torch.randn(width, 2 * hidden, generator=g)).to(dtype).to(device)
    w_out = (hidden ** -0.5 * torch.randn(hidden, width, generator=g)).to(dtype).to(device)
    return x, dy, w_in, w_out


def _mlp_case(x, dy, w_in, w_out, dtype):
    """{name: (value, tolerance before the output's rounding)} in float64, by the module docstring's count."""
    e = torch.finfo(dtype).eps / 2
    tiny = TINY[dtype]
    gu = x @ w_in
    gu_off = x.shape[1] * U * (np.abs(x) @ np.abs(w_in))
    half = gu.shape[1] // 2
    g, u = gu[:, :half], gu[:, half:]
    s, rest = M._sigmoid(g), M._sigmoid(-g)
    slope = np.abs(s * (1 + g * rest)) + gu_off[:, :half]      # silu's, which moves by at most half of gu_off
    silu = g * s
    (h, h_tol), _ = _gate_case(gu, np.zeros_like(g))
    h_off = h_tol + slope * gu_off[:, :half] * np.abs(u) + np.abs(silu) * gu_off[:, half:]
    h_all = h_off + e * (np.abs(h) + h_off) + tiny
    y = h @ w_out
    y_off = h_all @ np.abs(w_out) + hidden_sum(np.abs(h) + h_all, np.abs(w_out))
    dh = dy @ w_out.T
    dh_off = dy.shape[1] * U * (np.abs(dy) @ np.abs(w_out.T))
    _, (dgu, dgu_tol) = _gate_case(gu, dh)
    # how dg and du move with dh, g and u: |silu''| <= 0.5, |silu'| <= 1.1
    dg_off = dh_off * np.abs(u * s * (1 + g * rest)) + np.abs(dh) * (0.5 * np.abs(u) * gu_off[:, :half] + 1.1 * gu_off[:, half:])
    du_off = dh_off * np.abs(silu) + np.abs(dh) * 1.1 * gu_off[:, :half]
    off = dgu_tol + np.concatenate((dg_off, du_off), -1)
    d_all = off + e * (np.abs(dgu) + off) + tiny
    dx = dgu @ w_in.T
    dx_off = d_all @ np.abs(w_in.T) + hidden_sum(np.abs(dgu) + d_all, np.abs(w_in.T))
    dw_in = x.T @ dgu
    dwi_off = np.abs(x.T) @ d_all + hidden_sum(np.abs(x.T), np.abs(dgu) + d_all)
    dw_out = h.T @ dy
    dwo_off = h_all.T @ np.abs(dy) + hidden_sum((np.abs(h) + h_all).T, np.abs(dy))
    return {"y": (y, y_off), "dx": (dx, dx_off), "dw_in": (dw_in, dwi_off), "dw_out": (dw_out, dwo_off)}


def hidden_sum(a, b):
    """What float32 sums of the products' terms may be off by."""
    return a.shape[1] * U * (a @ b)


# Each product on each of its tiles (tests/test_mlp_host.py asserts which one a size takes): four row tiles, whose blocks
# touch their operands' lines ahead, five to seven, which sweep in two groups, and outputs that pass the caches by (past
# 80 MB; the gate's g and u); one stage of 64 terms, a ragged one after none, one and more whole stages.  The tokens'
# axis, inside in the fifth product, has any length.
SHORT, ODD = (64, 72, 136, 200, 328), (64, 71, 133, 200, 331)
TILES = [(product, tile, rows // 8 * 8 if product == mlp._MATMUL_AT else rows, cols, ODD if product == mlp._MATMUL_AT else inner)
         for product in (mlp._MATMUL, mlp._MATMUL_BT, mlp._MATMUL_AT, mlp._GATE_BACKWARD) for tile, rows, cols, inner in (
             ("256x256", 779, 12368, SHORT), ("256x256", 1547, 7600, SHORT), ("192x256", 779, 9352, SHORT),
             ("192x256", 8203, 928, SHORT), ("128x128 x2", 779, 4672, SHORT), ("128x128 deep", 1035, 304, SHORT))]
TILES += [(mlp._GATE, tile, rows, cols, SHORT) for tile, rows, cols in (
    ("256x256", 779, 6232), ("256x256", 1291, 4048), ("256x256", 267, 12368), ("192x256", 779, 4776), ("192x256", 1291, 3008),
    ("192x256", 267, 10912), ("128x128 x2", 779, 2384), ("128x128 deep", 779, 200))]
TILES += [(product, tile, rows, cols, (200,)) for product, tile, rows, cols in (
    (mlp._MATMUL, "256x256", 3347, 12576), (mlp._MATMUL_BT, "192x256", 3347, 13928), (mlp._MATMUL_AT, "256x256", 3344, 12576),
    (mlp._MATMUL_AT, "192x256", 3344, 13928), (mlp._GATE, "192x256", 2315, 4568), (mlp._GATE, "256x256", 779, 13512),
    (mlp._GATE, "256x256", 3347, 12576), (mlp._GATE_BACKWARD, "192x256", 2315, 4568), (mlp._GATE_BACKWARD, "256x256", 779, 13512),
    (mlp._GATE_BACKWARD, "128x128 x2", 1291, 10808))]
TILES += [(product, "128x128 deep split", 2072, 72, (1000,)) for product in range(5)]
TILES += [(product, "128x128 x2 split", 520, 2192, (4040,)) for product in range(1, 5)] + [(mlp._GATE, "128x128 x2 split", 267, 1832, (4040,))]
TILES += [(product, "128x32 split", 45, 200, (520,)) for product in range(4)]


def _inside(t):
    """t in the middle of a larger buffer of NaNs, rows 16-byte aligned."""
    wide = torch.full((t.shape[0] + 2, -(-t.shape[1] // 8) * 8 + 16), float("nan"), dtype=t.dtype, device=t.device)
    wide[1:-1, 8:8 + t.shape[1]] = t
    return wide[1:-1, 8:8 + t.shape[1]]


@pytest.mark.parametrize("product,tile,rows,cols,inners", TILES)
@pytest.mark.parametrize("dtype", BOTH)
def test_every_tile(device, product, tile, rows, cols, inners, dtype):
    """Whole numbers, whose sums are exact, inside NaNs that no result may hold.  The gate's g is at least 64, where
    1 + exp(-g) is 1: h = g u, dg = dh u and du = dh g in one float32 product each."""
    for inner in inners:
        print(f"product {product} {tile} rows={rows} cols={cols} inner={inner} {dtype}", flush=True)
        assert _lib.lib().flk_mlp_kernel(product, rows, cols, inner).decode() == tile
        ws, nbytes = mlp._workspace(product, rows, cols, inner, device)
        a = _inside(_whole(1, (rows, inner), dtype, device, 3))
        code, stream = mlp._dtype("a", a), _lib.stream_of(a)
        if product == mlp._GATE:
            a.abs_().add_(1.0)
            w = _inside(_whole(2, (inner, 2 * cols), dtype, device, 2))
            w[:, :cols].abs_().clamp_(1.0)
            w[:, cols:] *= 2.0 ** -10
            gu, h = torch.full((rows, 2 * cols), 77.0, device=device), _inside(torch.full((rows, cols), 77.0, dtype=dtype, device=device))
            want = (a.double() @ w.double()).float()
            for kept in (gu, None):
                h.fill_(77.0)
                _lib.run("flk_mlp_gate", (a, w, h, kept, ws), a.data_ptr(), a.stride(0), w.data_ptr(), w.stride(0), code, rows, inner,
                         cols, h.data_ptr(), h.stride(0), _lib.ptr(kept), _lib.ptr(ws), nbytes, stream)
                assert torch.equal(h, (want[:, :cols] * want[:, cols:]).to(dtype))
            assert torch.equal(gu, want)
            continue
        b = _inside(_whole(2, (cols, inner), dtype, device, 3))
        exact = (a.double() @ b.double().t()).float()
        if product == mlp._GATE_BACKWARD:
            g = torch.Generator(device).manual_seed(3)
            gu = torch.randn(rows, 2 * cols, generator=g, device=device)
            gu[:, :cols].abs_().add_(64.0)
            d = _inside(torch.full((rows, 2 * cols), 77.0, dtype=dtype, device=device))
            _lib.run("flk_mlp_gate_backward", (a, b, gu, d, ws), a.data_ptr(), a.stride(0), b.data_ptr(), b.stride(0), gu.data_ptr(),
                     code, rows, inner, cols, d.data_ptr(), d.stride(0), _lib.ptr(ws), nbytes, stream)
            assert torch.equal(d[:, :cols], (exact * gu[:, cols:]).to(dtype)) and torch.equal(d[:, cols:], (exact * gu[:, :cols]).to(dtype))
        else:
            d = _inside(torch.full((rows, cols), 77.0, dtype=dtype, device=device))
            a_t, b_t = product == mlp._MATMUL_AT, product == mlp._MATMUL_BT
            mlp._matmul(_inside(a.t()) if a_t else a, b if b_t else _inside(b.t()), d, a_t=a_t, b_t=b_t)
            assert torch.equal(d, exact.to(dtype))
        wide = d._base
        wide[1:-1, 8:8 + d.shape[1]] = float("nan")
        assert bool(wide.isnan().all())   # nothing beside the output is written


@pytest.mark.parametrize("dtype", BOTH)
def test_gate_on_large_tiles(device, dtype):
    """The gate and its gradients of ordinary values on 256 x 256 tiles, at the first and last rows."""
    rows, inner = 1291, 136
    for cols, scale in ((4048, 2.0 ** -6), (8104, 2.0 ** -6)):
        print(f"gate m={rows} width={inner} hidden={cols} {dtype}", flush=True)
        pick = torch.cat((torch.arange(20), torch.arange(rows - 20, rows))).to(device)
        x, w = _whole(1, (rows, inner), dtype, device, 3), _whole(2, (inner, 2 * cols), dtype, device, 1) * scale
        gu, h = torch.empty(rows, 2 * cols, device=device), torch.empty(rows, cols, dtype=dtype, device=device)
        _lib.run("flk_mlp_gate", (x, w, h, gu), x.data_ptr(), inner, w.data_ptr(), 2 * cols, mlp._dtype("x", x), rows, inner, cols,
                 h.data_ptr(), cols, gu.data_ptr(), None, 0, _lib.stream_of(x))
        want = _f64(x[pick]) @ _f64(w)
        assert np.array_equal(_f64(gu[pick]), want)
        _close("h", h[pick], *_gate_case(want, np.zeros((len(pick), cols)))[0])
        dy, w_out = _whole(3, (rows, inner), dtype, device, 3), _whole(4, (cols, inner), dtype, device, 2) * 2.0 ** -6
        dgu = torch.empty(rows, 2 * cols, dtype=dtype, device=device)
        _lib.run("flk_mlp_gate_backward", (dy, w_out, gu, dgu), dy.data_ptr(), inner, w_out.data_ptr(), inner, gu.data_ptr(),
                 mlp._dtype("x", x), rows, inner, cols, dgu.data_ptr(), 2 * cols, None, 0, _lib.stream_of(x))
        _close("dgu", dgu[pick], *_gate_case(want, _f64(dy[pick]) @ _f64(w_out).T)[1])


@pytest.mark.parametrize("m,width,hidden", [(1, 64, 64), (1, 512, 1536), (5, 256, 264), (24, 136, 320), (77, 512, 512),
                                            (200, 72, 136), (512, 256, 768), (1000, 200, 424)])
@pytest.mark.parametrize("dtype", BOTH)
def test_gated_mlp(device, m, width, hidden, dtype):
    print(f"gated_mlp m={m} width={width} hidden={hidden} {dtype}", flush=True)
    x, dy, w_in, w_out = _operands(m, m, width, hidden, dtype, device)
    want = _mlp_case(*map(_f64, (x, dy, w_in, w_out)), dtype)
    plain = mlp.gated_mlp(x, w_in, w_out)
    y, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    assert torch.equal(plain, y)
    got = dict(zip(("y", "dx", "dw_in", "dw_out"), (y, *mlp.gated_mlp_backward(dy, x, w_in, w_out, kept))))
    again = mlp.gated_mlp_backward(dy, x, w_in, w_out, kept)
    for name, value in got.items():
        _close(name, value, *want[name])
        # The terms' roundings are independent, so their sum's size is that of one rounding of each term:
        # about e / sqrt(3) of the output's norm from each of at most two (the inner and the output's), e in all
        off = np.linalg.norm(_f64(value) - want[name][0]) / np.linalg.norm(want[name][0])
        assert off < 1.5 * torch.finfo(dtype).eps / 2, (name, off)
    assert all(torch.equal(a, b) for a, b in zip(again, (got["dx"], got["dw_in"], got["dw_out"])))


@pytest.mark.parametrize("m,width,hidden", [(1, 256, 768), (77, 512, 136), (1291, 136, 4048)])
@pytest.mark.parametrize("dtype", BOTH)
def test_nothing_but_h_and_dgu_is_rounded_between_the_products(device, m, width, hidden, dtype):
    """y from the h that the call keeps, and the gradients from that h and dgu, are off by their float32 sums and
    their own rounding only."""
    print(f"gated_mlp m={m} width={width} hidden={hidden} {dtype}", flush=True)
    x, dy, w_in, w_out = _operands(m, m, width, hidden, dtype, device)
    y, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    dgu = torch.empty(m, 2 * hidden, dtype=dtype, device=device)
    ws, nbytes = mlp._workspace(mlp._GATE_BACKWARD, m, hidden, width, device)
    _lib.run("flk_mlp_gate_backward", (dy, w_out, kept.gu, dgu, ws), dy.data_ptr(), width, w_out.data_ptr(), width,
             kept.gu.data_ptr(), mlp._dtype("x", x), m, width, hidden, dgu.data_ptr(), 2 * hidden, _lib.ptr(ws), nbytes,
             _lib.stream_of(x))
    h, d, wi, wo, xs, g = map(_f64, (kept.h, dgu, w_in, w_out, x, dy))
    dx, dw_in, dw_out = mlp.gated_mlp_backward(dy, x, w_in, w_out, kept)
    for name, got, a, b in (("y", y, h, wo), ("dx", dx, d, wi.T), ("dw_in", dw_in, xs.T, d), ("dw_out", dw_out, h.T, g)):
        _close(name, got, a @ b, hidden_sum(np.abs(a), np.abs(b)))


def test_gated_mlp_shapes_and_views(device):
    """Batches, one token, rows of a wider buffer, weights inside wider ones, and the operands' gradients' shapes."""
    x, dy, w_in, w_out = _operands(3, 42, 64, 72, torch.bfloat16, device)
    want, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    grads = mlp.gated_mlp_backward(dy, x, w_in, w_out, kept)
    y3, kept3 = mlp.gated_mlp(x.view(2, 21, 64), w_in, w_out, keep=True)
    assert torch.equal(y3, want.view(2, 21, 64))
    got = mlp.gated_mlp_backward(dy.view(2, 21, 64), x.view(2, 21, 64), w_in, w_out, kept3)
    assert got[0].shape == (2, 21, 64) and all(torch.equal(a.reshape(-1), b.reshape(-1)) for a, b in zip(got, grads))
    wide = torch.full((42, 80), float("nan"), dtype=torch.bfloat16, device=device)
    wide[:, 8:72] = x
    ww = torch.full((64, 160), float("nan"), dtype=torch.bfloat16, device=device)
    ww[:, 8:152] = w_in
    out = torch.empty_like(x)
    assert mlp.gated_mlp(wide[:, 8:72], ww[:, 8:152], w_out, out=out) is out and torch.equal(out, want)
    assert torch.equal(mlp.gated_mlp(x.t().contiguous().t(), w_in, w_out.t().contiguous().t()), want)
    odd = torch.zeros(42, 65, dtype=torch.bfloat16, device=device)
    odd[:, 1:] = x
    assert torch.equal(mlp.gated_mlp(odd[:, 1:], w_in, w_out), want)   # rows that are not 16-byte aligned
    same = x.clone()
    assert torch.equal(mlp.gated_mlp(same, w_in, w_out, out=same), want)
    assert torch.equal(mlp.gated_mlp_backward(dy[:1].expand(42, 64), x, w_in, w_out, kept)[0],
                       mlp.gated_mlp_backward(dy[:1].repeat(42, 1), x, w_in, w_out, kept)[0])
    none = x[:0]
    y, kept = mlp.gated_mlp(none, w_in, w_out, keep=True)
    dx, dwi, dwo = mlp.gated_mlp_backward(none, none, w_in, w_out, kept)
    assert y.shape == dx.shape == (0, 64) and not dwi.any() and not dwo.any() and dwi.shape == w_in.shape
    assert torch.equal(mlp.gated_mlp(x[0], w_in, w_out), mlp.gated_mlp(x[:1], w_in, w_out)[0])


def test_rows_far_apart(device):
    """Each image's first token in place, whose rows are more than 2^22 elements apart."""
    x, dy, w_in, w_out = _operands(11, 3, 64, 72, torch.bfloat16, device)
    long = torch.zeros(2, 3, 2 ** 16 + 1, 64, dtype=torch.bfloat16, device=device)
    far_x, far_dy = long[0, :, 0], long[1, :, 0]
    far_x.copy_(x)
    far_dy.copy_(dy)
    want, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    y, far_kept = mlp.gated_mlp(far_x, w_in, w_out, keep=True)
    assert torch.equal(y, want)
    for got, exact in zip(mlp.gated_mlp_backward(far_dy, far_x, w_in, w_out, far_kept),
                          mlp.gated_mlp_backward(dy, x, w_in, w_out, kept)):
        assert torch.equal(got, exact)


def test_offsets_past_32_bits(device):
    """The last tokens of a call whose g and u hold more than 2^31 values, on whole numbers (g and u exact)."""
    m, width, hidden, last = 2 ** 17 + 300, 64, 8192 + 8, 300
    x, w_in = _whole(1, (last, width), torch.bfloat16, device, 3), _whole(2, (width, 2 * hidden), torch.bfloat16, device, 1) * 2.0 ** -4
    w_out, dy = _whole(3, (hidden, width), torch.bfloat16, device, 1) * 2.0 ** -6, _whole(4, (last, width), torch.bfloat16, device, 3)
    big_x, big_dy = (torch.zeros(m, width, dtype=torch.bfloat16, device=device) for _ in range(2))
    big_x[-last:], big_dy[-last:] = x, dy
    y, kept = mlp.gated_mlp(big_x, w_in, w_out, keep=True)
    want_y, want = mlp.gated_mlp(x, w_in, w_out, keep=True)
    assert torch.equal(kept.gu[-last:], want.gu) and torch.equal(kept.h[-last:], want.h) and not kept.gu[:-last].any()
    got = mlp.gated_mlp_backward(big_dy, big_x, w_in, w_out, kept)
    exact = _mlp_case(*map(_f64, (x, dy, w_in, w_out)), torch.bfloat16)
    assert not y[:-last].any() and not got[0][:-last].any()
    for name, value in (("y", y[-last:]), ("dx", got[0][-last:]), ("dw_in", got[1]), ("dw_out", got[2])):
        _close(name, value, *exact[name])


def test_more_tokens_than_small_tiles(device):
    """Tokens for more than 2^22 tiles of 128 rows, on whole numbers: the first and the last are those of a short call."""
    m, part = (1 << 29) + 136, 300
    x, w_in = _whole(1, (part, 8), torch.bfloat16, device, 3), _whole(2, (8, 16), torch.bfloat16, device, 1) * 2.0 ** -2
    w_out = _whole(3, (8, 8), torch.bfloat16, device, 1)
    long = torch.zeros(m, 8, dtype=torch.bfloat16, device=device)
    long[:part], long[-part:] = x, x
    want = mlp.gated_mlp(x, w_in, w_out)
    print(f"gated_mlp m={m}", flush=True)
    y = mlp.gated_mlp(long, w_in, w_out)
    assert torch.equal(y[:part], want) and torch.equal(y[-part:], want)
    assert not any(bool(rest.any()) for rest in y[part:-part].split(1 << 26))


def test_range_between_the_products(device):
    """h and dgu have the operands' type's range: in float16 h = 300 * 300 is infinite, and du = 2^-27 silu(1) zero."""
    def one(value, dtype):
        t = torch.zeros(1, 8, dtype=dtype, device=device)
        t[0, 0] = value
        return t
    for dtype, y, zero in ((torch.bfloat16, 90112.0, False), (torch.float16, float("inf"), True)):
        w_in, w_out = torch.zeros(8, 16, dtype=dtype, device=device), torch.eye(8, dtype=dtype, device=device)
        w_in[0, 0] = w_in[0, 8] = 1.0
        assert mlp.gated_mlp(one(300.0, dtype), w_in, w_out)[0, 0] == y   # 90000 to 8 bits: 176 * 512
        x, dy = one(1.0, dtype), one(2.0 ** -13, dtype)
        _, kept = mlp.gated_mlp(x, w_in, w_out * 2.0 ** -14, keep=True)
        dx, dw_in, _ = mlp.gated_mlp_backward(dy, x, w_in, w_out * 2.0 ** -14, kept)
        assert bool((dw_in == 0).all()) == bool((dx == 0).all()) == zero


def test_gated_mlp_not_finite(device):
    """A token's not-finite value stays in its row of y and dx, whatever rows share its tile."""
    x, dy, w_in, w_out = _operands(5, 40, 64, 64, torch.bfloat16, device)
    clean, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    dx = mlp.gated_mlp_backward(dy, x, w_in, w_out, kept)[0]
    bad = x.clone()
    bad[17, 3] = float("nan")
    got, kept = mlp.gated_mlp(bad, w_in, w_out, keep=True)
    rest = [i for i in range(40) if i != 17]
    assert got[17].isnan().all() and torch.equal(got[rest], clean[rest])
    got = mlp.gated_mlp_backward(dy, bad, w_in, w_out, kept)
    assert got[0][17].isnan().all() and torch.equal(got[0][rest], dx[rest])
    assert got[1].isnan().any()


@pytest.mark.parametrize("wanted", [(True, False, False), (False, True, False), (False, False, True), (True, True, False),
                                    (False, False, False)])
def test_gated_mlp_wanted_gradients(device, wanted):
    x, dy, w_in, w_out = _operands(6, 50, 64, 72, torch.bfloat16, device)
    _, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    every = mlp.gated_mlp_backward(dy, x, w_in, w_out, kept)
    for got, want, asked in zip(mlp.gated_mlp_backward(dy, x, w_in, w_out, kept, wanted=wanted), every, wanted, strict=True):
        assert torch.equal(got, want) if asked else got is None
    none = mlp.gated_mlp_backward(dy[:0], x[:0], w_in, w_out, mlp.Kept(kept.h[:0], kept.gu[:0]), wanted=wanted)
    assert [t is not None for t in none] == list(wanted) and not any(t.any() for t in none if t is not None)
    leaves = [t.clone().requires_grad_(a) for t, a in zip((x, w_in, w_out), wanted)]
    if any(wanted):
        autograd.gated_mlp(*leaves).backward(dy)
        for leaf, want, asked in zip(leaves, every, wanted):
            assert torch.equal(leaf.grad, want) if asked else leaf.grad is None


def test_gated_mlp_refusals(device):
    x, dy, w_in, w_out = _operands(1, 4, 64, 72, torch.bfloat16, device)
    with pytest.raises(TypeError, match="bfloat16 or float16"):
        mlp.gated_mlp(x.float(), w_in.float(), w_out.float())
    with pytest.raises(TypeError, match="like x"):
        mlp.gated_mlp(x, w_in.half(), w_out)
    with pytest.raises(ValueError, match="w_in must be"):
        mlp.gated_mlp(x, w_in[:, :72], w_out)
    with pytest.raises(ValueError, match="takes x"):
        mlp.gated_mlp(x, w_in[None], w_out)
    with pytest.raises(ValueError, match="multiples of 8"):
        mlp.gated_mlp(x[:, :60], w_in[:60], w_out[:, :60])
    with pytest.raises(ValueError, match="out must be"):
        mlp.gated_mlp(x, w_in, w_out, out=x[:2])
    with pytest.raises(ValueError, match="contiguous"):
        mlp.gated_mlp(x, w_in, w_out, out=torch.zeros(4, 128, dtype=x.dtype, device=device)[:, :64])
    _, kept = mlp.gated_mlp(x, w_in, w_out, keep=True)
    with pytest.raises(ValueError, match="dy must be"):
        mlp.gated_mlp_backward(dy[:2], x, w_in, w_out, kept)
    with pytest.raises(TypeError, match="like x"):
        mlp.gated_mlp_backward(dy.half(), x, w_in, w_out, kept)
    with pytest.raises(ValueError, match="kept.gu"):
        mlp.gated_mlp_backward(dy, x, w_in, w_out, kept._replace(gu=kept.gu[:2]))
    with pytest.raises(ValueError, match="kept.h"):
        mlp.gated_mlp_backward(dy, x, w_in, w_out, kept._replace(h=kept.h.float()))


def test_autograd_mlp_section(device):
    """modules.mlp_section (modulate, then the MLP) as a program trains it: its gradients are the explicit calls'."""
    g = torch.Generator().manual_seed(8)
    x = torch.randn(2, 21, 64, generator=g).to(torch.bfloat16).to(device).requires_grad_()
    shift, scale = (0.3 * torch.randn(2, 1, 64, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    shift.requires_grad_()
    scale.requires_grad_()
    _, dy, w_in, w_out = _operands(9, 42, 64, 72, torch.bfloat16, device)
    w_in.requires_grad_()
    w_out.requires_grad_()
    y = autograd.gated_mlp(autograd.modulate(x, shift, scale), w_in, w_out)
    assert torch.equal(y, modules.mlp_section(x.detach(), shift.detach(), scale.detach(), w_in.detach(), w_out.detach()))
    y.backward(dy.view(2, 21, 64))
    with torch.no_grad():
        mod = norm.modulate(x, shift, scale)
        _, kept = mlp.gated_mlp(mod, w_in, w_out, keep=True)
        dmod, dwi, dwo = mlp.gated_mlp_backward(dy.view(2, 21, 64), mod, w_in, w_out, kept)
        dx, dshift, dscale = norm.modulate_backward(dmod, x, shift, scale)
        assert not autograd.gated_mlp(mod, w_in, w_out).requires_grad
    for got, want in zip((x.grad, shift.grad, scale.grad, w_in.grad, w_out.grad), (dx, dshift, dscale, dwi, dwo)):
        assert torch.equal(got, want)


def _section(x, shift, scale, w_in, w_out, dy):
    mod = norm.modulate(x, shift, scale)
    y, kept = mlp.gated_mlp(mod, w_in, w_out, keep=True)
    dmod, dwi, dwo = mlp.gated_mlp_backward(dy, mod, w_in, w_out, kept)
    return y, dwi, dwo, *norm.modulate_backward(dmod, x, shift, scale)


def _section_inputs(seed, device, m=300):
    g = torch.Generator().manual_seed(seed)
    x, dy = (torch.randn(2, m, 64, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    shift, scale = (0.3 * torch.randn(2, 64, generator=g).to(torch.bfloat16).to(device) for _ in range(2))
    _, _, w_in, w_out = _operands(seed, 1, 64, 136, torch.bfloat16, device)
    return [x, shift, scale, w_in, w_out, dy]


@pytest.mark.parametrize("m", [1, 300])
def test_section_forward_and_backward_in_a_graph(device, m):
    """The explicit calls captured, two graphs of them replayed in turn with new inputs and eager work between: each
    replay equals the eager result of its inputs, and its workspaces are its own."""
    graphs = []
    for seed in (1, 2):
        static = _section_inputs(seed, device, m)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _section(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = _section(*static)
        graphs.append((graph, static, outs))
    for round_ in range(3):
        for i, (graph, static, outs) in enumerate(graphs):
            print(f"replay m={m} graph {i} round {round_}", flush=True)
            fresh = _section_inputs(10 + 2 * round_ + i, device, m)
            for dst, src in zip(static, fresh):
                dst.copy_(src)
            graph.replay()
        for graph, static, outs in graphs:
            want = _section(*[t.clone() for t in static])
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_side_stream(device):
    ins = _section_inputs(4, device)
    want = _section(*ins)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _section(*ins)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_autograd_refuses_capture_with_gradients(device):
    """Before anything is launched: the capture goes on and ends as it would have."""
    w = torch.ones(64, device=device, requires_grad=True)
    x = torch.randn(3, 64, device=device)
    norm.layer_norm(x, w.detach())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="explicit"):
            autograd.layer_norm(x, w)
        with torch.no_grad():
            out = autograd.layer_norm(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, norm.layer_norm(x, w.detach()))


@pytest.mark.parametrize("dtype", BOTH)
@pytest.mark.parametrize("m,width,hidden", [(1, 256, 264), (77, 72, 136), (600, 64, 64)])
def test_native_path_equals_the_python_path(device, monkeypatch, dtype, m, width, hidden):
    """Plain calls take the native path, and have the Python path's values, shapes and types."""
    x, dy, w_in, w_out = _operands(m, m, width, hidden, dtype, device)
    wide = torch.zeros(hidden, width + 8, dtype=dtype, device=device)
    wide[:, :width] = w_out
    w_out = wide[:, :width]
    x3, dy3 = x.view(1, m, width), dy.view(1, m, width)
    taken = mlp._native.gated_mlp(x3, w_in, w_out, True)
    assert taken is not None and mlp._native.gated_mlp(x3, w_in, w_out, False)[1:] == (None, None)
    assert mlp._native.gated_mlp_backward(dy3, x3, w_in, w_out, *taken[1:]) is not None
    y, kept = mlp.gated_mlp(x3, w_in, w_out, keep=True)
    got = (y, *kept, mlp.gated_mlp(x3, w_in, w_out), *mlp.gated_mlp_backward(dy3, x3, w_in, w_out, kept))
    monkeypatch.setattr(mlp, "_native", Declines())
    y, kept = mlp.gated_mlp(x3, w_in, w_out, keep=True)
    want = (y, *kept, mlp.gated_mlp(x3, w_in, w_out), *mlp.gated_mlp_backward(dy3, x3, w_in, w_out, kept))
    for a, b in zip(got, want, strict=True):
        assert a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous() and torch.equal(a, b)
