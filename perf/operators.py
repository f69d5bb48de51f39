"""The norm and MLP operators of the DiT blocks as programs call them, over the sizes they meet.

A Klein 4B block normalises its input, scales and shifts it by rows that belong to the image
(``modulate``), projects it, and adds the result back; its MLP is gated: one projection to twice
the MLP width, silu of the first half times the second, and a projection back.  Double blocks
run the whole MLP over each stream; single blocks project QKV and both MLP halves at once, so
there the gate reads its halves in place from the wide output.  Programs that fine-tune run
each of them backwards too.

A case is one such call:

  kind     what                                                         sizes
  modulate (1 + scale) * layer_norm(x) + shift, a row of each per image batch, tokens, width
  norm     layer_norm(x) * weight + bias                                batch, tokens, width
  swiglu   silu(g) * u of a view [g | u] into a wider row               batch, tokens, hidden, before
  mlp      (silu(x Wg) * (x Wu)) Wout                                   batch, tokens, width, hidden

``step`` is "forward", "backward" (the gradients of one incoming gradient), or for the mlp
"train": the forward pass and its gradients.  ``params`` is the type of scale, shift, weight and
bias.  The rows of the image grids are 16 pixels: 1024 pixels are 64 x 64 tokens.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
WIDTH, HIDDEN = 24 * 128, 3 * 24 * 128    # Klein 4B: hidden width, MLP width
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, kind, step, dtype, batch, tokens, **sizes):
    case = {"kind": kind, "step": step, "dtype": dtype, "batch": batch, "tokens": tokens, **sizes}
    return {"name": name, **case} if name else case


def listed():
    return [
        # The text stream's modulated norm: the smallest call of a block, where the launch counts.
        _case("modulate_text", "modulate", "forward", "bf16", 1, 512, width=WIDTH, params="bf16"),
        # Four 1024-pixel images through the same norm, each with its own rows.
        _case("modulate_1024px_b4", "modulate", "forward", "bf16", 4, 4096, width=WIDTH, params="bf16"),
        # Its gradients for one 1024-pixel image: dx, and both rows summed over 4608 tokens.
        _case("modulate_grad_1024px", "modulate", "backward", "bf16", 1, 4608, width=WIDTH, params="bf16"),
        # An affine norm with float32 activations of an odd width: no row is aligned.
        _case("norm_grad_odd_fp32", "norm", "backward", "fp32", 3, 1157, width=1111, params="fp32"),
        # A single block's gate at 1024 pixels, read in place behind the 9216 QKV columns.
        _case("swiglu_single_1024px", "swiglu", "forward", "bf16", 1, 4608, hidden=HIDDEN, before=3 * WIDTH),
        # Its gradient for two images of 1008 x 752 pixels with their text.
        _case("swiglu_grad_ragged", "swiglu", "backward", "bf16", 2, 3473, hidden=HIDDEN, before=3 * WIDTH),
        # One token through the MLP: the weights' bytes are all there is.
        _case("mlp_token", "mlp", "forward", "bf16", 1, 1, width=WIDTH, hidden=HIDDEN),
        # The text stream's MLP, and the image stream's at 1024 pixels.
        _case("mlp_text", "mlp", "forward", "bf16", 1, 512, width=WIDTH, hidden=HIDDEN),
        _case("mlp_1024px", "mlp", "forward", "bf16", 1, 4096, width=WIDTH, hidden=HIDDEN),
        # Fine-tuning: forward and gradients at 1024 pixels.
        _case("mlp_train_1024px", "mlp", "train", "bf16", 1, 4096, width=WIDTH, hidden=HIDDEN),
        # A narrower MLP in half precision, with sizes that no tile divides.
        _case("mlp_train_ragged_fp16", "mlp", "train", "fp16", 3, 987, width=1000, hidden=2728),
        # The largest: a 2048-pixel image's training step.
        _case("mlp_train_2048px", "mlp", "train", "bf16", 1, 16384, width=WIDTH, hidden=HIDDEN),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("modulate", "norm", "swiglu", "mlp", "mlp"))
    batch = rng.choice((1, 1, 1, 2, 3, 4))
    if kind == "mlp":
        step, dtype = rng.choice(("forward", "train")), rng.choice(("bf16", "bf16", "fp16"))
        tokens = _log_int(rng, 1, 16384 // batch)
        # widths are multiples of 8 elements: 16-byte rows
        width = 8 * _log_int(rng, 8, WIDTH // 8)
        hidden = 8 * _log_int(rng, max(8, width // 8), min(HIDDEN, 4 * width) // 8)
        return _case(None, kind, step, dtype, batch, tokens, width=width, hidden=hidden)
    step, dtype = rng.choice(("forward", "backward")), rng.choice(("bf16", "bf16", "fp16", "fp32"))
    tokens = _log_int(rng, 1, 16384 // batch)
    if kind == "swiglu":
        return _case(None, kind, step, dtype, batch, tokens, hidden=_log_int(rng, 8, HIDDEN),
                     before=rng.choice((0, 3 * WIDTH, rng.randrange(1, 3 * WIDTH))))
    return _case(None, kind, step, dtype, batch, tokens, width=_log_int(rng, 16, 8192),
                 params=rng.choice((dtype, "fp32")))


def work(case):
    rows, size = case["batch"] * case["tokens"], TYPES[case["dtype"]].itemsize
    forward = case["step"] == "forward"
    if case["kind"] == "swiglu":
        values = rows * case["hidden"]
        return {"bytes": (3 if forward else 5) * values * size, "flops": (6 if forward else 14) * values}
    width = case["width"]
    if case["kind"] == "mlp":
        weights, acts = 3 * width * case["hidden"] * size, rows * width * size
        flops = 2 * rows * 3 * width * case["hidden"]
        if forward:
            return {"bytes": weights + 2 * acts, "flops": flops}
        return {"bytes": 2 * weights + 4 * acts, "flops": 3 * flops}
    params = (case["batch"] if case["kind"] == "modulate" else 1) * width * TYPES[case["params"]].itemsize
    values = rows * width
    if forward:
        return {"bytes": 2 * values * size + 2 * params, "flops": 8 * values}
    return {"bytes": 3 * values * size + 3 * params, "flops": 18 * values}


def _random(gen, shape, dtype, scale=1.0):
    return (scale * torch.randn(shape, generator=gen, device="cuda")).to(dtype)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, batch, tokens = TYPES[case["dtype"]], case["batch"], case["tokens"]
    state = {"kind": case["kind"], "step": case["step"]}
    if case["kind"] == "swiglu":
        hidden, before = case["hidden"], case["before"]
        wide = _random(gen, (batch, tokens, before + 2 * hidden), dtype)
        state["gu"] = wide[..., before:]
        state["dh"] = _random(gen, (batch, tokens, hidden), dtype)
        return state
    width = case["width"]
    if case["kind"] == "mlp":
        hidden = case["hidden"]
        # a modulated norm's output, weights that keep its variance, a gradient of unit size
        state["x"] = _random(gen, (batch, tokens, width), dtype)
        state["w_in"] = _random(gen, (width, 2 * hidden), dtype, width ** -0.5)
        state["w_out"] = _random(gen, (hidden, width), dtype, hidden ** -0.5)
        state["dy"] = _random(gen, (batch, tokens, width), dtype)
        return state
    # a residual stream: tokens of different size, each off zero, one channel in a hundred large
    x = torch.randn((batch, tokens, width), generator=gen, device="cuda")
    x = x * torch.exp(0.5 * torch.randn((batch, tokens, 1), generator=gen, device="cuda"))
    x = x * torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    state["x"] = (x + 0.3 * torch.randn((batch, tokens, 1), generator=gen, device="cuda")).to(dtype)
    state["dy"] = _random(gen, (batch, tokens, width), dtype)
    params, rows = TYPES[case["params"]], (batch, 1, width) if case["kind"] == "modulate" else (width,)
    if case["kind"] == "modulate":
        state["shift"], state["scale"] = _random(gen, rows, params, 0.5), _random(gen, rows, params, 0.5)
    else:
        state["weight"] = (1 + 0.2 * torch.randn(rows, generator=gen, device="cuda")).to(params)
        state["bias"] = _random(gen, rows, params, 0.2)
    return state


def _normalised(x):
    centred = x - x.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + EPS)
    return centred * rstd, rstd


def _norm_grads(dy, x, factor, over):
    """Gradients of normalised(x) * factor + offset: of x, of the factor, of the offset."""
    normed, rstd = _normalised(x)
    t = dy * factor
    dx = rstd * (t - t.mean(-1, keepdim=True) - normed * (t * normed).mean(-1, keepdim=True))
    return dx, (dy * normed).sum(over), dy.sum(over)


def _gate(g, u):
    return g / (1 + torch.exp(-g)) * u


def _gate_grads(dh, g, u):
    s = 1 / (1 + torch.exp(-g))
    return torch.cat((dh * u * s * (1 + g * (1 - s)), dh * g * s), -1)


def _plain(s):
    """The operators in float32, each output rounded once."""
    forward = s["step"] == "forward"
    if s["kind"] == "swiglu":
        g, u = s["gu"].float().chunk(2, -1)
        out = _gate(g, u) if forward else _gate_grads(s["dh"].float(), g, u)
        return out.to(s["gu"].dtype)
    x = s["x"].float()
    if s["kind"] == "mlp":
        w_in, w_out = s["w_in"].float(), s["w_out"].float()
        flat = x.reshape(-1, x.shape[-1])
        gu = flat @ w_in
        g, u = gu.chunk(2, -1)
        h = _gate(g, u)
        y = (h @ w_out).to(s["x"].dtype).view(s["x"].shape)
        if forward:
            return y
        dy = s["dy"].float().reshape(flat.shape)
        dgu = _gate_grads(dy @ w_out.t(), g, u)
        dx = (dgu @ w_in.t()).to(s["x"].dtype).view(s["x"].shape)
        return y, dx, (flat.t() @ dgu).to(s["w_in"].dtype), (h.t() @ dy).to(s["w_out"].dtype)
    if s["kind"] == "modulate":
        factor, offset, over = 1 + s["scale"].float(), s["shift"].float(), 1
        params, rows = s["scale"].dtype, s["scale"].shape
    else:
        factor, offset, over = s["weight"].float(), s["bias"].float(), (0, 1)
        params, rows = s["weight"].dtype, s["weight"].shape
    if forward:
        return (_normalised(x)[0] * factor + offset).to(s["x"].dtype)
    dx, dfactor, doffset = _norm_grads(s["dy"].float(), x, factor, over)
    return dx.to(s["x"].dtype), dfactor.to(params).view(rows), doffset.to(params).view(rows)


def _framework(s):
    from flicker_amd import mlp, norm

    forward = s["step"] == "forward"
    if s["kind"] == "swiglu":
        return mlp.swiglu(s["gu"]) if forward else mlp.swiglu_backward(s["dh"], s["gu"])
    if s["kind"] == "mlp":
        if forward:
            return mlp.gated_mlp(s["x"], s["w_in"], s["w_out"])
        y, kept = mlp.gated_mlp(s["x"], s["w_in"], s["w_out"], keep=True)
        return (y, *mlp.gated_mlp_backward(s["dy"], s["x"], s["w_in"], s["w_out"], kept))
    if s["kind"] == "modulate":
        if forward:
            return norm.modulate(s["x"], s["shift"], s["scale"])
        dx, dshift, dscale = norm.modulate_backward(s["dy"], s["x"], s["shift"], s["scale"])
        return dx, dscale, dshift
    if forward:
        return norm.layer_norm(s["x"], s["weight"], s["bias"])
    return norm.layer_norm_backward(s["dy"], s["x"], s["weight"], s["bias"])


def run(state):
    return _framework(state) if own else _plain(state)


def exact(case, seed):
    """What run() returns, from the definitions in float64; gradients by differentiating the
    forward definition rather than from the formulas that the plain form uses."""
    s = prepare(case, seed)
    leaves = {k: v.double().requires_grad_() for k, v in s.items() if isinstance(v, torch.Tensor)}
    if s["kind"] == "swiglu":
        half = s["gu"].shape[-1] // 2
        out = leaves["gu"][..., :half] * torch.sigmoid(leaves["gu"][..., :half]) * leaves["gu"][..., half:]
        wanted, incoming = ("gu",), "dh"
    elif s["kind"] == "mlp":
        proj = torch.matmul(leaves["x"], leaves["w_in"])
        half = proj.shape[-1] // 2
        out = torch.matmul(proj[..., :half] * torch.sigmoid(proj[..., :half]) * proj[..., half:], leaves["w_out"])
        wanted, incoming = ("x", "w_in", "w_out"), "dy"
    else:
        x = leaves["x"]
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        out = (x - mean) * torch.rsqrt(var + EPS)
        if s["kind"] == "modulate":
            out, wanted = (1 + leaves["scale"]) * out + leaves["shift"], ("x", "scale", "shift")
        else:
            out, wanted = leaves["weight"] * out + leaves["bias"], ("x", "weight", "bias")
        incoming = "dy"
    if s["step"] == "forward":
        return out.detach()
    grads = torch.autograd.grad(out, [leaves[k] for k in wanted], leaves[incoming].detach())
    if s["step"] == "train":
        return (out.detach(), *grads)
    return grads[0] if s["kind"] == "swiglu" else tuple(grads)
