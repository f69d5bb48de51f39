"""The operators that training a DiT block's attention half adds, as programs call them.

A block prepares q, k and v from its projection (qk_prep: head split, RMS norm, rotation), attends, projects,
adds the result to its residual stream through a gate and normalises the sum for what comes next.  To
fine-tune it each of these has to run backwards; attention then keeps its rows' log-sum-exp, and a batch
whose prompts differ in length leaves their padding out with a mask over the keys.

A case is one such call:

  kind       what                                                             sizes
  attention  softmax(q k^T) v over the keys that the mask keeps; q is scaled  batch, heads, kv_heads, queries, keys
  qk_prep    the gradients of qk_prep: of the projection and of both scales   batch, tokens, heads, before
  residual   r = x + gate * branch, y = (1 + scale) * layer_norm(r) + shift   batch, tokens, width

``step`` is "forward", "backward" (the gradients of the incoming ones), or for attention "train": the
forward pass and its gradients.  ``mask`` says which keys are kept: "all"; "padding", where the first
``text`` keys belong to a prompt that ends before them; "random", seven in ten; "empty", as "padding" with
nothing at all kept of the last batch entry.  ``layout`` is "heads" for (B, H, L, D) in memory, "tokens"
for views of (B, L, H, D).  ``params`` is the type of the scales, gates and shifts.
"""

from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
HEADS, DIM = 24, 128                  # Klein 4B: heads and their width
WIDTH = HEADS * DIM
TEXT = 512                            # text tokens ahead of the image's in the joint sequence
LONGEST = TEXT + 128 * 128            # a 2048-pixel image with its text
MOST_PAIRS = HEADS * LONGEST ** 2     # of query and key, over heads and batch
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _case(name, kind, step, dtype, batch, **sizes):
    case = {"kind": kind, "step": step, "dtype": dtype, "batch": batch, **sizes}
    return {"name": name, **case} if name else case


def _attention(name, step, dtype, batch, heads, kv_heads, queries, keys, mask="all", text=0, layout="heads"):
    return _case(name, "attention", step, dtype, batch, heads=heads, kv_heads=kv_heads, queries=queries, keys=keys,
                 mask=mask, text=text, layout=layout)


def listed():
    tokens = {px: TEXT + (px // 16) ** 2 for px in (512, 1024, 2048)}
    return [
        # One new token against the keys of a 1024-pixel image and its text: latency, and the keys' bytes.
        _attention("attention_token", "forward", "bf16", 1, HEADS, HEADS, 1, tokens[1024]),
        # A sampling step for three images of 1008 x 752 pixels whose prompts end early, in the general form.
        _attention("attention_padded_b3", "forward", "bf16", 3, HEADS, HEADS, TEXT + 63 * 47, TEXT + 63 * 47,
                   mask="padding", text=TEXT),
        # Fine-tuning at 512 and at 1024 pixels.
        _attention("attention_train_512px", "train", "bf16", 1, HEADS, HEADS, tokens[512], tokens[512]),
        _attention("attention_train_1024px", "train", "bf16", 1, HEADS, HEADS, tokens[1024], tokens[1024]),
        # Half precision, shared key heads, views of token-major buffers, lengths that no tile divides, and a
        # batch entry with nothing to attend to.
        _attention("attention_train_ragged_fp16", "train", "fp16", 3, 12, 4, 987, 1203, mask="empty", text=301,
                   layout="tokens"),
        # The largest: a 2048-pixel image's training step.
        _attention("attention_train_2048px", "train", "bf16", 1, HEADS, HEADS, tokens[2048], tokens[2048]),
        # The text stream of a 1024-pixel double block: its rows of the joint gradients.
        _case("qk_prep_grad_text", "qk_prep", "backward", "bf16", 1, tokens=TEXT, heads=HEADS, before=0, after=64 * 64,
              params="bf16"),
        # The image streams of two such blocks, behind their text.
        _case("qk_prep_grad_1024px_b2", "qk_prep", "backward", "bf16", 2, tokens=64 * 64, heads=HEADS, before=TEXT,
              after=0, params="bf16"),
        # A block's first sum on its text stream, the smallest call of the section.
        _case("residual_text", "residual", "forward", "bf16", 1, tokens=TEXT, width=WIDTH, params="bf16"),
        # The same for four 1024-pixel images.
        _case("residual_1024px_b4", "residual", "forward", "bf16", 4, tokens=64 * 64, width=WIDTH, params="bf16"),
        # Its gradients for a 1024-pixel single block.
        _case("residual_grad_1024px", "residual", "backward", "bf16", 1, tokens=tokens[1024], width=WIDTH, params="bf16"),
        # In float32 at a width that no chunk divides.
        _case("residual_grad_odd_fp32", "residual", "backward", "fp32", 3, tokens=1157, width=1111, params="fp32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "qk_prep", "residual"))
    batch = rng.choice((1, 1, 1, 2, 3, 4))
    if kind == "attention":
        step, dtype = rng.choice(("forward", "train", "train")), rng.choice(("bf16", "bf16", "fp16"))
        kv_heads = rng.choice((1, 2, 3, 4, 6, 8, 12, 24))
        heads = kv_heads * rng.choice([g for g in (1, 1, 2, 3, 4) if g * kv_heads <= HEADS])
        if step == "forward" and rng.random() < 0.4:     # a few new tokens against what is there
            queries, keys = rng.randint(1, 16), _log_int(rng, 1, 65536)
        else:
            queries = _log_int(rng, 1, min(LONGEST, math.isqrt(MOST_PAIRS // (batch * heads))))
            keys = queries if rng.random() < 0.7 else _log_int(rng, 1, min(LONGEST, MOST_PAIRS // (batch * heads * queries)))
        keys = max(keys, 4)     # with one key kept the gradients of q and k are zero, and what is left of them is noise
        mask = rng.choice(("all", "all", "padding", "random" if keys >= 64 else "all", "empty"))
        text = rng.randint(0, min(keys - 4, TEXT)) if mask in ("padding", "empty") else 0
        return _attention(None, step, dtype, batch, heads, kv_heads, queries, keys, mask, text,
                          rng.choice(("heads", "tokens")))
    tokens = _log_int(rng, 1, LONGEST // batch)
    if kind == "qk_prep":
        before, after = rng.choice(((0, 0), (0, rng.randint(1, 4096)), (rng.randint(1, TEXT), 0)))
        return _case(None, kind, "backward", "bf16", batch, tokens=tokens, heads=rng.randint(1, HEADS), before=before,
                     after=after, params=rng.choice(("bf16", "fp32")))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    return _case(None, kind, rng.choice(("forward", "backward")), dtype, batch, tokens=tokens,
                 width=_log_int(rng, 16, 8192), params=rng.choice((dtype, "fp32")))


def _prompt(case, entry):
    """Tokens of batch entry's prompt: the rest of the first ``text`` keys is padding."""
    return case["text"] * (entry + 1) // (case["batch"] + 1)


def _kept(case):
    """Keys that the mask keeps, of each batch entry (of a random mask, the number to expect)."""
    if case["mask"] == "all":
        return [case["keys"]] * case["batch"]
    if case["mask"] == "random":
        return [0.7 * case["keys"]] * case["batch"]
    kept = [case["keys"] - case["text"] + _prompt(case, b) for b in range(case["batch"])]
    return kept[:-1] + [0] if case["mask"] == "empty" else kept


def work(case):
    size, batch = TYPES[case["dtype"]].itemsize, case["batch"]
    if case["kind"] == "attention":
        train = case["step"] == "train"
        kept = _kept(case)
        used = sum(1 for n in kept if n > 0) * case["queries"]         # an entry without keys needs no queries
        q = case["heads"] * DIM * size
        kv = 2 * case["kv_heads"] * DIM * size
        o = batch * case["queries"] * q
        mask = 0 if case["mask"] == "all" else batch * case["keys"]
        products = 2 * case["heads"] * case["queries"] * DIM * sum(kept)
        if train:   # q, k, v and the incoming gradient in; o and three gradients out
            return {"bytes": 2 * used * q + sum(kept) * kv + 2 * o + batch * case["keys"] * kv + mask,
                    "flops": 7 * products}
        return {"bytes": used * q + sum(kept) * kv + o + mask, "flops": 2 * products}
    rows = batch * case["tokens"]
    params = TYPES[case["params"]].itemsize
    if case["kind"] == "qk_prep":
        values = rows * case["heads"] * DIM
        # dq, dk, dv and the projection's q and k in, three sections out, two tables of a row per token
        return {"bytes": 8 * values * size + 2 * case["tokens"] * DIM * 4 + 4 * DIM * params, "flops": 2 * 18 * values}
    values = rows * case["width"]
    rows_of_params = batch * case["width"] * params
    if case["step"] == "forward":
        return {"bytes": 4 * values * size + 3 * rows_of_params, "flops": 10 * values}
    return {"bytes": 6 * values * size + 5 * rows_of_params, "flops": 26 * values}


def _randn(gen, *shape):
    return torch.randn(shape, generator=gen, device="cuda")


def _heads(gen, case, heads, length, scale):
    """(B, heads, length, DIM): RMS-normalised rows, as q and k arrive, or with scale None as v does."""
    t = _randn(gen, case["batch"], heads, length, DIM)
    if scale is not None:
        t = t / t.square().mean(-1, keepdim=True).sqrt() * (scale * (1 + 0.1 * _randn(gen, DIM)))
    t = t.to(TYPES[case["dtype"]])
    return t.transpose(1, 2).contiguous().transpose(1, 2) if case["layout"] == "tokens" else t


def _key_mask(gen, case):
    if case["mask"] == "all":
        return None
    batch, keys = case["batch"], case["keys"]
    if case["mask"] == "random":
        return torch.rand((batch, keys), generator=gen, device="cuda") < 0.7
    mask = torch.ones((batch, keys), dtype=torch.bool, device="cuda")
    for b in range(batch):
        mask[b, _prompt(case, b):case["text"]] = False
    if case["mask"] == "empty":
        mask[-1] = False
    return mask


def _lanes(tokens):
    """Rotation lanes of an image's tokens, row by row: four axes of 32 columns (none, row, column, none)."""
    side = math.isqrt(tokens - 1) + 1
    at = torch.arange(tokens, device="cuda", dtype=torch.float64)
    zero = torch.zeros_like(at)
    freqs = 2000.0 ** (-torch.arange(0, 32, 2, device="cuda", dtype=torch.float64) / 32)
    angles = torch.cat([p[:, None] * freqs for p in (zero, at // side, at % side, zero)], 1)
    cos = torch.cos(angles).repeat_interleave(2, 1)
    sin = torch.stack((-torch.sin(angles), torch.sin(angles)), -1).flatten(1)
    return cos.float(), sin.float()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype, batch = TYPES[case["dtype"]], case["batch"]
    state = {"kind": case["kind"], "step": case["step"]}
    if case["kind"] == "attention":
        # norm scales of 1.2: logits with a deviation of 1.4; q comes scaled by 1 / sqrt(DIM)
        state["q"] = _heads(gen, case, case["heads"], case["queries"], 1.2 / math.sqrt(DIM))
        state["k"] = _heads(gen, case, case["kv_heads"], case["keys"], 1.2)
        state["v"] = _heads(gen, case, case["kv_heads"], case["keys"], None)
        state["mask"] = _key_mask(gen, case)
        if case["step"] == "train":
            state["do"] = _randn(gen, batch, case["queries"], case["heads"] * DIM).to(dtype)
        return state
    tokens, params = case["tokens"], TYPES[case["params"]]
    if case["kind"] == "qk_prep":
        heads, before = case["heads"], case["before"]
        joint = (batch, heads, before + tokens + case["after"], DIM)
        state["dq"], state["dk"], state["dv"] = (_randn(gen, *joint).to(dtype) for _ in range(3))
        # a projection whose heads differ in size
        size = torch.exp(0.5 * _randn(gen, 3 * heads, 1)).expand(-1, DIM).reshape(-1)
        state["qkv"] = (_randn(gen, batch, tokens, 3 * heads * DIM) * size).to(dtype)
        state["q_scale"], state["k_scale"] = ((1 + 0.2 * _randn(gen, DIM)).to(params) for _ in range(2))
        state["cos"], state["sin"] = _lanes(tokens)
        state["gain"], state["heads"], state["before"] = 1 / math.sqrt(DIM), heads, before
        return state
    width = case["width"]
    # a residual stream: tokens of different size, each off zero, one channel in a hundred large
    x = _randn(gen, batch, tokens, width) * torch.exp(0.5 * _randn(gen, batch, tokens, 1))
    x = x * torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    state["x"] = (x + 0.3 * _randn(gen, batch, tokens, 1)).to(dtype)
    state["branch"] = _randn(gen, batch, tokens, width).to(dtype)
    for name in ("gate", "shift", "scale"):
        state[name] = (0.5 * _randn(gen, batch, 1, width)).to(params)
    if case["step"] == "backward":
        state["dr"], state["dy"] = (_randn(gen, batch, tokens, width).to(dtype) for _ in range(2))
    return state


def _plain_attention(s):
    q, k, v, mask = s["q"], s["k"], s["v"], s["mask"]
    (batch, heads, queries, dim), (_, kv_heads, keys, _) = q.shape, k.shape
    group, train = heads // kv_heads, s["step"] == "train"
    o = torch.empty((batch, queries, kv_heads, group, dim), dtype=q.dtype, device=q.device)
    grads = [torch.empty_like(t) for t in (q, k, v)] if train else None
    # as many key heads at once as keep a float32 matrix of their logits near 2 GiB
    step = max(1, 2 ** 29 // (group * queries * keys))
    for b in range(batch):
        for h in range(0, kv_heads, step):
            kv, of_q = slice(h, h + step), slice(h * group, (h + step) * group)
            kf, vf, qf = k[b, kv].float(), v[b, kv].float(), q[b, of_q].float().reshape(-1, group * queries, dim)
            logits = qf @ kf.transpose(1, 2).contiguous()
            if mask is not None:
                logits = torch.where(mask[b], logits, -math.inf)
            top = logits.amax(-1, keepdim=True)
            p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
            del logits
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            out = p @ vf
            o[b, :, kv] = out.view(-1, group, queries, dim).permute(2, 0, 1, 3).to(o.dtype)
            if not train:
                continue
            do = s["do"][b].view(queries, heads, dim)[:, of_q].transpose(0, 1).float().reshape(qf.shape)
            ds = p * (do @ vf.transpose(1, 2).contiguous() - (do * out).sum(-1, keepdim=True))
            grads[0][b, of_q] = (ds @ kf).view(-1, queries, dim).to(q.dtype)
            grads[1][b, kv] = (ds.transpose(1, 2) @ qf).to(k.dtype)
            grads[2][b, kv] = (p.transpose(1, 2) @ do).to(v.dtype)
    o = o.view(batch, queries, heads * dim)
    return (o, *grads) if train else o


def _plain_qk_prep(s):
    qkv, heads, before = s["qkv"], s["heads"], s["before"]
    batch, tokens, _ = qkv.shape
    x = qkv.view(batch, tokens, 3, heads, DIM)
    rows = slice(before, before + tokens)
    cos, sin = s["cos"][:, None], s["sin"][:, None]
    sections, scales = [], []
    for i, (grad, scale, gain) in enumerate(((s["dq"], s["q_scale"], s["gain"]), (s["dk"], s["k_scale"], 1.0))):
        dr = gain * grad[:, :, rows].transpose(1, 2).float()
        turned = sin * dr
        dy = cos * dr + torch.stack((turned[..., 1::2], turned[..., 0::2]), -1).flatten(-2)
        xf = x[:, :, i].float()
        inv = 1 / torch.sqrt(xf.square().mean(-1, keepdim=True) + EPS)
        normed = xf * inv
        dn = dy * scale.float()
        sections.append((inv * (dn - normed * (dn * normed).mean(-1, keepdim=True))).to(qkv.dtype))
        scales.append((dy * normed).sum((0, 1, 2)).to(scale.dtype))
    sections.append(s["dv"][:, :, rows].transpose(1, 2))
    return torch.stack(sections, 2).flatten(2), *scales


def _plain_residual(s):
    x, dtype, params = s["x"], s["x"].dtype, s["gate"].dtype
    branch, gate = s["branch"].float(), s["gate"].float()
    r = x.float() + gate * branch
    centred = r - r.mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(centred.square().mean(-1, keepdim=True) + EPS)
    normed, factor = centred * rstd, 1 + s["scale"].float()
    if s["step"] == "forward":
        return r.to(dtype), (normed * factor + s["shift"].float()).to(dtype)
    dy = s["dy"].float()
    t = dy * factor
    dr = s["dr"].float() + rstd * (t - t.mean(-1, keepdim=True) - normed * (t * normed).mean(-1, keepdim=True))
    sums = ((dr * branch).sum(1, keepdim=True), dy.sum(1, keepdim=True), (dy * normed).sum(1, keepdim=True))
    return dr.to(dtype), (gate * dr).to(dtype), *(t.to(params) for t in sums)


def _plain(s):
    """The operators in float32, each output rounded once."""
    return {"attention": _plain_attention, "qk_prep": _plain_qk_prep, "residual": _plain_residual}[s["kind"]](s)


def _framework(s):
    if s["kind"] == "attention":
        from flicker_amd import attention
        if s["step"] == "forward":
            return attention.attention(s["q"], s["k"], s["v"], key_mask=s["mask"])
        o, kept = attention.attention(s["q"], s["k"], s["v"], key_mask=s["mask"], keep=True)
        return o, *attention.attention_backward(s["do"], s["q"], s["k"], s["v"], kept, key_mask=s["mask"])
    if s["kind"] == "qk_prep":
        from flicker_amd import kernels
        freqs = kernels.Freqs(s["cos"], s["sin"], s["gain"])
        return kernels.qk_prep_backward(s["dq"], s["dk"], s["dv"], s["qkv"], s["q_scale"], s["k_scale"], freqs,
                                        s["heads"], offset=s["before"])
    from flicker_amd import norm
    if s["step"] == "forward":
        return norm.residual_modulate(s["x"], s["branch"], s["gate"], s["shift"], s["scale"])
    return norm.residual_modulate_backward(s["dr"], s["dy"], s["x"], s["branch"], s["gate"], s["shift"], s["scale"])


def run(state):
    return _framework(state) if own else _plain(state)


def _exact_attention(s):
    """Head by head, the gradients by differentiating softmax."""
    train, mask = s["step"] == "train", s["mask"]
    q, k, v = (s[n].double() for n in "qkv")
    (batch, heads, queries, dim), group = q.shape, s["q"].shape[1] // s["k"].shape[1]
    o = torch.zeros((batch, queries, heads, dim), dtype=torch.float64, device=q.device)
    grads = [torch.zeros_like(t) for t in (q, k, v)]
    for b in range(batch):
        kept = slice(None) if mask is None else mask[b].nonzero().flatten()
        if mask is not None and kept.numel() == 0:
            continue
        for h in range(heads):
            leaves = [t.detach().requires_grad_(train) for t in (q[b, h], k[b, h // group][kept], v[b, h // group][kept])]
            out = torch.softmax(torch.matmul(leaves[0], leaves[1].transpose(0, 1)), -1) @ leaves[2]
            o[b, :, h] = out.detach()
            if train:
                incoming = s["do"].view(batch, queries, heads, dim)[b, :, h].double()
                dq, dk, dv = torch.autograd.grad(out, leaves, incoming)
                grads[0][b, h] = dq
                grads[1][b, h // group][kept] += dk
                grads[2][b, h // group][kept] += dv
    o = o.flatten(2)
    return (o, *grads) if train else o


def exact(case, seed):
    """What run() returns, from the definitions in float64; gradients by differentiating the
    forward definition rather than from the formulas that the plain form uses."""
    s = prepare(case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    leaves = {n: t.double().requires_grad_() for n, t in s.items() if isinstance(t, torch.Tensor)}
    if case["kind"] == "qk_prep":
        batch, tokens, _ = s["qkv"].shape
        rows = slice(s["before"], s["before"] + tokens)
        parts = leaves["qkv"].view(batch, tokens, 3, s["heads"], DIM).unbind(2)
        outs = []
        for x, scale, gain in zip(parts, ("q_scale", "k_scale"), (s["gain"], 1.0)):
            y = x * torch.rsqrt((x * x).mean(-1, True) + EPS)
            pairs = torch.view_as_complex((y * leaves[scale]).unflatten(-1, (-1, 2)))
            turn = torch.complex(s["cos"][:, 0::2].double(), s["sin"][:, 1::2].double())[:, None]
            outs.append(gain * torch.view_as_real(pairs * turn).flatten(-2).transpose(1, 2))
        outs.append(parts[2].transpose(1, 2))
        return torch.autograd.grad(outs, [leaves[n] for n in ("qkv", "q_scale", "k_scale")],
                                   [leaves[n].detach()[:, :, rows] for n in ("dq", "dk", "dv")])
    r = torch.addcmul(leaves["x"], leaves["gate"], leaves["branch"])
    var, mean = torch.var_mean(r, -1, correction=0, keepdim=True)
    y = (1 + leaves["scale"]) * ((r - mean) * torch.rsqrt(var + EPS)) + leaves["shift"]
    if case["step"] == "forward":
        return r.detach(), y.detach()
    wanted = [leaves[n] for n in ("x", "branch", "gate", "shift", "scale")]
    return torch.autograd.grad((r, y), wanted, (leaves["dr"].detach(), leaves["dy"].detach()))
