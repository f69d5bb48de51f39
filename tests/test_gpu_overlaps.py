"""An `out` over memory that the call still reads is refused, the small operands' among it."""

import pytest
import torch

from flicker_amd import attention, kernels

pytestmark = pytest.mark.gpu
D = 128


def test_attention_out_over_the_mask(device):
    q = torch.randn(2, 2, 40, D, device=device, dtype=torch.bfloat16)
    buffer = torch.zeros(2, 40, 2 * D, device=device, dtype=torch.bfloat16)
    mask = buffer.view(-1).view(torch.bool)[1000:1080].view(2, 40)
    mask[:, ::2] = True
    with pytest.raises(ValueError, match="shares memory with key_mask"):
        attention.attention(q, q, q, key_mask=mask, out=buffer)
    apart = buffer[:, :40].clone()
    assert attention.attention(q, q, q, key_mask=mask, out=apart) is apart


@pytest.mark.parametrize("which", ["q_scale", "k_scale", "cos", "sin"])
def test_qk_prep_backward_out_over_scales_and_tables(device, which):
    length, heads = 16, 2
    qkv = torch.randn(1, length, 3 * heads * D, device=device, dtype=torch.bfloat16)
    grads = torch.randn(3, 1, heads, length, D, device=device, dtype=torch.bfloat16)
    buffer = torch.zeros(1, length, 3 * heads * D, device=device, dtype=torch.bfloat16)
    ops = {n: torch.ones(D, device=device, dtype=torch.bfloat16) for n in ("q_scale", "k_scale")}
    ops.update({n: torch.ones(length, D, device=device) for n in ("cos", "sin")})
    t = ops[which]
    ops[which] = buffer.view(-1)[512:].view(t.dtype)[:t.numel()].view(t.shape).copy_(t)
    freqs = kernels.Freqs(ops["cos"], ops["sin"], 0.5)
    with pytest.raises(ValueError, match=f"shares memory with {which}"):
        kernels.qk_prep_backward(*grads, qkv, ops["q_scale"], ops["k_scale"], freqs, heads, out=buffer)
    apart = torch.empty_like(buffer)
    got = kernels.qk_prep_backward(*grads, qkv, ops["q_scale"], ops["k_scale"], freqs, heads, out=apart)
    want = kernels.qk_prep_backward(*grads, qkv, ops["q_scale"], ops["k_scale"], freqs, heads)
    assert got[0] is apart and all(torch.equal(a, b) for a, b in zip(got, want))
