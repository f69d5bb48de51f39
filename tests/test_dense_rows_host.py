"""Operands whose rows do not start on 16 bytes are copied to where they do, contiguous ones among them."""

import pytest
import torch

from flicker_amd import kernels


def _views():
    flat = torch.arange(2 * 3 * 8 * 16 + 64, dtype=torch.float32).to(torch.bfloat16)
    yield "contiguous, off 16 bytes", flat[1:1 + 2 * 3 * 8 * 16].view(2, 3, 8, 16), True
    yield "one entry, odd batch stride", torch.as_strided(flat, (1, 3, 8, 16), (3 * 8 * 16 + 3, 8 * 16, 16, 1)), True
    yield "odd rows", torch.as_strided(flat, (2, 2, 4, 16), (400, 160, 20, 1)), True
    yield "strided columns", flat[:2 * 3 * 8 * 16].view(2, 3, 8, 16)[..., ::2], True
    yield "as it is", flat[:2 * 3 * 8 * 16].view(2, 3, 8, 16).transpose(1, 2), False


@pytest.mark.parametrize("name,t,copied", list(_views()), ids=lambda x: x if isinstance(x, str) else "")
def test_dense_rows(name, t, copied):
    got = kernels._dense_rows(t)
    assert torch.equal(got, t) and (got is not t) == copied
    assert got.data_ptr() % 16 == 0 and got.stride(-1) == 1 and all(s % 8 == 0 for s in got.stride()[:-1])
