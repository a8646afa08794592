"""Rotary positions and their table at the ends of their arguments' ranges, on the GPU."""

import ctypes

import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


def test_rows_past_one_grid(gpu):
    """More (token, head) rows off the 16-byte grid than the waves of one launch: 2^21 tokens of 33 heads, whose
    waves have 2^32 work-items and more."""
    import torch

    mod, lib = R.binding()
    tokens, heads = 2 ** 21, 33
    assert tokens * heads * 64 > 2 ** 32
    g = torch.Generator(device="cuda:0").manual_seed(1)
    x = torch.randn((tokens, heads, 2), generator=g, device="cuda:0").half()
    y = torch.zeros_like(x)
    table = R.dev(R.rope_table(100, 2).astype("float32"))
    pos = torch.randint(0, 100, (tokens,), generator=g, device="cuda:0", dtype=torch.int32)
    p = mod.RopeParams(tokens=tokens, heads=heads, head_dim=2, X=R.ptr(x), x_token_stride=2 * heads,
                       x_head_stride=2, Y=R.ptr(y), y_token_stride=2 * heads, y_head_stride=2,
                       positions=R.ptr(pos), map=R.rope_map(mod, table, 2, False))
    assert lib.op("rope_f16", "get_error")(ctypes.byref(p)) is None
    lib.op("rope_f16", "run")(ctypes.byref(p))
    # the arithmetic is defined to the bit: f32 products and sums, one rounding
    t = table[pos.long()]
    a, b, c, s = x[..., 0].float(), x[..., 1].float(), t[:, :1], t[:, 1:]
    assert torch.equal(y[..., 0], (a * c - b * s).half())
    assert torch.equal(y[..., 1], (b * c + a * s).half())
