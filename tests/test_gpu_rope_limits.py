"""Rotary positions, their table and the append at the ends of their arguments' ranges, on the GPU."""

import ctypes

import numpy as np
import pytest

import paged_ref as R
from test_gpu_rope_append import run_append, table_freq

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


@pytest.mark.parametrize("name", ["qsi8dx_f16", "qsi8dx_bf16"])
@pytest.mark.parametrize("rot", [0, 64])
@pytest.mark.parametrize("pads", [(0, 0, 0), (1, 0, 0)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_int8_not_finite_reads_back_as_nan(gpu, name, rot, bad, pads):
    """Every element of a key's or value's row with a NaN or an infinity, that one's own among them."""
    r = np.random.default_rng(1).standard_normal((4, 3, 64))
    r[1, 1, 17] = r[2, 2, 40] = bad  # a key, a value
    g = run_append(name, 4, 1, 1, 64, rot, rows=r, pads=pads)
    for cache, scale, token in (("k", "sk", 1), ("v", "sv", 2)):
        back = g[cache].double() * g[scale].double().transpose(1, 2)[..., None]
        back = back.reshape(-1, 64)[R.dev(g["slots"])].cpu().numpy()
        assert np.isnan(back[token]).all()
        assert np.isfinite(np.delete(back, token, 0)).all()


@pytest.mark.parametrize("factor,amplitude", [(0.5, 1.0), (1e-5, 1.0), (1.0, 1.0), (4.0, 0.1 * np.log(4.0) + 1)])
def test_ramp_amplitude(gpu, factor, amplitude):
    """The ramp's amplitude grows with factors above 1 and is 1 for the others."""
    import torch

    mod, lib = R.binding()
    t = torch.zeros((500, 32), device="cuda:0")
    p = mod.RopeTableParams(table=R.ptr(t), max_pos=500, rotary_dim=32, scaling=mod.ROPE_RAMP, base=10000.0,
                            factor=factor, original_max_pos=4096.0, low_turns=1, high_turns=32)
    lib.op("rope_table_f32", "run")(ctypes.byref(p))
    want = amplitude * R.rope_table(500, 32, freq=table_freq(32, 3, 10000.0, factor, 4096.0, 1, 32))
    # one rounding to f32; the angles' own error in f64 is below 500 / 1e-5 * 2^-50
    assert np.abs(R.host(t) - want).max() <= amplitude * 2.0 ** -24 + 5e7 * 2.0 ** -50
