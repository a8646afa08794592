"""Rotary positions and the append to a paged cache on the GPU, against plain forms in 64 bits (with bounds from
the roundings the operators are defined by) and, where the arithmetic is defined to the last bit, exactly."""

import ctypes

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


def strided(x, kind, pad_head=0, pad_token=0, offset=0):
    """x [tokens, heads, d] on the GPU as a view with gaps after every head and token."""
    import torch

    t, h, d = x.shape
    ts = h * (d + pad_head) + pad_token
    buf = torch.full((offset + t * ts + 8,), 7.0, dtype=R.torch_type(kind), device="cuda:0")
    view = buf.as_strided((t, h, d), (ts, d + pad_head, 1), offset)
    view.copy_(R.dev(x))
    return buf, view


def run_rope(kind, x, pos, table, rot, interleaved, inverse=False, pads=(0, 0, 0), in_place=False):
    import torch

    mod, lib = R.binding()
    buf, xv = strided(x, kind, *pads)
    before = buf.clone()
    ybuf, yv = (buf, xv) if in_place else strided(np.zeros_like(x), kind, *pads)
    dpos, dt = R.dev(pos.astype(np.int32)), None if table is None else R.dev(table.astype(np.float32))
    p = mod.RopeParams(tokens=x.shape[0], heads=x.shape[1], head_dim=x.shape[2], X=R.ptr(xv),
                       x_token_stride=xv.stride(0), x_head_stride=xv.stride(1), Y=R.ptr(yv),
                       y_token_stride=yv.stride(0), y_head_stride=yv.stride(1), positions=R.ptr(dpos),
                       map=R.rope_map(mod, dt, rot, interleaved, inverse))
    given = R.host(xv)
    lib.op("rope_" + kind, "run")(ctypes.byref(p))
    # nothing outside the heads is written
    mask = torch.ones_like(ybuf, dtype=torch.bool)
    mask.as_strided(yv.shape, yv.stride(), pads[2]).fill_(False)
    assert torch.equal(ybuf[mask], before[mask])
    return given, R.host(yv)


def check_rope(kind, tokens, heads, d, rot, interleaved, inverse=False, **kw):
    rng = np.random.default_rng(tokens * 131 + heads * 17 + d + rot)
    x = rng.standard_normal((tokens, heads, d))
    table = R.rope_table(300, rot).astype(np.float32) if rot else None
    pos = rng.integers(0, 300, tokens)
    given, got = run_rope(kind, x, pos, table, rot, interleaved, inverse, **kw)
    want, size = R.rope(given, pos, table, rot, interleaved, inverse)
    u, tiny = R.ROUND[kind]
    # two products and a sum in f32, then one rounding to the type
    assert (np.abs(got - want) <= size * 2.0 ** -23 + np.abs(want) * u * 1.01 + tiny).all()
    np.testing.assert_array_equal(got[..., rot:], given[..., rot:])


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,d,rot", [
    (1, 1, 16, 16), (1, 32, 128, 128), (3, 5, 64, 32), (37, 7, 80, 80), (5, 3, 256, 64), (9, 2, 96, 80),
    (2, 3, 48, 0), (700, 40, 128, 96),
    # off the 16-element grid: odd heads, rotations that end inside one
    (4, 3, 10, 10), (3, 2, 7, 4), (6, 5, 72, 36), (2, 2, 130, 66), (3, 4, 64, 2), (2, 1, 1, 0)])
def test_rope(gpu, kind, interleaved, tokens, heads, d, rot):
    check_rope(kind, tokens, heads, d, rot, interleaved)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("pads", [(0, 16, 0), (16, 8, 8), (1, 0, 0), (0, 0, 1), (3, 5, 2)])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rope_strides_alignment_in_place(gpu, kind, pads, in_place, interleaved):
    check_rope(kind, 11, 6, 64, 48, interleaved, pads=pads, in_place=in_place)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot", [(64, 64), (80, 48), (30, 18)])
def test_rope_gradient(gpu, interleaved, d, rot):
    """The inverse is the gradient: against the formula (the transposed rotation, by check_rope) and
    against differences of the forward pass in a random direction."""
    check_rope("f32", 9, 4, d, rot, interleaved, inverse=True)
    rng = np.random.default_rng(d)
    x, u, g = (rng.standard_normal((5, 3, d)).astype(np.float32) for _ in range(3))
    table = (R.rope_table(64, rot) * 1.3).astype(np.float32)  # a table with an amplitude
    pos = rng.integers(0, 64, 5)
    _, hi = run_rope("f32", x + u, pos, table, rot, interleaved)
    _, lo = run_rope("f32", x - u, pos, table, rot, interleaved)
    _, grad = run_rope("f32", g, pos, table, rot, interleaved, inverse=True)
    by_difference = ((hi - lo) / 2 * g).sum()
    # linear: the difference has no error but roundings, about 2^-23 of each of the 15 d terms
    assert abs(by_difference - (grad * u).sum()) <= 15 * d * 2.0 ** -20


def test_rope_position_outside_table(gpu):
    table = R.rope_table(16, 32)
    x = np.random.default_rng(0).standard_normal((5, 2, 48))
    for d in (48, 47):  # the kernel for the 16-byte grid, and the other
        given, got = run_rope("f32", x[..., :d], np.array([15, 16, -1, 2 ** 31 - 1, 0]), table, 32, False)
        for t, ok in enumerate([True, False, False, False, True]):
            assert np.isfinite(got[t]).all() if ok else np.isnan(got[t, :, :32]).all()
            np.testing.assert_array_equal(got[t, :, 32:], given[t, :, 32:])


def test_rope_nothing_to_do(gpu):
    mod, lib = R.binding()
    run = lib.op("rope_f16", "run")
    run(None)
    run(ctypes.byref(mod.RopeParams(tokens=0, heads=4, head_dim=64)))
    run(ctypes.byref(mod.RopeParams(tokens=4, heads=0, head_dim=64)))


def table_freq(rot, scaling, base, factor, orig, low, high):
    """The frequencies of tqt_rope_table_params, written out."""
    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / rot)
    if scaling == 1:
        return f / factor
    if scaling == 2:
        return (base * factor ** (rot / (rot - 2))) ** (-2.0 * i / rot)
    if scaling == 3:
        at = lambda turns: rot * np.log(orig / (turns * 2 * np.pi)) / (2 * np.log(base))  # noqa: E731
        lo, hi = max(np.floor(at(high)), 0), min(np.ceil(at(low)), rot - 1)
        ramp = np.clip((i - lo) / max(hi - lo, 0.001), 0, 1)
        return f / factor * ramp + f * (1 - ramp)
    if scaling == 4:
        smooth = np.clip((orig * f / (2 * np.pi) - low) / (high - low), 0, 1)
        return f / factor * (1 - smooth) + f * smooth
    return f


@pytest.mark.parametrize("scaling,low,high", [(0, 0, 0), (1, 0, 0), (2, 0, 0), (3, 1, 32), (4, 1, 4)])
@pytest.mark.parametrize("rot,max_pos,base", [(128, 5000, 10000.0), (4, 9, 100.0),
                                              (64, 70000, 500000.0)])
def test_rope_table(gpu, scaling, low, high, rot, max_pos, base):
    import torch

    mod, lib = R.binding()
    t = torch.full((max_pos + 1, rot), 5.0, device="cuda:0")
    p = mod.RopeTableParams(table=R.ptr(t), max_pos=max_pos, rotary_dim=rot, scaling=scaling, base=base,
                            factor=8.0, original_max_pos=4096.0, low_turns=low, high_turns=high)
    lib.op("rope_table_f32", "run")(ctypes.byref(p))
    amp = 0.1 * np.log(8.0) + 1 if scaling == 3 else 1.0
    want = amp * R.rope_table(max_pos, rot, freq=table_freq(rot, scaling, base, 8.0, 4096.0, low, high))
    # one rounding to f32; the angles' own error in f64 is below 70000 * 2^-50
    assert np.abs(R.host(t[:max_pos]) - want).max() <= amp * 2.0 ** -24 + 70000 * 2.0 ** -50
    assert (t[max_pos] == 5.0).all()


# ------------------------------------------------------------------------------------------
# Append
# ------------------------------------------------------------------------------------------

KINDS = ["f16_f16", "bf16_bf16", "f16_f32", "bf16_f32", "qsi8dx_f16", "qsi8dx_bf16"]


def run_append(name, tokens, heads, kv_heads, d, rot, interleaved=False, page=16, pages=8, queries=True,
               heads_first=False, pads=(0, 0, 0), rows=None, slots=None, stream=None):
    """(what was given, what the cache holds before and after) of one call."""
    import torch

    mod, lib = R.binding()
    cache, src = name.split("_")
    rng = np.random.default_rng(tokens * 31 + heads + d)
    n = heads + 2 * kv_heads
    x = rng.standard_normal((tokens, n, d)) if rows is None else rows
    _, xv = strided(x, src, *pads)
    given = R.host(xv)
    qt = R.torch_type(cache if src == "f32" else src)
    q_out = torch.full((tokens, heads, d + pads[0]), 7.0, dtype=qt, device="cuda:0")
    shape = (pages, kv_heads, page, d) if heads_first else (pages, page, kv_heads, d)
    k, v = (torch.randint(-99, 99, shape, device="cuda:0").to(R.torch_type(cache)) for _ in range(2))
    sk = sv = None
    if cache == "qsi8dx":
        sk, sv = (torch.rand((pages, kv_heads, page), device="cuda:0") for _ in range(2))
    old = [None if t is None else t.clone() for t in (k, v, sk, sv)]
    if slots is None:
        slots = rng.permutation(pages * page)[:tokens]
    pos = rng.integers(0, 100, tokens)
    table = R.rope_table(100, rot).astype(np.float32) if rot else None
    dt, dpos, dslots = None if table is None else R.dev(table), R.dev(pos.astype(np.int32)), R.dev(
        slots.astype(np.int64))
    p = mod.KVAppendRopeParams(
        tokens=tokens, K=R.ptr(xv[:, heads:]), k_token_stride=xv.stride(0), k_head_stride=xv.stride(1),
        V=R.ptr(xv[:, heads + kv_heads:]), v_token_stride=xv.stride(0), v_head_stride=xv.stride(1),
        q_heads=heads if queries else 0, Q=R.ptr(xv), q_token_stride=xv.stride(0),
        q_head_stride=xv.stride(1), Q_out=R.ptr(q_out), qo_token_stride=q_out.stride(0),
        qo_head_stride=q_out.stride(1), positions=R.ptr(dpos), slots=R.ptr(dslots),
        map=R.rope_map(mod, dt, rot, interleaved), kv=R.paged(mod, k, v, sk, sv, heads_first=heads_first))
    assert lib.op("kv_append_rope_" + name, "get_error")(ctypes.byref(p)) is None
    if stream is None:
        lib.op("kv_append_rope_" + name, "run")(ctypes.byref(p))
    else:
        lib.op("kv_append_rope_" + name, "run_async")(ctypes.byref(p), stream)
        torch.cuda.synchronize()
    if heads_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
        old[0], old[1] = old[0].transpose(1, 2), old[1].transpose(1, 2)
    return dict(x=given, q=q_out, k=k, v=v, sk=sk, sv=sv, old=old, slots=slots, pos=pos, table=table)


def check_append(name, tokens, heads, kv_heads, d, rot, interleaved=False, page=16, **kw):
    import torch

    cache, src = name.split("_")
    g = run_append(name, tokens, heads, kv_heads, d, rot, interleaved, page, **kw)
    x32 = g["x"].astype(np.float32)
    turned, _ = R.rope(x32, g["pos"], g["table"], rot, interleaved, dtype=np.float32)
    rows = dict(k=turned[:, heads:heads + kv_heads], v=x32[:, heads + kv_heads:])
    if kw.get("queries", True):
        # the arithmetic is defined to the bit: f32 products and sums, one rounding
        want = R.dev(turned[:, :heads]).to(g["q"].dtype)
        assert torch.equal(g["q"][..., :d], want)
        assert (g["q"][..., d:] == 7).all()
    else:
        assert (g["q"] == 7).all()
    pages = g["k"].shape[0]
    kept = np.ones(pages * page, bool)
    use = (g["slots"] >= 0) & (g["slots"] < pages * page)
    at = g["slots"][use]
    kept[at] = False
    for name_, scale, old, old_scale in (("k", "sk", 0, 2), ("v", "sv", 1, 3)):
        flat = g[name_].reshape(pages * page, kv_heads, d)
        was = g["old"][old].reshape(pages * page, kv_heads, d)
        r = rows[name_][use]
        assert torch.equal(flat[R.dev(np.nonzero(kept)[0])], was[R.dev(np.nonzero(kept)[0])])
        got = flat[R.dev(at)]
        if cache == "qsi8dx":
            q, s = R.quantize_rows(r)
            np.testing.assert_array_equal(got.cpu().numpy(), q)
            sc = g[scale].transpose(1, 2).reshape(pages * page, kv_heads)
            np.testing.assert_array_equal(sc[R.dev(at)].cpu().numpy().view(np.uint32),
                                          s.view(np.uint32))
            was_sc = g["old"][old_scale].transpose(1, 2).reshape(pages * page, kv_heads)
            assert torch.equal(sc[R.dev(np.nonzero(kept)[0])], was_sc[R.dev(np.nonzero(kept)[0])])
        else:
            assert torch.equal(got, R.dev(r).to(got.dtype))


@pytest.mark.parametrize("name", KINDS)
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot", [
    (1, 1, 1, 16, 16), (1, 32, 8, 128, 128), (13, 6, 2, 80, 80), (40, 7, 7, 64, 32), (9, 4, 2, 256, 128),
    (21, 3, 1, 96, 48), (5, 2, 1, 192, 192), (3, 2, 2, 112, 0), (7, 3, 1, 48, 22)])
def test_append(gpu, name, tokens, heads, kv_heads, d, rot):
    check_append(name, tokens, heads, kv_heads, d, rot)


@pytest.mark.parametrize("name", KINDS)
@pytest.mark.parametrize("page,pages", [(1, 64), (24, 3), (64, 2), (7, 9)])
@pytest.mark.parametrize("heads_first", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append_pages(gpu, name, page, pages, heads_first, interleaved):
    check_append(name, 33, 6, 3, 64, 64, interleaved, page, pages=pages, heads_first=heads_first)


@pytest.mark.parametrize("name", KINDS)
@pytest.mark.parametrize("pads", [(16, 8, 0), (8, 16, 8), (1, 0, 0), (0, 3, 1)])
def test_append_strides(gpu, name, pads):
    check_append(name, 12, 4, 2, 64, 64, pads=pads)


@pytest.mark.parametrize("name", KINDS)
def test_append_many(gpu, name):
    """Enough threads for the form that takes four heads a thread."""
    check_append(name, 1201, 24, 8, 128, 64, page=32, pages=40)


@pytest.mark.parametrize("name", KINDS)
def test_append_without_queries_padding_slots(gpu, name):
    slots = np.array([3, -1, 0, 128, 2 ** 40, 127, -2 ** 63, 64])
    check_append(name, 8, 5, 2, 64, 64, slots=slots, queries=False)
    check_append(name, 8, 5, 2, 64, 22, slots=slots)


@pytest.mark.parametrize("name,rot", [("qsi8dx_f16", 0), ("qsi8dx_bf16", 0)])
@pytest.mark.parametrize("pads", [(0, 0, 0), (1, 0, 0)])
def test_append_int8_special_rows(gpu, name, rot, pads):
    """Rows of zeros, of one value, ties, the type's smallest and largest values."""
    d = 64
    big, small = (65504.0, 2.0 ** -24) if name.endswith("f16") and "bf16" not in name else (3e38, 1e-40)
    r = np.zeros((6, 3, d))
    r[1] = 1.0
    r[2] = np.linspace(-127, 127, d).round() + 0.5
    r[2, :, 0] = 127
    r[3, :, ::2] = small
    r[4] = -big
    r[5, 1, 5] = 3
    check_append(name, 6, 1, 1, d, rot, rows=r, pads=pads)


@pytest.mark.parametrize("pads", [(0, 0, 0), (1, 0, 0)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_int8_not_finite(gpu, bad, pads):
    """A row with a NaN or an infinity reads back as NaN, and only that row does."""
    r = np.random.default_rng(1).standard_normal((4, 3, 64))
    r[2, 1, 17] = bad
    g = run_append("qsi8dx_f16", 4, 1, 1, 64, 0, rows=r, pads=pads)
    back = g["k"].double() * g["sk"].double().transpose(1, 2)[..., None]
    back = back.reshape(-1, 64)[R.dev(g["slots"])].cpu().numpy()
    assert not np.isfinite(back[2]).any()
    assert np.isfinite(back[[0, 1, 3]]).all()


def test_append_in_place_queries_on_a_stream(gpu):
    """Q and Q_out of one tensor, on a stream other than the default one."""
    import torch

    mod, lib = R.binding()
    stream = torch.cuda.Stream()
    x = np.random.default_rng(4).standard_normal((20, 10, 64))
    with torch.cuda.stream(stream):
        qkv = R.dev(x, "bf16")
        given = R.host(qkv)
        k, v = (torch.zeros((2, 16, 2, 64), dtype=torch.bfloat16, device="cuda:0") for _ in range(2))
        table = R.rope_table(64, 64).astype(np.float32)
        pos = np.arange(20)
        dt, dpos, slots = R.dev(table), R.dev(pos.astype(np.int32)), R.dev(np.arange(20))
        p = mod.KVAppendRopeParams(
            tokens=20, K=R.ptr(qkv[:, 6:]), k_token_stride=640, k_head_stride=64, V=R.ptr(qkv[:, 8:]),
            v_token_stride=640, v_head_stride=64, q_heads=6, Q=R.ptr(qkv), q_token_stride=640,
            q_head_stride=64, Q_out=R.ptr(qkv), qo_token_stride=640, qo_head_stride=64,
            positions=R.ptr(dpos), slots=R.ptr(slots), map=R.rope_map(mod, dt, 64, False),
            kv=R.paged(mod, k, v))
        lib.op("kv_append_rope_bf16_bf16", "run_async")(ctypes.byref(p), stream.cuda_stream)
        stream.synchronize()
    turned, _ = R.rope(given.astype(np.float32), pos, table, 64, False, dtype=np.float32)
    assert torch.equal(qkv[:, :6], R.dev(turned[:, :6], "bf16"))
    assert torch.equal(qkv[:, 6:], R.dev(given[:, 6:], "bf16"))
    assert torch.equal(k.reshape(32, 2, 64)[:20], R.dev(turned[:, 6:8], "bf16"))
