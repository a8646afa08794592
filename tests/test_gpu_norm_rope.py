"""The norm of heads with its rotation, its gradient, and both on the way into a paged cache, on the GPU against plain
forms in 64 bits (drafted_ref.py, which derives the bounds from the operators' roundings)."""

import ctypes

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R
from test_gpu_rope_append import strided

pytestmark = pytest.mark.gpu
KINDS = ["f32", "f16", "bf16"]
# (tokens, heads, head_dim, rotary_dim): a token, odd heads, several workgroups, and off the 16-element grid
SHAPES = [(1, 1, 16, 16), (1, 32, 128, 128), (3, 5, 64, 32), (37, 7, 80, 80), (5, 3, 256, 64), (9, 2, 96, 80),
          (2, 3, 48, 0), (300, 40, 128, 96), (3, 2, 1024, 512), (2, 2, 1040, 16),
          (4, 3, 10, 10), (3, 2, 7, 4), (6, 5, 72, 36), (2, 2, 130, 66), (5, 4, 80, 40), (2, 1, 1, 0)]


def check_outside(buf, before, view, offset):
    import torch

    mask = torch.ones_like(buf, dtype=torch.bool)
    mask.as_strided(view.shape, view.stride(), offset).fill_(False)
    assert torch.equal(buf[mask], before[mask])


class Call:
    """Inputs of one call, rows with gaps `pads` after every head and token and before the first."""

    def __init__(self, kind, tokens, heads, d, rot, inter=False, weight=True, shift=0.0, eps=1e-5, inverse=False,
                 pads=(0, 0, 0), size=2.0, seed=0):
        self.mod, self.lib = R.binding()
        rng = np.random.default_rng(seed + tokens * 131 + heads * 17 + d + rot)
        self.kind, self.rot, self.inter, self.inverse = kind, rot, inter, inverse
        self.pads, self.shift, self.eps, self.d = pads, shift, eps, d
        self.buf, self.x = strided(rng.standard_normal((tokens, heads, d)) * size, kind, *pads)
        self.dbuf, self.dy = strided(rng.standard_normal((tokens, heads, d)), kind, *pads)
        self.w = (rng.standard_normal(d) * 0.3 + 1 - shift).astype(np.float32) if weight else None
        self.table = (R.rope_table(300, rot) * 1.1).astype(np.float32) if rot else None
        self.pos = rng.integers(0, 300, tokens)
        self.dw_, self.dtable = None if self.w is None else R.dev(self.w), \
            None if self.table is None else R.dev(self.table)

    def params(self, x, y, dpos, weight=None):
        w = self.dw_ if weight is None else weight
        mod = self.mod
        return mod.NormRopeParams(
            rope=mod.RopeParams(tokens=x.shape[0], heads=x.shape[1], head_dim=x.shape[2], X=R.ptr(x),
                                x_token_stride=x.stride(0), x_head_stride=x.stride(1), Y=R.ptr(y),
                                y_token_stride=0 if y is None else y.stride(0),
                                y_head_stride=0 if y is None else y.stride(1), positions=R.ptr(dpos),
                                map=R.rope_map(mod, self.dtable, self.rot, self.inter, self.inverse)),
            norm=D.head_norm(mod, w, self.shift, self.eps))

    def forward(self, in_place=False, weight=None):
        import torch

        given = R.host(self.x)
        ybuf, y = (self.buf, self.x) if in_place else strided(np.zeros(self.x.shape), self.kind, *self.pads)
        before, dpos = ybuf.clone(), R.dev(self.pos.astype(np.int32))
        D.run("norm_rope_" + self.kind, self.params(self.x, y, dpos, weight))
        check_outside(ybuf, before, y, self.pads[2])
        got = R.host(y)
        if in_place:
            self.x.copy_(torch.from_numpy(given).to(self.x.dtype))
        return given, got

    def backward(self, dweight=True, into=None, weight=None):
        """dX, dweight; `into`: "dy" or "x", where dX goes in its place."""
        import torch

        given = R.host(self.x), R.host(self.dy)
        obuf, dx = {None: lambda: strided(np.zeros(self.x.shape), self.kind, *self.pads),
                    "x": lambda: (self.buf, self.x), "dy": lambda: (self.dbuf, self.dy)}[into]()
        before, dpos = obuf.clone(), R.dev(self.pos.astype(np.int32))
        dw = torch.full((self.d + 2,), 7.0, device="cuda:0")
        p = self.mod.NormRopeGradParams(
            forward=self.params(self.x, None, dpos, weight), dY=R.ptr(self.dy), dy_token_stride=self.dy.stride(0),
            dy_head_stride=self.dy.stride(1), dX=R.ptr(dx), dx_token_stride=dx.stride(0),
            dx_head_stride=dx.stride(1), dweight=dw.data_ptr() + 4 if dweight else None)
        space, size = D.workspace(self.lib, "norm_rope_grad", p)
        assert dweight or size == 0
        D.run("norm_rope_grad_" + self.kind, p)
        assert torch.isnan(space[size // 4:]).all()
        check_outside(obuf, before, dx, self.pads[2])
        assert dw[0] == 7.0 and dw[-1] == 7.0 and (dweight or (dw == 7.0).all())
        return given, R.host(dx), R.host(dw[1:-1])

    def check(self, rows_in_f32=1, **kw):
        u, tiny = R.ROUND[self.kind]
        args = (self.pos, self.table, self.rot, self.inter, self.w, self.shift, self.eps)
        given, got = self.forward(**kw)
        want, tol = D.norm_rope(given, *args, inverse=self.inverse)
        assert (np.abs(got - want) <= tol + (np.abs(want) + tol) * u * 1.01 + tiny).all()
        (x, dy), dx, dw = self.backward(**{k: v for k, v in kw.items() if k == "weight"})
        want, want_w, tol, tol_w = D.norm_rope_grad(x, dy, *args, rows_in_f32, inverse=self.inverse)
        assert (np.abs(dx - want) <= tol + (np.abs(want) + tol) * u * 1.01 + tiny).all()
        assert (np.abs(dw - want_w) <= tol_w).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("tokens,heads,d,rot", SHAPES)
def test_shapes(gpu, kind, inter, tokens, heads, d, rot):
    # 12000 heads at most: up to 32768 rows (16 threads a head, 1024 workgroups) or 4096 (a wave a head)
    # are each a thread's only one
    Call(kind, tokens, heads, d, rot, inter).check(rows_in_f32=1 if tokens * heads <= 4096 else 3)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("weight,shift,inverse", [(False, 0.0, False), (False, 1.0, False), (True, 1.0, False),
                                                  (True, 0.0, True)])
@pytest.mark.parametrize("d,rot", [(64, 64), (72, 36)])
def test_weights(gpu, kind, weight, shift, inverse, d, rot):
    Call(kind, 7, 5, d, rot, weight=weight, shift=shift, inverse=inverse).check()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("pads", [(0, 16, 0), (16, 8, 8), (1, 0, 0), (0, 0, 1), (3, 5, 2)])
@pytest.mark.parametrize("inter", [False, True])
def test_strides_alignment_in_place(gpu, kind, pads, inter):
    c = Call(kind, 11, 6, 64, 48, inter, pads=pads)
    c.check()
    plain, dx = c.forward()[1], c.backward()[1]
    np.testing.assert_array_equal(c.forward(in_place=True)[1], plain)
    for into in ("dy", "x"):
        c = Call(kind, 11, 6, 64, 48, inter, pads=pads)
        np.testing.assert_array_equal(c.backward(into=into)[1], dx)
    c = Call(kind, 11, 6, 64, 48, inter, pads=pads)
    np.testing.assert_array_equal(c.backward(dweight=False)[1], dx)


def test_weight_off_the_grid(gpu):
    import torch

    c = Call("f16", 9, 4, 64, 64)
    w = torch.zeros(65, device="cuda:0")[1:]
    w.copy_(c.dw_)
    c.check(weight=w)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d", [128, 130])
def test_many_rows_give_the_same_bits(gpu, kind, d):
    """Several heads a thread: dweight's sums in a fixed order."""
    c = Call(kind, 1500, 24, d, 64)  # 36000 heads: 3 a thread with 8 a head, 9 a wave
    c.check(rows_in_f32=9)
    first = c.backward()
    for _ in range(3):
        again = c.backward()
        np.testing.assert_array_equal(first[1], again[1])
        np.testing.assert_array_equal(first[2], again[2])


@pytest.mark.parametrize("d", [64, 66])
def test_sizes_at_the_type_limits(gpu, d):
    """Squares that f32 does not hold, and rows so small that eps decides."""
    c = Call("f32", 4, 2, d, 32, size=1e30)
    given, got = c.forward()
    want, tol = D.norm_rope(given, c.pos, c.table, 32, False, c.w, 0.0, c.eps)
    # r is subnormal-free here (1e-30); the bound is the usual one
    assert (np.abs(got - want) <= tol + np.abs(want) * 2.0 ** -23).all()
    Call("bf16", 4, 2, d, 32, size=1e18).check()
    Call("f32", 4, 2, d, 32, size=1e-4, eps=1e-6).check()
    c = Call("f16", 4, 2, d, 32)
    c.x.zero_()
    assert (c.forward()[1] == 0).all()
    (_, dy), dx, dw = c.backward()
    assert np.isfinite(dx).all() and (dw == 0).all()


@pytest.mark.parametrize("d", [64, 60])
def test_values_that_are_no_numbers(gpu, d):
    """A head with a NaN is NaN, one with an infinity is NaN there and at its partner, else 0; others are as ever."""
    c = Call("f16", 3, 4, d, 32)
    _, plain = c.forward()
    c.x[1, 2, 5], c.x[2, 0, 40] = float("inf"), float("nan")
    _, got = c.forward()
    assert np.isnan(got[2, 0]).all() and np.isnan(got[1, 2, [5, 21]]).all()
    rest = np.ones(d, bool)
    rest[[5, 21]] = False
    assert (got[1, 2, rest] == 0).all()
    fine = np.ones((3, 4), bool)
    fine[1, 2] = fine[2, 0] = False
    np.testing.assert_array_equal(got[fine], plain[fine])


@pytest.mark.parametrize("d", [48, 47])
def test_position_outside_table(gpu, d):
    c = Call("f32", 5, 2, d, 32)
    c.pos = np.array([299, 300, -1, 2 ** 31 - 1, 0])
    _, y = c.forward()
    _, dx, dw = c.backward()
    for t, ok in enumerate([True, False, False, False, True]):
        assert np.isfinite(y[t]).all() if ok else np.isnan(y[t, :, :32]).all() and np.isfinite(y[t, :, 32:]).all()
        assert np.isfinite(dx[t]).all() if ok else np.isnan(dx[t]).all()
    assert np.isnan(dw[:32]).all() and np.isfinite(dw[32:]).all()


@pytest.mark.parametrize("d,rot", [(64, 64), (30, 18)])
def test_gradient_against_differences(gpu, d, rot):
    """The kernel's gradient in a direction against differences of the forward pass in 64 bits."""
    c = Call("f32", 6, 3, d, rot)
    (x, dy), dx, dw = c.backward()
    rng = np.random.default_rng(1)
    v, vw = rng.standard_normal(x.shape), rng.standard_normal(d)
    loss = lambda h: (D.norm_rope(x + h * v, c.pos, c.table, rot, False, c.w + h * vw, 0.0,  # noqa: E731
                                  c.eps)[0] * dy).sum()
    h = 1e-5
    diff = (loss(h) - loss(-h)) / (2 * h)
    _, _, tol, tol_w = D.norm_rope_grad(x, dy, c.pos, c.table, rot, False, c.w, 0.0, c.eps, 1)
    size = np.abs(dx * v).sum() + np.abs(dw * vw).sum()
    # the bounds of each gradient, its rounding, and the difference's own error (h^2, 2^-53 / h)
    bound = (tol * np.abs(v)).sum() + (tol_w * np.abs(vw)).sum() + size * (2.0 ** -24 + 1e-7)
    assert abs(diff - (dx * v).sum() - (dw * vw).sum()) <= bound


def test_nothing_to_do(gpu):
    import torch

    mod, lib = R.binding()
    run = lib.op("norm_rope_f16", "run")
    run(ctypes.byref(mod.NormRopeParams(rope=mod.RopeParams(tokens=0, heads=4, head_dim=64))))
    dw = torch.full((64,), 7.0, device="cuda:0")
    p = mod.NormRopeGradParams(dweight=dw.data_ptr())
    p.forward.rope = mod.RopeParams(tokens=0, heads=4, head_dim=64)
    lib.op("norm_rope_grad_f16", "run")(ctypes.byref(p))
    assert (dw == 0).all()  # the sum of no rows


# ------------------------------------------------------------------------------------------
# On the way into a cache
# ------------------------------------------------------------------------------------------

def run_append(name, tokens, heads, kv_heads, d, rot, inter=False, page=16, weights=(True, True), shift=0.0,
               pad=0, heads_first=False, stream=None):
    """A call with slots all over the cache, a negative one and one past it among them; returns what a check needs."""
    import torch

    mod, lib = R.binding()
    cache, src = name.split("_")
    rng = np.random.default_rng(tokens + d + heads)
    n = heads + 2 * kv_heads
    qkv = R.dev(rng.standard_normal((tokens, n, d)) * 2, src)
    if pad:
        wide = torch.zeros((tokens, n, d + pad), dtype=qkv.dtype, device="cuda:0")
        wide[..., :d] = qkv
        qkv = wide[..., :d]
    pages = tokens // page + 4
    shape = (pages, kv_heads, page, d) if heads_first else (pages, page, kv_heads, d)
    k, v = (torch.full(shape, 5, dtype=R.torch_type(cache), device="cuda:0") for _ in range(2))
    sk = sv = None
    if cache == "qsi8dx":
        sk, sv = (torch.full((pages, kv_heads, page), 5.0, device="cuda:0") for _ in range(2))
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 2:
        slots[1], slots[2] = -1, pages * page
    pos = rng.integers(0, 200, tokens).astype(np.int32)
    table = R.rope_table(200, rot).astype(np.float32) if rot else None
    w = [(rng.standard_normal(d) * 0.3 + 1 - shift).astype(np.float32) if on else None for on in weights]
    qo = torch.full((tokens, max(heads, 1), d), 5.0, device="cuda:0",
                    dtype=R.torch_type(cache if src == "f32" else src))
    keep = [R.dev(x) if x is not None else None for x in (slots, pos, table, *w)]
    at = lambda h: qkv.data_ptr() + h * qkv.stride(1) * qkv.element_size()  # noqa: E731
    p = mod.KVAppendNormRopeParams(
        append=mod.KVAppendRopeParams(
            tokens=tokens, K=at(heads), k_token_stride=qkv.stride(0), k_head_stride=qkv.stride(1),
            V=at(heads + kv_heads), v_token_stride=qkv.stride(0), v_head_stride=qkv.stride(1), q_heads=heads,
            Q=at(0) if heads else None, q_token_stride=qkv.stride(0), q_head_stride=qkv.stride(1), Q_out=R.ptr(qo),
            qo_token_stride=qo.stride(0), qo_head_stride=qo.stride(1), positions=R.ptr(keep[1]),
            slots=R.ptr(keep[0]), map=R.rope_map(mod, keep[2], rot, inter),
            kv=R.paged(mod, k, v, sk, sv, heads_first=heads_first)),
        q_norm=D.head_norm(mod, keep[3], shift, 1e-5), k_norm=D.head_norm(mod, keep[4], shift, 1e-5))
    if not heads:
        p.q_norm = mod.HeadNorm()
    D.run("kv_append_norm_rope_" + name, p, stream)
    x = R.host(qkv)
    args = (pos, table, rot, inter)
    q, tq = D.norm_rope(x[:, :heads], *args, w[0], shift, 1e-5)
    kk, tk = D.norm_rope(x[:, heads:heads + kv_heads], *args, w[1], shift, 1e-5)
    vv = x[:, heads + kv_heads:]
    if heads_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return slots, page, (qo, q, tq), (k, sk, kk, tk), (v, sv, vv, np.zeros_like(vv)), heads


def check_append(name, *a, **kw):
    cache, src = name.split("_")
    slots, page, (qo, q, tq), k, v, heads = run_append(name, *a, **kw)
    if heads:
        u, tiny = R.ROUND[cache if src == "f32" else src]
        got = R.host(qo)
        assert (np.abs(got - q) <= tq + (np.abs(q) + tq) * u * 1.01 + tiny).all()
    for c, s, want, tol in (k, v):
        got = R.host(c).reshape(-1, *c.shape[2:])
        ok = (slots >= 0) & (slots < got.shape[0])
        at, want, tol = slots[ok], want[ok], tol[ok]
        untouched = np.ones(got.shape[0], bool)
        untouched[at] = False
        assert (got[untouched] == 5).all()
        if cache == "qsi8dx":
            sc = R.host(s).transpose(0, 2, 1).reshape(got.shape[:2])
            assert (sc[untouched] == 5).all()
            amax = np.abs(want).max(-1)
            # a scale is amax / 127 with two roundings, a value off by half a step at most beside its row's error (which
            # the quotient may carry over the border of a step)
            assert (np.abs(sc[at] - amax / 127) <= (tol.max(-1) + amax * 3 * 2.0 ** -24) / 127).all()
            got = got * sc[..., None]
            step = sc[at][..., None]
            assert (np.abs(got[at] - want) <= step * (0.5 + 127 * 2.0 ** -22) + tol).all()
        else:
            u, tiny = R.ROUND[cache]
            assert (np.abs(got[at] - want) <= tol + (np.abs(want) + tol) * u * 1.01 + tiny).all()


APPENDS = ["f16_f16", "bf16_bf16", "f16_f32", "bf16_f32", "qsi8dx_f16", "qsi8dx_bf16"]


@pytest.mark.parametrize("name", APPENDS)
@pytest.mark.parametrize("tokens,heads,kv_heads,d,rot,inter", [
    (1, 32, 8, 128, 128, False), (7, 4, 2, 64, 32, True), (33, 3, 3, 80, 80, False), (5, 0, 2, 96, 96, False),
    (70, 6, 1, 256, 64, True), (3, 2, 1, 16, 0, False), (4, 4, 2, 192, 192, False), (6, 2, 2, 80, 40, True),
    (200, 8, 4, 64, 64, False)])
def test_append(gpu, name, tokens, heads, kv_heads, d, rot, inter):
    check_append(name, tokens, heads, kv_heads, d, rot, inter)


@pytest.mark.parametrize("name", APPENDS)
def test_append_weights_strides_layout(gpu, name):
    check_append(name, 9, 4, 2, 64, 64, weights=(False, True))
    check_append(name, 9, 4, 2, 64, 64, weights=(True, False), shift=1.0)
    check_append(name, 9, 4, 2, 64, 64, pad=16, page=24)
    check_append(name, 9, 4, 2, 64, 64, pad=3, heads_first=True)


def test_append_rows_that_are_no_numbers(gpu):
    """As in the append without a norm: an int8 row with a NaN or an infinity gets a NaN for its scale."""
    import torch

    mod, lib = R.binding()
    x = torch.ones((2, 1, 32), dtype=torch.float16, device="cuda:0")
    x[0, 0, 3], x[1, 0, 4] = float("nan"), float("inf")
    k, v = (torch.zeros((1, 16, 1, 32), dtype=torch.int8, device="cuda:0") for _ in range(2))
    sk, sv = (torch.zeros((1, 1, 16), device="cuda:0") for _ in range(2))
    slots = torch.tensor([3, 4], device="cuda:0")
    a = mod.KVAppendRopeParams(tokens=2, K=R.ptr(x), k_token_stride=32, k_head_stride=32, V=R.ptr(x),
                               v_token_stride=32, v_head_stride=32, slots=R.ptr(slots), kv=R.paged(mod, k, v, sk, sv))
    p = mod.KVAppendNormRopeParams(append=a, k_norm=mod.HeadNorm(eps=1e-5))
    D.run("kv_append_norm_rope_qsi8dx_f16", p)
    assert torch.isnan(sk[0, 0, 3:5]).all() and torch.isnan(sv[0, 0, 3:5]).all()
    assert (sk[0, 0, :3] == 0).all() and (sk[0, 0, 5:] == 0).all()


def test_on_another_stream_and_in_a_graph(gpu):
    """Forward and gradient captured together and replayed with new rows."""
    import torch

    c = Call("bf16", 40, 8, 128, 128)
    mod, lib = c.mod, c.lib
    y, dx = torch.empty_like(c.x), torch.empty_like(c.x)
    dw, dpos = torch.empty(128, device="cuda:0"), R.dev(c.pos.astype(np.int32))
    f = c.params(c.x, y, dpos)
    g = mod.NormRopeGradParams(forward=f, dY=R.ptr(c.dy), dy_token_stride=c.dy.stride(0),
                               dy_head_stride=c.dy.stride(1), dX=R.ptr(dx), dx_token_stride=dx.stride(0),
                               dx_head_stride=dx.stride(1), dweight=dw.data_ptr())
    space, _ = D.workspace(lib, "norm_rope_grad", g)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        s = torch.cuda.current_stream().cuda_stream
        D.run("norm_rope_bf16", f, s)
        D.run("norm_rope_grad_bf16", g, s)
    for seed in range(3):
        c.x.normal_()
        for t in (y, dx, dw, space):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        (_, _), want_dx, want_dw = c.backward()
        np.testing.assert_array_equal(R.host(y), c.forward()[1])
        np.testing.assert_array_equal(R.host(dx), want_dx)
        np.testing.assert_array_equal(R.host(dw), want_dw)
