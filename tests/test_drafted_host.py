"""The checks of the operators of a step with drafted tokens that need no GPU: the binding's structs lie as the headers'
do, what the operators refuse is refused with its reason before anything is launched, launch rules, and the
plain forms that the GPU tests compare with."""

import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R
import test_paged_host as H

ROOT = H.ROOT
STRUCTS = {"tqt_head_norm": "HeadNorm", "tqt_norm_rope_params": "NormRopeParams",
           "tqt_norm_rope_grad_params": "NormRopeGradParams",
           "tqt_kv_append_norm_rope_params": "KVAppendNormRopeParams",
           "tqt_paged_plan_params": "PagedPlanParams", "tqt_kv_keep_params": "KVKeepParams",
           "tqt_attn_tree_params": "AttnTreeParams"}
HEADERS = ["tqt_kv_append_norm_rope_gfx950.h", "tqt_paged_plan_gfx950.h", "tqt_kv_keep_gfx950.h",
           "tqt_attn_tree_gfx950.h"]


@pytest.mark.skipif(not os.path.exists(H.CLANG), reason="no C compiler")
def test_structs_lie_as_the_headers_say(tmp_path):
    mod, _ = R.binding()
    lines = []
    for c, py in STRUCTS.items():
        lines.append('printf("%s %%zu\\n", sizeof(struct %s));' % (c, c))
        for field, _ in getattr(mod, py)._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(struct %s, %s));' % (c, field, c, field))
    src = tmp_path / "lay.c"
    src.write_text("%s\n#include <stdio.h>\nint main(void){%s return 0;}\n" % (
        "\n".join('#include "%s"' % h for h in HEADERS), "\n".join(lines)))
    subprocess.run([H.CLANG, "-std=c11", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), "-o",
                    str(tmp_path / "lay"), str(src)], check=True)
    out = subprocess.run([str(tmp_path / "lay")], capture_output=True, text=True, check=True).stdout
    said = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for c, py in STRUCTS.items():
        cls = getattr(mod, py)
        assert int(said[c]) == ctypes.sizeof(cls), c
        for field, _ in cls._fields_:
            assert int(said["%s.%s" % (c, field)]) == getattr(cls, field).offset, (c, field)


def norm_params():
    mod, _ = R.binding()
    return mod.NormRopeParams(rope=H.rope_params(), norm=mod.HeadNorm(weight=4096, shift=0.0, eps=1e-6))


NORMS = ["norm_rope_" + k for k in ("f32", "f16", "bf16")]
ROPE_REFUSED = [dict(X=None), dict(positions=None), dict(map__table=None), dict(map__rotary_dim=63),
                dict(map__rotary_dim=66), dict(map__max_pos=0), dict(tokens=2 ** 31), dict(heads=2 ** 20),
                dict(head_dim=2 ** 20)]
NAN, INF = float("nan"), float("inf")
NORM_REFUSED = [dict(eps=0.0), dict(eps=-1.0), dict(eps=NAN), dict(eps=INF), dict(shift=INF), dict(shift=NAN)]


def inside(prefix, changes):
    return [{prefix + "__" + k: v for k, v in c.items()} for c in changes]


@pytest.mark.parametrize("change", inside("rope", ROPE_REFUSED + [dict(Y=None)]) + inside("norm", NORM_REFUSED))
def test_norm_refusals(change):
    for name in NORMS:
        assert H.refusal(name, norm_params()) is None
        assert H.refusal(name, H.changed(norm_params, **change))


@pytest.mark.parametrize("change", [dict(rope__tokens=0, norm__eps=0.0), dict(rope__heads=0), dict(norm__weight=None),
                                    dict(norm__weight=4100), dict(norm__shift=1.0), dict(rope__X=4097),
                                    dict(rope__head_dim=4096, rope__map__rotary_dim=0)])
def test_norm_takes(change):
    for name in NORMS:
        assert H.refusal(name, H.changed(norm_params, **change)) is None


def grad_params():
    mod, _ = R.binding()
    p = mod.NormRopeGradParams(forward=norm_params(), dY=4096, dy_token_stride=128, dy_head_stride=64, dX=8192,
                               dx_token_stride=128, dx_head_stride=64, dweight=4096, workspace=4096,
                               workspace_size=1 << 30)
    p.forward.rope.Y = None
    return p


GRADS = ["norm_rope_grad_" + k for k in ("f32", "f16", "bf16")]


@pytest.mark.parametrize("change", inside("forward__rope", ROPE_REFUSED) + inside("forward__norm", NORM_REFUSED) + [
    dict(dY=None), dict(dX=None), dict(workspace=None), dict(workspace=4100), dict(workspace_size=0),
    dict(forward__rope__tokens=2 ** 20, forward__rope__heads=2 ** 11)])
def test_grad_refusals(change):
    for name in GRADS:
        assert H.refusal(name, grad_params()) is None
        assert H.refusal(name, H.changed(grad_params, **change))


def test_grad_takes():
    for name in GRADS:
        for change in (dict(dweight=None, workspace=None, workspace_size=0),
                       dict(forward__rope__tokens=0, forward__rope__X=None, dY=None, dX=None, workspace=None,
                            workspace_size=0), dict(forward__rope__head_dim=0), dict(dY=4097)):
            assert H.refusal(name, H.changed(grad_params, **change)) is None, change


def append_norm_params():
    mod, _ = R.binding()
    n = lambda: mod.HeadNorm(weight=4096, shift=0.0, eps=1e-6)  # noqa: E731
    return mod.KVAppendNormRopeParams(append=H.append_params(), q_norm=n(), k_norm=n())


APPENDS = ["kv_append_norm_rope_" + k for k in H.APPENDS]


@pytest.mark.parametrize("change", inside("append", H.KV_REFUSED + [
    dict(K=None), dict(V=None), dict(slots=None), dict(positions=None), dict(Q=None), dict(Q_out=None),
    dict(map__table=None), dict(map__rotary_dim=65), dict(tokens=2 ** 31), dict(q_heads=2 ** 20)]) +
    inside("q_norm", NORM_REFUSED) + inside("k_norm", NORM_REFUSED))
def test_append_refusals(change):
    for name in APPENDS:
        assert H.refusal(name, append_norm_params()) is None
        assert H.refusal(name, H.changed(append_norm_params, **change)), name


def test_append_takes():
    for name in APPENDS:
        for change in (dict(append__tokens=0, k_norm__eps=0.0),
                       dict(append__q_heads=0, append__Q=None, append__Q_out=None, q_norm__eps=0.0),
                       dict(q_norm__weight=None, k_norm__weight=None), dict(k_norm__weight=4100)):
            assert H.refusal(name, H.changed(append_norm_params, **change)) is None, (name, change)
        int8 = "qsi8dx" in name
        assert bool(H.refusal(name, H.changed(append_norm_params, append__kv__scale_k=None))) == int8


def plan_params():
    mod, _ = R.binding()
    arrays = ("new_len kv_len kv_len_out held held_out block_table free_pages free_count free_count_out refused q_start "
              "positions slots").split()
    return mod.PagedPlanParams(batch=3, tokens=7, page_size=16, num_pages=9, ld_table=4, free_capacity=9,
                               **{k: 4096 + 256 * i for i, k in enumerate(arrays)})


@pytest.mark.parametrize("change", [{k: None} for k in (
    "new_len kv_len kv_len_out held held_out block_table free_pages free_count free_count_out refused q_start "
    "positions slots").split()] + [
    dict(batch=2 ** 16), dict(tokens=2 ** 30), dict(page_size=0), dict(num_pages=2 ** 31),
    dict(num_pages=2 ** 20, page_size=2 ** 11), dict(ld_table=2 ** 31), dict(free_capacity=2 ** 31),
    dict(mask=4096), dict(parent=4096), dict(ld_mask=1), dict(parent=4096, mask=4096),
    dict(parent=4096, ld_mask=1), dict(parent=4096, mask=4096, ld_mask=2 ** 25),
    dict(tokens=2 ** 20), dict(batch=2000, workspace=4100, workspace_size=1 << 20)])
def test_plan_refusals(change):
    assert H.refusal("paged_plan", plan_params()) is None
    assert H.refusal("paged_plan", H.changed(plan_params, **change))


@pytest.mark.parametrize("change", [
    dict(batch=0, new_len=None, kv_len=None, kv_len_out=None, held=None, held_out=None, block_table=None),
    dict(tokens=0, positions=None, slots=None), dict(free_capacity=0, free_pages=None),
    dict(ld_table=0, block_table=None), dict(num_pages=0), dict(parent=4096, mask=4096, ld_mask=1),
    dict(tokens=2 ** 20, workspace=4096, workspace_size=48)])
def test_plan_takes(change):
    assert H.refusal("paged_plan", H.changed(plan_params, **change)) is None


def keep_params():
    mod, _ = R.binding()
    return mod.KVKeepParams(batch=3, max_keep=4, q_start=4096, kv_len=8192, kv_len_out=12288, keep=4096, ld_keep=4,
                            keep_len=4096, block_table=4096, ld_table=4, layers=2, layer_stride=8192,
                            scale_layer_stride=128, kv=H.paged_kv())


KEEPS = ["kv_keep_" + k for k in ("f16", "bf16", "qsi8dx")]


@pytest.mark.parametrize("change", H.KV_REFUSED + [
    dict(q_start=None), dict(kv_len=None), dict(keep=None), dict(keep_len=None), dict(block_table=None),
    dict(batch=2 ** 16), dict(layers=2 ** 16), dict(max_keep=2 ** 31, ld_keep=2 ** 31), dict(ld_table=2 ** 31),
    dict(max_keep=5), dict(layer_stride=8193), dict(kv_len_out=8192), dict(kv_len_out=8200), dict(kv_len_out=8184),
    dict(batch=2 ** 15, layers=2 ** 15), dict(slots=4096, tokens=2 ** 31)])
def test_keep_refusals(change):
    for name in KEEPS:
        assert H.refusal(name, keep_params()) is None
        assert H.refusal(name, H.changed(keep_params, **change)), name


def test_keep_takes():
    for name in KEEPS:
        for change in (dict(batch=0, q_start=None), dict(layers=0, kv_len=None), dict(kv_len_out=None),
                       dict(max_keep=0, keep=None), dict(layers=1, layer_stride=3), dict(kv_len_out=8204),
                       dict(slots=4096, tokens=7), dict(slots=None, tokens=2 ** 31)):
            assert H.refusal(name, H.changed(keep_params, **change)) is None, (name, change)


def tree_params():
    mod, _ = R.binding()
    return mod.AttnTreeParams(attn=H.attn_params(), mask=4096, ld_mask=1)


TREES = ["attn_tree_" + k for k in H.ATTNS]


@pytest.mark.parametrize("change", inside("attn", H.KV_REFUSED + [
    dict(Q=None), dict(D=None), dict(q_start=None), dict(kv_len=None), dict(block_table=None), dict(q_heads=5),
    dict(max_kv_len=65), dict(Q=4104), dict(D=4100), dict(q_token_stride=260), dict(d_head_stride=65),
    dict(scale=NAN), dict(scale=INF), dict(causal=0), dict(causal=2), dict(batch=2 ** 24),
    dict(q_tokens=2 ** 31)]) + [
    dict(mask=None), dict(ld_mask=0), dict(ld_mask=2 ** 25), dict(attn__max_q_len=33)])
def test_tree_refusals(change):
    base = lambda: H.changed(tree_params, attn__max_kv_len=64, attn__batch=2)  # noqa: E731
    for name in TREES:
        assert H.refusal(name, base()) is None
        assert H.refusal(name, H.changed(base, **change)), name


@pytest.mark.parametrize("change", inside("attn", [dict(workspace=None), dict(workspace=4100),
                                                   dict(workspace_size=0)]))
def test_tree_workspace(change):
    """Keys that are split need a workspace; spans that one workgroup takes whole need none."""
    long = lambda: H.changed(tree_params, attn__max_kv_len=2 ** 16, attn__ld_table=2 ** 12)  # noqa: E731
    short = lambda: H.changed(tree_params, attn__max_kv_len=64)  # noqa: E731
    _, lib = R.binding()
    size = lib.op("attn_tree", "get_workspace_size")
    assert size(ctypes.byref(long())) > 0 and size(ctypes.byref(short())) == 0
    for name in TREES:
        assert H.refusal(name, long()) is None
        assert H.refusal(name, H.changed(long, **change)), name
        assert H.refusal(name, H.changed(short, **change)) is None, name


def test_tree_takes():
    for name in TREES:
        for change in (dict(attn__batch=0, attn__Q=None, mask=None), dict(attn__max_q_len=0, ld_mask=0),
                       dict(attn__window=2 ** 40), dict(attn__scale=-1.0), dict(attn__max_q_len=32)):
            assert H.refusal(name, H.changed(tree_params, **change)) is None, (name, change)


def test_null_params():
    _, lib = R.binding()
    for name in NORMS + GRADS + APPENDS + ["paged_plan"] + KEEPS + TREES:
        assert lib.op(name, "get_error")(None)
        lib.op(name, "run_async")(None, None)  # returns at once
        lib.op(name, "run")(None)
    for name in ("norm_rope_grad", "paged_plan", "attn_tree"):
        assert lib.op(name, "get_workspace_size")(None) == 0


@pytest.mark.parametrize("name,build,change", [
    ("norm_rope_f16", "norm_params", dict(norm__eps=0.0)), ("norm_rope_grad_f32", "grad_params", dict(dX=None)),
    ("kv_append_norm_rope_f16_f16", "append_norm_params", dict(append__slots=None)),
    ("paged_plan", "plan_params", dict(page_size=0)), ("kv_keep_qsi8dx", "keep_params", dict(keep=None)),
    ("attn_tree_f16_f16", "tree_params", dict(mask=None))])
def test_a_refused_run_aborts_with_its_reason(name, build, change):
    code = ("import sys, ctypes; sys.path.insert(0, %r); import paged_ref as R, test_drafted_host as T\n"
            "p = T.H.changed(T.%s, **%r); R.binding()[1].op(%r, 'run_async')(ctypes.byref(p), None)\n"
            "print('returned')" % (os.path.join(ROOT, "tests"), build, change, name))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == -6 and "returned" not in r.stdout
    assert H.refusal(name, H.changed(globals()[build], **change)).decode() in r.stderr


# ------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("shift", [0.0, 1.0])
def test_gradient_of_the_plain_form_is_that_of_differences(inter, inverse, shift):
    rng = np.random.default_rng(3)
    x, dy, v = rng.standard_normal((3, 5, 4, 24))
    w, vw = rng.standard_normal((2, 24))
    table, pos = R.rope_table(40, 16) * 1.2, rng.integers(0, 40, 5)
    loss = lambda h: (D.norm_rope(x + h * v, pos, table, 16, inter, w + h * vw, shift, 1e-3,  # noqa: E731
                                  inverse)[0] * dy).sum()
    dx, dw, _, _ = D.norm_rope_grad(x, dy, pos, table, 16, inter, w, shift, 1e-3, 1, inverse)
    h = 1e-5  # the difference's own error: h^2 of a third derivative, and 2^-53 / h of the sum
    assert abs((loss(h) - loss(-h)) / (2 * h) - (dx * v).sum() - (dw * vw).sum()) < 1e-7 * np.abs(dx * v).sum()


def test_plan_of_a_small_step_by_hand():
    """Page size 4; sequence 0 grows by one token into its last page, 1 takes two pages, 2 has ended, 3 asks for more
    than is left, 4 needs none."""
    table = np.array([[5, 6, -1, -1], [7, -1, -1, -1], [8, -1, 9, -1], [-1, -1, -1, -1], [4, -1, -1, -1]], np.int32)
    free = np.array([0, 1, 0, 0, 0, 0], np.int32)
    got = D.plan(np.array([1, 6, -1, 9, 2]), np.array([6, 4, 9, 0, 1]), np.array([2, 1, 3, 0, 1]), table, free, 2, 20,
                 4, 10)
    # 8 and 9 go on the stack (0 1 8 9); 1 takes 9, 8; 3 needs 3 of the 2 left
    assert got["table"].tolist() == [[5, 6, -1, -1], [7, 9, 8, -1], [8, -1, 9, -1], [-1, -1, -1, -1], [4, -1, -1, -1]]
    assert got["free"].tolist() == [0, 1, 8, 9, 0, 0] and got["free_count_out"] == [2] and got["refused"] == [1]
    assert got["kv_len_out"].tolist() == [7, 10, 0, 0, 3] and got["held_out"].tolist() == [2, 3, 0, 0, 1]
    assert got["q_start"].tolist() == [0, 1, 7, 7, 16, 18]
    assert got["slots"].tolist() == [26, 36, 37, 38, 39, 32, 33] + [-1] * 9 + [17, 18, -1, -1]
    assert got["positions"].tolist() == [6, 4, 5, 6, 7, 8, 9] + list(range(9)) + [1, 2, 0, 0]


def test_tree_of_a_small_step_by_hand():
    parent = np.array([-1, 0, 0, 1, 5, -7, 2], np.int32)  # token 4's parent lies after it, 5's is no token: -1
    table = np.array([[3, 1]], np.int32)
    got = D.plan(np.array([7]), np.array([5]), np.array([2]), table, np.zeros(1, np.int32), 0, 7, 8, 4, parent, 1)
    assert got["mask"][:, 0].tolist() == [1, 3, 5, 11, 16, 32, 69]
    assert got["positions"].tolist() == [5, 6, 6, 7, 5, 5, 7]
    assert got["slots"].tolist() == [29, 30, 31, 8, 9, 10, 11]
    see = D.visible_tree(got["mask"], 7, 12, 0)
    assert see[3].nonzero()[0].tolist() == [0, 1, 2, 3, 4, 5, 6, 8]
    assert D.visible_tree(got["mask"], 7, 12, 4)[3].nonzero()[0].tolist() == [4, 5, 6, 8]


def test_kept_lists():
    assert D.kept([0, 2, 5, 6], 4, 7, 4) == [0, 2, 5, 6]
    assert D.kept([0, 2, 2, 6], 4, 7, 4) == [0, 2]
    assert D.kept([0, 2, 7, 8], 4, 7, 4) == [0, 2]
    assert D.kept([-1, 2], 2, 7, 4) == []
    assert D.kept([1, 2, 3], 3, 7, 2) == [1, 2]
    assert D.kept([1, 2, 3], -3, 7, 2) == []
