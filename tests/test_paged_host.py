"""The rotary, cache-append and attention operators' checks that need no GPU: the binding's structs lie as the
headers' do, and what the operators refuse is refused with its reason before anything is launched."""

import ctypes
import os
import subprocess
import sys

import pytest

import paged_ref as R

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang"
STRUCTS = {"tqt_rope_map": "RopeMap", "tqt_rope_params": "RopeParams",
           "tqt_rope_table_params": "RopeTableParams", "tqt_paged_kv": "PagedKV",
           "tqt_kv_append_rope_params": "KVAppendRopeParams", "tqt_attn_paged_params": "AttnPagedParams"}


@pytest.mark.skipif(not os.path.exists(CLANG), reason="no C compiler")
def test_structs_lie_as_the_headers_say(tmp_path):
    mod, _ = R.binding()
    lines = []
    for c, py in STRUCTS.items():
        lines.append('printf("%s %%zu\\n", sizeof(struct %s));' % (c, c))
        for field, _ in getattr(mod, py)._fields_:
            lines.append('printf("%s.%s %%zu\\n", offsetof(struct %s, %s));' % (c, field, c, field))
    src = tmp_path / "lay.c"
    src.write_text('#include "tqt_attn_paged_gfx950.h"\n#include <stdio.h>\nint main(void){%s return 0;}\n'
                   % "\n".join(lines))
    subprocess.run([CLANG, "-std=c11", "-Wall", "-Werror", "-I" + os.path.join(ROOT, "include"), "-o",
                    str(tmp_path / "lay"), str(src)], check=True)
    out = subprocess.run([str(tmp_path / "lay")], capture_output=True, text=True, check=True).stdout
    said = dict(line.rsplit(" ", 1) for line in out.splitlines())
    for c, py in STRUCTS.items():
        cls = getattr(mod, py)
        assert int(said[c]) == ctypes.sizeof(cls), c
        for field, _ in cls._fields_:
            assert int(said["%s.%s" % (c, field)]) == getattr(cls, field).offset, (c, field)


def refusal(name, p):
    _, lib = R.binding()
    return lib.op(name, "get_error")(ctypes.byref(p))


def changed(build, **changes):
    p = build()
    for path, value in changes.items():
        at, *names = p, *path.split("__")
        for n in names[:-1]:
            at = getattr(at, n)
        setattr(at, names[-1], value)
    return p


def rope_params():
    mod, _ = R.binding()
    return mod.RopeParams(tokens=3, heads=2, head_dim=64, X=4096, x_token_stride=128, x_head_stride=64,
                          Y=8192, y_token_stride=128, y_head_stride=64, positions=16,
                          map=mod.RopeMap(table=4096, max_pos=10, rotary_dim=64))


@pytest.mark.parametrize("change", [
    dict(X=None), dict(Y=None), dict(positions=None), dict(map__table=None), dict(map__rotary_dim=63),
    dict(map__rotary_dim=66), dict(map__max_pos=0), dict(map__max_pos=2 ** 31), dict(tokens=2 ** 31),
    dict(heads=2 ** 20), dict(head_dim=2 ** 20)])
def test_rope_refusals(change):
    for kind in ("f32", "f16", "bf16"):
        assert refusal("rope_" + kind, rope_params()) is None
        assert refusal("rope_" + kind, changed(rope_params, **change))


@pytest.mark.parametrize("change", [dict(), dict(tokens=0, X=None), dict(heads=0), dict(head_dim=0),
                                    dict(map__rotary_dim=0, map__table=None, positions=None),
                                    dict(X=4097), dict(x_head_stride=65), dict(x_head_stride=0)])
def test_rope_takes(change):
    assert refusal("rope_f16", changed(rope_params, **change)) is None


def append_params():
    mod, _ = R.binding()
    return mod.KVAppendRopeParams(
        tokens=3, K=4096, k_token_stride=128, k_head_stride=64, V=4096, v_token_stride=128,
        v_head_stride=64, q_heads=4, Q=4096, q_token_stride=256, q_head_stride=64, Q_out=4096,
        qo_token_stride=256, qo_head_stride=64, positions=16, slots=16,
        map=mod.RopeMap(table=4096, max_pos=10, rotary_dim=64), kv=paged_kv())


def paged_kv():
    mod, _ = R.binding()
    return mod.PagedKV(k=4096, v=8192, scale_k=16, scale_v=16, num_pages=4, page_size=16, kv_heads=2,
                       head_dim=64, page_stride=2048, token_stride=128, head_stride=64)


KV_REFUSED = [dict(kv__k=None), dict(kv__v=None), dict(kv__page_size=0), dict(kv__kv_heads=0),
              dict(kv__head_dim=0), dict(kv__head_dim=72), dict(kv__head_dim=272), dict(kv__k=4104),
              dict(kv__v=4100), dict(kv__page_stride=2044), dict(kv__token_stride=132),
              dict(kv__head_stride=63), dict(kv__num_pages=2 ** 31),
              dict(kv__num_pages=2 ** 20, kv__page_size=2 ** 11), dict(kv__kv_heads=2 ** 16)]
APPENDS = ["f16_f16", "bf16_bf16", "f16_f32", "bf16_f32", "qsi8dx_f16", "qsi8dx_bf16"]


@pytest.mark.parametrize("change", KV_REFUSED + [
    dict(K=None), dict(V=None), dict(slots=None), dict(positions=None), dict(Q=None), dict(Q_out=None),
    dict(map__table=None), dict(map__rotary_dim=65), dict(tokens=2 ** 31), dict(q_heads=2 ** 20)])
def test_append_refusals(change):
    for kind in APPENDS:
        assert refusal("kv_append_rope_" + kind, append_params()) is None
        assert refusal("kv_append_rope_" + kind, changed(append_params, **change)), kind


def test_append_scales_and_int8_grid():
    for kind in APPENDS:
        int8 = kind.startswith("qsi8dx")
        for change in (dict(kv__scale_k=None), dict(kv__scale_v=None), dict(kv__head_stride=72)):
            assert bool(refusal("kv_append_rope_" + kind, changed(append_params, **change))) == int8
        assert refusal("kv_append_rope_" + kind, changed(append_params, q_heads=0, Q=None, Q_out=None)) is None
        assert refusal("kv_append_rope_" + kind, changed(append_params, K=4097, k_head_stride=65)) is None


def attn_params():
    mod, lib = R.binding()
    p = mod.AttnPagedParams(
        batch=2, q_tokens=2, q_heads=4, max_q_len=1, max_kv_len=64, Q=4096, q_token_stride=256,
        q_head_stride=64, D=8192, d_token_stride=256, d_head_stride=64, lse=None, q_start=16, kv_len=16,
        block_table=16, ld_table=4, scale=0.125, causal=1, window=0, kv=paged_kv())
    p.workspace, p.workspace_size = 4096, 1 << 40
    return p


ATTNS = ["f16_f16", "bf16_bf16", "f16_qsi8dx", "bf16_qsi8dx"]


@pytest.mark.parametrize("change", KV_REFUSED + [
    dict(Q=None), dict(D=None), dict(q_start=None), dict(kv_len=None), dict(block_table=None),
    dict(q_heads=5), dict(q_heads=2 ** 16), dict(max_kv_len=65), dict(Q=4104), dict(D=4100),
    dict(q_token_stride=260), dict(q_head_stride=65), dict(d_token_stride=260), dict(d_head_stride=65),
    dict(scale=float("nan")), dict(scale=float("inf")), dict(window=5, causal=0), dict(batch=2 ** 24),
    dict(q_tokens=2 ** 31), dict(max_q_len=2 ** 31), dict(max_q_len=2 ** 30 + 1)])
def test_attention_refusals(change):
    for kind in ATTNS:
        assert refusal("attn_paged_" + kind, attn_params()) is None
        assert refusal("attn_paged_" + kind, changed(attn_params, **change)), kind


def test_attention_takes():
    for kind in ATTNS:
        for change in (dict(batch=0, Q=None), dict(q_tokens=0, Q=None), dict(q_heads=0, Q=None),
                       dict(max_kv_len=0, block_table=None), dict(window=2 ** 40), dict(scale=-1.0)):
            assert refusal("attn_paged_" + kind, changed(attn_params, **change)) is None, (kind, change)


def test_null_params():
    _, lib = R.binding()
    for name in (["rope_f32", "rope_table_f32"] + ["kv_append_rope_" + k for k in APPENDS] +
                 ["attn_paged_" + k for k in ATTNS]):
        assert lib.op(name, "get_error")(None)
        lib.op(name, "run_async")(None, None)  # returns at once
        lib.op(name, "run")(None)


@pytest.mark.parametrize("change", [dict(table=None), dict(rotary_dim=3), dict(base=1.0),
                                    dict(base=float("nan")), dict(scaling=5), dict(scaling=-1),
                                    dict(factor=0.0), dict(scaling=3, low_turns=0.0),
                                    dict(scaling=4, high_turns=1.0), dict(scaling=3, original_max_pos=0.0),
                                    dict(max_pos=2 ** 31)])
def test_table_refusals(change):
    mod, _ = R.binding()

    def build():
        return mod.RopeTableParams(table=4096, max_pos=10, rotary_dim=8, scaling=1, base=1e4, factor=2.0,
                                   original_max_pos=100.0, low_turns=1.0, high_turns=4.0)

    assert refusal("rope_table_f32", build()) is None
    assert refusal("rope_table_f32", changed(build, **change))


@pytest.mark.parametrize("name,build,change", [
    ("rope_f16", "rope_params", dict(X=None)), ("kv_append_rope_f16_f16", "append_params", dict(slots=None)),
    ("attn_paged_f16_f16", "attn_params", dict(q_heads=5))])
def test_a_refused_run_aborts_with_its_reason(name, build, change):
    """As every entry point of the library does: file:line and the reason on stderr, then abort."""
    code = ("import sys, ctypes; sys.path.insert(0, %r); import paged_ref as R, test_paged_host as H\n"
            "p = H.changed(H.%s, **%r); R.binding()[1].op(%r, 'run_async')(ctypes.byref(p), None)\n"
            "print('returned')" % (os.path.join(ROOT, "tests"), build, change, name))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert r.returncode == -6 and "returned" not in r.stdout
    assert refusal(name, changed(globals()[build], **change)).decode() in r.stderr
