"""The attention's and the append's index rules at the ends of their ranges (the HIP-free headers of torq-tile_amd/csrc),
evaluated on the CPU."""

import ctypes
import os
import random
import subprocess
import sys

import pytest

import paged_ref as R
import test_paged_host as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("limits")
    (d / "r.cpp").write_text('''
#include "attn_route.hpp"
#include "rope_route.hpp"
using namespace tqt;
extern "C" {
int r_first_key(int pos, int window) { return attn_first_key(pos, window); }
long long r_span(long long q, long long kv, long long w) { return attn_span(q, kv, w); }
int r_tile_rows() { return kAttnTileRows; }
void r_split(long long tiles, long long kv_heads, long long span, long long d, int *out)
{
    const AttnSplit s = attn_call_split(tiles, kv_heads, span, d, 1000);
    out[0] = s.chunk;
    out[1] = s.splits;
}
void r_rope(long long heads, long long d, int grid16, int pow2, long long *out)
{
    const RopeLaunch r = rope_launch(heads, d, grid16, pow2);
    out[0] = r.rows;
    out[1] = r.per_head;
    out[2] = r.tokens;
}
}
''')
    subprocess.run([CLANG, "-O2", "-std=c++17", "-fwrapv", "-fPIC", "-shared", "-Wall", "-I" +
                    os.path.join(ROOT, "torq-tile_amd", "csrc"), "-o", str(d / "r.so"), str(d / "r.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(d / "r.so"))
    lib.r_first_key.argtypes = [ctypes.c_int] * 2
    lib.r_span.argtypes, lib.r_span.restype = [ctypes.c_longlong] * 3, ctypes.c_longlong
    lib.r_split.argtypes = [ctypes.c_longlong] * 4 + [ctypes.c_void_p]
    lib.r_rope.argtypes = [ctypes.c_longlong] * 2 + [ctypes.c_int] * 2 + [ctypes.c_void_p]
    return lib


POSITIONS = [1 - 2 ** 31, -2 ** 30, -70, -2, -1, 0, 1, 63, 64, 99, 2 ** 30 - 1]


@pytest.mark.parametrize("window", [0, 1, 2, 64, 100, 2 ** 30, 2 ** 31 - 2, 2 ** 31 - 1])
def test_first_key_of_a_window(rules, window):
    """Queries before every key (negative positions) beside windows up to the largest."""
    for pos in POSITIONS:
        want = max(pos - window + 1, 0) if window else 0
        assert rules.r_first_key(pos, window) == want, (pos, window)


# rows of a token up to those of the widest calls: rope's 2^20 - 1 heads, the append's queries, keys and values
@pytest.mark.parametrize("heads", [1, 33, 48, 1 << 16, (1 << 20) - 1, (1 << 20) - 1 + 2 * ((1 << 16) - 1)])
@pytest.mark.parametrize("d", [1, 16, 20, 80, 128, 256, 1 << 15, (1 << 20) - 16])
def test_rope_launches_fit(rules, heads, d):
    """Every launch's work-items stay below 2^32 and its indexes below 2^31, and it has a token at least."""
    for grid16 in (0, 1):
        for pow2 in (0, 1):
            if grid16 and d % 16 or pow2 and d > 256:
                continue
            out = (ctypes.c_longlong * 3)()
            rules.r_rope(heads, d, grid16, pow2, out)
            rows, per_head, tokens = out
            assert tokens >= 1 and (grid16 or not rows)
            threads = tokens * heads * per_head * (1 if rows else 64)
            assert -(-threads // 256) * 256 < 2 ** 32 and tokens * heads * per_head < 2 ** 31
            if rows:
                assert per_head * 16 >= d and (not pow2 or per_head & (per_head - 1) == 0)


def test_ordinary_rope_calls_take_one_launch(rules):
    for heads, d, grid16 in ((32, 128, 1), (48, 128, 1), (32, 72, 0)):
        out = (ctypes.c_longlong * 3)()
        rules.r_rope(heads, d, grid16, 0, out)
        assert out[0] == grid16 and out[2] >= 8192


@pytest.mark.parametrize("d", [64, 256])
def test_buffers_of_many_rows_are_not_split(d):
    """q_tokens of a large buffer, of which a call's sequences use few rows: no parts, whose join would have a
    workgroup for every row of the buffer."""
    _, lib = R.binding()

    def need(tokens):
        p = H.changed(H.attn_params, batch=1, q_tokens=tokens, q_heads=16, kv__kv_heads=2, max_q_len=64,
                      max_kv_len=100000, ld_table=6250, kv__num_pages=6250, kv__head_dim=d)
        size = lib.op("attn_paged", "get_workspace_size")(ctypes.byref(p))
        assert H.refusal("attn_paged_f16_f16", H.changed(lambda: p, workspace_size=size)) is None
        return size

    splits = need(64) // (64 * 16 * (d + 2) * 4)
    assert splits > 16
    assert need(2 ** 19 - 1) == splits * (2 ** 19 - 1) * 16 * (d + 2) * 4
    assert need(2 ** 19) == need(2 ** 20) == 0


def table_params():
    mod, _ = R.binding()
    return mod.RopeTableParams(table=4096, max_pos=10, rotary_dim=8, base=1e4)


@pytest.mark.parametrize("max_pos,rot", [
    (2 ** 31 - 1, 2), (2 ** 31 - 1, 4), (2 ** 31 - 1, 6), (2 ** 26 - 4, 128), (2 ** 26 - 3, 128), (2 ** 26, 128),
    (2 ** 13, 2 ** 20 - 2), (2 ** 13 + 1, 2 ** 20 - 2)])
def test_tables_past_one_launch_are_refused(max_pos, rot):
    """Whether a run would take it is what get_error says: its workgroups of 256 threads, one per pair, are of fewer
    than 2^32 threads."""
    said = H.refusal("rope_table_f32", H.changed(table_params, max_pos=max_pos, rotary_dim=rot))
    assert (said is None) == (-(-max_pos * (rot // 2) // 256) * 256 < 2 ** 32)


def test_a_refused_table_aborts_in_both_forms():
    """Also where there is nothing to write."""
    for action in ("run", "run_async"):
        code = ("import sys, ctypes; sys.path.insert(0, %r); import paged_ref as R\n"
                "mod, lib = R.binding(); p = mod.RopeTableParams(table=4096, max_pos=0, rotary_dim=3, base=1e4)\n"
                "lib.op('rope_table_f32', %r)(ctypes.byref(p)%s)\nprint('returned')"
                % (os.path.join(ROOT, "tests"), action, ", None" if action == "run_async" else ""))
        r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
        assert r.returncode == -6 and "returned" not in r.stdout
        assert H.refusal("rope_table_f32", H.changed(table_params, rotary_dim=3)).decode() in r.stderr


@pytest.mark.parametrize("scale,taken", [(2.3e38, True), (-2.3e38, True), (2.4e38, False), (-3.4e38, False),
                                         (0.0, True), (1e-45, True)])
def test_scales_whose_log2_form_overflows_are_refused(scale, taken):
    for kind in H.ATTNS:
        assert (H.refusal("attn_paged_" + kind, H.changed(H.attn_params, scale=scale)) is None) == taken


def split(rules, tiles, kv_heads, span, d):
    out = (ctypes.c_int * 2)()
    rules.r_split(tiles, kv_heads, span, d, out)
    return tuple(out)


@pytest.mark.parametrize("d", [16, 64, 128, 144, 192, 256])
def test_splits_cover_every_tile_at_every_head_dim(rules, d):
    """The spans of a tile's keys, from a multiple of 64 on, fit the splits that are launched."""
    rng = random.Random(d)
    m = rules.r_tile_rows()
    several = 0
    for _ in range(1500):
        group = rng.choice([1, 3, 4, 8, 16, 50])
        max_q, max_kv = rng.randint(1, 3000), rng.randint(1, 200000)
        window = rng.choice([0, 0, rng.randint(1, 5000)])
        tiles, heads = rng.randint(1, 60), rng.choice([1, 2, 8, 32])
        span = rules.r_span(min(max_q, m // group + 2), max_kv, window)
        chunk, splits = split(rules, tiles, heads, span, d)
        assert chunk % 64 == 0 and splits >= 1
        several += splits > 1
        nq, kv = rng.randint(1, max_q), rng.randint(1, max_kv)
        for tile in range(-(-nq * group // m)):
            t0, t1 = tile * m // group, (min((tile + 1) * m, nq * group) - 1) // group
            lo = max(kv - nq + t0 - window + 1, 0) if window else 0
            hi = min(max(kv - nq + t1 + 1, 0), kv)
            n = max(1, -(-(hi - lo // 64 * 64) // chunk))
            assert n <= splits, (group, nq, kv, window, tile, chunk, splits)
    assert several > 200


@pytest.mark.parametrize("d,workgroups", [(64, 512), (128, 512), (192, 256), (256, 256)])
def test_split_of_few_tiles_by_head_dim(rules, d, workgroups):
    """As many workgroups as the chip holds of a head size; none where that many tiles are there already."""
    assert split(rules, 4, 8, 2 ** 20, d)[1] in (workgroups // 32, workgroups // 32 + 1)
    assert split(rules, workgroups // 8, 8, 2 ** 20, d)[1] == 1
    for span in (1, 63, 64, 65, 300):
        chunk, splits = split(rules, 1, 1, span, d)
        assert splits == 1 and chunk >= span + 63


def test_units_of_the_last_run_fit_32_bits():
    """512 workgroups take equal runs of units, the last of which ends at or past the last unit: that end has to fit
    32 bits too."""
    def said(units):  # of 462 sequences with a key head each
        assert units % 462 == 0
        p = H.changed(H.attn_params, batch=462, q_tokens=462, q_heads=1, kv__kv_heads=1, ld_table=2 ** 23,
                      kv__page_size=128, kv__num_pages=2 ** 20, max_kv_len=(units // 462 - 1) * 128)
        return H.refusal("attn_paged_f16_f16", p)

    top = 2 ** 31 - 2  # a multiple of 462
    assert -(-(top - 2 * 462) // 512) * 512 < 2 ** 31 and said(top - 2 * 462) is None
    for units in (top, top - 462):
        assert -(-units // 512) * 512 >= 2 ** 31 and "too large" in said(units).decode()
