"""The plan of the attention over a paged cache (torq-tile_amd/csrc/attn_route.hpp, fast_div.hpp), evaluated on the
CPU: what the launcher decides from the host's bounds covers what the kernels then find."""

import ctypes
import os
import random
import subprocess

import pytest

import paged_ref as R
import test_paged_host as H

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"
FEW = 16


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("route")
    (d / "r.cpp").write_text('''
#include "attn_route.hpp"
#include "fast_div.hpp"
using namespace tqt;
extern "C" {
long long r_span(long long q, long long kv, long long w) { return attn_span(q, kv, w); }
long long r_tiles(long long b, long long t, long long q, long long g) { return attn_tiles(b, t, q, g); }
int r_chunk(long long t, long long h, long long s) { return attn_tile_split(t, h, s).chunk; }
int r_splits(long long t, long long h, long long s) { return attn_tile_split(t, h, s).splits; }
int r_few(long long u, int p) { return attn_few_row_workgroups(u, p); }
int r_tile_rows() { return kAttnTileRows; }
long long r_div(unsigned n, unsigned d) { unsigned r; unsigned q = fast_div(n, make_fast_div(d), r);
                                          return (long long)q << 32 | r; }
}
''')
    subprocess.run([CLANG, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-I" +
                    os.path.join(ROOT, "torq-tile_amd", "csrc"), "-o", str(d / "r.so"), str(d / "r.cpp")],
                   check=True)
    lib = ctypes.CDLL(str(d / "r.so"))
    ll = ctypes.c_longlong
    for name, args in (("r_span", [ll] * 3), ("r_tiles", [ll] * 4), ("r_chunk", [ll] * 3),
                       ("r_splits", [ll] * 3), ("r_few", [ll, ctypes.c_int]),
                       ("r_div", [ctypes.c_uint] * 2)):
        getattr(lib, name).argtypes = args
    for name in ("r_span", "r_tiles", "r_div"):
        getattr(lib, name).restype = ll
    return lib


def test_fast_division(rules):
    rng = random.Random(1)
    ds = list(range(1, 70)) + [2 ** k + e for k in range(7, 31) for e in (-1, 0, 1)]
    ds += [2 ** 31 - 1] + [rng.randrange(1, 2 ** 31) for _ in range(300)]
    for d in ds:
        top = (2 ** 31 - 1) // d * d
        for n in [0, 1, d - 1, d, d + 1, top - 1, top, 2 ** 31 - 1] + [rng.randrange(2 ** 31) for _ in range(20)]:
            if 0 <= n < 2 ** 31:
                assert rules.r_div(n, d) == (n // d << 32 | n % d), (n, d)


def test_tiles_cover_every_batch(rules):
    """The bound on tiles holds for any lengths within the bounds."""
    rng = random.Random(2)
    m = rules.r_tile_rows()
    for _ in range(2000):
        group = rng.choice([1, 2, 3, 4, 7, 8, 16, 20])
        q = [rng.choice([0, 1, 2, rng.randint(1, 40), rng.randint(1, 3000)]) for _ in range(rng.randint(1, 70))]
        need = sum(-(-x * group // m) for x in q)
        assert need <= rules.r_tiles(len(q), sum(q), max(q), group)
        assert need <= rules.r_tiles(len(q) + 3, sum(q) + 50, max(q) + 9, group)


def test_splits_cover_every_tile(rules):
    """The spans of a tile's keys, from a multiple of 64 on, fit the splits that are launched."""
    rng = random.Random(3)
    m = rules.r_tile_rows()
    for _ in range(3000):
        group = rng.choice([1, 3, 4, 8, 16, 50])
        max_q, max_kv = rng.randint(1, 3000), rng.randint(1, 200000)
        window = rng.choice([0, 0, rng.randint(1, 5000)])
        tiles, heads = rng.randint(1, 60), rng.choice([1, 2, 8, 32])
        span = rules.r_span(min(max_q, m // group + 2), max_kv, window)
        chunk, splits = rules.r_chunk(tiles, heads, span), rules.r_splits(tiles, heads, span)
        assert chunk % 64 == 0 and splits >= 1
        nq, kv = rng.randint(1, max_q), rng.randint(1, max_kv)
        for tile in range(-(-nq * group // m)):
            t0, t1 = tile * m // group, (min((tile + 1) * m, nq * group) - 1) // group
            lo = max(kv - nq + t0 - window + 1, 0) if window else 0
            hi = min(max(kv - nq + t1 + 1, 0), kv)
            n = max(1, -(-(hi - lo // 64 * 64) // chunk))
            assert n <= splits, (group, nq, kv, window, tile, chunk, splits)


def test_split_of_few_tiles_alone(rules):
    """Many keys of few tiles are split; few keys, or tiles that fill the chip, are not."""
    assert rules.r_splits(6, 2, 3001) == 12 and rules.r_chunk(6, 2, 3001) == 256
    assert rules.r_splits(16, 8, 512) == 1 and rules.r_splits(64, 8, 10 ** 6) == 1
    for span in (1, 63, 64, 65, 300):
        assert rules.r_splits(1, 1, span) == 1 and rules.r_chunk(1, 1, span) >= span + 63


def test_few_row_workgroups(rules):
    assert rules.r_few(1, 2) == 1 and rules.r_few(100, 2) == 100
    assert rules.r_few(10 ** 9, 2) == 512 and rules.r_few(10 ** 9, 1) == 256


def workspace(**sizes):
    mod, lib = R.binding()
    p = H.changed(H.attn_params, **sizes)
    return lib.op("attn_paged", "get_workspace_size")(ctypes.byref(p))


def test_workspace_size():
    """Depends on the sizes alone, and is refused when short, absent or off the grid."""
    mod, lib = R.binding()
    assert lib.op("attn_paged", "get_workspace_size")(None) == 0
    assert workspace(batch=0) == 0 and workspace(q_heads=3) == 0
    sizes = dict(max_kv_len=4096, ld_table=256, kv__num_pages=4096)
    need = workspace(**sizes)
    assert need > 0 and need % 8 == 0
    assert need == workspace(workspace=None, workspace_size=0, Q=None, **sizes)
    name = "attn_paged_f16_f16"
    for change, ok in ((dict(workspace_size=need), True), (dict(workspace_size=need - 1), False),
                       (dict(workspace=None), False), (dict(workspace=4104), False)):
        assert (H.refusal(name, H.changed(H.attn_params, **sizes, **change)) is None) == ok, change
    # a prompt that fills the chip without a split needs none
    assert workspace(batch=1, q_tokens=8192, max_q_len=8192, max_kv_len=8192, ld_table=512,
                     q_heads=32, kv__kv_heads=8, kv__num_pages=512) == 0


@pytest.mark.parametrize("change", [
    dict(batch=2 ** 16), dict(max_kv_len=2 ** 30, ld_table=2 ** 30), dict(q_tokens=2 ** 30, q_heads=4),
    dict(batch=60000, kv__kv_heads=2, q_heads=2, max_kv_len=10 ** 7, ld_table=10 ** 6),
    dict(batch=60000, kv__kv_heads=2 ** 7, q_heads=2 ** 7)])
def test_sizes_past_the_kernels_indexes(change):
    for kind in H.ATTNS:
        assert H.refusal("attn_paged_" + kind, H.changed(H.attn_params, **change))
