"""Trees of a ragged batch in equal spans of each sequence's own: the host's rule (torq-tile_amd/csrc/attn_route.hpp), and
what the kernel makes of it (attn_find_work in attn_tile.hpp, restated here): the grid and the workspace that the host
lays out hold every tile's spans, whatever the lengths."""

import ctypes
import os
import random
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CLANG = "/opt/rocm/llvm/bin/clang++"
TILE, LEAST, COST = 128, 256, 512


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no C++ compiler")
    d = tmp_path_factory.mktemp("even")
    (d / "r.cpp").write_text('''
#include "attn_route.hpp"
using namespace tqt;
extern "C" {
long long r_tiles(long long b, long long t, long long q, long long g) { return attn_tiles(b, t, q, g); }
long long r_span(long long q, long long kv, long long w) { return attn_span(q, kv, w); }
int r_first(int pos, int window) { return attn_first_key(pos, window); }
int r_few(int d) { return attn_tree_few_rows(d); }
long long r_round(long long d) { return attn_tile_workgroups(d); }
int r_constants() { return kAttnTileRows == 128 && kAttnTileLeast == 256 && kAttnEvenCost == 512; }
int r_even(long long b, long long tiles, long long kvh, long long span, long long d, long long rows)
{
    return attn_even_parts(b, tiles * kvh, attn_call_split(tiles, kvh, span, d, rows), span, d, rows);
}
}
''')
    subprocess.run([CLANG, "-O2", "-std=c++17", "-fPIC", "-shared", "-Wall", "-I" +
                    os.path.join(ROOT, "torq-tile_amd", "csrc"), "-o", str(d / "r.so"), str(d / "r.cpp")], check=True)
    lib = ctypes.CDLL(str(d / "r.so"))
    ll = ctypes.c_longlong
    for name, n in (("r_tiles", 4), ("r_span", 3), ("r_round", 1), ("r_even", 6)):
        getattr(lib, name).argtypes = [ll] * n
        getattr(lib, name).restype = ctypes.c_int if name == "r_even" else ll
    assert lib.r_constants()
    return lib


def spans(lib, seqs, max_q, max_kv, words, group, kv_heads, d, window, q_tokens):
    """None, or (workgroups of the grid, most parts, [(tiles, keys, spans)] of the sequences, rounds)."""
    tiles = lib.r_tiles(len(seqs), q_tokens, max_q, group)
    span = lib.r_span(32 * words + 1, max_kv, window)
    most = lib.r_even(len(seqs), tiles, kv_heads, span, d, q_tokens * group * kv_heads)
    if most == 0:
        return None
    turn, longest = lib.r_round(d), span + 63
    least = max(LEAST, (-(-longest // most) + 63) // 64 * 64)
    works = []
    for q, kv in seqs:
        rows = min(q, max_q) * group
        n, keys = -(-rows // TILE) if rows > lib.r_few(d) else 0, 0
        if n:
            pos0 = kv - q
            first = min(lib.r_first(pos0 - 1, window), max(pos0, 0)) & ~63
            keys = max(min(kv, pos0 + 32 * words) - first, 0)
        works.append((n, keys))
    parts = lambda keys, each: min(max(-(-keys // each), 1), most)  # noqa: E731

    def smallest(workgroups):
        lo, hi = least >> 6, (longest + 127) // 64
        while lo < hi:
            mid = (lo + hi) >> 1
            if sum(n * parts(keys, mid << 6) for n, keys in works) * kv_heads <= workgroups:
                hi = mid
            else:
                lo = mid + 1
        return lo << 6

    one, two = smallest(turn), smallest(2 * turn)
    each, out = two if 2 * two + COST < one else one, []
    for n, keys in works:
        own = max((-(-keys // parts(keys, each)) + 63) & ~63, 64)
        out.append((n, keys, own))
    return 2 * turn // kv_heads * kv_heads, most, out, 1 + (2 * two + COST < one)


def test_grid_and_workspace_hold_every_span(rules):
    rng, seen = random.Random(3), [0, 0, 0]
    for _ in range(30000):
        d, kv_heads = rng.choice([64, 128, 256]), rng.choice([1, 2, 3, 4, 6, 8, 16, 40])
        group, batch, words = rng.choice([1, 2, 4, 5, 8]), rng.randint(1, 70), rng.randint(1, 8)
        max_q, max_kv = rng.randint(1, 32 * words), rng.choice([300, 1000, 5000, 20000, 100000, 2 ** 30 - 1])
        window = rng.choice([0, 0, 0, 100, 2000])
        seqs = [(rng.randint(0, max_q), rng.randint(0, max_kv)) for _ in range(batch)]
        if rng.random() < 0.2:
            seqs = [(max_q, max_kv)] * batch
        got = spans(rules, seqs, max_q, max_kv, words, group, kv_heads, d, window,
                    sum(q for q, _ in seqs) + rng.randint(0, 50))
        if got is None:
            seen[0] += 1
            continue
        grid, most, works, rounds = got
        seen[rounds] += 1
        assert 2 <= batch <= 64
        for n, keys, own in works:
            assert own % 64 == 0 and (max(keys, 1) - 1) // own < most
        assert sum(n * ((max(keys, 1) - 1) // own + 1) for n, keys, own in works) * kv_heads <= grid
    assert min(seen) > 100, seen  # every form was met


def test_one_length_makes_one_round(rules):
    """Equal lengths that fill a round are not cut further."""
    for batch, nodes, kv, most_parts in ((16, 63, 8192, 2), (8, 63, 16384, 4), (32, 63, 8192, 1)):
        _, _, works, rounds = spans(rules, [(nodes, kv)] * batch, nodes, kv, 2, 4, 8, 128, 0, batch * nodes)
        assert rounds == 1
        assert all(-(-keys // own) == most_parts for _, keys, own in works)
