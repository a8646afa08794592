"""Attention over a paged cache at the ends of its arguments' ranges, on the GPU against the plain form in 64
bits."""

import numpy as np
import pytest

import paged_ref as R
from test_gpu_attn_paged import NAMES, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 5, 2 ** 31 - 1])
def test_widest_windows(gpu, name, window):
    """Windows past every length, with queries that stand before every key beside others, for both kernels."""
    Case(name, [(4, 1), (3, 200), (7, 2)], 4, 2, 64, window=window).run().check()
    Case(name, [(9, 4), (40, 7), (70, 1), (33, 300)], 4, 2, 64, window=window).run().check()


def test_few_rows_of_a_large_buffer(gpu):
    """One sequence of 50 tokens over 20000 keys in a buffer of 2^20 rows: the others are not touched."""
    import torch

    mod, _ = R.binding()
    heads, kv_heads, d, page, n, nk = 16, 2, 16, 64, 50, 20000
    rng = np.random.default_rng(5)
    q = torch.zeros((2 ** 20, heads, d), dtype=torch.float16, device="cuda:0")
    q[:n] = R.dev(rng.standard_normal((n, heads, d)), "f16")
    out, lse = torch.full_like(q, 9.0), torch.full(q.shape[:2], 9.0, device="cuda:0")
    k, v = (R.dev(rng.standard_normal((-(-nk // page), page, kv_heads, d)), "f16") for _ in range(2))
    table = np.arange(k.shape[0], dtype=np.int32)[None]
    R.run_attention("f16_f16", q, R.paged(mod, k, v), R.dev(np.array([0, n], np.int32)),
                    R.dev(np.array([nk], np.int32)), R.dev(table), out, lse, 0.25)
    assert (out[n:] == 9.0).all() and (lse[n:] == 9.0).all()
    kk, vv = (R.host(t).reshape(-1, kv_heads, d)[:nk] for t in (k, v))
    want = R.attention(R.host(q[:n]), kk, vv, R.visible(n, nk, True, 0), 0.25)
    tol, tol_lse = R.attention_bound("f16", d, *want)
    assert (np.abs(R.host(out[:n]) - want[0]) <= tol).all()
    assert (np.abs(R.host(lse[:n]) - want[1]) <= tol_lse).all()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("max_q", [1, 2, 5, 20, 33])
def test_queries_past_max_q_len_are_left_out(gpu, name, max_q):
    """They keep what was there, and the others stand where they stood."""
    lengths = [(50, 90), (3, 100), (1, 40), (34, 20)]
    c = Case(name, lengths, 4, 2, 64).run(max_q=max_q)
    for b, (nq, nk) in enumerate(lengths):
        lo, n = int(c.starts[b]), min(nq, max_q)
        assert (c.out[lo + n:lo + nq] == 9.0).all() and (c.lse[lo + n:lo + nq] == 9.0).all()
        k, v, kept = c.keys(b)
        see = (R.visible(nq, nk, True, 0) & kept[None])[:n]
        want = R.attention(c.q[lo:lo + n], k, v, see, c.scale)
        tol, tol_lse = R.attention_bound(c.kind, c.d, *want)
        assert (np.abs(R.host(c.out[lo:lo + n]) - want[0]) <= tol).all()
        seen = np.isfinite(want[1])
        got = R.host(c.lse[lo:lo + n])
        assert (np.abs(got[seen] - want[1][seen]) <= tol_lse[seen]).all() and np.isneginf(got[~seen]).all()
