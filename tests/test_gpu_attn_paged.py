"""Attention over a paged cache on the GPU against a plain form in 64 bits, at the sizes and masks where it can go
wrong. The bounds follow from the roundings the operator is defined with (paged_ref.attention_bound)."""

import ctypes
import math

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu

NAMES = ["f16_f16", "bf16_bf16", "f16_qsi8dx", "bf16_qsi8dx"]


class Case:
    """A batch with random contents. lengths: (new tokens, keys) of every sequence."""

    def __init__(self, name, lengths, heads, kv_heads, d, page=16, causal=True, window=0, seed=0,
                 heads_first=False, spread=1.5, spare=float("nan"), pad=0):
        import torch

        self.name, self.lengths, self.d = name, lengths, d
        self.heads, self.kv_heads, self.page = heads, kv_heads, page
        self.causal, self.window = causal, window
        kind, cache = name.split("_")
        self.kind = kind
        rng = np.random.default_rng(seed + 7 * d + heads)
        starts = np.concatenate(([0], np.cumsum([q for q, _ in lengths]))).astype(np.int32)
        self.starts = starts
        per = max([1] + [-(-kv // page) for _, kv in lengths])
        need = sum(-(-kv // page) for _, kv in lengths)
        pages = need + 3
        order = rng.permutation(pages)
        table = np.full((len(lengths), per), -1, np.int32)
        at = 0
        for b, (_, kv) in enumerate(lengths):
            n = -(-kv // page)
            table[b, :n] = order[at:at + n]
            at += n
        self.table = table
        # the cache, with what no key uses left at `spare`
        q = R.dev(rng.standard_normal((int(starts[-1]), heads, d)) * spread, kind)
        self.q = R.host(q)
        self.dq = q
        if pad:
            buf = torch.zeros((q.shape[0], heads, d + pad), dtype=q.dtype, device="cuda:0")
            buf[..., :d] = q
            self.dq = buf[..., :d]
        kv = []
        for _ in range(2):
            x = R.dev(rng.standard_normal((pages, page, kv_heads, d)))
            sc = None
            if cache == "qsi8dx":
                c = torch.randint(-127, 128, x.shape, dtype=torch.int8, device="cuda:0")
                sc = torch.rand((pages, kv_heads, page), device="cuda:0") * 0.02 + 0.003
                val = R.host(c) * R.host(sc).transpose(0, 2, 1)[..., None]
            else:
                c = x.to(R.torch_type(cache))
                val = R.host(c)
            kv.append((c, sc, val))
        used = np.zeros((pages, page), bool)
        for b, (_, n) in enumerate(lengths):
            for j in range(n):
                used[table[b, j // page], j % page] = True
        self.used = used
        (k, sk, self.k), (v, sv, self.v) = kv
        unused = R.dev(~used)
        if sk is None:
            k[unused] = spare
            v[unused] = spare
        else:
            sk.transpose(1, 2)[unused] = spare
            sv.transpose(1, 2)[unused] = spare
        if heads_first:
            k, v = k.transpose(1, 2).contiguous(), v.transpose(1, 2).contiguous()
        self.dk, self.dv, self.dsk, self.dsv, self.heads_first = k, v, sk, sv, heads_first
        self.scale = 1.0 / math.sqrt(d)

    def run(self, **kw):
        import torch

        mod, _ = R.binding()
        t = int(self.starts[-1])
        self.out = torch.full((t, self.heads, self.d), 9.0, dtype=self.dq.dtype, device="cuda:0")
        self.lse = torch.full((t, self.heads), 9.0, device="cuda:0")
        kv = R.paged(mod, self.dk, self.dv, self.dsk, self.dsv, heads_first=self.heads_first)
        lens = R.dev(np.array([n for _, n in self.lengths], np.int32))
        R.run_attention(self.name, self.dq, kv, R.dev(self.starts), lens, R.dev(self.table), self.out,
                        None if kw.pop("no_lse", False) else self.lse, self.scale, self.causal,
                        self.window, **kw)
        return self

    def keys(self, b):
        """k, v [kv_len, kv_heads, d] of a sequence and which of its keys are kept."""
        n = self.lengths[b][1]
        j = np.arange(n)
        p = self.table[b, j // self.page]
        kept = (p >= 0) & (p < self.k.shape[0])
        p = np.where(kept, p, 0)
        return self.k[p, j % self.page], self.v[p, j % self.page], kept

    def check(self, lse=True):
        got, got_lse = R.host(self.out), R.host(self.lse)
        for b, (nq, nk) in enumerate(self.lengths):
            lo = int(self.starts[b])
            k, v, kept = self.keys(b)
            see = R.visible(nq, nk, self.causal, self.window) & kept[None]
            want = R.attention(self.q[lo:lo + nq], k, v, see, self.scale)
            tol, tol_lse = R.attention_bound(self.kind, self.d, *want)
            out, l = got[lo:lo + nq], got_lse[lo:lo + nq]
            off = np.abs(out - want[0])
            assert (off <= tol).all(), (b, np.nanmax(off / tol), np.argwhere(~(off <= tol))[:4])
            if lse:
                none = np.isneginf(want[1])
                np.testing.assert_array_equal(np.isneginf(l), none)
                assert (np.abs(l - want[1])[~none] <= tol_lse[~none]).all()
        return self


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (8, 2), (6, 6), (7, 1), (32, 2), (40, 2)])
def test_one_token(gpu, name, heads, kv_heads):
    Case(name, [(1, 1), (1, 33), (1, 300), (1, 16)], heads, kv_heads, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("d", [16, 32, 48, 64, 80, 96, 112, 128, 144, 160, 192, 208, 240, 256])
def test_head_dims(gpu, name, d):
    Case(name, [(1, 70), (1, 5)], 4, 2, d).run().check()
    Case(name, [(23, 70), (65, 65)], 4, 2, d).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 100, 256])
@pytest.mark.parametrize("heads_first", [False, True])
def test_pages(gpu, name, page, heads_first):
    Case(name, [(1, 131), (1, 63)], 4, 2, 64, page, heads_first=heads_first).run().check()
    Case(name, [(40, 131), (2, 257)], 4, 2, 64, page, heads_first=heads_first).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("nq,nk", [(2, 2), (3, 200), (4, 5), (16, 16), (17, 90), (31, 64), (33, 33),
                                   (64, 64), (65, 129), (127, 128), (130, 400)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(gpu, name, nq, nk, causal):
    Case(name, [(nq, nk)], 6, 2, 128, causal=causal).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("d", [64, 128, 192, 256])
@pytest.mark.parametrize("window", [0, 1700])
def test_few_tiles_over_many_keys(gpu, name, d, window):
    """The keys of a tile are split and the parts joined, beside sequences that are not split; the second's
    last pages are not kept, so that whole parts of it have no key."""
    c = Case(name, [(40, 3001), (17, 1500), (1, 2000), (70, 30)], 4, 2, d, window=window)
    c.table[1, 40:] = -1
    c.run().check()


@pytest.mark.parametrize("name", ["f16_f16", "bf16_qsi8dx"])
@pytest.mark.parametrize("window", [1, 2, 15, 64, 100, 1000])
@pytest.mark.parametrize("lengths", [[(1, 300), (1, 40)], [(90, 300), (1, 129), (33, 33)]])
def test_windows(gpu, name, window, lengths):
    Case(name, lengths, 4, 2, 64, window=window).run().check()


@pytest.mark.parametrize("name", NAMES)
def test_rows_that_see_nothing(gpu, name):
    """No keys at all, more new tokens than keys (the first ones stand before every key), no new
    tokens: zeros and -infinity, and the other rows as ever."""
    c = Case(name, [(1, 0), (3, 0), (1, 5), (0, 20), (9, 4), (40, 7), (70, 1)], 4, 2, 64).run().check()
    out, lse = R.host(c.out), R.host(c.lse)
    assert (out[:4] == 0).all() and np.isneginf(lse[:4]).all()
    Case(name, [(1, 0), (1, 9)], 4, 2, 64).run().check()
    Case(name, [(1, 0)], 4, 2, 64).run().check()
    Case(name, [(5, 0)], 32, 2, 64, causal=False).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("lengths", [[(1, 200), (1, 90)], [(50, 200), (20, 90)]])
def test_pages_not_kept(gpu, name, lengths):
    """Entries that name no page: with a window that has passed them, and as holes."""
    c = Case(name, lengths, 4, 2, 64, window=60)
    c.table[0, :4] = [-1, 2 ** 31 - 1, -2 ** 31, c.k.shape[0]]
    c.run().check()
    c = Case(name, lengths, 4, 2, 64)
    c.table[0, 3:7] = [-1, 2 ** 31 - 1, -2 ** 31, c.k.shape[0]]
    c.table[1, :] = -1
    c.run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("q_len", [1, 70])
def test_unused_memory_is_not_used(gpu, name, bad, q_len):
    """Past kv_len and in other pages lie NaN or infinities (int8: in the scales): the same results."""
    a = Case(name, [(q_len, 75), (q_len, 130)], 4, 2, 64, spare=0.0).run().check()
    b = Case(name, [(q_len, 75), (q_len, 130)], 4, 2, 64, spare=bad).run()
    b.dk.copy_(a.dk) if a.dsk is not None else None
    b.dv.copy_(a.dv) if a.dsv is not None else None
    if a.dsk is not None:
        unused = R.dev(~a.used)
        for x, y in ((b.dsk, a.dsk), (b.dsv, a.dsv)):
            x.copy_(y)
            x.transpose(1, 2)[unused] = bad
    b.run()
    import torch

    assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)


@pytest.mark.parametrize("name", ["f16_f16", "bf16_bf16"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("window", [0, 20])
def test_not_finite_reaches_only_who_sees_it(gpu, name, which, bad, window):
    """A NaN or infinity at one key: rows that do not see the key are as without it, bit for bit."""
    import torch

    lengths, at = [(90, 150)], 101
    a = Case(name, lengths, 4, 2, 64, window=window).run().check()
    b = Case(name, lengths, 4, 2, 64, window=window)
    t = b.dk if which == "k" else b.dv
    t[b.table[0, at // 16], at % 16, 1, 7] = bad
    b.run()
    see = R.visible(*lengths[0], True, window)[:, at]
    blind = R.dev(np.nonzero(~see)[0])
    assert torch.equal(a.out[blind], b.out[blind]) and torch.equal(a.lse[blind], b.lse[blind])
    assert torch.equal(a.out[:, :2], b.out[:, :2])  # the other key head's queries
    seen = R.dev(np.nonzero(see)[0])
    if which == "v":
        got = R.host(b.out[seen])[:, 2:]
        assert (np.isnan(got[..., 7]) if np.isnan(bad) else got[..., 7] == bad).all()
        got[..., 7] = 0
        assert np.isfinite(got).all()
    elif np.isnan(bad):
        assert torch.isnan(b.out[seen][:, 2:]).all()


@pytest.mark.parametrize("name", ["f16_qsi8dx", "bf16_qsi8dx"])
@pytest.mark.parametrize("which", ["dsk", "dsv"])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("lengths,at", [((90, 150), 101), ((4, 150), 147)])
def test_scale_not_finite_reaches_only_who_sees_it(gpu, name, which, bad, lengths, at):
    """The scale of one key is no number: rows that see the key are none either, the others as ever."""
    c = Case(name, [lengths], 4, 2, 64, window=30)
    getattr(c, which)[c.table[0, at // 16], 1, at % 16] = bad
    c.run()
    see = R.visible(*lengths, True, 30)[:, at]
    k, v, kept = c.keys(0)
    want = R.attention(c.q, k, v, R.visible(*lengths, True, 30), c.scale)
    tol, tol_lse = R.attention_bound(c.kind, c.d, *want)
    out, lse = R.host(c.out), R.host(c.lse)
    fine = np.ones(out.shape[:2], bool)
    fine[see, 2:] = False  # the heads that read key head 1
    assert (np.abs(out - want[0]) <= tol)[fine].all()
    assert (np.abs(lse - want[1]) <= tol_lse)[fine].all()
    # an infinite key makes a score of either sign: a row that has -infinity there is as without the key
    if which == "dsv" or np.isnan(bad):
        assert not np.isfinite(out[~fine]).all(axis=-1).any()


@pytest.mark.parametrize("name", ["f16_f16", "bf16_bf16"])
@pytest.mark.parametrize("q_len", [1, 40])
def test_scores_at_the_type_limits(gpu, name, q_len):
    """Scores of the types' largest magnitude (sums that pass f16's range), and keys with a score of
    -infinity beside others and alone."""
    c = Case(name, [(q_len, 120)], 2, 1, 64, spread=1.0)
    c.dk.mul_(200)
    c.k = R.host(c.dk)
    c.run().check()
    c = Case(name, [(q_len, 120)], 2, 1, 64)
    c.dq.fill_(1.0)
    c.q = R.host(c.dq)
    for j in range(0, 120, 3):
        c.dk[c.table[0, j // 16], j % 16] = -np.inf
    c.k = R.host(c.dk)
    with np.errstate(invalid="ignore"):
        want = R.attention(c.q, *c.keys(0)[:2], R.visible(q_len, 120, True, 0), c.scale)
    c.run()
    terms = np.full_like(want[4], 64.0)
    tol, tol_lse = R.attention_bound(c.kind, 64, *want[:4], terms)
    assert (np.abs(R.host(c.out) - want[0]) <= tol).all()
    assert (np.abs(R.host(c.lse) - want[1]) <= tol_lse).all()
    c.dk.fill_(-np.inf)
    c.run()
    assert (c.out == 0).all() and torch_isneginf(c.lse)


def torch_isneginf(t):
    import torch

    return bool(torch.isneginf(t).all())


@pytest.mark.parametrize("name", NAMES)
def test_mixed_batch_and_strides(gpu, name):
    """Decoded tokens, chunks and prompts in one call; heads of Q with gaps between them."""
    lengths = [(1, 500), (40, 40), (1, 3), (130, 300), (0, 0), (1, 1), (5, 260), (17, 18)]
    Case(name, lengths, 8, 2, 80, pad=16).run().check()
    Case(name, lengths, 3, 3, 128, pad=8).run().check()
    Case(name, lengths, 48, 1, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("decode", [True, False])
def test_many_sequences(gpu, name, decode):
    """More sequences than a wave has lanes, of all kinds, empty ones among them."""
    rng = np.random.default_rng(9)
    lengths = []
    for b in range(203):
        kv = int(rng.choice([0, 1, 7, 40, 129, 300]))
        q = 1 if decode or b % 5 else int(rng.integers(0, 60))
        lengths.append((q, kv))
    Case(name, lengths, 4, 2, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
def test_long_split_axis(gpu, name):
    """One token over a long cache: split over workgroups and joined."""
    Case(name, [(1, 20011)], 4, 2, 64, page=32).run().check()
    Case(name, [(1, 9001), (1, 17), (2, 5000)], 4, 2, 128, page=64).run().check()
    Case(name, [(60, 6000)], 2, 1, 64, page=32).run().check()


@pytest.mark.parametrize("name", ["f16_f16", "f16_qsi8dx"])
def test_lengths_below_their_bounds(gpu, name):
    """max_q_len and max_kv_len are bounds only: larger ones give the same rows (the split may differ);
    more keys than max_kv_len count as that many, and queries past max_q_len are not written."""
    c = Case(name, [(1, 100), (1, 30)], 4, 2, 64)
    c.table = np.concatenate((c.table, np.full((2, 600), -1, np.int32)), 1)
    c.run(max_q=40, max_kv=9000).check()
    c = Case(name, [(3, 100), (50, 90)], 4, 2, 64)
    c.run(max_q=64, max_kv=112).check()
    c = Case(name, [(1, 100), (1, 64)], 4, 2, 64)
    c.run(max_kv=64)
    c.lengths = [(1, 64), (1, 64)]
    c.check()


@pytest.mark.parametrize("q_len", [1, 50])
def test_without_lse(gpu, q_len):
    c = Case("f16_f16", [(q_len, 80)], 4, 2, 64).run()
    out = c.out
    c.run(no_lse=True)
    import torch

    assert torch.equal(out, c.out) and (c.lse == 9.0).all()


@pytest.mark.parametrize("name", ["f16_f16", "bf16_qsi8dx"])
def test_same_bits_every_time(gpu, name):
    """No result depends on the order in which workgroups run."""
    import torch

    c = Case(name, [(1, 3000), (70, 900), (1, 40)], 8, 2, 64, page=32).run()
    first, lse = c.out, c.lse
    for _ in range(5):
        c.run()
        assert torch.equal(first, c.out) and torch.equal(lse, c.lse)


@pytest.mark.parametrize("lengths", [[(1, 900), (1, 77)], [(1, 500), (60, 200)]])
def test_graph_replay_with_changing_lengths(gpu, lengths):
    """A captured call replayed as the lengths in device memory change, with eager work in between."""
    import torch

    mod, lib = R.binding()
    c = Case("f16_f16", [(q, 1000) for q, _ in lengths], 8, 2, 64, page=16)
    kv = R.paged(mod, c.dk, c.dv)
    starts, table = R.dev(c.starts), R.dev(c.table)
    lens = R.dev(np.array([1000, 1000], np.int32))
    out = torch.zeros((int(c.starts[-1]), 8, 64), dtype=torch.float16, device="cuda:0")
    lse = torch.zeros((int(c.starts[-1]), 8), device="cuda:0")
    keep = []
    R.run_attention("f16_f16", c.dq, kv, starts, lens, table, out, lse, c.scale, keep=keep)
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        lib.op("attn_paged_f16_f16", "run_async")(ctypes.byref(keep[0][0]),
                                                  torch.cuda.current_stream().cuda_stream)
    for n0, n1 in [(900, 77), (1, 1000), (500, 499), (61, 60)]:
        lens.copy_(R.dev(np.array([n0, n1], np.int32)))
        out.fill_(9.0)
        lse.fill_(9.0)
        keep[0][1].fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        c.lengths = [(lengths[0][0], n0), (lengths[1][0], n1)]
        c.out, c.lse = out, lse
        c.check()


def test_cache_past_32_bit_offsets(gpu):
    """Pages whose element offsets pass 2^31 and byte offsets pass 2^32 (strides, not memory of that
    size times two: keys and values share one tensor)."""
    import torch

    mod, _ = R.binding()
    page, d, kvh, stride = 16, 64, 2, 3 * 2 ** 28  # elements between pages
    pages = 4
    big = torch.empty(pages * stride, dtype=torch.float16, device="cuda:0")
    view = big.as_strided((pages, page, kvh, d), (stride, kvh * d, d, 1))
    x = np.random.default_rng(3).standard_normal((pages, page, kvh, d))
    view.copy_(R.dev(x, "f16"))
    k = R.host(view)
    q = R.dev(np.random.default_rng(4).standard_normal((21, 4, d)), "f16")
    for lengths in ([(1, 64)], [(20, 64)]):
        nq, nk = lengths[0]
        out = torch.zeros((nq, 4, d), dtype=torch.float16, device="cuda:0")
        lse = torch.zeros((nq, 4), device="cuda:0")
        table = np.array([[3, 1, 2, 0]], np.int32)
        R.run_attention("f16_f16", q[:nq], R.paged(mod, view, view), R.dev(np.array([0, nq], np.int32)),
                        R.dev(np.array([nk], np.int32)), R.dev(table), out, lse, 0.125)
        kk = k[table[0]].reshape(64, kvh, d)
        want = R.attention(R.host(q[:nq]), kk, kk, R.visible(nq, nk, True, 0), 0.125)
        tol, _ = R.attention_bound("f16", d, *want)
        assert (np.abs(R.host(out) - want[0]) <= tol).all()


def test_nothing_to_do(gpu):
    mod, lib = R.binding()
    run = lib.op("attn_paged_f16_f16", "run")
    run(None)
    run(ctypes.byref(mod.AttnPagedParams(batch=0, q_tokens=5, q_heads=4)))
    run(ctypes.byref(mod.AttnPagedParams(batch=2, q_tokens=0, q_heads=4)))
