"""Attention of trees of drafted tokens over a paged cache on the GPU, against a plain form in 64 bits, with the bounds
that hold for the attention without trees (paged_ref.attention_bound)."""

import ctypes

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R
from test_gpu_attn_paged import NAMES, Case

pytestmark = pytest.mark.gpu


class Tree(Case):
    """A batch whose new tokens are random trees, unless rows (sets of bits for every row of Q) are given."""

    def __init__(self, name, lengths, *a, words=None, rows=None, chain=0.3, **kw):
        super().__init__(name, lengths, *a, **kw)
        rng = np.random.default_rng(len(lengths) + self.d)
        if rows is None:
            rows = []
            for nq, _ in lengths:
                parents = D.random_parents(rng, nq, chain)
                rows += [D.path(parents, i) for i in range(nq)]
        most = max([1] + [q for q, _ in lengths])
        self.mask = D.pack(rows, words or -(-most // 32))

    def params(self, max_q=None, max_kv=None, no_lse=False, noise=True):
        import torch

        mod, lib = R.binding()
        t = int(self.starts[-1])
        self.out = torch.full((t, self.heads, self.d), 9.0, dtype=self.dq.dtype, device="cuda:0")
        self.lse = torch.full((t, self.heads), 9.0, device="cuda:0")
        mask = self.mask.copy()
        if noise:  # bits past a sequence's new tokens are not looked at
            for b, (nq, _) in enumerate(self.lengths):
                lo, hi = self.starts[b], self.starts[b + 1]
                for w in range(mask.shape[1]):
                    past = np.uint32((0xffffffff << min(max(nq - 32 * w, 0), 32)) & 0xffffffff)
                    mask[lo:hi, w] |= past
        self.args = [R.dev(self.starts), R.dev(np.array([n for _, n in self.lengths], np.int32)),
                     R.dev(self.table), R.dev(mask.view(np.int32))]
        q, out = self.dq, self.out
        p = mod.AttnTreeParams(
            attn=mod.AttnPagedParams(
                batch=len(self.lengths), q_tokens=t, q_heads=self.heads,
                max_q_len=max([0] + [n for n, _ in self.lengths]) if max_q is None else max_q,
                max_kv_len=max(n for _, n in self.lengths) if max_kv is None else max_kv, Q=R.ptr(q),
                q_token_stride=q.stride(0), q_head_stride=q.stride(1), D=R.ptr(out), d_token_stride=out.stride(0),
                d_head_stride=out.stride(1), lse=None if no_lse else R.ptr(self.lse), q_start=R.ptr(self.args[0]),
                kv_len=R.ptr(self.args[1]), block_table=R.ptr(self.args[2]), ld_table=self.table.shape[1],
                scale=self.scale, causal=1, window=self.window,
                kv=R.paged(mod, self.dk, self.dv, self.dsk, self.dsv, heads_first=self.heads_first)),
            mask=R.ptr(self.args[3]), ld_mask=self.mask.shape[1])
        self.space, self.size = D.workspace(lib, "attn_tree", p, p.attn)
        return p

    def run(self, **kw):
        import torch

        D.run("attn_tree_" + self.name, self.params(**kw))
        assert torch.isnan(self.space[self.size // 4 + 4:]).all()
        return self

    def see(self, b):
        lo = int(self.starts[b])
        nq, nk = self.lengths[b]
        return D.visible_tree(self.mask[lo:lo + nq], nq, nk, self.window)

    def check(self, only=None):
        got, got_lse = R.host(self.out), R.host(self.lse)
        for b, (nq, nk) in enumerate(self.lengths):
            lo = int(self.starts[b])
            k, v, kept = self.keys(b)
            want = R.attention(self.q[lo:lo + nq], k, v, self.see(b) & kept[None], self.scale)
            tol, tol_lse = R.attention_bound(self.kind, self.d, *want)
            n = nq if only is None else min(nq, only)  # queries past max_q_len are left out
            off = np.abs(got[lo:lo + n] - want[0][:n])
            assert (off <= tol[:n]).all(), (b, np.nanmax(off / tol[:n]), np.argwhere(~(off <= tol[:n]))[:4])
            assert (got[lo + n:lo + nq] == 9).all()
            none, l = np.isneginf(want[1][:n]), got_lse[lo:lo + n]
            np.testing.assert_array_equal(np.isneginf(l), none)
            assert (np.abs(l - want[1][:n])[~none] <= tol_lse[:n][~none]).all()
        return self


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 1), (8, 2), (6, 6), (7, 1), (40, 2)])
@pytest.mark.parametrize("nodes", [1, 3, 4, 7, 9, 16])
def test_heads_and_nodes(gpu, name, heads, kv_heads, nodes):
    """Rows of a key head from 1 to 320: few rows, many, and in between."""
    Tree(name, [(nodes, nodes), (nodes, 33 + nodes), (nodes, 300), (1, 1), (0, 9)], heads, kv_heads, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("d", [16, 48, 64, 80, 96, 112, 128, 144, 192, 208, 256])
def test_head_dims(gpu, name, d):
    Tree(name, [(3, 70), (2, 5)], 4, 2, d).run().check()
    Tree(name, [(11, 170), (9, 9)], 4, 2, d).run().check()
    Tree(name, [(23, 70), (65, 65)], 4, 2, d).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("page", [1, 3, 16, 24, 100])
@pytest.mark.parametrize("heads_first", [False, True])
def test_pages(gpu, name, page, heads_first):
    for nodes in (4, 13, 40):
        Tree(name, [(nodes, 131), (2, 63)], 4, 2, 64, page, heads_first=heads_first).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("nodes", [1, 5, 8, 15, 16, 17, 31, 32, 33, 63, 64, 65, 96, 100, 128, 200])
@pytest.mark.parametrize("context", [0, 1, 31, 32, 63, 64, 100])
def test_trees_at_every_place_of_a_tile(gpu, name, nodes, context):
    """The tree's keys begin and end at the borders of words and tiles and beside them."""
    Tree(name, [(nodes, nodes + context)], 4, 2, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
def test_masks_of_all_kinds(gpu, name):
    """No bit, not even the own one; all bits; every second; chains (the causal rule)."""
    nq, nk = 21, 60
    for rows in ([set()] * nq, [range(nq)] * nq, [range(i % 2, nq, 2) for i in range(nq)],
                 [{nq - 1 - i} for i in range(nq)]):
        Tree(name, [(nq, nk)], 4, 2, 64, rows=list(rows)).run().check()
        Tree(name, [(nq, nq)], 4, 2, 64, rows=list(rows)).run().check()
        Tree(name, [(3, 40)], 4, 2, 64, rows=[[x for x in r if x < 3] for r in list(rows)[:3]]).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("lengths", [[(1, 100)], [(3, 200), (4, 50)], [(9, 700)], [(70, 150), (33, 33)]])
def test_a_chain_is_the_causal_rule(gpu, name, lengths):
    """The same rows as the attention without trees, within its bounds."""
    c = Tree(name, lengths, 4, 2, 64, chain=1.0).run().check()
    Case.check(c)


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("window", [1, 2, 5, 15, 64, 100, 1000, 2 ** 31 - 1, 2 ** 33])
@pytest.mark.parametrize("lengths", [[(3, 300), (2, 40)], [(12, 300), (9, 40)], [(90, 300), (5, 129), (33, 33)]])
def test_windows(gpu, name, window, lengths):
    """The context's keys are hidden by a token's depth, new tokens never."""
    Tree(name, lengths, 4, 2, 64, window=window).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [0, 1700])
def test_few_trees_over_many_keys(gpu, name, d, window):
    """Keys split over workgroups and joined; the second's last context pages are not kept."""
    c = Tree(name, [(40, 3001), (17, 1500), (3, 2000), (70, 80), (7, 2500)], 4, 2, d, window=window)
    c.table[1, 40:80] = -1
    c.run().check()
    Tree(name, [(13, 9001)], 4, 2, d, page=32, window=window).run().check()
    Tree(name, [(4, 9001)], 4, 2, d, page=32, window=window).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("short", [3, 9])
def test_whole_sequences_beside_split_tiles(gpu, name, short):
    """Many sequences of few rows, whose keys are not split, beside a tree of tiles whose keys are (short 9: rows of a
    tile, of two columns at heads of 64)."""
    rng = np.random.default_rng(short)
    lengths = [(short, int(rng.integers(short, 500))) for _ in range(70)] + [(40, 1900), (1, 1), (70, 1300)]
    Tree(name, lengths, 4, 2, 64).run().check()
    Tree(name, lengths[40:], 8, 4, 128, window=900).run().check()


@pytest.mark.parametrize("name", NAMES)
def test_rows_that_see_nothing(gpu, name):
    """No keys, or more new tokens than keys, so that some of the new ones' own keys do not exist."""
    for chain in (0.0, 1.0):
        lengths = [(1, 0), (3, 0), (2, 5), (0, 20), (9, 4), (40, 7), (70, 1)]
        Tree(name, lengths, 4, 2, 64, chain=chain).run().check()
        Tree(name, [(9, 4)], 4, 2, 64, chain=chain, window=3).run().check()
    c = Tree(name, [(5, 0), (11, 0)], 32, 2, 64).run().check()
    assert (c.out == 0).all()


@pytest.mark.parametrize("name", NAMES)
def test_pages_not_kept(gpu, name):
    for lengths in ([(3, 200), (2, 90)], [(12, 200), (9, 90)], [(50, 200), (20, 90)]):
        c = Tree(name, lengths, 4, 2, 64)
        c.table[0, 3:7] = [-1, 2 ** 31 - 1, -2 ** 31, c.k.shape[0]]
        c.table[0, -1] = -1  # new tokens' own keys among them
        c.table[1, :] = -1
        c.run().check()


@pytest.mark.parametrize("name", ["f16_f16", "bf16_bf16"])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("nodes", [4, 14, 90])
def test_not_finite_reaches_only_who_sees_it(gpu, name, which, bad, nodes):
    """A NaN or infinity at a new token's key: rows that do not see it are as without it, bit for bit."""
    import torch

    nk, token = nodes + 70, nodes // 2
    a = Tree(name, [(nodes, nk)], 4, 2, 64).run().check()
    b = Tree(name, [(nodes, nk)], 4, 2, 64)
    at = nk - nodes + token
    (b.dk if which == "k" else b.dv)[b.table[0, at // 16], at % 16, 1, 7] = bad
    b.run()
    see = b.see(0)[:, at]
    assert see.any() and not see.all()
    blind, seen = R.dev(np.nonzero(~see)[0]), R.dev(np.nonzero(see)[0])
    assert torch.equal(a.out[blind], b.out[blind]) and torch.equal(a.lse[blind], b.lse[blind])
    assert torch.equal(a.out[:, :2], b.out[:, :2])  # the other key head's queries
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
@pytest.mark.parametrize("nodes", [4, 14, 90])
def test_scale_not_finite_reaches_only_who_sees_it(gpu, name, which, bad, nodes):
    nk, token = nodes + 70, nodes // 2
    c = Tree(name, [(nodes, nk)], 4, 2, 64)
    k, v, _ = c.keys(0)
    want = R.attention(c.q, k, v, c.see(0), c.scale)
    at = nk - nodes + token
    getattr(c, which)[c.table[0, at // 16], 1, at % 16] = bad
    c.run()
    tol, tol_lse = R.attention_bound(c.kind, c.d, *want)
    out, lse = R.host(c.out), R.host(c.lse)
    fine = np.ones(out.shape[:2], bool)
    fine[c.see(0)[:, at], 2:] = False  # the heads that read key head 1
    assert fine[:, 2:].any() and not fine.all()
    assert (np.abs(out - want[0]) <= tol)[fine].all()
    assert (np.abs(lse - want[1]) <= tol_lse)[fine].all()
    if which == "dsv" or np.isnan(bad):
        assert not np.isfinite(out[~fine]).all(axis=-1).any()


@pytest.mark.parametrize("name", NAMES)
def test_unused_memory_is_not_used(gpu, name):
    """Past kv_len and in other pages lie NaN (the cases' default) or zeros: the same bits."""
    import torch

    for nodes in (4, 14, 70):
        a = Tree(name, [(nodes, 75), (nodes, 130)], 4, 2, 64, spare=0.0).run().check()
        b = Tree(name, [(nodes, 75), (nodes, 130)], 4, 2, 64, spare=0.0)
        if a.dsk is not None:
            for x, y in ((b.dk, a.dk), (b.dv, a.dv), (b.dsk, a.dsk), (b.dsv, a.dsv)):
                x.copy_(y)
            for x in (b.dsk, b.dsv):
                x.transpose(1, 2)[R.dev(~b.used)] = float("nan")
        else:
            for x in (b.dk, b.dv):
                x[R.dev(~b.used)] = float("nan")
        b.run()
        assert torch.equal(a.out, b.out) and torch.equal(a.lse, b.lse)


@pytest.mark.parametrize("name", NAMES)
def test_mixed_batch_and_strides(gpu, name):
    lengths = [(1, 500), (40, 40), (4, 30), (130, 300), (0, 0), (1, 1), (8, 260), (17, 18), (12, 1000)]
    Tree(name, lengths, 8, 2, 80, pad=16).run().check()
    Tree(name, lengths, 3, 3, 128, pad=8).run().check()
    Tree(name, lengths, 48, 1, 64).run().check()
    Tree(name, lengths, 34, 1, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("most", [4, 8, 30])
def test_many_sequences(gpu, name, most):
    """More sequences than a wave has lanes, of all kinds, empty ones among them."""
    rng = np.random.default_rng(9)
    lengths = [(int(rng.integers(0, most + 1)), int(rng.choice([0, 1, 7, 40, 129, 300]))) for _ in range(203)]
    Tree(name, lengths, 4, 2, 64).run().check()


@pytest.mark.parametrize("name", NAMES)
def test_bounds(gpu, name):
    """Larger bounds than the lengths, more keys than max_kv_len, more queries than max_q_len (which are not written,
    while the others still see the keys that their masks name), and masks of fewer words than new tokens."""
    c = Tree(name, [(3, 100), (6, 30)], 4, 2, 64, words=5)
    c.table = np.concatenate((c.table, np.full((2, 600), -1, np.int32)), 1)
    c.run(max_q=140, max_kv=9000).check()
    c = Tree(name, [(3, 100), (3, 64)], 4, 2, 64)
    c.run(max_kv=64)
    c.lengths = [(3, 64), (3, 64)]
    c.check()
    for window in (0, 40):
        for most in (2, 7, 30):
            c = Tree(name, [(50, 90), (3, 40), (40, 200)], 4, 2, 64, words=1, window=window,
                     rows=[range(50)] * 50 + [range(3)] * 3 + [range(40)] * 40)
            c.run(max_q=most, noise=False).check(only=most)


@pytest.mark.parametrize("nodes", [3, 9, 50])
def test_without_lse_and_the_same_bits_every_time(gpu, nodes):
    import torch

    for name in NAMES:
        c = Tree(name, [(nodes, 3000), (nodes, 80)], 4, 2, 64, page=32).run().check()
        out, lse = c.out, c.lse
        for _ in range(3):
            c.run()
            assert torch.equal(out, c.out) and torch.equal(lse, c.lse)
        c.run(no_lse=True)
        assert torch.equal(out, c.out) and (c.lse == 9.0).all()


@pytest.mark.parametrize("lengths", [[(4, 900), (2, 77)], [(9, 500), (13, 200)], [(40, 500), (60, 200)]])
def test_graph_replay_with_changing_lengths_and_trees(gpu, lengths):
    import torch

    c = Tree("f16_f16", [(q, 1000) for q, _ in lengths], 8, 2, 64)
    p = c.params()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        D.run("attn_tree_f16_f16", p, torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(2)
    for n0, n1 in [(900, 77), (20, 1000), (500, 499), (61, 90)]:
        rows = []
        for q, _ in lengths:
            parents = D.random_parents(rng, q)
            rows += [D.path(parents, i) for i in range(q)]
        c.mask = D.pack(rows, c.mask.shape[1])
        c.args[1].copy_(R.dev(np.array([n0, n1], np.int32)))
        c.args[3].copy_(R.dev(c.mask.view(np.int32)))
        c.out.fill_(9.0)
        c.lse.fill_(9.0)
        c.space.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        c.lengths = [(lengths[0][0], n0), (lengths[1][0], n1)]
        c.check()


# 8 key heads with two query heads each: 17 to 64 tokens are a tile, so 8 to 16 sequences are 64 to 128 workgroups, whose
# keys are cut into equal spans of each sequence's own
EVEN = [[(40, 2000), (33, 500), (64, 1400), (20, 64), (17, 17), (50, 900), (5, 700), (0, 30), (30, 1100), (64, 64), (21, 0)],
        [(30, 1500)] * 9, [(17 + 5 * i, 40 + 131 * i) for i in range(10)], [(65, 1800), (100, 130), (128, 1300), (70, 71)]]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("lengths", EVEN)
@pytest.mark.parametrize("d,window", [(64, 0), (128, 0), (144, 0), (64, 150)])
def test_spans_of_each_sequence(gpu, name, lengths, d, window):
    kv = {"max_kv": 6000} if window == 0 else {}
    c = Tree(name, lengths, 16, 8, d, window=window)
    per = -(-6000 // c.page)
    if kv:  # the bound is far above the lengths; the table has to hold it
        wide = np.zeros((len(lengths), per), np.int32)
        wide[:, :c.table.shape[1]] = c.table
        c.table = wide
    c.run(**kv).check()


@pytest.mark.parametrize("name", NAMES)
def test_spans_of_a_round(gpu, name):
    """Half a round of workgroups and more (64 sequences of one tile, 8 key heads), and one length over all others."""
    lengths = [(17 + b % 40, 17 + b % 40 + 5 * b) for b in range(62)] + [(40, 4100), (3, 900)]
    c = Tree(name, lengths, 16, 8, 64)
    wide = np.zeros((len(lengths), 8200 // c.page + 1), np.int32)
    wide[:, :c.table.shape[1]] = c.table
    c.table = wide
    c.run(max_kv=8200).check()


@pytest.mark.parametrize("name", NAMES)
def test_spans_replayed_as_lengths_change(gpu, name):
    """One graph, eager calls between its replays: equal lengths, one long one, short ones, the bounds' own."""
    import torch

    longest = [(64, 3000)] * 10
    c = Tree(name, longest, 16, 8, 64)
    p = c.params(max_kv=3000)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        D.run("attn_tree_" + name, p, torch.cuda.current_stream().cuda_stream)
    q_len = [q for q, _ in longest]
    for lengths in (longest, [(64, 3000)] + [(64, 70)] * 9, [(64, 64 + 300 * b) for b in range(10)], [(64, 64)] * 10):
        assert [q for q, _ in lengths] == q_len
        c.lengths = lengths
        c.args[1].copy_(R.dev(np.array([n for _, n in lengths], np.int32)))
        for replay in range(2):
            c.out.fill_(9.0)
            if replay:
                D.run("attn_tree_" + name, p)
            graph.replay()
            torch.cuda.synchronize()
            c.check()


@pytest.mark.parametrize("name", NAMES)
def test_two_at_once(gpu, name):
    """Calls on streams of their own, with parts in workspaces of their own."""
    import torch

    both = [Tree(name, [(5, 1500), (3, 700)], 4, 2, 64), Tree(name, [(40, 1200), (20, 900)], 4, 2, 64)]
    params, streams = [c.params() for c in both], [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for _ in range(3):
        for p, s in zip(params, streams):
            D.run("attn_tree_" + name, p, s.cuda_stream)
    torch.cuda.synchronize()
    for c in both:
        assert c.size > 0
        c.check()


def test_nothing_to_do(gpu):
    mod, lib = R.binding()
    run = lib.op("attn_tree_f16_f16", "run")
    run(None)
    for kw in (dict(batch=0, q_tokens=5, q_heads=4), dict(batch=2, q_tokens=0, q_heads=4)):
        run(ctypes.byref(mod.AttnTreeParams(attn=mod.AttnPagedParams(**kw))))
