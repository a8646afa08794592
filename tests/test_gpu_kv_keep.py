"""The cache's rows of accepted tokens on the GPU, bit for bit, against a plain move."""

import ctypes

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R

pytestmark = pytest.mark.gpu
KINDS = ["f16", "bf16", "qsi8dx"]


class Keep:
    """lengths: (drafted tokens, tokens in the cache) of every sequence; keep: a list for each."""

    def __init__(self, kind, lengths, keep, kv_heads=2, d=64, page=16, layers=1, heads_first=False, max_keep=None,
                 keep_len=None):
        import torch

        self.kind, self.page, self.layers, self.lengths = kind, page, layers, lengths
        rng = np.random.default_rng(len(lengths) + d + page)
        per = max([1] + [-(-n // page) for _, n in lengths]) + 1
        pages = per * len(lengths) + 2
        self.pages = pages
        self.table = rng.permutation(pages)[:per * len(lengths)].reshape(-1, per).astype(np.int32)
        self.heads_first = heads_first
        shape = (layers, pages, kv_heads, page, d) if heads_first else (layers, pages, page, kv_heads, d)
        self.c = [torch.randint(-127, 128, shape, dtype=torch.int8, device="cuda:0") if kind == "qsi8dx" else
                  torch.randn(shape, device="cuda:0").to(R.torch_type(kind)) for _ in range(2)]
        self.s = [torch.rand((layers, pages, kv_heads, page), device="cuda:0") if kind == "qsi8dx" else None
                  for _ in range(2)]
        self.max_keep = max([1] + [len(k) for k in keep]) if max_keep is None else max_keep
        self.keep = np.full((len(lengths), max([1] + [len(k) for k in keep]) + 1), -3, np.int32)
        for b, k in enumerate(keep):
            self.keep[b, :len(k)] = k
        self.keep_len = np.array([len(k) for k in keep] if keep_len is None else keep_len, np.int32)

    def rows(self, x):
        """A cache tensor as [layers, slots, ...] on the host."""
        x = x.cpu().float().numpy()
        if x.ndim == 4:  # scales
            return x.transpose(0, 1, 3, 2).reshape(self.layers, -1, x.shape[2])
        x = x.transpose(0, 1, 3, 2, 4) if self.heads_first else x
        return x.reshape(self.layers, -1, *x.shape[3:])

    def want(self):
        got = [None if x is None else self.rows(x).copy() for x in self.c + self.s]
        before = [None if x is None else x.copy() for x in got]
        kv_len = []
        for b, (nq, n) in enumerate(self.lengths):
            base = n - nq
            if base < 0:
                kv_len.append(0)
                continue
            path = D.kept(self.keep[b], self.keep_len[b], nq, self.max_keep)
            kv_len.append(base + len(path))
            for j, i in enumerate(path):
                src, dst = base + i, base + j
                ps, pd = self.table[b, src // self.page], self.table[b, dst // self.page]
                if 0 <= ps < self.pages and 0 <= pd < self.pages:
                    for x, y in zip(got, before):
                        if x is not None:
                            x[:, pd * self.page + dst % self.page] = y[:, ps * self.page + src % self.page]
        return got, kv_len

    def params(self, kv_len_out=True):
        import torch

        mod, _ = R.binding()
        starts = np.concatenate(([0], np.cumsum([q for q, _ in self.lengths]))).astype(np.int32)
        self.out = torch.full((len(self.lengths) + 1,), 77, dtype=torch.int32, device="cuda:0")
        self.dev = [R.dev(x) for x in (starts, np.array([n for _, n in self.lengths], np.int32), self.keep,
                                       self.keep_len, self.table)]
        kv = R.paged(mod, self.c[0][0], self.c[1][0], None if self.s[0] is None else self.s[0][0],
                     None if self.s[1] is None else self.s[1][0], heads_first=self.heads_first)
        return mod.KVKeepParams(
            batch=len(self.lengths), max_keep=self.max_keep, q_start=R.ptr(self.dev[0]), kv_len=R.ptr(self.dev[1]),
            kv_len_out=R.ptr(self.out) if kv_len_out else None, keep=R.ptr(self.dev[2]),
            ld_keep=self.keep.shape[1], keep_len=R.ptr(self.dev[3]), block_table=R.ptr(self.dev[4]),
            ld_table=self.table.shape[1], layers=self.layers, layer_stride=self.c[0].stride(0),
            scale_layer_stride=0 if self.s[0] is None else self.s[0].stride(0), kv=kv)

    def check(self, **kw):
        want, kv_len = self.want()
        D.run("kv_keep_" + self.kind, self.params(**kw))
        for x, y in zip(self.c + self.s, want):
            if x is not None:
                np.testing.assert_array_equal(self.rows(x), y)
        assert self.out.tolist() == (kv_len if kw.get("kv_len_out", True) else [77] * len(kv_len)) + [77]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("d,kv_heads,page,heads_first", [(64, 2, 16, False), (16, 1, 1, False), (256, 3, 24, True),
                                                         (80, 8, 16, True), (128, 5, 3, False)])
@pytest.mark.parametrize("layers", [1, 3])
def test_paths(gpu, kind, d, kv_heads, page, heads_first, layers):
    """Paths that stay, move by one, overlap their own places, are long, empty, cross pages."""
    lengths = [(7, 50), (7, 23), (1, 1), (26, 26), (40, 95), (5, 90), (0, 12), (33, 64)]
    keep = [[0, 2, 5], [0, 1, 2], [0], [1, 2, 3, 4, 5, 20, 21, 22, 23, 24, 25], list(range(3, 40)), [], [], [32]]
    Keep(kind, lengths, keep, kv_heads, d, page, layers, heads_first).check()


@pytest.mark.parametrize("kind", KINDS)
def test_random_paths(gpu, kind):
    rng = np.random.default_rng(5)
    lengths, keep = [], []
    for b in range(90):
        nq = int(rng.integers(0, 60))
        lengths.append((nq, nq + int(rng.integers(0, 90))))
        keep.append(sorted(rng.permutation(nq)[:rng.integers(0, nq + 1)].tolist()))
    Keep(kind, lengths, keep, layers=2).check()


@pytest.mark.parametrize("kind", KINDS)
def test_lists_that_break_their_order(gpu, kind):
    """A list ends before an entry that is not above the last, or no drafted token; lengths out of range."""
    lengths = [(9, 40)] * 8 + [(9, 4)]
    keep = [[0, 3, 3, 5], [2, 1, 4], [4, 9, 10], [-1, 2], [0, 2, 2 ** 31 - 1, 8], [1, 3, 5, 7], [8], [0, 4, 5], [1, 2]]
    Keep(kind, lengths, keep, keep_len=[4, 3, 3, 2, 4, 9, -3, 2, 2], max_keep=3).check()
    Keep(kind, lengths, keep, max_keep=0).check()
    Keep(kind, lengths, keep).check(kv_len_out=False)


@pytest.mark.parametrize("kind", KINDS)
def test_pages_not_kept(gpu, kind):
    """Rows from or to an entry that names no page are not moved; others of the path are."""
    c = Keep(kind, [(30, 70)], [[1, 5, 12, 20, 25, 29]], page=4)
    c.table[0, 10], c.table[0, 13] = -1, 10 ** 9
    c.check()


@pytest.mark.parametrize("kind", KINDS)
def test_sequences_that_brought_nothing(gpu, kind):
    """With slots: a first row without one leaves its sequence as it is, whatever its list names; rows past the slots
    are none."""
    lengths = [(7, 50), (5, 23), (0, 12), (6, 40), (4, 3), (9, 33), (3, 20)]
    keep = [[0, 2, 5], [1, 3], [], [2, 4, 5], [0, 1], [8], [1, 2]]
    c = Keep(kind, lengths, keep, layers=2)
    starts = np.concatenate(([0], np.cumsum([q for q, _ in lengths])))
    tokens = int(starts[6])  # the last sequence's rows are past the buffer
    slots = np.arange(tokens, dtype=np.int64)
    slots[starts[0] + 1] = slots[starts[0] + 3] = -1  # rows past the first do not matter
    out = [1, 3, 4, 6]
    for b in (1, 3, 4):
        slots[starts[b]] = -1
    c.lengths = [(0, n) if b in out else (q, n) for b, (q, n) in enumerate(lengths)]
    want, kv_len = c.want()
    assert [kv_len[b] for b in out] == [23, 40, 3, 20]
    c.lengths = lengths
    p = c.params()
    dev = R.dev(slots)
    p.slots, p.tokens = R.ptr(dev), tokens
    D.run("kv_keep_" + kind, p)
    for x, y in zip(c.c + c.s, want):
        if x is not None:
            np.testing.assert_array_equal(c.rows(x), y)
    assert c.out.tolist() == kv_len + [77]


def test_longer_than_the_table(gpu):
    """A kv_len past the block table counts as its end."""
    c = Keep("f16", [(6, 30)], [[1, 3, 5]])
    c.table = c.table[:, :1].copy()
    c.lengths = [(6, 16)]
    want, kv_len = c.want()
    p = c.params()
    c.dev[1].fill_(10 ** 6)
    D.run("kv_keep_f16", p)
    np.testing.assert_array_equal(c.rows(c.c[0]), want[0])
    assert c.out.tolist() == kv_len + [77]


def test_past_32_bit_offsets(gpu):
    """Layers whose byte offsets pass 2^32."""
    import torch

    mod, _ = R.binding()
    page, d, stride = 16, 64, 2 ** 31 + 2 ** 20
    big = torch.empty(stride + 2 ** 20, dtype=torch.float16, device="cuda:0")
    view = big.as_strided((2, 4, page, 2, d), (stride, page * 2 * d, 2 * d, d, 1))
    view.copy_(torch.randn(view.shape, device="cuda:0"))
    c = Keep("f16", [(8, 40)], [[0, 4, 7]])
    c.layers, c.c, c.pages = 2, [view, view], 4
    c.table = np.array([[2, 3, 0, 1]], np.int32)
    want, _ = c.want()
    D.run("kv_keep_f16", c.params())
    np.testing.assert_array_equal(c.rows(view), want[0])


def test_replayed_as_lists_change(gpu):
    import torch

    c = Keep("bf16", [(20, 60), (20, 45)], [[0] * 6, [0] * 6])
    p = c.params()
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        D.run("kv_keep_bf16", p, torch.cuda.current_stream().cuda_stream)
    rng = np.random.default_rng(0)
    for _ in range(4):
        for b in range(2):
            c.keep[b, :6] = np.sort(rng.permutation(20)[:6])
        c.keep_len = rng.integers(0, 7, 2).astype(np.int32)
        c.dev[2].copy_(R.dev(c.keep))
        c.dev[3].copy_(R.dev(c.keep_len))
        want, kv_len = c.want()
        graph.replay()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(c.rows(c.c[0]), want[0])
        np.testing.assert_array_equal(c.rows(c.c[1]), want[1])
        assert c.out.tolist() == kv_len + [77]


def test_two_at_once(gpu):
    """Calls of two caches on streams of their own."""
    import torch

    both = [Keep("f16", [(20, 60)] * 40, [[1, 4, 9, 15]] * 40), Keep("qsi8dx", [(30, 95)] * 30, [[0, 2, 29]] * 30)]
    want = [c.want() for c in both]
    params = [c.params() for c in both]
    streams = [torch.cuda.Stream() for _ in both]
    torch.cuda.synchronize()
    for c, p, s in zip(both, params, streams):
        D.run("kv_keep_" + c.kind, p, s.cuda_stream)
    torch.cuda.synchronize()
    for c, (rows, kv_len) in zip(both, want):
        for x, y in zip(c.c + c.s, rows):
            if x is not None:
                np.testing.assert_array_equal(c.rows(x), y)
        assert c.out.tolist() == kv_len + [77]


def test_nothing_to_do(gpu):
    mod, lib = R.binding()
    run = lib.op("kv_keep_f16", "run")
    run(None)
    run(ctypes.byref(mod.KVKeepParams(batch=0, layers=1)))
    run(ctypes.byref(mod.KVKeepParams(batch=1, layers=0)))
