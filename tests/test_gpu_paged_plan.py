"""A step's plan (pages, block tables, slots, positions, tree masks) on the GPU, exactly, against drafted_ref.plan."""

import ctypes

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R

pytestmark = pytest.mark.gpu


class Plan:
    """A step's arrays; random ones from a seed unless they are given."""

    def __init__(self, new, kv, page, ld=None, spare=40, seed=0, held=None, parent=None, words=None, tokens=None,
                 holes=()):
        rng = np.random.default_rng(seed)
        new, kv = np.asarray(new, np.int32), np.asarray(kv, np.int32)
        self.new, self.kv, self.page = new, kv, page
        batch = len(new)
        own = -(-np.maximum(kv, 0) // page)
        held = own + rng.integers(0, 2, batch) if held is None else np.asarray(held)
        self.held = held.astype(np.int32)
        most = int(max([1] + [-(-(max(int(k), 0) + max(int(n), 0)) // page) for k, n in zip(kv, new)]))
        self.ld = ld or most + 2
        used = int(np.minimum(np.maximum(self.held, 0), self.ld).sum())
        self.pages = used + spare + 3
        order = rng.permutation(self.pages).astype(np.int32)
        self.table = np.full((batch, self.ld), -5, np.int32)
        at = 0
        for b in range(batch):
            n = min(max(int(self.held[b]), 0), self.ld)
            self.table[b, :n] = order[at:at + n]
            at += n
        for b, j, page_id in holes:
            self.table[b, j] = page_id
        self.free = np.full(self.pages, -9, np.int32)
        self.free[:spare] = order[at:at + spare]
        self.count = spare
        self.tokens = int(np.maximum(new, 0).sum()) if tokens is None else tokens
        self.parent = parent
        self.words = 0 if parent is None else words or max(1, -(-int(max(new.max(), 1)) // 32))

    def want(self):
        return D.plan(self.new, self.kv, self.held, self.table, self.free, self.count, self.tokens, self.page,
                      self.pages, self.parent, self.words)

    def params(self, in_place=False):
        import torch

        mod, lib = R.binding()
        full = lambda n, t=torch.int32: torch.full((n + 2,), 77, dtype=t, device="cuda:0")  # noqa: E731
        b = len(self.new)
        self.dev = {k: R.dev(np.asarray(v, np.int32)) for k, v in (
            ("new_len", self.new), ("kv_len", self.kv), ("held", self.held), ("block_table", self.table),
            ("free_pages", self.free), ("free_count", [self.count]))}
        out = dict(kv_len_out=full(b), held_out=full(b), free_count_out=full(1), refused=full(1), q_start=full(b + 1),
                   positions=full(self.tokens), slots=full(self.tokens, torch.int64))
        if in_place:
            for k in ("kv_len", "held", "free_count"):
                out[k + "_out"] = self.dev[k]
        if self.parent is not None:
            self.dev["parent"] = R.dev(np.asarray(self.parent, np.int32))
            out["mask"] = full(self.tokens * self.words)
        self.out = out
        p = mod.PagedPlanParams(batch=b, tokens=self.tokens, page_size=self.page, num_pages=self.pages,
                                ld_table=self.ld, free_capacity=len(self.free), ld_mask=self.words,
                                **{k: R.ptr(v) for k, v in list(self.dev.items()) + list(out.items())})
        self.space, self.size = D.workspace(lib, "paged_plan", p)
        return p

    def check(self, in_place=False, p=None):
        import torch

        if p is None:
            D.run("paged_plan", self.params(in_place))
        want = self.want()
        got = {k: v.cpu().numpy() for k, v in self.out.items()}
        if self.parent is None:
            want.pop("mask")
        else:
            got["mask"] = got["mask"].view(np.uint32)
            want["mask"] = want["mask"].ravel()
        for k, v in got.items():
            n = want[k].size
            np.testing.assert_array_equal(v[:n], want[k], k)
            if not (in_place and k in ("kv_len_out", "held_out", "free_count_out")):
                assert (v[n:] == 77).all(), k
        np.testing.assert_array_equal(self.dev["block_table"].cpu().numpy(), want["table"])
        np.testing.assert_array_equal(self.dev["free_pages"].cpu().numpy(), want["free"])
        assert torch.isnan(self.space[self.size // 4:]).all()
        return want


def random_step(rng, batch, new, kv):
    n = rng.integers(0, new + 1, batch)
    n[rng.random(batch) < 0.15] = -1
    return n, rng.integers(0, kv + 1, batch)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("new,kv", [([1], [0]), ([1], [16]), ([0], [5]), ([-1], [33]), ([5, 0, -1, 17], [15, 16, 9, 0]),
                                    ([1] * 70, list(range(70))), ([64, 1, 1], [0, 1000, 31])])
def test_small_steps(gpu, new, kv, in_place):
    Plan(new, kv, 16).check(in_place)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 256, 2 ** 16])
@pytest.mark.parametrize("batch,new", [(5, 40), (64, 9), (300, 3), (1024, 4), (3, 4000), (64, 300), (1025, 2),
                                       (2100, 5)])
def test_random_steps(gpu, page, batch, new):
    """One launch and two, batches of several rounds of threads, growing and ended sequences."""
    rng = np.random.default_rng(batch + new + page)
    n, kv = random_step(rng, batch, new, 500)
    Plan(n, kv, page, spare=batch * (new // page + 1) + 5, seed=page).check(in_place=bool(batch % 2))


@pytest.mark.parametrize("batch,new", [(40, 30), (1500, 20)])
def test_too_few_pages(gpu, batch, new):
    """Sequences without pages are refused, those that need none are not."""
    rng = np.random.default_rng(batch)
    n, kv = random_step(rng, batch, new, 100)
    Plan(n, kv, 8, spare=batch, seed=1).check()  # the first finds enough with what ended sequences return
    want = Plan(np.where(n < 0, 0, n), kv, 8, spare=batch // 4, seed=1).check()
    assert 0 < want["refused"][0] < batch
    want = Plan(np.where(n < 0, 0, n), kv, 8, spare=0).check()
    assert 0 < want["refused"][0] < batch and want["free_count_out"][0] == 0


def test_returned_pages_are_taken_in_the_same_step(gpu):
    """An empty stack that ended sequences fill; entries that name no page are left out."""
    want = Plan([-1, 40, -1, 3], [50, 4, 70, 8], 8, spare=0, held=[7, 1, 9, 1],
                holes=[(0, 2, -1), (2, 0, 10 ** 9), (2, 8, -2 ** 31)]).check()
    assert want["refused"][0] == 0 and want["free_count_out"][0] > 0
    rng = np.random.default_rng(0)
    n = np.where(rng.random(1300) < 0.6, -1, 3)
    Plan(n, rng.integers(0, 900, 1300), 4, spare=0, seed=2).check(in_place=True)


def test_tables_rows_and_lengths_that_do_not_fit(gpu):
    Plan([9, 9, 9], [8, 16, 20], 8, ld=3, held=[1, 2, 3]).check()  # the last would need a fourth entry
    Plan([5, 6, 7], [0, 0, 0], 4, tokens=12).check()               # the last one's rows do not fit
    Plan([5, 6, 7], [0, 0, 0], 4, tokens=3).check()
    Plan([5, 6], [0, 3], 4, tokens=30).check()                     # rows behind the last sequence
    Plan([3000, 2000], [0, 3], 4, tokens=6000, spare=1300).check()
    Plan([5, 2, 1], [-7, 3, 2], 4, held=[-3, 900, 0]).check()      # lengths and held pages out of range
    Plan([2 ** 31 - 1, 2], [5, 2 ** 30], 2 ** 20, ld=2000, held=[1, 1024], tokens=9).check()


def test_counts_out_of_range(gpu):
    a = Plan([9, 3], [4, 5], 4, spare=5)
    a.count = -4
    a.check()
    a = Plan([9, 3], [4, 5], 4, spare=5)
    a.free[:] = np.arange(len(a.free))
    a.count = 10 ** 6
    a.check()
    a = Plan([-1, -1], [40, 50], 4, spare=5)  # more pages than the stack holds
    a.free = a.free[:12]
    a.check()


def test_nothing(gpu):
    import torch

    mod, lib = R.binding()
    lib.op("paged_plan", "run")(None)
    out = torch.full((6,), 7, dtype=torch.int32, device="cuda:0")
    slots = torch.full((3,), 7, dtype=torch.int64, device="cuda:0")
    count = torch.tensor([0], dtype=torch.int32, device="cuda:0")
    at = out.data_ptr()
    p = mod.PagedPlanParams(batch=0, tokens=3, page_size=4, free_count=R.ptr(count), free_count_out=at, refused=at + 4,
                            q_start=at + 8, positions=at + 12, slots=R.ptr(slots))
    lib.op("paged_plan", "run")(ctypes.byref(p))
    assert out.tolist() == [0, 0, 0, 0, 0, 0] and slots.tolist() == [-1] * 3


@pytest.mark.parametrize("batch,new,chain", [(1, 7, 0.0), (1, 64, 0.5), (5, 130, 0.3), (64, 26, 0.2), (3, 300, 1.0),
                                             (70, 100, 0.9), (1100, 5, 0.3)])
@pytest.mark.parametrize("words", [None, 1, 12])
def test_trees(gpu, batch, new, chain, words):
    """Masks of one word and several, of fewer bits than tokens and of more, deep chains."""
    rng = np.random.default_rng(batch + new)
    n, kv = random_step(rng, batch, new, 200)
    n[0] = new
    parent = np.concatenate([D.random_parents(rng, x, chain) for x in np.maximum(n, 0)]).astype(np.int32)
    Plan(n, kv, 16, spare=batch * (new // 16 + 2), parent=parent, words=words).check()


def test_parents_that_are_none(gpu):
    """Entries not below the row's own number count as -1, whatever they are."""
    parent = np.array([0, 5, 1, -2 ** 31, 2 ** 31 - 1, 4, -3, 0, 0, 1], np.int32)
    Plan([7, 3], [5, 9], 4, parent=parent).check()
    Plan([7, 3], [5, 9], 4, parent=np.append(parent, [7, 7, 7]), tokens=13).check()


def test_two_at_once(gpu):
    """Calls on streams of their own: one launch each, and two."""
    import torch

    rng = np.random.default_rng(8)
    plans = [Plan(*random_step(rng, batch, new, 300), 16, spare=4000, seed=batch)
             for batch, new in ((90, 20), (200, 40), (90, 20), (200, 40))]
    params, streams = [c.params() for c in plans], [torch.cuda.Stream() for _ in plans]
    torch.cuda.synchronize()
    for p, s in zip(params, streams):
        D.run("paged_plan", p, s.cuda_stream)
    torch.cuda.synchronize()
    for c, p in zip(plans, params):
        c.check(p=p)


def test_replayed_with_changing_lengths(gpu):
    """A captured step whose lengths, held pages and stack are its own outputs, over several replays."""
    import torch

    for batch, most in ((9, 20), (1100, 6)):
        rng = np.random.default_rng(batch)
        a = Plan(rng.integers(0, most, batch), rng.integers(0, 50, batch), 8, spare=9000, ld=64)
        a.tokens = most * batch
        p = a.params(in_place=True)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            D.run("paged_plan", p, torch.cuda.current_stream().cuda_stream)
        for step in range(6):
            a.new = random_step(rng, batch, most, 1)[0].astype(np.int32)
            a.dev["new_len"].copy_(R.dev(a.new))
            a.space.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            want = a.check(in_place=True, p=p)
            a.kv, a.held = (want[k].astype(np.int32) for k in ("kv_len_out", "held_out"))
            a.table, a.free, a.count = want["table"], want["free"], int(want["free_count_out"][0])
