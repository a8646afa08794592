"""Held pages that disagree with the lengths, on the GPU: they count as the pages of kv_len at least and as ld_table at
most, in ended sequences and in those that go on. Expected values are worked by hand from that rule."""

import numpy as np
import pytest

import drafted_ref as D
from test_gpu_paged_plan import Plan

pytestmark = pytest.mark.gpu


def outcome(c, in_place=False):
    """What a plan writes, as lists; rows of `c.table` and the stack among them."""
    D.run("paged_plan", c.params(in_place))
    got = {k: v.tolist()[:len(v) - (0 if in_place and k in ("kv_len_out", "held_out", "free_count_out") else 2)]
           for k, v in c.out.items()}
    return dict(got, table=c.dev["block_table"].tolist(), free=c.dev["free_pages"].tolist())


@pytest.mark.parametrize("in_place", [False, True])
def test_ended_sequences_return_the_pages_of_their_tokens(gpu, in_place):
    """Ended: 8 tokens of pages of 4 with held 0, 1, -5; 5 tokens with held 7 (all of them), 0 tokens with held 0."""
    c = Plan([-1, -1, -1, -1, -1, 1], [8, 8, 8, 5, 0, 4], 4, ld=8, held=[0, 1, -5, 7, 0, 1], spare=2)
    c.pages = 40
    c.table[:] = np.arange(48).reshape(6, 8) % 40
    c.free = np.full(40, -9, np.int32)
    c.free[:2] = [38, 39]
    got = outcome(c, in_place)
    stack = [38, 39, 0, 1, 8, 9, 16, 17] + list(range(24, 31))
    assert got["free"][:15] == stack and got["free"][15:] == [-9] * 25
    # the last sequence takes the top one
    assert got["free_count_out"] == [14] and got["table"][5][:2] == [0, 30]
    assert got["kv_len_out"] == [0, 0, 0, 0, 0, 5] and got["held_out"] == [0, 0, 0, 0, 0, 2]
    assert got["slots"] == [30 * 4] and got["refused"] == [0]


def test_many_ended_sequences(gpu):
    """More than a round of threads; every ended one has held 0 and tokens on two pages."""
    n = 1500
    c = Plan([-1] * n, [5] * n, 4, ld=3, held=[0] * n, spare=0)
    c.pages = 2 * n
    c.table[:, :2] = np.arange(2 * n).reshape(n, 2)
    c.free = np.full(2 * n, -9, np.int32)
    got = outcome(c)
    assert got["free_count_out"] == [2 * n] and np.array_equal(got["free"], np.arange(2 * n))


def test_ended_tables_shorter_than_the_tokens(gpu):
    """40 tokens of pages of 4 with a table of 2: it is the two that go back."""
    c = Plan([-1, -1], [40, 2 ** 31 - 1], 4, ld=2, held=[0, 1], spare=0)
    c.pages = 9
    c.table[:] = [[5, 6], [7, 8]]
    c.free = np.full(9, -9, np.int32)
    got = outcome(c)
    assert got["free"] == [5, 6, 7, 8] + [-9] * 5 and got["free_count_out"] == [4]


@pytest.mark.parametrize("in_place", [False, True])
def test_tables_shorter_than_the_tokens(gpu, in_place):
    """40 tokens of pages of 4 with a table of 2: refused, new tokens or none, and held is 2; 8 and 7 tokens fit."""
    c = Plan([3, 0, 1, 1, 0], [40, 40, 8, 7, 8], 4, ld=2, held=[0, 900, 2, 2, 0], spare=3, tokens=7)
    got = outcome(c, in_place)
    assert got["refused"] == [3] and got["held_out"] == [2, 2, 2, 2, 2]
    assert got["kv_len_out"] == [40, 40, 8, 8, 8] and got["free_count_out"] == [3]
    assert got["q_start"] == [0, 3, 3, 4, 5, 5]
    page = int(c.table[3, 1])
    assert got["slots"] == [-1, -1, -1, -1, page * 4 + 3, -1, -1] and got["positions"] == [40, 41, 42, 8, 7, 0, 0]
    assert got["table"] == c.table.tolist()


def test_no_table(gpu):
    """ld_table 0: nobody holds a page, and only empty sequences that stay so are served."""
    c = Plan([0, 0, 1, -1], [0, 4, 0, 9], 4, held=[5, 1, 0, 2], spare=3)
    c.ld = 0
    p = c.params()
    p.ld_table = 0
    D.run("paged_plan", p)
    assert c.out["held_out"].tolist()[:4] == [0] * 4 and c.out["refused"].tolist()[:1] == [2]
    assert c.out["kv_len_out"].tolist()[:4] == [0, 4, 0, 0] and c.out["free_count_out"].tolist()[:1] == [3]
