"""The accepted rows of a step as its plan left it, on the GPU: which sequences the plan refused is told from its positions,
and from its slots wherever a page is left to tell it by. Rows whose page is no page of the cache have no slot either."""

import numpy as np
import pytest

import drafted_ref as D
import paged_ref as R
from test_gpu_paged_plan import Plan

pytestmark = pytest.mark.gpu
PAGE = 4


def step(new, kv, keep, bad_free=(), holes=(), spare=40, by="positions"):
    """Plans the step, keeps `keep` of every sequence; the lengths, and (rows of the cache, expected rows)."""
    import torch

    mod, _ = R.binding()
    c = Plan(new, kv, PAGE, spare=spare, holes=holes, held=[-(-n // PAGE) for n in kv])
    for at, page in bad_free:  # from the stack's top
        c.free[spare - 1 - at] = page
    p = c.params()
    D.run("paged_plan", p)
    after = c.check(p=p)
    cache = torch.arange(c.pages * PAGE, device="cuda:0").to(torch.float16)[:, None].repeat(1, 16)
    cache = cache.view(c.pages, PAGE, 1, 16).contiguous()
    k, v = cache.clone(), -cache
    lists = np.full((len(new), 8), -1, np.int32)
    for b, x in enumerate(keep):
        lists[b, :len(x)] = x
    out = torch.full((len(new),), 77, dtype=torch.int32, device="cuda:0")
    dev = [R.dev(x) for x in (lists, np.array([len(x) for x in keep], np.int32))]
    q = mod.KVKeepParams(
        batch=len(new), max_keep=8, q_start=R.ptr(c.out["q_start"]), kv_len=R.ptr(c.out["kv_len_out"]),
        kv_len_out=R.ptr(out), keep=R.ptr(dev[0]), ld_keep=8, keep_len=R.ptr(dev[1]),
        block_table=R.ptr(c.dev["block_table"]), ld_table=c.ld, layers=1, tokens=c.tokens,
        kv=R.paged(mod, k, v))
    setattr(q, by, R.ptr(c.out[by]))
    D.run("kv_keep_f16", q)
    want = cache.cpu().numpy().reshape(-1, 16).copy()
    was, lens = want.copy(), []
    for b, (n, length) in enumerate(zip(new, kv)):
        if after["kv_len_out"][b] != length + n:
            lens.append(length)
            continue
        lens.append(length + len(keep[b]))
        for j, i in enumerate(keep[b]):
            src, dst = length + i, length + j
            ps, pd = (after["table"][b, x // PAGE] for x in (src, dst))
            if 0 <= ps < c.pages and 0 <= pd < c.pages:
                want[pd * PAGE + dst % PAGE] = was[ps * PAGE + src % PAGE]
    for x, sign in ((k, 1), (v, -1)):
        np.testing.assert_array_equal(sign * x.cpu().numpy().reshape(-1, 16), want)
    return out.tolist(), lens, after


@pytest.mark.parametrize("by", ["positions", "slots"])
@pytest.mark.parametrize("bad", [-1, 10 ** 6, 2 ** 31 - 1])
def test_served_rows_without_a_page(gpu, by, bad):
    """The stack holds entries that name no page: all of a sequence's drafted rows fall on one, or the first, or the last."""
    got, want, after = step([3, 7, 6, 2], [8, 5, 4, 7], [[0, 2], [0, 3, 6], [2, 3, 5], [1]],
                            bad_free=[(0, bad), (4, bad)], by=by)
    assert after["refused"] == [0]
    assert (after["slots"][:3] == -1).all()  # page 0 of the stack: the first sequence's
    assert got == want == [10, 8, 7, 8]


@pytest.mark.parametrize("by", ["positions", "slots"])
def test_served_rows_behind_a_tail_without_a_page(gpu, by):
    """The last page of the context is none: the first drafted rows are on it, the next ones on a page of the stack."""
    got, want, after = step([5, 2, 4], [6, 6, 6], [[1, 2, 4], [1], []], holes=[(0, 1, -1), (1, 1, 99999)], by=by)
    assert after["refused"] == [0] and after["slots"][0] == -1 and after["slots"][2] >= 0
    assert (after["slots"][5:7] == -1).all()
    assert got == want == [9, 7, 6]


@pytest.mark.parametrize("by", ["positions", "slots"])
def test_refused_sequences_beside_served_ones(gpu, by):
    """Few pages: some are refused, one with fewer tokens than it brings, one with early pages that are not kept."""
    new, kv = [4, 9, 2, 9, 1, 0], [8, 3, 5, 41, 3, 9]
    got, want, after = step(new, kv, [[1, 3], [0, 5], [1], [2], [0], []], holes=[(3, 0, -1), (3, 1, -1)], spare=1, by=by)
    assert after["refused"] == [2]
    assert got == want == [10, 3, 6, 41, 4, 9]


def test_refused_with_a_tail_without_a_page(gpu):
    """Positions tell it where the last tokens of a refused sequence have no page either."""
    got, want, after = step([4, 3], [8, 8], [[1, 3], [0, 2]], holes=[(0, 1, -1), (1, 1, -1)], spare=0)
    assert after["refused"] == [2] and got == want == [8, 8]


def test_positions_decide_over_slots(gpu):
    """With both, positions; rows past the buffer belong to a refused sequence."""
    import torch

    mod, _ = R.binding()
    k = torch.arange(64, device="cuda:0").to(torch.float16).view(4, 16, 1, 1).repeat(1, 1, 1, 16).contiguous()
    v, out = k.clone(), torch.full((3,), 77, dtype=torch.int32, device="cuda:0")
    dev = [torch.tensor(x, dtype=torch.int32, device="cuda:0") for x in (
        [0, 2, 4, 6], [10, 12, 9], [[1], [1], [1]], [1, 1, 1], [[0], [1], [2]], [8, 9, 12, 13])]
    slots = torch.tensor([-1, -1, 5, 6], device="cuda:0")
    p = mod.KVKeepParams(batch=3, max_keep=1, q_start=R.ptr(dev[0]), kv_len=R.ptr(dev[1]), kv_len_out=R.ptr(out),
                         keep=R.ptr(dev[2]), ld_keep=1, keep_len=R.ptr(dev[3]), block_table=R.ptr(dev[4]), ld_table=1,
                         layers=1, kv=R.paged(mod, k, v), slots=R.ptr(slots), tokens=4, positions=R.ptr(dev[5]))
    D.run("kv_keep_f16", p)
    assert out.tolist() == [9, 12, 9]
    want = torch.arange(64)
    want[8] = 9
    assert torch.equal(k[:, :, 0, 0].flatten().cpu().long(), want)
