"""Int8 caches whose value scales lie far apart, on the GPU against the plain form in 64 bits: a row's result depends on
the keys that it sees alone, and on a key no more than its probability times its scale does."""

import numpy as np
import pytest

import paged_ref as R
from test_gpu_attn_paged import Case

pytestmark = pytest.mark.gpu

INT8 = ["f16_qsi8dx", "bf16_qsi8dx"]
# new tokens and keys: tiles, with the keys of one workgroup and split over several; few rows, in one and in
# several workgroups
TILES = [(90, 150), (40, 3001)]
FEW = [(8, 100), (5, 3001)]


def values(c):
    """The value scales in device memory have changed: the plain form's values anew."""
    c.v = R.host(c.dv) * R.host(c.dsv).transpose(0, 2, 1)[..., None]
    return c


def at(c, key):
    return c.table[0, key // c.page], key % c.page


def check_unseen(name, lengths, d, factor, window):
    """One key's value scale, 3 keys before the end of what the last row sees: rows blind to it keep their bits."""
    import torch

    key = lengths[1] - 3
    c = Case(name, [lengths], 4, 2, d, window=window).run().check()
    out, lse = c.out, c.lse
    page, off = at(c, key)
    c.dsv[page, :, off] = factor
    c.run()
    blind = R.dev(np.nonzero(~R.visible(*lengths, True, window)[:, key])[0])
    assert len(blind) > 0
    assert torch.equal(out[blind], c.out[blind]) and torch.equal(lse[blind], c.lse[blind])


def check_zero_row(name, lengths, d, factor):
    """A seen row of zeros has a scale that means nothing: any finite one gives the same bits."""
    import torch

    c = Case(name, [lengths], 4, 2, d)
    page, off = at(c, 5)
    c.dv[page, off] = 0
    c.dsv[page, :, off] = 0.01
    values(c).run().check()
    out, lse = c.out, c.lse
    c.dsv[page, :, off] = factor
    values(c).run().check()
    assert torch.equal(out, c.out) and torch.equal(lse, c.lse)


def check_low_score(name, lengths, d, factor):
    """A seen key of a score far below the others', with a scale far above theirs."""
    c = Case(name, [lengths], 4, 2, d)
    c.dq.abs_()
    c.q = R.host(c.dq)
    page, off = at(c, 7)
    c.dk[page, off] = -127
    c.k = R.host(c.dk) * R.host(c.dsk).transpose(0, 2, 1)[..., None]
    c.dsv[page, :, off] = factor
    values(c).run().check()


def check_far_apart(lengths, d, low, high, period):
    """Scales of 2^low and, every `period` keys, of 2^high among the same row's keys (bf16: its range has both).
    Rows before the first of these see the low ones alone."""
    c = Case("bf16_qsi8dx", [lengths], 4, 2, d)
    c.dv.masked_fill_(c.dv == 0, 1)
    for key in range(lengths[1]):
        page, off = at(c, key)
        c.dsv[page, :, off] = 2.0 ** (high if key % period == period - 1 else low)
    values(c).run().check()


def check_negative(name, lengths, d):
    """Scales of either sign."""
    c = Case(name, [lengths], 4, 2, d)
    c.dsv[::2] *= -50.0
    values(c).run().check()


def check_not_finite_underflow(name, lengths, d, bad):
    """A value scale that is no number, at a key whose probability is below f32's range: NaN all the same."""
    c = Case(name, [lengths], 4, 2, d)
    c.dq.abs_()
    c.dq.mul_(20)
    page, off = at(c, lengths[1] - 3)
    c.dk[page, off] = -127
    c.dsv[page, 1, off] = bad
    c.run()
    see = R.visible(*lengths, True, 0)[:, lengths[1] - 3]
    out, lse = R.host(c.out), R.host(c.lse)
    assert np.isnan(out[see][:, 2:]).all() and np.isnan(lse[see][:, 2:]).all()
    assert np.isfinite(out[~see]).all() and np.isfinite(out[:, :2]).all()


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", TILES)
@pytest.mark.parametrize("d", [64, 96, 256])
@pytest.mark.parametrize("factor,window", [(2.0 ** 20, 0), (2.0 ** 30, 40), (3e38, 0)])
def test_tiles_unseen(gpu, name, lengths, d, factor, window):
    check_unseen(name, lengths, d, factor, window)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", TILES)
@pytest.mark.parametrize("factor", [1.0, 2.0 ** 20, 2.0 ** 100])
def test_tiles_zero_row(gpu, name, lengths, factor):
    check_zero_row(name, lengths, 64, factor)
    check_zero_row(name, lengths, 192, factor)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", TILES)
@pytest.mark.parametrize("factor", [2.0 ** 8, 2.0 ** 14])
def test_tiles_low_score(gpu, name, lengths, factor):
    check_low_score(name, lengths, 64, factor)
    check_low_score(name, lengths, 128, factor)


@pytest.mark.parametrize("lengths", TILES)
@pytest.mark.parametrize("low,high", [(-7, 20), (-50, 100), (-30, 110)])
@pytest.mark.parametrize("period", [75, 1])
def test_tiles_far_apart(gpu, lengths, low, high, period):
    check_far_apart(lengths, 64, low, high, period)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", TILES)
def test_tiles_negative(gpu, name, lengths):
    check_negative(name, lengths, 64)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", TILES)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_tiles_not_finite_underflow(gpu, name, lengths, bad):
    check_not_finite_underflow(name, lengths, 64, bad)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", FEW)
@pytest.mark.parametrize("d", [64, 96, 256])
@pytest.mark.parametrize("factor,window", [(2.0 ** 20, 0), (2.0 ** 30, 40), (3e38, 0)])
def test_few_rows_unseen(gpu, name, lengths, d, factor, window):
    check_unseen(name, lengths, d, factor, window)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", FEW + [(1, 700)])
@pytest.mark.parametrize("factor", [1.0, 2.0 ** 20, 2.0 ** 100])
def test_few_rows_zero_row(gpu, name, lengths, factor):
    check_zero_row(name, lengths, 64, factor)
    check_zero_row(name, lengths, 192, factor)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", FEW + [(1, 700)])
@pytest.mark.parametrize("factor", [2.0 ** 8, 2.0 ** 14])
def test_few_rows_low_score(gpu, name, lengths, factor):
    check_low_score(name, lengths, 64, factor)
    check_low_score(name, lengths, 128, factor)


@pytest.mark.parametrize("lengths", FEW + [(1, 700)])
@pytest.mark.parametrize("low,high", [(-7, 20), (-50, 100), (-30, 110)])
@pytest.mark.parametrize("period", [75, 1])
def test_few_rows_far_apart(gpu, lengths, low, high, period):
    check_far_apart(lengths, 64, low, high, period)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", FEW)
def test_few_rows_negative(gpu, name, lengths):
    check_negative(name, lengths, 64)


@pytest.mark.parametrize("name", INT8)
@pytest.mark.parametrize("lengths", FEW)
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_few_rows_not_finite_underflow(gpu, name, lengths, bad):
    check_not_finite_underflow(name, lengths, 64, bad)
