"""What kv_keep takes and refuses of a step's positions (no GPU)."""

import pytest

import test_drafted_host as T


@pytest.mark.parametrize("change,refused", [
    (dict(positions=4096, tokens=7), False), (dict(positions=4096, slots=4096, tokens=7), False),
    (dict(positions=4096, tokens=2 ** 31), True), (dict(positions=None, tokens=2 ** 31), False)])
def test_positions(change, refused):
    for name in T.KEEPS:
        assert bool(T.H.refusal(name, T.H.changed(T.keep_params, **change))) == refused
