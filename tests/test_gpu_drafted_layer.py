"""The operators of a step with drafted tokens together as a program uses them: examples/drafted_layer.py (plan,
products, append with norm, tree attention, kept rows; sequences that end and begin) against the layer in 64 bits."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# The bounds of the layer without trees (test_gpu_attention_layer.py): the same roundings, 11 bits each of the cache's
# rows, the probabilities and the result; int8 rows with a step of amax / 127, normalised rows having the same ratio of
# amax to their size. The norm itself is in f32.
def example():
    spec = importlib.util.spec_from_file_location("drafted_layer", os.path.join(ROOT, "examples", "drafted_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("int8_cache", [False, True])
def test_refused_sequence_stays_as_it_is(gpu, int8_cache):
    """A step with pages for one sequence of two: the other's length and rows are the same after append and keep, and
    the next step, with pages again, goes on from them."""
    import torch

    mod = example()
    layer, n = mod.Layer(2, int8_cache), 2 * mod.PAGE
    g = torch.Generator(device="cuda").manual_seed(1)
    hidden = lambda rows: torch.randn((rows, mod.HIDDEN), generator=g, device="cuda").half()  # noqa: E731
    layer.step(hidden(2 * n), [n, n], mod.MAX_LEN)
    layer.kv_len.copy_(layer.with_drafted)
    caches = [x for x in (layer.k, layer.v, layer.sk, layer.sv) if x is not None]
    pages = layer.blocks[1, :2].long()
    before = [x[pages].clone() for x in caches]
    for pages_left, refused, kv_len in ((1, 1, [n + 2, n]), (layer.num_pages - 5, 0, [n + 4, n + 2])):
        layer.free_count.fill_(pages_left)
        layer.step(hidden(10), [5, 5], mod.MAX_LEN, mod.ints([-1, 0, 1, 1, 0] * 2))
        assert int(layer.refused) == refused
        layer.keep(mod.ints([[0, 4], [0, 1]]), mod.ints([2, 2]))
        assert layer.kv_len.tolist() == kv_len
        assert layer.blocks[1, :2].tolist() == pages.tolist()
        for x, y in zip(caches, before):
            assert torch.equal(x[pages], y)


@pytest.mark.parametrize("int8_cache,bound", [(False, 4 * 2.0 ** -11), (True, 0.03)])
def test_layer(gpu, int8_cache, bound):
    seen = list(example().run(int8_cache))
    assert len(seen) == 18
    for step, b, n, err in seen:
        assert err <= bound, (step, b, n, err)
