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
@pytest.mark.parametrize("int8_cache,bound", [(False, 4 * 2.0 ** -11), (True, 0.03)])
def test_layer(gpu, int8_cache, bound):
    spec = importlib.util.spec_from_file_location("drafted_layer", os.path.join(ROOT, "examples", "drafted_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    seen = list(mod.run(int8_cache))
    assert len(seen) == 18
    for step, b, n, err in seen:
        assert err <= bound, (step, b, n, err)
