"""The operators together as a program uses them: examples/attention_layer.py (products, append with rotation, paged
attention, output product; prompts in chunks beside decoded tokens) against the layer in 64 bits."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# f16: the rows of the cache, the probabilities and the attention's result are each rounded to 11 bits
# (2^-11), which random signs keep near that in the sums: 4 of them. int8: a row's step is amax / 127, at 64
# normal values about 2.5 / 127 of their size, uniform (1 / sqrt 12), for keys and values: about 0.01.
@pytest.mark.parametrize("int8_cache,bound", [(False, 4 * 2.0 ** -11), (True, 0.03)])
def test_layer(gpu, int8_cache, bound):
    spec = importlib.util.spec_from_file_location("attention_layer",
                                                  os.path.join(ROOT, "examples", "attention_layer.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    seen = list(mod.run(int8_cache))
    assert sorted(b for b, _, _ in seen) == [0, 1, 2]
    for b, n, err in seen:
        assert err <= bound, (b, n, err)
