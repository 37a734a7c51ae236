"""The decoder-layer example end to end: prompts, then single tokens, against the layer in 64 bits."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_layer.py")


# 16-bit caches: keys and values rounded to 11 or 8 bits; 8-bit: to half a step of max|x| / 127, up to 1 / 60 of
# a value's standard deviation.  An output sums hundreds of such values with weights of their own.
@pytest.mark.parametrize("cache,most", [("f16", 1e-2), ("bf16", 5e-2), ("i8", 1e-1)])
def test_layer(cache, most):
    spec = importlib.util.spec_from_file_location("decode_layer", PATH)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.run(4, cache) < most
