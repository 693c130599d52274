"""The 4-bit operators as one decode loop (examples/decode_4bit.py): ragged
prompts, steps in which requests end, pages that go back to the pool, and
logits against torch on the same quantised weights and cache.

Bound: both sides take the same quantised keys, values and routing, so what
differs is fp32 rounding through the layers.  A layer's products, attention and
norms each contribute a few 1e-6 of their result (K <= 512 terms at 2^-23, 22
operand bits), and the residual stream passes them on: 1e-4 leaves a factor of
about ten for two layers and the head.
"""
import importlib.util
import sys

import pytest

from conftest import ROOT


def load_example():
    spec = importlib.util.spec_from_file_location("decode_4bit", ROOT / "examples" / "decode_4bit.py")
    mod = importlib.util.module_from_spec(spec)
    sys.modules["decode_4bit"] = mod
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.gpu
@pytest.mark.parametrize("requests,new_tokens,seed", [(1, 3, 1), (5, 12, 0), (9, 6, 2)])
def test_decode_matches_torch(requests, new_tokens, seed):
    out, worst, same, total, whole = load_example().decode(requests, new_tokens, True, seed)
    assert whole, "every page is back in the pool"
    assert worst <= 1e-4
    assert same == total == sum(len(o) for o in out)


@pytest.mark.gpu
def test_decode_repeats():
    ex = load_example()
    assert ex.decode(4, 6, False, 3)[0] == ex.decode(4, 6, False, 3)[0]
