"""examples/decode.py: a prompt, single tokens and a tree of drafts on one cache."""
import importlib.util
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
def test_a_trees_logits_are_those_of_its_tokens():
    spec = importlib.util.spec_from_file_location("decode_example", os.path.join(ROOT, "examples", "decode.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # The two ways sum in other orders and split x differently for batches of
    # other sizes (1.6e-5 of a block's largest a product, seven products deep,
    # each at most doubled by the layer after it): 2e-3 of the largest logit.
    # A key quantized across a rounding boundary moves by 1/127 or 1/8 of its
    # block's largest value, which softmax and later layers hand on: 5e-2.
    assert example.main() < 5e-2
