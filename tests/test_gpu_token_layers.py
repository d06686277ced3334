"""The example model trains and writes: every operator and every gradient together, as a program has them."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_example_learns(tb, monkeypatch):
    monkeypatch.syspath_prepend(os.path.join(ROOT, "examples"))
    monkeypatch.setattr(sys, "argv", ["token_layers.py", "--steps", "40"])
    import token_layers
    losses = token_layers.main()
    # each token has two successors: log 2 = 0.69 is what can be learnt of log 211 = 5.35; a model that learns gets half way in forty steps
    assert losses[0] > 4 and losses[-1] < 3
