"""The vocabulary operators together, as the example uses them: the encoder's states, distillation, given tokens, answers."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "distill_vocabulary.py")


def test_example_learns(igdev):
    spec = importlib.util.spec_from_file_location("distill_vocabulary", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, nll, agree = mod.main(steps=40, log=lambda *_: None)
    assert losses[-1] < 0.5 * losses[0]
    assert nll[-1] < nll[0]
    assert agree > 0.5
