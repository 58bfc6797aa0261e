"""The policy-training example: all the training operators in one step, as a user would run them."""
import os
import sys

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(ROOT, "examples"))


def test_the_policy_learns():
    from policy_training import train
    first, last = train(steps=40, verbose=False)
    assert first < 0.45          # five actions, untrained
    assert last > first + 0.15
