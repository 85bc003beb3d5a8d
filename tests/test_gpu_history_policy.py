"""The example policy (examples/train_history_policy.py): training through the control step runs and lowers its loss, and
the control loop over cached histories gives the training rollout's controls."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def example():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")
    spec = importlib.util.spec_from_file_location("train_history_policy", os.path.join(ROOT, "examples", "train_history_policy.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_training_and_control_loop(example):
    net, losses, (state, friction, com, height) = example.train(worlds=64, steps=4, updates=8, report=lambda s: print(s, flush=True))
    assert all(x == x for x in losses) and losses[-1] < losses[0], losses
    with torch.no_grad():
        _, trained = example.rollout(net, state, friction, com, 4)
    _, looped = example.control_loop(net, state, friction, com, 4)
    # the first controls differ by the attention's roundings alone (bfloat16: 2^-8 of values that a norm, a product with
    # weights of about 0.01 x sqrt(128) and 0.3 tanh follow); later ones also by the states that came of them
    assert (trained[0] - looped[0]).abs().max() < 2e-3
    assert (trained[3] - looped[3]).abs().max() < 2e-2


def test_training_is_the_same_every_time(example):
    a, b = (example.train(worlds=33, steps=3, updates=2, report=lambda s: None) for _ in range(2))
    assert a[1] == b[1]
