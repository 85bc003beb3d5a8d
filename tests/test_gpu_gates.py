"""The sigmoid of the recurrence's gates in float32, each side to its own last places."""
import pytest
import torch

from nablaengine_amd import policy

pytestmark = pytest.mark.gpu
# The exponential is off by 2^-23, the correction of its argument, the sum and the product by 2^-24 each, the reciprocal by 2^-23: 7 2^-24
SMALL = 8 * 2.0 ** -24


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")


def test_small_sides_of_gates():
    """take = 1 - a of a state of 0 and an input of 1, keep = a of a state of 1 and an input of 0, one token, float32, over the
    whole range: both within SMALL of themselves."""
    g = torch.cat([torch.linspace(-87.0, 87.0, 100001, dtype=torch.float64), torch.logspace(-6, 1, 1001, dtype=torch.float64)]).float().cuda()[None]
    one, zero = torch.ones_like(g), torch.zeros_like(g)
    for name, x, s, want in (("take", one, zero, torch.sigmoid(-g.double())), ("keep", zero, one, torch.sigmoid(g.double()))):
        got = policy.recurrence_step(x, g, s)[1].double()
        off = ((got - want) / want).abs().max().item()
        assert off <= SMALL, (name, off)
        assert torch.equal(policy.recurrence(x, g, torch.tensor([0, 1], dtype=torch.int32, device="cuda"), s)[1].double(), got)
