"""The recurrence at the ends of its sizes."""
import pytest
import torch

from nablaengine_amd import policy

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")


def test_channels_past_one_launch_of_the_chain():
    """2^25 channels and a few over two chunks: the kernel that carries states over chunks has 128 work-items a channel, 2^32 in
    all, more than a launch. One row for all tokens; some channels, the last ones among them, are bit for bit those of a narrow call."""
    n, c = 128, 2 ** 25 + 24
    print("channels", c, flush=True)
    g = torch.Generator(device="cuda").manual_seed(1)
    x, f, dh = (torch.randn((1, c), generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    initial, dlast = (torch.randn((1, c), generator=g, device="cuda") for _ in range(2))
    a = torch.tensor([0, n], dtype=torch.int32, device="cuda")

    def run(at):
        leaves = [x[:, at].expand(n, -1).detach().requires_grad_(), f[:, at].expand(n, -1).detach().requires_grad_(),
                  initial[:, at].contiguous().requires_grad_()]
        h, last = policy.recurrence(leaves[0], leaves[1], a, leaves[2])
        return [h.detach(), last.detach(),
                *torch.autograd.grad((h, last), leaves, (dh[:, at].expand(n, -1), dlast[:, at].contiguous()))]
    whole = run(slice(None))
    for first in (0, 2 ** 24, 2 ** 25 - 64, c - 64):
        for one, all_ in zip(run(slice(first, first + 64)), whole):
            assert torch.equal(one, all_[:, first:first + 64])
