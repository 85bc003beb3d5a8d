"""The C entries of the recurrence in forms that the Python calls do not use."""
import pytest
import torch

from nablaengine_amd import torch_ffi

pytestmark = pytest.mark.gpu
TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


@pytest.fixture(autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("worlds,channels", [(1, 1), (5, 3), (4, 4), (1000, 5), (3000, 8), (5000, 9), (16384, 99), (16384, 100), (8192, 130),
                                             (4000, 513), (3000, 1001), (3, 100001)])
def test_next_states_in_the_states_own_memory(dtype, worlds, channels):
    """The next states over the states, bit for bit those beside them: at widths that are no multiple of a thread's 16 bytes the
    last elements of a row are taken once all the same. (The step is a function of its inputs: a second one of the same inputs
    gives the same.)"""
    print("in place", dtype, worlds, channels, flush=True)
    dll = torch_ffi.load_library()
    g = torch.Generator(device="cuda").manual_seed(channels)
    x, f = (torch.randn((worlds, channels), generator=g, device="cuda").to(dtype) for _ in range(2))
    state = torch.randn((worlds, channels), generator=g, device="cuda")

    def step(states, to):
        h = torch.full_like(x, 7.0)
        rc = dll.dk_recurrence_step(torch.cuda.current_stream().cuda_stream, TYPES[dtype], worlds, channels, x.data_ptr(), channels,
                                    f.data_ptr(), channels, states.data_ptr(), channels, h.data_ptr(), to.data_ptr())
        assert rc == 0
        return h, to
    h, beside = step(state, torch.full_like(state, 7.0))
    for _ in range(3):
        copy = state.clone()
        h2, over = step(copy, copy)
        assert torch.equal(h, h2) and torch.equal(beside, over)
    keep = torch.sigmoid(f.double())
    want = keep * state.double() + (1 - keep) * x.double()
    assert ((beside.double() - want).abs() <= 2.0 ** -18 * (state.double().abs() + x.double().abs())).all()
