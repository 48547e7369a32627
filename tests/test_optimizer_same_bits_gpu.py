"""GPU: a value's update does not depend on where it lies or on what stands beside it."""
import pytest
import torch

from tests.test_optimizers_gpu import HYPER, parameters_of, set_gradients
from torchtitan_amd.optimizers import AdamW

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-8, 1e-12])
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True)])
def test_the_same_bits_whatever_the_list(device, bits, eps, dtype, master):
    """Alone, and beside a parameter that makes the list a long one with larger chunks."""
    some = parameters_of(device, [(8191,), (2048,), (40,)], (dtype,), seed=5)
    twins = [torch.nn.Parameter(p.detach().clone()) for p in some] + parameters_of(device, [(1200, 1001)], (dtype,), seed=6)
    kw = dict(HYPER, eps=eps, state_bits=bits, master_weights=master, seed=1)
    a, b = AdamW(some, **kw), AdamW(twins, **kw)
    for step in range(3):
        set_gradients(some, step)
        set_gradients(twins, step)
        a.step()
        b.step()
        for p, q in zip(some, twins):
            assert torch.equal(p, q)
            for name, value in a.state[p].items():
                assert value == b.state[q][name] if name == "step" else torch.equal(value, b.state[q][name])


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-8, 1e-12])
@pytest.mark.parametrize("size", [3 * 4096 + 1000, (1 << 20) + 1000])
def test_the_same_bits_wherever_a_value_lies(device, bits, eps, size):
    """Equal values in whole chunks and in the ragged last one (a first step: no moments that were rounded by chance)."""
    period = 1024
    g, w = (torch.randn(period, generator=torch.Generator(device=device).manual_seed(i), device=device) for i in (1, 2))
    repeated = lambda t: t.repeat(-(-size // period))[:size].clone()
    p = torch.nn.Parameter(repeated(w))
    p.grad = repeated(g * 1e-2)
    AdamW([p], **dict(HYPER, eps=eps), state_bits=bits).step()
    assert torch.equal(p.detach(), repeated(p.detach()[:period]))
