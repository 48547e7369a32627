"""GPU: AdamW with gradients of another type than their parameters."""
import pytest
import torch

from tests.test_optimizers_gpu import HYPER, SHAPES, check_steps, parameters_of
from torchtitan_amd import ops
from torchtitan_amd.optimizers import AdamW

pytestmark = pytest.mark.gpu


def gradients_in(dtype, std=1e-2):
    def set_grads(params, seed):
        for i, p in enumerate(params):
            g = torch.Generator(device=p.device).manual_seed(seed * 1000 + i)
            p.grad_dtype = None  # (any type)
            p.grad = (torch.randn(p.shape, generator=g, device=p.device) * std).to(dtype)

    return set_grads


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_float32_gradients_of_bf16_parameters_keep_their_bits(device, bits, master):
    """Beside float32 parameters in the same list, small lists and long ones, clipped."""
    for shapes in (SHAPES, [*SHAPES, (1200, 1001), (4095,), (8191,)]):
        params = parameters_of(device, shapes)
        check_steps(AdamW(params, **HYPER, weight_decay=0.1, state_bits=bits, master_weights=master, seed=3), params, steps=2,
                    norm=torch.tensor(7.0, device=device), limit=2.0, set_grads=gradients_in(torch.float32))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float16, torch.float64])
def test_gradients_of_other_types_are_read_in_float32(device, bits, dtype):
    """(float64: the step is that of their rounding to float32.)"""
    params = parameters_of(device, SHAPES)

    def set_grads(params, seed):
        gradients_in(torch.float32)(params, seed)
        for p in params:
            p.grad = p.grad.half().to(dtype)

    check_steps(AdamW(params, **HYPER, weight_decay=0.1, state_bits=bits), params, steps=2, set_grads=set_grads)


@pytest.mark.parametrize("bits", [32, 8])
def test_the_same_moments_on_the_cpu_and_in_one_launch(device, bits):
    params = parameters_of(device, SHAPES, (torch.bfloat16,))
    twins = [torch.nn.Parameter(p.detach().cpu()) for p in params]
    kw = dict(**HYPER, weight_decay=0.1, state_bits=bits, master_weights=True, seed=5)
    a, b = AdamW(params, **kw), AdamW(twins, **kw)
    for step in range(3):
        gradients_in(torch.float32)(params, step)
        for p, q in zip(params, twins):
            q.grad_dtype = None
            q.grad = p.grad.cpu()
        timer = ops.KernelTimer()
        if step:
            ops.set_kernel_timer(timer)
        try:
            a.step()
        finally:
            ops.set_kernel_timer(None)
        b.step()
        assert not step or timer.summary()["adamw"][0] == 1
        for p, q in zip(params, twins):
            for name in a.state[p]:
                if name.startswith("exp_avg"):
                    assert torch.equal(a.state[p][name].cpu(), b.state[q][name]), name


def test_views_and_orders(device):
    """float32 gradients at any element and in another order than their parameter's."""
    grads = torch.zeros(3 + 1000, device=device)
    params = [torch.nn.Parameter(torch.randn(1000, device=device).bfloat16()),
              torch.nn.Parameter(torch.randn(40, 30, device=device).bfloat16().t())]

    def set_grads(params, seed):
        grads.normal_()
        for p in params:
            p.grad_dtype = None
        params[0].grad = grads[3:]
        params[1].grad = torch.randn(30, 40, device=device)

    check_steps(AdamW(params, **HYPER, weight_decay=0.1), params, set_grads=set_grads)


def test_a_captured_step(device):
    p = torch.nn.Parameter(torch.randn(5000, device=device).bfloat16())
    q = torch.nn.Parameter(p.detach().clone())
    for t in (p, q):
        t.grad_dtype = torch.float32
        t.grad = torch.zeros(5000, device=device)
    a, b = AdamW([p], **HYPER, capturable=True), AdamW([q], **HYPER)
    a.step()
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for replay in range(3):
        p.grad.normal_()
        q.grad.copy_(p.grad)
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])
        assert torch.equal(a.state[p]["exp_avg_sq"], b.state[q]["exp_avg_sq"])
