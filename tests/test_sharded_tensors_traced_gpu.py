"""Distributed tensors through the traced operators: as eager, in torch operations."""
import pytest
import torch
import torch.distributed as dist

from torchtitan_amd.modules import residual_rms_norm, scaled_embedding

pytestmark = pytest.mark.gpu


@pytest.fixture
def mesh(device):
    """One rank; nothing is sent."""
    from torch.distributed.device_mesh import DeviceMesh

    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        yield DeviceMesh("cuda", [0])
    finally:
        dist.destroy_process_group()


def test_distributed_tensors_are_traced_in_torch_operations(device, mesh):
    from torch.distributed.tensor import DTensor, Replicate

    spread = lambda t: DTensor.from_local(t, mesh, [Replicate()], run_check=False)
    ids = torch.randint(0, 9, (5,), device=device)
    weight, h = torch.randn((9, 64), device=device), torch.randn((5, 64), device=device)
    pre = torch.randn(64, device=device)

    def step(ids, weight, h, pre):
        x = scaled_embedding(ids, weight, 2.0)
        return residual_rms_norm(h, x, pre_weight=pre)

    operands = [spread(t) for t in (ids, weight, h, pre)]
    want = step(*operands)
    torch._dynamo.reset()
    try:
        got = torch.compile(step, backend="aot_eager")(*operands)
    finally:
        torch._dynamo.reset()
    for a, b in zip(got, want):
        assert isinstance(a, DTensor) and torch.equal(a.to_local(), b.to_local())


class Named(torch.Tensor):
    """No operation of its own: torch's operations keep the type."""


def test_subclasses_without_a_dispatch_keep_their_type_when_traced(device):
    ids = torch.randint(0, 9, (5,), device=device)
    weight, h = torch.randn((9, 64), device=device).as_subclass(Named), torch.randn((5, 64), device=device)

    def step(ids, weight, h):
        return residual_rms_norm(h, scaled_embedding(ids, weight, 2.0))[0]

    want = step(ids, weight, h)
    torch._dynamo.reset()
    try:
        got = torch.compile(step, backend="aot_eager")(ids, weight, h)
    finally:
        torch._dynamo.reset()
    assert type(got) is type(want) is Named and torch.equal(got.as_subclass(torch.Tensor), want.as_subclass(torch.Tensor))
