"""CPU: the groups that AdamW takes."""
import pytest
import torch

from torchtitan_amd.optimizers import AdamW


@pytest.mark.parametrize("bad", [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(state_bits=16),
                                 dict(seed=-1), dict(seed=1 << 64), dict(lr=torch.ones(2))])
def test_a_groups_own_numbers_are_checked(bad):
    """As the constructor's are: when it is made and when a group is added; a refused group is not there."""
    p, q = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError):
        AdamW([dict(params=[p], **bad)])
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[q], **bad))
    assert len(opt.param_groups) == 1
    opt.add_param_group(dict(params=[q], state_bits=8, lr=0.5))
    for t in (p, q):
        t.grad = torch.ones(4)
    opt.step()
    assert opt.state[p]["exp_avg"].dtype == torch.float32 and opt.state[q]["exp_avg"].dtype == torch.uint8
    # (first steps: the learning rate, but for eps, and the decay)
    assert torch.allclose(p.detach(), torch.full((4,), 1 - 1e-3 - 1e-5)) and torch.allclose(q.detach(), torch.full((4,), 0.5 - 0.005))


def test_numbers_without_a_group_of_them():
    """What every group says for itself need not be right in the defaults, which torch's optimizers check all the same."""
    p = torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError):
        AdamW([dict(params=[p], lr=1e-3)], lr=-1.0)


@pytest.mark.filterwarnings("ignore:optimizer contains")
def test_a_parameter_is_in_a_group_once():
    """Listed twice it would be one state that two entries of a launch update, with one step's correction for both."""
    p, q = torch.nn.Parameter(torch.ones(4)), torch.nn.Parameter(torch.ones(4))
    with pytest.raises(ValueError, match="twice"):
        AdamW([p, q, p])
    opt = AdamW([p])
    with pytest.raises(ValueError, match="twice"):
        opt.add_param_group(dict(params=[q, q]))
    with pytest.raises(ValueError, match="more than one"):
        opt.add_param_group(dict(params=[p]))
    assert len(opt.param_groups) == 1


def test_types_of_a_table():
    """Of parameter and gradient: what is none of the three, and a float32 gradient at half of an element, is refused in front of any launch."""
    import ctypes

    from torchtitan_amd import _lib

    lib = _lib.load()

    def adamw(types, gradient=0x2000, parameter=0x1000):
        row = [parameter, types, gradient, 0x3000, 0x4000, 0, 0, 0, 10, 1, 0]
        table = (ctypes.c_int64 * len(row))(*row)
        return lib.mx_adamw(1, ctypes.cast(table, ctypes.c_void_p), 0, 1e-3, 0.9, 0.95, 1e-8, 0.0, 0, None, 0.0, 0, None, None, None, None)

    assert adamw(3) == 1 and adamw(-1) == 1
    assert adamw(2, gradient=0x2002) == 2 and adamw(2, parameter=0x1001) == 2 and adamw(1, parameter=0x1002) == 2
