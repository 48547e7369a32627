"""CPU: what AdamW takes when it loads a state or is given a group, as torch's optimizers do."""
import copy

import pytest
import torch

from torchtitan_amd.optimizers import AdamW


def stepped(cls=AdamW, steps=3, shape=(7, 9), **options):
    p = torch.nn.Parameter(torch.randn(shape, generator=torch.Generator().manual_seed(4)))
    opt = cls([p], lr=1e-2, **options)
    for step in range(steps):
        p.grad = torch.randn(shape, generator=torch.Generator().manual_seed(step))
        opt.step()
    return p, opt


@pytest.mark.parametrize("bits", [32, 8])
def test_what_a_hook_returns_is_loaded(bits):
    """A hook in front of the loading renames, moves on and replaces; one behind it sees and changes the states that are kept."""
    _, source = stepped(state_bits=32)
    saved = copy.deepcopy(source.state_dict())
    saved["state"][0]["first"] = saved["state"][0].pop("exp_avg")
    p, opt = stepped(steps=1, state_bits=bits)
    want = torch.full((7, 9), 0.5)

    def rename(optimizer, state_dict):
        one = dict(state_dict["state"][0])
        one.pop("first")
        return {**state_dict, "state": {0: dict(one, exp_avg=want, step=50)}}

    seen = []

    def behind(optimizer):
        state = optimizer.state[p]
        seen.append((state["step"], {name: t.dtype for name, t in state.items() if name != "step"}))
        state["exp_avg_sq"] = torch.ones_like(state["exp_avg_sq"])

    opt.register_load_state_dict_pre_hook(rename)
    opt.register_load_state_dict_post_hook(behind)
    opt.load_state_dict(saved)
    state = opt.state[p]
    assert state["step"] == 50 and (state["exp_avg_sq"] == 1).all()
    held = torch.float32 if bits == 32 else torch.uint8
    assert seen == [(50, {name: held for name in state if name != "step"})]
    assert torch.equal(opt.moments(torch.float32)[0][0], want)  # (0.5 is a code)
    assert "first" in saved["state"][0] and "exp_avg" not in saved["state"][0]
    assert len(opt._optimizer_load_state_dict_pre_hooks) == len(opt._optimizer_load_state_dict_post_hooks) == 1


def test_a_hook_in_place_and_groups_of_another_number():
    """A hook that changes the dict that it is given; a state dict that does not fit leaves the optimizer as it was."""
    p, opt = stepped()
    saved = copy.deepcopy(opt.state_dict())

    def in_place(optimizer, state_dict):
        state_dict["state"] = {0: dict(state_dict["state"][0], step=9)}

    handle = opt.register_load_state_dict_pre_hook(in_place)
    opt.load_state_dict(saved)
    assert opt.state[p]["step"] == 9
    handle.remove()
    with pytest.raises(ValueError, match="number of parameter groups"):
        opt.load_state_dict({**saved, "param_groups": saved["param_groups"] * 2})
    assert opt.state[p]["step"] == 9 and not opt._optimizer_load_state_dict_pre_hooks and not opt._optimizer_load_state_dict_post_hooks
    opt.load_state_dict(saved)
    assert opt.state[p]["step"] == 3


def test_entries_of_no_parameter_are_kept():
    """As torch's optimizers keep them."""
    _, opt = stepped()
    saved = copy.deepcopy(opt.state_dict())
    saved["state"]["note"] = {"run": 7}
    opt.load_state_dict(saved)
    assert opt.state["note"] == {"run": 7}


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("saved_bits", [32, 8])
def test_a_state_of_other_shapes_leaves_the_optimizer_as_it_was(bits, saved_bits):
    p, opt = stepped(state_bits=bits)
    _, other = stepped(state_bits=saved_bits, shape=(8, 9))
    before, numbers = copy.deepcopy(opt.state[p]), dict(opt.param_groups[0])
    saved = other.state_dict()
    saved["param_groups"][0]["lr"] = 0.5
    with pytest.raises(ValueError, match="shape"):
        opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] == numbers["lr"] and set(opt.state) == {p}
    assert all(value == before[name] if name == "step" else torch.equal(value, before[name]) for name, value in opt.state[p].items())
    p.grad = torch.ones(7, 9)
    opt.step()
    assert opt.state[p]["step"] == 4


def test_a_state_with_the_largest_second_moments_is_refused():
    """AdamW has no amsgrad: going on without it would be another optimizer."""
    p, opt = stepped()
    _, other = stepped(torch.optim.AdamW, amsgrad=True)
    with pytest.raises(ValueError, match="amsgrad"):
        opt.load_state_dict(other.state_dict())
    assert opt.state[p]["step"] == 3 and "amsgrad" not in opt.param_groups[0]
    _, plain = stepped(torch.optim.AdamW, steps=5)
    opt.load_state_dict(plain.state_dict())
    assert opt.state[p]["step"] == 5
