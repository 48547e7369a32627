"""CPU: the AdamW step in torch operations against float64, its 8-bit moments, states and refusals."""
import copy
import ctypes
import math

import pytest
import torch

from torchtitan_amd import _lib
from torchtitan_amd.optimizers import _FIRST, _SECOND, AdamW, _decode, _encode, _random_bits

U = 2.0 ** -24


def step64(p, g, m, v, step, lr, betas, eps, decay, factor=1.0):
    """(p, m, v) after one step, from the formula in 64 bits."""
    p, g, m, v = (t.detach().double().cpu() for t in (p, g, m, v))
    b1, b2 = betas
    g = g * factor
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    update = lr / (1 - b1 ** step) * m / ((v / (1 - b2 ** step)).sqrt() + eps)
    return (1 - lr * decay) * p - update, m, v


def step_bounds(p, g, m, v, step, lr, betas, eps, decay, factor=1.0, half=0.0):
    """How far float32 may be from that: a rounding (U of the value) of every constant, product, sum, root and quotient; `half`:
    of p's own rounding."""
    p, g, m, v = (t.detach().double().cpu().abs() for t in (p, g, m, v))
    b1, b2 = betas
    g = g * factor  # (the factor: a sum, a quotient and the product, 4 roundings)
    m_size, v_new = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    m_off, v_off = 7 * U * m_size, 13 * U * v_new
    below = (v_new / (1 - b2 ** step)).sqrt() + eps
    scale = lr / (1 - b1 ** step)
    # (half of v_off under the root; the root and the reciprocal within an ulp, 2 roundings, each; root's factor, its product, the
    # sum, the quotient's product, the step and its product)
    update_off = scale * m_off / below + scale * m_size / below * (6.5 + 2 * 2 + 6) * U
    p_off = 3 * U * p + update_off + (half + U) * (p + scale * m_size / below)
    return p_off + 1e-44, m_off + 1e-44, v_off + 1e-44  # (denormal results: half of 2^-149)


def test_eight_bit_codes_stand_for_the_documented_values():
    codes = torch.arange(256, dtype=torch.uint8).view(8, 32)
    for scale in (0, 1, 100, 127, 140, 254):
        scales = torch.full((8,), scale, dtype=torch.uint8)
        first = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double() * 2.0 ** (scale - 127)
        got = _decode(codes, scales, _FIRST, 256).double()
        known = ~torch.isnan(first)  # (7F and FF are not written)
        fits = known & (first.abs() < 2.0 ** 128)
        assert torch.equal(got[fits], first[fits])
        c = torch.arange(256)
        e, f = (c >> 3).double(), (c & 7).double()
        second = torch.where(e == 0, f * 2.0 ** -17, (1 + f / 8) * 2.0 ** (e - 15)) * 2.0 ** (scale - 127)
        fits = second < 2.0 ** 128
        assert torch.equal(_decode(codes, scales, _SECOND, 256).double()[fits], torch.where(second < 2.0 ** -149, 0.0, second)[fits])
    assert torch.isnan(_decode(codes, torch.full((8,), 255, dtype=torch.uint8), _FIRST, 256)).all()


@pytest.mark.parametrize("form", [_FIRST, _SECOND])
@pytest.mark.parametrize("std", [1e-30, 1e-3, 1.0, 1e15])
def test_eight_bit_rounding_is_to_a_neighbour_and_right_in_the_mean(form, std):
    g = torch.Generator().manual_seed(3)
    n, tries = 32 * 40 + 5, 1024
    x = torch.randn(n, generator=g) * std * torch.exp(torch.randn(n, generator=g))
    x = x if form is _FIRST else x.square() if std < 1e10 else x.abs()
    x[64:96] = 0.0
    mean, seen = torch.zeros(n, dtype=torch.float64), []
    amax = torch.nn.functional.pad(x.abs(), (0, -n % 32)).view(-1, 32).amax(1).double()
    for t in range(tries):
        codes, scales = _encode(x, form, _random_bits(n, 11, t + 1, 5, x.device))
        value = _decode(codes, scales, form, n).double()
        if t < 64:
            # the scale is the smallest whose largest code holds the block's largest value
            largest = 448.0 if form is _FIRST else 122880.0
            s = scales.double() - 127
            assert (amax <= largest * 2 ** s).all() and ((amax > largest * 2 ** (s - 1)) | (scales == 0)).all()
            assert (value[x == 0] == 0).all() and (value * x.double() >= 0).all()
        mean += value / tries
    # a code's step at x: 1/8 of its power of two, or the smallest code
    at = (scales.double() - 127).repeat_interleave(32)[:n]
    low = -6 if form is _FIRST else -14
    unit = 2.0 ** (torch.floor(torch.log2((x.double().abs() * 2 ** -at).clamp(min=1e-300))).clamp(min=low) - 3 + at)
    assert ((value - x.double()).abs() < unit).all()
    # sums of `tries` roundings, each off by less than a step with a deviation of at most half of one; 16 bits of chance round to
    # 2^-17 of a step; a second moment below half of the smallest code is raised to it
    raised = (x > 0) & (x.double() < unit) if form is _SECOND else torch.zeros(n, dtype=torch.bool)
    off = (mean - x.double()).abs()[~raised]
    assert (off <= unit[~raised] * (6 * 0.5 / math.sqrt(tries) + 2.0 ** -17) + 1e-44).all()
    assert (value[raised] == unit[raised]).all()


def test_eight_bit_blocks_with_an_infinity_or_nan_are_nan():
    x = torch.ones(96)
    x[3], x[70] = math.inf, math.nan
    for form in (_FIRST, _SECOND):
        codes, scales = _encode(x, form, _random_bits(96, 0, 1, 0, x.device))
        value = _decode(codes, scales, form, 96)
        assert scales.tolist()[0::2] == [255, 255] and torch.isnan(value[:32]).all() and torch.isnan(value[64:]).all()
        assert torch.equal(value[32:64], torch.ones(32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64, torch.float16])
@pytest.mark.parametrize("master", [False, True])
def test_steps_in_torch_operations_against_64_bits(dtype, master):
    g = torch.Generator().manual_seed(1)
    p = torch.nn.Parameter(torch.randn(37, 21, generator=g).to(dtype))
    hyper = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8)
    opt = AdamW([p], **hyper, weight_decay=0.1, master_weights=master)
    for step in range(1, 4):
        p.grad = (torch.randn(37, 21, generator=g) * 1e-2).to(dtype)
        state = opt.state.get(p) or dict(exp_avg=torch.zeros(37, 21), exp_avg_sq=torch.zeros(37, 21))
        before = copy.deepcopy([state.get("master", p.detach()), p.grad, state["exp_avg"], state["exp_avg_sq"]])
        opt.step()
        want = step64(*before, step, *hyper.values(), 0.1)
        held = opt.state[p].get("master", p)
        half = torch.finfo(dtype).eps / 2 if held is p else 0.0
        for got, w, b in zip((held, opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"]), want,
                             step_bounds(*before, step, *hyper.values(), 0.1, half=half)):
            assert ((got.detach().double() - w).abs() <= b).all()
        if held is not p:
            assert torch.equal(p.detach(), held.to(dtype))
    assert ("master" in opt.state[p]) == (master and dtype in (torch.bfloat16, torch.float16))


def test_the_step_is_torchs():
    g = torch.Generator().manual_seed(2)
    ours, theirs = ([torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(5), dtype=torch.float64))
                     for s in ((5, 7), (3,))] for _ in range(2))
    a = AdamW(ours, lr=1e-2, weight_decay=0.2, maximize=True)
    b = torch.optim.AdamW(theirs, lr=1e-2, weight_decay=0.2, maximize=True)
    for _ in range(5):
        for p, q in zip(ours, theirs):
            p.grad = torch.randn(p.shape, generator=g, dtype=torch.float64)
            q.grad = p.grad.clone()
        assert a.step(lambda: 3.0) == 3.0
        b.step()
    for p, q in zip(ours, theirs):
        assert torch.allclose(p, q, rtol=1e-13, atol=1e-15)  # (float64 throughout)
    # a state saved by torch's optimizer goes on here
    c = AdamW(ours, lr=1e-2, weight_decay=0.2, maximize=True)
    c.load_state_dict(b.state_dict())
    assert all(torch.equal(c.state[p]["exp_avg"], b.state[q]["exp_avg"]) and c.state[p]["step"] == 5 for p, q in zip(ours, theirs))


def test_clipping_factor_and_missing_gradients():
    p, q = (torch.nn.Parameter(torch.ones(40)) for _ in range(2))
    p.grad = torch.full((40,), 0.5)
    opt = AdamW([p, q], lr=0.1, betas=(0.5, 0.5), weight_decay=0.0)
    opt.step(total_norm=torch.tensor(4.0), max_norm=1.0)
    f = 1.0 / (4.0 + 1e-6)
    assert torch.allclose(opt.state[p]["exp_avg"], torch.full((40,), 0.25 * f)) and torch.equal(p.grad, torch.full((40,), 0.5))
    assert torch.equal(q.detach(), torch.ones(40)) and q not in opt.state
    opt.step(total_norm=torch.tensor(0.25), max_norm=1.0)
    assert torch.allclose(opt.state[p]["exp_avg"], torch.full((40,), 0.125 * f + 0.25))


@pytest.mark.parametrize("n", [1, 31, 32, 33, 1000])
def test_eight_bit_steps_round_the_moments_of_the_formula(n):
    g = torch.Generator().manual_seed(n)
    p = torch.nn.Parameter(torch.randn(n, generator=g))
    opt = AdamW([p], lr=1e-2, betas=(0.9, 0.95), state_bits=8, seed=3)
    assert opt.moments() == [None]
    m = v = torch.zeros(n)
    for step in range(1, 5):
        p.grad = torch.randn(n, generator=g) * 0.1
        want = step64(p, p.grad, m, v, step, 1e-2, (0.9, 0.95), 1e-8, 1e-2)
        bound = step_bounds(p, p.grad, m, v, step, 1e-2, (0.9, 0.95), 1e-8, 1e-2)
        opt.step()
        assert ((p.detach().double() - want[0]).abs() <= bound[0]).all()
        ((m, v),) = opt.moments(torch.float32)
        assert torch.equal(m, opt.moments()[0][0].float()) and torch.equal(v, opt.moments()[0][1].float())
        for got, w, (_, most, top, _, _) in ((m, want[1], _FIRST), (v, want[2], _SECOND)):
            size = torch.nn.functional.pad(w.abs(), (0, -n % 32)).view(-1, 32).amax(1, keepdim=True).expand(-1, 32).reshape(-1)[:n]
            # a code is off by less than 1/8 of the value, or by the smallest code: 2^-18 of the largest value and twice that for
            # its scale's rounding up (first moment), 2^-34 (second)
            assert ((got.double() - w).abs() <= w.abs() / 8 * 1.0001 + size * 2.0 ** -(16 if top == 8 else 32)).all()
    assert opt.state[p]["exp_avg"].shape == (-(-n // 32), 32) and opt.state[p]["exp_avg_sq_scale"].shape == (-(-n // 32),)


def test_eight_bit_second_moment_follows_smaller_gradients():
    """Rounded to nearest, a moment whose step is a thousandth would stay where it is."""
    p = torch.nn.Parameter(torch.zeros(4096))
    opt = AdamW([p], lr=1e-3, betas=(0.9, 0.99), state_bits=8)
    for step in range(400):
        p.grad = torch.full((4096,), 1.0 if step < 100 else 0.01)
        opt.step()
    exact = (1 - 0.99 ** 100) * 0.99 ** 300 + 1e-4 * (1 - 0.99 ** 300)
    mean = float(opt.moments(torch.float32)[0][1].double().mean())
    # 4096 chains of roundings: a step in 99 is off by a code (up to 1/8) and is forgotten after a hundred, so that one of them
    # deviates by less than half of its value, and their mean by six times that over 64
    assert abs(mean - exact) <= 6 * 0.5 * exact / 64


def test_state_dicts_keep_their_types_and_are_converted():
    g = torch.Generator().manual_seed(0)
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=torch.Generator().manual_seed(9)).bfloat16()) for s in ((9, 9), (70,))]
    grads = [torch.randn(9, 9, generator=g).bfloat16(), torch.randn(70, generator=g).bfloat16()]

    def run(params, opt):
        for p, grad in zip(params, grads):
            p.grad = grad
        opt.step()

    for bits in (32, 8):
        kw = dict(state_bits=bits, master_weights=True, seed=5)
        a_params, b_params = make(), make()
        a, b = AdamW(a_params, **kw), AdamW(b_params, **kw)
        run(a_params, a)
        run(a_params, a)
        b.load_state_dict(copy.deepcopy(a.state_dict()))
        for p, q in zip(a_params, b_params):
            q.data.copy_(p.data)
            for name, value in a.state[p].items():
                other = b.state[q][name]
                assert other == value if name == "step" else other.dtype == value.dtype and torch.equal(other, value)
        run(a_params, a)
        run(b_params, b)
        for p, q in zip(a_params, b_params):
            assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])
        # to the other number of bits, and back
        other_params = make()
        other = AdamW(other_params, **dict(kw, state_bits=40 - bits))
        other.load_state_dict(copy.deepcopy(a.state_dict()))
        for (m, v), (m2, v2) in zip(a.moments(torch.float32), other.moments(torch.float32)):
            if bits == 8:
                assert torch.equal(m, m2) and torch.equal(v, v2)
            else:
                size = float(m.abs().max())
                assert ((m - m2).abs() <= m.abs() / 8 + size * 2.0 ** -16).all()
                assert ((v - v2).abs() <= v / 8 + float(v.max()) * 2.0 ** -32).all()
    twin = copy.deepcopy(a)
    assert isinstance(twin, AdamW) and len(twin.state) == 2


@pytest.fixture
def mesh():
    """One rank; nothing is sent."""
    import torch.distributed as dist
    from torch.distributed.device_mesh import DeviceMesh

    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        yield DeviceMesh("cpu", [0])
    finally:
        dist.destroy_process_group()


def test_distributed_parameters_are_updated_shard_by_shard(mesh):
    from torch.distributed.tensor import DTensor, Replicate, Shard

    plain = torch.nn.Parameter(torch.randn(8, 6, generator=torch.Generator().manual_seed(0)))
    spread = torch.nn.Parameter(DTensor.from_local(plain.detach().clone(), mesh, [Shard(0)], run_check=False))
    a, b = AdamW([plain]), AdamW([spread])
    for step in range(3):
        plain.grad = torch.randn(8, 6, generator=torch.Generator().manual_seed(step))
        spread.grad = DTensor.from_local(plain.grad.clone(), mesh, [Shard(0) if step < 2 else Replicate()], run_check=False)
        norm = torch.tensor(3.0)
        a.step(total_norm=norm, max_norm=1.0)
        b.step(total_norm=DTensor.from_local(norm, mesh, [Replicate()], run_check=False), max_norm=1.0)
    assert isinstance(spread.data, DTensor) and torch.equal(spread.to_local(), plain)
    assert isinstance(b.state[spread]["exp_avg"], DTensor) and torch.equal(b.state[spread]["exp_avg"].to_local(), a.state[plain]["exp_avg"])
    c = AdamW([spread])
    c.load_state_dict(b.state_dict())
    assert c.state[spread]["step"] == 3 and torch.equal(c.state[spread]["exp_avg_sq"].to_local(), a.state[plain]["exp_avg_sq"])
    with pytest.raises(ValueError, match="plain contiguous"):
        AdamW([spread], state_bits=8).step()


def test_hooks_schedulers_and_a_compiled_caller():
    p = torch.nn.Parameter(torch.ones(10))
    opt = AdamW([p], lr=0.1, weight_decay=0.0)
    seen = []
    opt.register_step_post_hook(lambda *a: seen.append(float(p[0])))
    schedule = torch.optim.lr_scheduler.LambdaLR(opt, lambda step: 0.5 ** step)

    @torch.compile(backend="eager")
    def update(g):
        p.grad = g
        opt.step()

    try:
        for _ in range(2):
            update(torch.ones(10))
            schedule.step()
    finally:
        torch._dynamo.reset()
    # (a constant gradient moves by the learning rate, 0.1 and 0.05, but for eps and some roundings)
    assert len(seen) == 2 and abs(seen[0] - 0.9) < 1e-6 and abs(seen[1] - 0.85) < 1e-6


def test_refusals():
    p = torch.nn.Parameter(torch.ones(4, 4))
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-0.1), dict(state_bits=16), dict(seed=-1),
                dict(lr=torch.ones(2))):
        with pytest.raises(ValueError):
            AdamW([p], **bad)
    opt = AdamW([p])
    with pytest.raises(ValueError, match="together"):
        opt.step(max_norm=1.0)
    with pytest.raises(TypeError):
        opt.moments(torch.float16)
    q = torch.nn.Parameter(torch.ones(4, 6).t())
    q.grad = torch.ones(6, 4)
    with pytest.raises(ValueError, match="contiguous"):
        AdamW([q], state_bits=8).step()
    c = torch.nn.Parameter(torch.ones(2, dtype=torch.complex64))
    c.grad = torch.ones(2, dtype=torch.complex64)
    with pytest.raises(TypeError, match="complex"):
        AdamW([c]).step()
    p.grad = torch.ones(4, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        AdamW([p], capturable=True).step()


def test_entry_points_refuse_before_any_launch():
    lib = _lib.load()
    P, I = ctypes.c_void_p, ctypes.c_int64

    def adamw(row, n=1, eight=0, betas=(0.9, 0.95), steps=None, corrections=None, lr_device=None, norm=None):
        table = (I * len(row))(*row)
        return lib.mx_adamw(n, ctypes.cast(table, P), eight, 1e-3, *betas, 1e-8, 0.0, 0, norm, 0.0, 0, steps, lr_device, corrections, None)

    good = [0x1000, 1, 0x2000, 0x3000, 0x4000, 0, 0, 0, 10, 1, 0]
    change = lambda **at: [at.get(f"f{i}", x) for i, x in enumerate(good)]
    assert lib.mx_adamw(0, None, 0, 1e-3, 0.9, 0.95, 1e-8, 0.0, 0, None, 0.0, 0, None, None, None, None) == 0
    assert adamw(change(f8=0)) == 0                                   # nothing to update
    assert adamw(good, n=-1) == 1 and lib.mx_adamw(1, None, 0, 1e-3, 0.9, 0.95, 1e-8, 0.0, 0, None, 0.0, 0, None, None, None, None) == 1
    for bad in (change(f0=0), change(f2=0), change(f3=0), change(f4=0), change(f8=-1), change(f9=0), change(f10=-1)):
        assert adamw(bad) == 1
    assert adamw(good, eight=1) == 1                                  # no scales
    assert adamw(good, betas=(1.0, 0.9)) == 1 and adamw(good, betas=(0.9, float("nan"))) == 1
    for bad in (change(f0=0x1002), change(f2=0x2001), change(f3=0x3002), change(f7=0x5001), change(f1=0, f0=0x1001)):
        assert adamw(bad) == 2
    assert adamw(change(f3=0x3004, f5=0x6000, f6=0x7000), eight=1) == 2   # codes are 8-byte aligned
    assert adamw(good, steps=P(0x8000)) == 1 and adamw(good, lr_device=P(0x8000)) == 1
    assert adamw(good, steps=P(0x8000), corrections=P(0x9008)) == 2 and adamw(good, norm=P(0x8001)) == 2
    assert adamw(change(f8=1 << 33)) == 4
    one = lambda t, v: (t * 1)(v)
    moments = lambda codes=0x1000, scales=0x2000, n=10, kind=0, out=0x3000: lib.mx_adamw_moments(
        1, one(P, codes), one(P, scales), one(I, n), one(ctypes.c_int32, kind), one(P, out), None)
    assert lib.mx_adamw_moments(0, None, None, None, None, None, None) == 0 and moments(n=0) == 0
    assert moments(kind=4) == 1 and moments(codes=None) == 1 and moments(n=-1) == 1
    assert moments(codes=0x1004) == 2 and moments(out=0x3002, kind=2) == 2 and moments(n=1 << 33) == 4
