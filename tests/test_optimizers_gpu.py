"""GPU: the AdamW kernels against float64 and against the same formula in torch operations."""
import copy
import math

import pytest
import torch

from tests.test_optimizers_cpu import step64, step_bounds
from torchtitan_amd import ops
from torchtitan_amd.mx_tensor import MXFP8Config, wrap_parameter
from torchtitan_amd.optimizers import _FIRST, _SECOND, AdamW, _decode

pytestmark = pytest.mark.gpu

HYPER = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8)
SHAPES = [(1,), (7,), (3, 5), (0,), (31,), (32,), (33,), (64, 65), (2048,), (4097,), (300, 301), (2, 3, 511)]


def parameters_of(device, shapes, dtypes=(torch.bfloat16, torch.float32), seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, generator=g, device=device).to(dtypes[i % len(dtypes)])) for i, s in enumerate(shapes)]


def set_gradients(params, seed, std=1e-2):
    for i, p in enumerate(params):
        g = torch.Generator(device=p.device).manual_seed(seed * 1000 + i)
        p.grad = (torch.randn(p.shape, generator=g, device=p.device) * std).to(p.dtype)


def check_steps(opt, params, steps=3, decay=0.1, norm=None, limit=None, set_grads=set_gradients):
    """Every step of the optimizer against float64, from the state that it began with."""
    kw = {} if norm is None else dict(total_norm=norm, max_norm=limit)
    factor = 1.0 if norm is None else min(1.0, limit / (float(norm) + 1e-6))
    for _ in range(steps):
        set_grads(params, int(torch.randint(0, 999, ())))
        before = []
        for p in params:
            state = opt.state.get(p) or {}
            eight = "exp_avg_scale" in state
            m, v = (torch.zeros(p.shape, device=p.device) if not state else
                    _decode(state[n], state[n + "_scale"], f, p.numel()).view(p.shape) if eight else state[n].clone()
                    for n, f in (("exp_avg", _FIRST), ("exp_avg_sq", _SECOND)))
            before.append((state.get("master", p.detach()).clone(), p.grad.clone(), m, v, int(state.get("step", 0)) + 1))
        opt.step(**kw)
        for p, (w0, g, m, v, step) in zip(params, before):
            state = opt.state[p]
            want = step64(w0, g, m, v, step, *HYPER.values(), decay, factor)
            held = state.get("master", p)
            half = torch.finfo(p.dtype).eps / 2 if held is p else 0.0
            bounds = step_bounds(w0, g, m, v, step, *HYPER.values(), decay, factor, half)
            assert int(state["step"]) == step and torch.equal(g, p.grad)
            pairs = [(held.detach(), want[0], bounds[0])]
            if "exp_avg_scale" not in state:
                pairs += [(state["exp_avg"], want[1], bounds[1]), (state["exp_avg_sq"], want[2], bounds[2])]
            for got, w, b in pairs:
                assert ((got.double().cpu() - w).abs() <= b).all()
            if held is not p:
                assert torch.equal(p.detach(), held.to(p.dtype))


@pytest.mark.parametrize("dtypes", [(torch.bfloat16,), (torch.float32,), (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_steps_against_64_bits(device, dtypes, bits, master):
    params = parameters_of(device, SHAPES, dtypes)
    check_steps(AdamW(params, **HYPER, weight_decay=0.1, state_bits=bits, master_weights=master, seed=7), params)


@pytest.mark.parametrize("norm", [0.5, 12.0, math.inf, 0.0])
@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_steps(device, norm, bits):
    params = parameters_of(device, [(130, 33), (5,)])
    check_steps(AdamW(params, **HYPER, weight_decay=0.1, state_bits=bits), params, steps=2,
                norm=torch.tensor(norm, device=device), limit=2.0)


def test_a_norm_that_is_not_a_number_reaches_every_parameter(device):
    params = parameters_of(device, [(130, 33), (5,)])
    set_gradients(params, 0)
    AdamW(params).step(total_norm=torch.tensor(math.nan, device=device), max_norm=1.0)
    assert all(torch.isnan(p).all() for p in params)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_eight_bit_moments_are_the_same_bits_in_torch_operations(device, dtype):
    """Products, sums and the chances of rounding are the same on the CPU."""
    params = parameters_of(device, SHAPES, (dtype,))
    twins = [torch.nn.Parameter(p.detach().cpu()) for p in params]
    kw = dict(**HYPER, weight_decay=0.1, state_bits=8, master_weights=True, seed=(3 << 40) + 5)
    a, b = AdamW(params, **kw), AdamW(twins, **kw)
    norm = torch.tensor(7.0)
    for step in range(4):
        set_gradients(params, step, 10.0 ** (1 - 3 * step))
        for p, q in zip(params, twins):
            q.grad = p.grad.cpu()
        a.step(total_norm=norm.to(device), max_norm=3.0)
        b.step(total_norm=norm, max_norm=3.0)
        for p, q in zip(params, twins):
            for name in ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale"):
                assert torch.equal(a.state[p][name].cpu(), b.state[q][name]), name
    for out in (torch.bfloat16, torch.float32):
        for (m, v), (m2, v2) in zip(a.moments(out), b.moments(out)):
            assert torch.equal(m.cpu(), m2) and torch.equal(v.cpu(), v2)


@pytest.mark.parametrize("bits", [32, 8])
def test_values_that_are_not_finite(device, bits):
    p = torch.nn.Parameter(torch.ones(96, device=device))
    opt = AdamW([p], state_bits=bits)
    p.grad = torch.full((96,), 0.1, device=device)
    p.grad[3], p.grad[40] = math.nan, math.inf
    opt.step()
    bad = torch.zeros(96, dtype=torch.bool, device=device)
    bad[3] = bad[40] = True
    assert torch.equal(torch.isnan(p), bad)
    ((m, v),) = opt.moments(torch.float32)
    if bits == 32:
        assert torch.equal(~torch.isfinite(m), bad) and torch.equal(~torch.isfinite(v), bad)
    else:
        assert torch.isnan(m[:64]).all() and torch.isnan(v[:64]).all() and torch.isfinite(m[64:]).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("first", [0, 1, 3])
def test_views_at_any_element_and_neighbours_left_alone(device, bits, first):
    """Parameters and gradients may begin at any element; nothing around them is written."""
    for dtype in (torch.bfloat16, torch.float32):
        buffer = torch.full((first + 1000 + 9,), 7.0, device=device, dtype=dtype)
        grads = torch.full((first + 1000 + 9,), 7.0, device=device, dtype=dtype)
        p = torch.nn.Parameter(buffer[first:first + 1000])
        opt = AdamW([p], **HYPER, weight_decay=0.1, state_bits=bits)

        def set_grads(params, seed):
            grads[first:first + 1000] = torch.randn(1000, device=device).to(dtype)
            params[0].grad = grads[first:first + 1000]

        check_steps(opt, [p], set_grads=set_grads)
        assert (buffer[:first] == 7).all() and (buffer[first + 1000:] == 7).all()


def test_other_layouts(device):
    """Permuted dense parameters keep their order; gradients in another order, or of another type, are laid out first."""
    params = [torch.nn.Parameter(torch.randn(40, 30, device=device).t()), torch.nn.Parameter(torch.randn(40, 30, device=device)),
              torch.nn.Parameter(torch.randn(10, 12, device=device)[:, ::2])]

    def set_grads(params, seed):
        for p in params:
            p.grad = torch.randn(tuple(reversed(p.shape)), device=device).t()

    opt = AdamW(params, **HYPER, weight_decay=0.1)
    check_steps(opt, params, set_grads=set_grads)
    assert opt.state[params[0]]["exp_avg"].stride() == params[0].stride()


def test_parameters_that_share_memory_are_updated_one_after_the_other(device):
    base = torch.randn(5000, device=device)
    twin = base.clone()
    pair = [torch.nn.Parameter(base), torch.nn.Parameter(base)]
    single = torch.nn.Parameter(twin)
    opt = AdamW(pair, **HYPER)
    for p in pair:
        p.grad = torch.full_like(p, 0.5)
    opt.step()
    for _ in range(2):  # the same two first steps of an optimizer, on one parameter
        single.grad = torch.full_like(single, 0.5)
        AdamW([single], **HYPER).step()
    assert torch.equal(pair[0].detach(), single.detach())


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_take_several_launches(device, bits):
    params = parameters_of(device, [(i * 37 % 91 + 1, i % 7 + 1) for i in range(150)])
    check_steps(AdamW(params, **HYPER, weight_decay=0.1, state_bits=bits), params, steps=2)


def test_a_large_tensor_and_groups_with_their_own_numbers(device):
    """More values than one launch has chunks' worth of waves in flight; the same bits whatever the list around them."""
    params = parameters_of(device, [(3000, 5001), (70,)], (torch.float32,))
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    kw = dict(**HYPER, state_bits=8, seed=9)
    a, b = AdamW(params, **kw), AdamW([dict(params=twins[:1]), dict(params=twins[1:], lr=1e-2)], **kw)
    for step in range(2):
        set_gradients(params, step)
        set_gradients(twins, step)
        a.step()
        b.step()
    for p, q in zip(params, twins):
        assert torch.equal(p, q) and torch.equal(a.state[p]["exp_avg"], b.state[q]["exp_avg"])
    check_steps(a, params, steps=1, decay=1e-2)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_odd_sizes_in_a_list_of_more_than_a_million_values(device, bits, master):
    """Longer lists have larger chunks: the ends of small tensors inside them."""
    params = parameters_of(device, [*SHAPES, (1200, 1001), (4095,), (4096,), (8191,), (2047, 3)])
    check_steps(AdamW(params, **HYPER, weight_decay=0.1, state_bits=bits, master_weights=master, seed=3), params, steps=2)
    if bits == 8 and master:
        # the same list beside nothing: the same bits in smaller chunks
        some = parameters_of(device, [(8191,)], (torch.float32,), seed=5)
        twins = [torch.nn.Parameter(p.detach().clone()) for p in some] + parameters_of(device, [(1200, 1001)], seed=6)
        a, b = AdamW(some, state_bits=8), AdamW(twins, state_bits=8)
        set_gradients(some, 1)
        set_gradients(twins, 1)
        a.step()
        b.step()
        assert torch.equal(a.state[some[0]]["exp_avg"], b.state[twins[0]]["exp_avg"])
        assert torch.equal(a.state[some[0]]["exp_avg_sq"], b.state[twins[0]]["exp_avg_sq"])


def test_converted_weights_are_updated_and_their_versions_counted(device):
    plain = parameters_of(device, [(64, 96)], (torch.bfloat16,))[0]
    twin = torch.nn.Parameter(plain.detach().clone())
    weight = wrap_parameter(plain, MXFP8Config())
    a, b = AdamW([weight], **HYPER), AdamW([twin], **HYPER)
    for step in range(2):
        set_gradients([twin], step)
        weight.grad = twin.grad.clone()
        version = weight._version
        a.step()
        b.step()
        assert weight._version > version
    assert torch.equal(weight.detach().as_subclass(torch.Tensor), twin.detach())
    assert type(a.state[weight]["exp_avg"]) is torch.Tensor


@pytest.mark.parametrize("bits", [32, 8])
def test_captured_steps_go_on_counting(device, bits):
    """A captured step replayed is the steps of the eager loop, with a learning rate that changes on the device; two optimizers'
    graphs in turn."""
    def setup(seed):
        params = parameters_of(device, SHAPES, seed=seed)
        set_gradients(params, seed)
        return params

    lr = torch.tensor(1e-2, device=device)
    runs = []
    for seed in (1, 2):
        params = setup(seed)
        opt = AdamW(params, lr=lr, betas=(0.9, 0.95), state_bits=bits, capturable=True, seed=seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt.step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        twins = setup(seed)
        eager = AdamW(twins, lr=1e-2, betas=(0.9, 0.95), state_bits=bits, seed=seed)
        eager.step()
        runs.append((params, opt, graph, twins, eager))
    for replay in range(4):
        rate = 1e-2 / (replay + 1)
        lr.fill_(rate)
        for params, opt, graph, twins, eager in runs:
            for p, q in zip(params, twins):
                g = torch.randn(p.shape, device=device).to(p.dtype)
                p.grad.copy_(g)
                q.grad.copy_(g)
            graph.replay()
            eager.param_groups[0]["lr"] = float(torch.tensor(rate))
            eager.step()
            torch.cuda.synchronize()
            for p, q in zip(params, twins):
                assert float(opt.state[p]["step"]) == replay + 2 == eager.state[q]["step"]
                assert torch.equal(opt.state[p]["exp_avg"], eager.state[q]["exp_avg"])
                # the corrections in 64 bits differ in a last bit of pow, their roundings to float32 now and then by a step
                size = q.detach().float().abs() + 1
                assert ((p.detach().float() - q.detach().float()).abs() <= size * (torch.finfo(p.dtype).eps if p.dtype == torch.bfloat16 else 2.0 ** -22)).all()
    # a saved state goes on in an optimizer that counts on the host
    params, opt = runs[0][:2]
    later = AdamW(params, state_bits=bits)
    later.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert all(later.state[p]["step"] == 5 for p in params)


def test_capture_is_refused_where_a_step_would_be_wrong(device):
    params = parameters_of(device, [(100,)])
    set_gradients(params, 0)
    opt = AdamW(params)
    opt.step()
    fresh = AdamW(params, capturable=True)
    before = params[0].detach().clone()
    with pytest.raises(RuntimeError, match="capturable=True"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    with pytest.raises(RuntimeError, match="outside"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh.step()
    torch.cuda.synchronize()
    assert torch.equal(params[0].detach(), before) and opt.state[params[0]]["step"] == 1
    opt.step()
    assert opt.state[params[0]]["step"] == 2


def test_on_another_stream_after_work_there(device):
    params = parameters_of(device, [(2000, 1000)], (torch.float32,))
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    set_gradients(twins, 1)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    a, b = AdamW(params, state_bits=8), AdamW(twins, state_bits=8)
    with torch.cuda.stream(stream):
        set_gradients(params, 1)
        a.step()
    b.step()
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(params[0], twins[0])


def test_state_that_does_not_fit_is_refused(device):
    p = parameters_of(device, [(64,)], (torch.float32,))[0]
    set_gradients([p], 0)
    opt = AdamW([p])
    opt.step()
    for bad in (torch.zeros(63, device=device), torch.zeros(64, device=device, dtype=torch.bfloat16), torch.zeros(64)):
        opt.state[p]["exp_avg"] = bad
        with pytest.raises(ValueError, match="does not fit"):
            opt.step()
    with pytest.raises(ValueError, match="does not fit|wants"):
        ops.adamw_moments([(torch.zeros(31, dtype=torch.uint8, device=device), torch.zeros(1, dtype=torch.uint8, device=device), 0,
                            torch.zeros(32, device=device))])


def test_the_timer_and_other_types_take_their_paths(device):
    """The launches under a kernel timer are the same; float16 and float64 parameters run in torch operations."""
    params = parameters_of(device, [(130, 33), (5,)])
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = AdamW(params, state_bits=8, seed=1), AdamW(twins, state_bits=8, seed=1)
    timer = ops.KernelTimer()
    for step in range(2):
        set_gradients(params, step)
        set_gradients(twins, step)
        a.step()
        ops.set_kernel_timer(timer)
        try:
            b.step()
        finally:
            ops.set_kernel_timer(None)
    assert timer.summary()["adamw"][0] == 2
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    others = parameters_of(device, [(40, 3), (9,)], (torch.float16, torch.float64))
    check_steps(AdamW(others, **HYPER, weight_decay=0.1), others)


def test_distributed_parameters_run_on_their_shards(device):
    import torch.distributed as dist
    from torch.distributed.device_mesh import DeviceMesh
    from torch.distributed.tensor import DTensor, Shard

    dist.init_process_group("gloo", store=dist.HashStore(), rank=0, world_size=1)
    try:
        mesh = DeviceMesh("cuda", [0])
        plain = torch.nn.Parameter(torch.randn(300, 70, device=device).bfloat16())
        spread = torch.nn.Parameter(DTensor.from_local(plain.detach().clone(), mesh, [Shard(0)], run_check=False))
        a, b = AdamW([plain], master_weights=True), AdamW([spread], master_weights=True)
        timer = ops.KernelTimer()
        for step in range(2):
            set_gradients([plain], step)
            spread.grad = DTensor.from_local(plain.grad.clone(), mesh, [Shard(0)], run_check=False)
            a.step()
            ops.set_kernel_timer(timer)
            try:
                b.step()
            finally:
                ops.set_kernel_timer(None)
        assert timer.summary()["adamw"][0] == 2
        assert torch.equal(spread.to_local(), plain) and isinstance(b.state[spread]["master"], DTensor)
    finally:
        dist.destroy_process_group()


def test_other_types_are_not_captured_either(device):
    p = torch.nn.Parameter(torch.randn(10, device=device).half())
    p.grad = torch.ones_like(p)
    opt = AdamW([p])
    opt.step()
    with pytest.raises(RuntimeError, match="capturable=True"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            opt.step()
    with pytest.raises(RuntimeError, match="one GPU"):
        AdamW([p], capturable=True).step()


def test_a_compiled_caller(device):
    params = parameters_of(device, [(64, 33)], (torch.float32,))
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    a, b = AdamW(params, state_bits=8), AdamW(twins, state_bits=8)

    @torch.compile(backend="eager")
    def update(g):
        twins[0].grad = g * 2
        b.step()

    try:
        for step in range(3):
            set_gradients(params, step)
            update(params[0].grad / 2)
            a.step()
    finally:
        torch._dynamo.reset()
    assert torch.equal(params[0], twins[0]) and a.state[params[0]]["step"] == b.state[twins[0]]["step"] == 3


def test_more_values_than_31_bits_count(device):
    """2^31 and some parameters with 8-bit moments: the last ones are updated and rounded as the first."""
    n = (1 << 31) + (1 << 13) + 5
    p = torch.nn.Parameter(torch.ones(n, dtype=torch.bfloat16, device=device))
    p.grad = torch.zeros(n, dtype=torch.bfloat16, device=device)
    ends = [slice(0, 4096), slice(n - 4096, n)]
    for i, at in enumerate(ends):
        g = torch.Generator(device=device).manual_seed(i)
        p.grad[at] = (torch.randn(4096, generator=g, device=device) * 1e-2).bfloat16()
    opt = AdamW([p], **HYPER, weight_decay=0.1, state_bits=8)
    opt.step()
    ((m, v),) = opt.moments()
    assert m.shape == (n,) and not m[4096:8192].any() and not opt.state[p]["exp_avg_sq"][1 << 20].any()
    for at in ends:
        zero = torch.zeros(4096, device=device)
        args = (torch.ones(4096, device=device), p.grad[at], zero, zero, 1, *HYPER.values(), 0.1)
        want, bounds = step64(*args), step_bounds(*args, half=torch.finfo(torch.bfloat16).eps / 2)
        assert ((p.detach()[at].double().cpu() - want[0]).abs() <= bounds[0]).all()
        # a code is off by less than an eighth of the value, or by the smallest code
        for got, w, least in ((m[at], want[1], 2.0 ** -16), (v[at], want[2], 2.0 ** -32)):
            assert ((got.double().cpu() - w).abs() <= w.abs() / 8 * 1.0001 + w.abs().max() * least).all()


def test_states_that_are_there_but_empty(device):
    """Asking an optimizer for the state of a parameter without one leaves an empty dict."""
    params = parameters_of(device, [(40,), (50,)])
    for capturable in (False, True):
        opt = AdamW(params, capturable=capturable)
        assert not opt.state[params[0]] and not opt.state[params[1]]
        set_gradients(params, 1)
        params[1].grad = None
        opt.step()
        opt.step()
        assert float(opt.state[params[0]]["step"]) == 2 and not opt.state[params[1]]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps,std", [(1e-8, 1e-18), (1e-12, 1e-14), (1e-15, 1e-18), (0.0, 1e-15), (1e-8, 1e6)])
def test_tiny_and_large_gradients_with_any_eps(device, bits, eps, std):
    """First steps from gradients whose squares are near float32's smallest numbers, or beyond 1e12; whole chunks and a ragged end."""
    for dtype in (torch.bfloat16, torch.float32):
        p = torch.nn.Parameter(torch.zeros(2 * 2048 * 4 + 1000, device=device, dtype=dtype))
        g = torch.randn(p.shape, generator=torch.Generator(device=device).manual_seed(1), device=device)
        p.grad = ((g + g.sign()) * std).to(dtype)
        opt = AdamW([p], lr=1e-2, betas=(0.9, 0.95), eps=eps, weight_decay=0.0, state_bits=bits)
        opt.step()
        zero = torch.zeros_like(p)
        args = (zero, p.grad, zero, zero, 1, 1e-2, (0.9, 0.95), eps, 0.0)
        want, bounds = step64(*args), step_bounds(*args, half=torch.finfo(dtype).eps / 2)
        # a second moment below 2^-126 is held to 2^-150 of its square's roundings; the root of 3 * 2^-150 where it stands over eps
        lost = 3 * 2.0 ** -150
        v = want[2]
        root = (v / 0.05).sqrt()
        moved = 1e-2 * (0.1 * p.grad.double().cpu().abs() / 0.1) * (lost / 0.05 / (2 * root.clamp(min=1e-30))) / (root + eps).clamp(min=1e-30) ** 2
        assert ((p.detach().double().cpu() - want[0]).abs() <= bounds[0] + moved).all()
