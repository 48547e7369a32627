"""The global gradient norm and clipping against float64 and torch's own functions."""
import math

import pytest
import torch

from torchtitan_amd import ops
from torchtitan_amd.gradients import clip_grad_norm_, clip_grads_with_norm_, get_total_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def grads_of(device, dtypes, sizes, seed=0, std=1e-2):
    g = torch.Generator(device=device).manual_seed(seed)
    return [(torch.randn(s, generator=g, device=device) * std).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


def exact_norm(grads, kind):
    flat = [t.double().abs().reshape(-1) for t in grads if t.numel()]
    if not flat:
        return 0.0
    if kind == math.inf:
        return max(float(t.max()) for t in flat)
    return math.fsum(float((t ** kind).sum()) for t in flat) ** (1 / kind)


def parameters_of(grads):
    out = []
    for t in grads:
        p = torch.nn.Parameter(torch.empty(t.shape, dtype=t.dtype, device=t.device))
        p.grad = t
        out.append(p)
    return out


def check(grads, max_norm, kind=2.0):
    before = [t.clone() for t in grads]
    want = exact_norm(grads, kind)
    params = parameters_of(grads)
    norm = clip_grad_norm_(params, max_norm, norm_type=kind)
    assert norm.dtype == torch.float32 and norm.shape == ()
    assert abs(float(norm) - want) <= 2 * U * want  # float64 sums, one rounding
    factor = min(1.0, max_norm / (want + 1e-6))
    for t, b in zip(grads, before):
        half = 0.0 if t.dtype == torch.float32 else torch.finfo(t.dtype).eps / 2
        # the factor: the norm's rounding, a sum and a quotient in float32; one product; the result's rounding
        bound = (b.double() * factor).abs() * (half + 6 * U) + 1e-38
        assert ((t.double() - b.double() * factor).abs() <= bound).all()
        if max_norm > 1.01 * want:
            assert torch.equal(t, b)


SIZES = [(1,), (7,), (3, 5), (0,), (64, 64), (4096,), (8192 * 2 + 1,), (128, 1000), (2, 3, 511), (0, 9), (300, 301)]


@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtypes", [[torch.bfloat16], [torch.float32], [torch.float32, torch.bfloat16]])
@pytest.mark.parametrize("count", [1, 2, 11, 159, 160, 161, 400])
def test_lists(device, count, dtypes, kind):
    grads = grads_of(device, dtypes, [SIZES[i % len(SIZES)] for i in range(count)], count)
    norm = exact_norm(grads, kind)
    check(grads, 0.37 * norm, kind)
    check(grads, 100.0 * norm, kind)
    check(grads, 1e-3 * norm, kind)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_one_large_tensor(device, dtype):
    """More chunks than a launch has workgroups."""
    check(grads_of(device, [dtype], [(2053, 32768 + 3)]), 0.5)


def test_unaligned_and_strided(device):
    buf = torch.randn(200000, device=device)
    half = torch.randn(200001, device=device).to(torch.bfloat16)
    grads = [buf[1:1001], buf[2001:2001 + 64 * 65].view(64, 65).t(), half[1:30000], half[40001:40001 + 4000].view(40, 100),
             buf[50000:150000].view(100, 1000)[:, ::3], half[60001:160001].view(100, 1000)[:, 1:900]]
    frame = buf.clone(), half.clone()
    check(grads, 1.0)
    untouched = torch.ones(200000, dtype=torch.bool, device=device)
    for lo, hi in ((1, 1001), (2001, 2001 + 64 * 65)):
        untouched[lo:hi] = False
    untouched[50000:150000].view(100, 1000)[:, ::3] = False
    assert torch.equal(buf[untouched], frame[0][untouched])
    untouched = torch.ones(200001, dtype=torch.bool, device=device)
    untouched[1:30000] = untouched[40001:44001] = False
    untouched[60001:160001].view(100, 1000)[:, 1:900] = False
    assert torch.equal(half[untouched], frame[1][untouched])


def test_very_large_and_very_small_values(device):
    for size in (1e30, 1e-30, 3e38):
        grads = [torch.full((1000,), size, device=device), torch.full((10, 10), -size, device=device)]
        norm = get_total_norm(grads)
        want = exact_norm(grads, 2.0)
        if want < 3.4e38:
            assert abs(float(norm) - want) <= 2 * U * want
        else:
            assert norm.isinf()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_what_is_not_finite(device, dtype, kind, bad):
    """As torch's functions: the norm is not finite, an infinite one makes zeros (and NaN of infinities), a NaN NaN."""
    ours = grads_of(device, [dtype], [(5000,), (64, 1000)])
    ours[1][63, 999] = bad
    ours[1][0, 0] = 1.0
    theirs = parameters_of([t.clone() for t in ours])
    params = parameters_of(ours)
    with pytest.raises(RuntimeError, match="non-finite"):
        clip_grad_norm_(params, 1.0, norm_type=kind, error_if_nonfinite=True)
    a = clip_grad_norm_(params, 1.0, norm_type=kind)
    b = torch.nn.utils.clip_grad_norm_(theirs, 1.0, norm_type=kind, foreach=False)
    assert a.isnan() == b.isnan() and a.isinf() == b.isinf()
    for p, q in zip(params, theirs):
        assert torch.equal(p.grad.isnan(), q.grad.isnan()) and torch.equal(p.grad[~p.grad.isnan()], q.grad[~q.grad.isnan()])


def test_a_gradient_listed_twice_is_scaled_twice(device):
    """As a loop over the list would: counted in the norm and scaled once for every place it has in the list."""
    ours, theirs = (parameters_of(grads_of(device, [torch.float32], [(100, 1000), (50,), (9,)], 4)) for _ in range(2))
    ours.append(ours[0]), theirs.append(theirs[0])
    theirs[0].grad, ours[0].grad = theirs[0].grad.clone(), ours[0].grad.clone()
    a = clip_grad_norm_(ours, 0.5)
    b = torch.nn.utils.clip_grad_norm_(theirs, 0.5, foreach=False)
    # torch sums 100 000 squares in float32 parts
    assert abs(float(a) - float(b)) <= 1e-5 * float(b)
    for p, q in zip(ours, theirs):
        assert (p.grad - q.grad).abs().max() <= 4e-5 * q.grad.abs().max()


def test_without_gradients_and_other_types(device):
    p = torch.nn.Parameter(torch.zeros(3, device=device))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and float(get_total_norm([])) == 0.0
    p.grad = torch.full((3,), 2.0, device=device)
    assert abs(float(clip_grad_norm_(p, 1.0)) - math.sqrt(12)) <= 1e-6  # a tensor in place of a list
    assert (p.grad - 2 / math.sqrt(12)).abs().max() <= 1e-6
    h = torch.nn.Parameter(torch.zeros(3, device=device, dtype=torch.float64))
    h.grad = torch.full((3,), 2.0, device=device, dtype=torch.float64)
    p.grad = torch.full((3,), 2.0, device=device)
    norm = clip_grad_norm_([p, h], 1.0)  # through torch's functions
    assert abs(float(norm) - math.sqrt(24)) <= 1e-6
    assert abs(float(get_total_norm([p.grad], 3.0)) - float(p.grad.norm(3.0))) <= 1e-6


def test_a_norm_of_the_callers_own(device):
    """Shards of gradients: the norms of all ranks joined by the caller."""
    grads = grads_of(device, [torch.bfloat16, torch.float32], [(64, 999), (7,)], 5)
    before = [t.clone() for t in grads]
    total = (get_total_norm(grads) ** 2 * 4).sqrt()
    versions = [t._version for t in grads]
    clip_grads_with_norm_(parameters_of(grads), 0.1, total)
    assert all(t._version > v for t, v in zip(grads, versions))
    for t, b in zip(grads, before):
        want = b.double() * (0.1 / (float(total) + 1e-6))
        half = 0.0 if t.dtype == torch.float32 else torch.finfo(t.dtype).eps / 2
        assert ((t.double() - want).abs() <= want.abs() * (half + 6 * U) + 1e-38).all()


def test_a_side_stream_and_a_captured_graph(device):
    grads = grads_of(device, [torch.float32, torch.bfloat16], [(300, 1000), (17,), (64, 64)], 6)
    start = [t.clone() for t in grads]
    params = parameters_of(grads)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = clip_grad_norm_(params, 0.1)
    torch.cuda.current_stream().wait_stream(side)
    result = [t.clone() for t in grads]
    for t, s in zip(grads, start):
        t.copy_(s)
    b = clip_grad_norm_(params, 0.1)
    assert torch.equal(a, b) and all(torch.equal(t, r) for t, r in zip(grads, result))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm_(params, 0.1)
    for seed in range(4):
        new = grads_of(device, [torch.float32, torch.bfloat16], [(300, 1000), (17,), (64, 64)], 10 + seed)
        for t, s in zip(grads, new):
            t.copy_(s)
        graph.replay()
        want = clip_grad_norm_(parameters_of(new), 0.1)
        torch.cuda.synchronize()
        assert torch.equal(norm, want) and all(torch.equal(t, s) for t, s in zip(grads, new))


def test_refusals(device):
    t = torch.zeros(4, device=device)
    with pytest.raises(TypeError):
        ops.grad_norm([t, t.half()])
    with pytest.raises(ValueError):
        ops.grad_norm([torch.zeros((4, 4), device=device)[:, ::2]])
    with pytest.raises(KeyError):
        ops.grad_norm([t], 3.0)
    with pytest.raises(TypeError):
        ops.grad_scale_([t], torch.zeros((), device=device, dtype=torch.float64), 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_place_in_the_list_scales(device, dtype):
    """A column slice listed twice, a part of it a third time through a view of its own and its frame once: every element times the factor
    as often as it is listed."""
    frame = torch.randn((64, 100), device=device).to(dtype)
    other = torch.randn(33, device=device).to(dtype)
    lists = ([frame[:, 3:40]] * 2 + [other], [frame[:, 3:40], frame[:32, 10:90], other, frame], [frame[:, ::2], frame[:, 1::2], other],
             [frame.t()[2:50], frame, frame.t()[2:50]])
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    for grads in lists:
        before, before_other = frame.double(), other.double()
        places = torch.zeros((64, 100), device=device)
        mirror = lambda t: places.as_strided(t.shape, t.stride(), t.storage_offset())
        for t in grads:
            if t is not other:
                mirror(t).add_(1)
        exact = float(sum(t.double().square().sum() for t in grads)) ** 0.5
        norm = clip_grad_norm_(parameters_of(grads), exact / 2)
        assert abs(float(norm) - exact) <= 2 * U * exact
        factor = exact / 2 / (exact + 1e-6)
        listed = torch.full((33,), float(any(t is other for t in grads)), dtype=torch.float64, device=device)
        for now, was, times in ((frame, before, places.double()), (other, before_other, listed)):
            want = was * factor ** times
            # the factor to 6 U and a rounding to the type for every place in the list
            assert ((now.double() - want).abs() <= want.abs() * (times * (half + 7 * U) * 1.01) + 1e-30).all()
        clip_grads_with_norm_(parameters_of(grads), 1e9, norm)  # a factor of 1: nothing changes
        assert ((frame.double() - before * factor ** places).abs() <= before.abs() * (places * (half + 7 * U) * 1.01) + 1e-30).all()
