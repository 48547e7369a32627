"""Gradients of the norms around a block where only `stream` has one: nothing of the norm behind the sum is in them, so what
is not finite in the sum stays out of them."""
import itertools

import pytest
import torch

from torchtitan_amd.modules import residual_rms_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
EPS = 1e-5
INF, NAN = float("inf"), float("nan")
TYPES = [(torch.float32,) * 3, (torch.bfloat16,) * 3, (torch.bfloat16, torch.float32, torch.float32)]
KINDS = [k for k in itertools.product((True, False), repeat=3)]  # post, gate, pre


def formula(h, post, gate, scale, ds):
    """Gradients of `stream` alone in float64 and the sums of their terms' absolute values."""
    one = torch.ones((), dtype=torch.float64, device=h.device)
    q, g = ds * (one if gate is None else gate), {"residual": (scale * ds, (scale * ds).abs())}
    if post is None:
        g["h"], n = (q, q.abs()), h
    else:
        s = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS)
        k, e = h * s, q * post
        g["h"] = (s * (e - k * (e * k).mean(1, keepdim=True)), s * (e.abs() + k.abs() * (e * k).abs().mean(1, keepdim=True)))
        g["post_weight"], n = ((q * k).sum(0), (q * k).abs().sum(0)), k * post
    if gate is not None:
        g["gate"] = ((ds * n).sum(0), (ds * n).abs().sum(0))
    return g


def check(device, dim, kind, types, bad):
    """`bad`: values that are put into the operands, as (operand, value)."""
    h_type, r_type, w_type = types
    post, gate, pre = kind
    g = torch.Generator(device=device).manual_seed(dim)
    n = lambda shape, t: torch.randn(shape, generator=g, device=device).to(t)
    rows = 7
    h, r, ds = n((rows, dim), h_type), n((rows, dim), r_type), n((rows, dim), r_type)
    vec = lambda: (1 + 0.3 * torch.randn(dim, generator=g, device=device)).to(w_type)
    weights = {name: vec() for name, there in zip(("post_weight", "gate", "pre_weight"), kind) if there}
    for i, (where, value) in enumerate(bad):
        {"h": h, "residual": r}[where][1 + 2 * i, (dim // 2 + i) % dim] = value
    leaves = {"h": h, "residual": r, **weights}
    for t in leaves.values():
        t.requires_grad_(True)
    stream, normed = residual_rms_norm(h, r, **weights, residual_scale=0.7, eps=EPS)
    got = dict(zip(leaves, torch.autograd.grad(stream, list(leaves.values()), ds, allow_unused=True)))
    wide = lambda t: None if t is None else t.detach().double()
    want = formula(wide(h), wide(weights.get("post_weight")), wide(weights.get("gate")), 0.7, wide(ds))
    if pre:
        unused = got.pop("pre_weight")
        assert unused is None or not unused.any()
    # The norm's sum over a row and its mean: a lane adds up to 20 products in turn, 64 lanes in 6 steps, 16 waves in turn,
    # 42 roundings at most; some twenty more around each, and 7 rows
    terms = 3 * 42 + 40 + rows
    assert set(got) == set(want)
    for name, grad in got.items():
        value, absolute = want[name]
        half = 0.0 if grad.dtype == torch.float32 else torch.finfo(grad.dtype).eps / 2
        grad, there = grad.double(), value.isfinite()
        assert torch.equal(grad.isnan(), value.isnan()), name
        assert torch.equal(grad[value.isinf()], value[value.isinf()]), name
        bound = value.abs() * half + terms * U * absolute + 1e-38
        assert ((grad - value).abs() <= bound)[there].all(), name


@pytest.mark.parametrize("kind", KINDS, ids=lambda k: "".join("pgn"[i] if v else "-" for i, v in enumerate(k)))
@pytest.mark.parametrize("dim", [5, 12, 640, 4096, 9001, 16400])
def test_what_is_not_finite_in_the_residual(device, dim, kind):
    for types in TYPES:
        check(device, dim, kind, types, [])
        check(device, dim, kind, types, [("residual", INF), ("residual", NAN), ("residual", -INF)])


@pytest.mark.parametrize("kind", [k for k in KINDS if k[0] or not k[1]], ids=lambda k: "".join("pgn"[i] if v else "-" for i, v in enumerate(k)))
@pytest.mark.parametrize("dim", [5, 12, 640, 4096, 9001, 16400])
def test_what_is_not_finite_in_the_block_output(device, dim, kind):
    """Behind a norm it takes its own row and its column's sums; without one nothing."""
    for types in TYPES:
        for value in (INF, NAN, -INF):
            check(device, dim, kind, types, [("h", value)])


@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("dim", [5, 12, 640, 4096, 9001, 16400])
def test_what_is_not_finite_behind_a_gate(device, dim, pre):
    """A gate without a norm in front of it: the block's gradient has nothing of the block's output in it."""
    for types in TYPES:
        for value in (INF, NAN, -INF):
            check(device, dim, (False, True, pre), types, [("h", value)])


@pytest.mark.parametrize("dim", [640, 2048])
def test_a_gate_for_every_row(device, dim):
    """The lanes of a row take gates of their own."""
    rows = 4099
    g = torch.Generator(device=device).manual_seed(dim)
    h, r, ds, gate = (torch.randn((rows, dim), generator=g, device=device) for _ in range(4))
    post = 1 + 0.3 * torch.randn(dim, generator=g, device=device)
    h[5, 7], r[9, 3], r[4000, dim - 1] = INF, INF, NAN
    for weight in (None, post):
        leaves = [t.detach().requires_grad_(True) for t in (h, r, gate)]
        stream, _ = residual_rms_norm(leaves[0], leaves[1], gate=leaves[2], post_weight=weight, residual_scale=0.5)
        got = torch.autograd.grad(stream, leaves, ds)
        k = h.double()
        s = torch.ones((rows, 1), dtype=torch.float64, device=device) if weight is None else torch.rsqrt(k.square().mean(1, keepdim=True) + EPS)
        n, p = k * s, 1.0 if weight is None else weight.double()
        q = ds.double() * gate.double() * p
        mean = 0.0 if weight is None else (q * n).mean(1, keepdim=True)
        dh = q if weight is None else s * (q - n * mean)
        room = s * (q.abs() + (0.0 if weight is None else n.abs() * (q * n).abs().mean(1, keepdim=True)))
        assert torch.equal(got[1], 0.5 * ds)
        for a, b, absolute in ((got[0].double(), dh, room), (got[2].double(), ds.double() * n * p, (ds.double() * n * p).abs())):
            assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a[b.isinf()], b[b.isinf()])
            assert ((a - b).abs() <= 170 * U * absolute)[b.isfinite()].all()
