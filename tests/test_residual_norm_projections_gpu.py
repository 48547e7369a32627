"""Gradients of the norms around a block where the projections behind both norms are as large as everything else.

With gradients that are noise the means over a row, which the norms subtract, are small beside it, and a kernel that loses a
part of one would pass.  Here the outputs' gradients lie along the normalised rows, and the room for errors counts the
roundings that one value passes, not the terms of a sum."""
import pytest
import torch

from torchtitan_amd import ops

U = 2.0 ** -24  # float32 rounds by at most this, relative to the value
EPS = 1e-5
BF, F32 = torch.bfloat16, torch.float32
TYPES = [(BF, BF, BF), (F32, F32, F32), (BF, F32, F32)]
WIDTHS = [1, 2, 7, 8, 9, 63, 64, 65, 127, 128, 130, 255, 256, 257, 500, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 5119, 5120, 6144,
          6150, 8192, 8193, 9000, 12001, 16384, 16385, 17000, 20000]

# Roundings of a sum over a row: a lane adds up to 20 products in turn (16 in registers), the lanes of a wave are joined in 6
# steps, 16 waves in turn: 42.  With D for them, relative to the sums of absolute values: s1 D/2 + 4, t D/2 + 8, s2 (whose
# mean is over t) D + 12, t s2 3/2 D + 22, the mean of u t s2 5/2 D + 24, e 5 D + 62; for h's gradient once more s1, h s1
# and a mean: 7.5 D + 81; for the weights' sums e, h s1 and the rows in turn.
D = 42
ROUNDINGS = 8 * D + 100


def operands(device, rows, dim, types, gates=0, seed=0):
    """(h, r, post, gate, pre, dstream, dnormed): dstream along h s1, dnormed along the normalised stream."""
    h_type, r_type, w_type = types
    g = torch.Generator(device=device).manual_seed(seed + 131 * dim + rows)
    n = lambda *s: torch.randn(s, generator=g, device=device)
    h, r = (2 * n(rows, dim)).to(h_type), (3 * n(rows, dim)).to(r_type)
    post, pre = ((1 + 0.3 * n(dim)).to(w_type) for _ in range(2))
    gate = (1 + 0.3 * n(gates or 1, dim)).to(w_type)
    side = n(rows, 1).sign()
    k = h.double() * torch.rsqrt(h.double().square().mean(1, keepdim=True) + EPS)
    t = 0.7 * r.double() + gate.double().repeat_interleave(rows // gate.shape[0], 0) * k * post.double()
    hat = t * torch.rsqrt(t.square().mean(1, keepdim=True) + EPS)
    return h, r, post, gate, pre, (n(rows, dim) + 3 * side * k).to(r_type), (n(rows, dim) - 2 * side * hat).to(h_type)


def gradients(h, r, post, gate, pre, dstream, dnormed, behind=1.0, front=1.0):
    """{name: (value, sum of its terms' absolute values)} in float64.  `behind` and `front` are what is kept of the
    means behind the block's norm and of the norm in front of the next block: 1."""
    rows, groups = h.shape[0], gate.shape[0]
    h, r, post, pre, ds, dy = (t.double() for t in (h, r, post, pre, dstream, dnormed))
    g = gate.double().repeat_interleave(rows // groups, 0)
    mean = lambda x: x.mean(1, keepdim=True)
    s1 = torch.rsqrt(mean(h.square()) + EPS)
    k = h * s1
    t, t_abs = 0.7 * r + g * k * post, (0.7 * r).abs() + (g * k * post).abs()
    s2 = torch.rsqrt(mean(t.square()) + EPS)
    spread = 1 + mean(t_abs * t.abs()) * s2.square()
    hat, hat_abs, u = t * s2, t_abs * s2 * spread, dy * pre
    e = ds + s2 * (u - front * hat * mean(u * hat))
    e_abs = ds.abs() + s2 * spread * (u.abs() + hat_abs * mean(u.abs() * hat_abs))
    q, q_abs = e * g, e_abs * g.abs()
    dh = s1 * (q * post - behind * k * mean(q * post * k))
    dh_abs = s1 * (q_abs * post.abs() + k.abs() * mean(q_abs * post.abs() * k.abs()))
    by_gate = lambda x: x.view(groups, rows // groups, -1).sum(1)
    return {"h": (dh, dh_abs), "residual": (0.7 * e, 0.7 * e_abs), "post": ((q * k).sum(0), (q_abs * k.abs()).sum(0)),
            "gate": (by_gate(e * k * post), by_gate(e_abs * (k * post).abs())), "pre": ((dy * hat).sum(0), (dy.abs() * hat_abs).sum(0))}


def outside(got, want, rows):
    """Names of the gradients that are further off than their roundings."""
    bad = []
    for name, value in got.items():
        exact, absolute = want[name]
        half = 0.0 if value.dtype in (F32, torch.float64) else torch.finfo(value.dtype).eps / 2
        bound = exact.abs() * half + (ROUNDINGS + rows) * U * absolute * 1.01 + 1e-38
        if not ((value.double() - exact).abs() <= bound).all():
            bad.append(name)
    return bad


@pytest.mark.gpu
@pytest.mark.parametrize("types", TYPES, ids=["bf16", "f32", "mixed"])
@pytest.mark.parametrize("dim", WIDTHS)
def test_projections(device, dim, types):
    for rows, gates in ((5, 0), (6, 3)):
        inputs = operands(device, rows, dim, types, gates)
        h, r, post, gate, pre, ds, dy = inputs
        _, _, rstd = ops.residual_norm(h, r, post, gate, pre, 0.7, EPS, want_rstd=True)
        got = dict(zip(("h", "residual", "post", "gate", "pre"), ops.residual_norm_bwd(h, r, post, gate, pre, 0.7, rstd, ds, dy)))
        assert not outside(got, gradients(*inputs), rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [500, 1025, 4097, 8193, 16384, 17000])
def test_projections_without_a_side(device, dim):
    """One norm alone: the same gradients with the other's side left out."""
    for types in TYPES:
        h, r, post, _, pre, ds, dy = operands(device, 5, dim, types)
        one = torch.ones((1, dim), device=device, dtype=post.dtype)
        _, _, rstd = ops.residual_norm(h, r, post, None, None, 0.7, EPS, want_rstd=True)
        dh, dr, dpost, _, _ = ops.residual_norm_bwd(h, r, post, None, None, 0.7, rstd, ds, None)
        want = gradients(h, r, post, one, torch.zeros_like(pre), ds, dy)
        assert not outside({"h": dh, "residual": dr, "post": dpost}, want, 5)
        _, _, rstd = ops.residual_norm(h, r, None, None, pre, 0.7, EPS, want_rstd=True)
        dh, dr, _, _, dpre = ops.residual_norm_bwd(h, r, None, None, pre, 0.7, rstd, ds, dy)
        # t = 0.7 r + h: its gradient e is h's, and 0.7 e residual's
        wide = [t.double() for t in (h, r, pre, ds, dy)]
        t, t_abs = 0.7 * wide[1] + wide[0], (0.7 * wide[1]).abs() + wide[0].abs()
        s2 = torch.rsqrt(t.square().mean(1, keepdim=True) + EPS)
        spread = 1 + (t_abs * t.abs()).mean(1, keepdim=True) * s2.square()
        hat, hat_abs, u = t * s2, t_abs * s2 * spread, wide[4] * wide[2]
        e = wide[3] + s2 * (u - hat * (u * hat).mean(1, keepdim=True))
        e_abs = wide[3].abs() + s2 * spread * (u.abs() + hat_abs * (u.abs() * hat_abs).mean(1, keepdim=True))
        assert not outside({"h": dh, "residual": dr, "pre": dpre},
                           {"h": (e, e_abs), "residual": (0.7 * e, 0.7 * e_abs),
                            "pre": ((wide[4] * hat).sum(0), (wide[4].abs() * hat_abs).sum(0))}, 5)


@pytest.mark.parametrize("types", TYPES, ids=["bf16", "f32", "mixed"])
@pytest.mark.parametrize("dim", WIDTHS)
def test_what_lacks_a_part_of_a_mean_is_outside(dim, types):
    """The oracle without one of the means, and with a sixteenth of one missing (a wave's share of the widest rows): the
    check above fails for it at every width; with both it holds."""
    rounded = lambda grads: {n: v[0].to(t) for (n, v), t in zip(grads.items(), (types[0], types[1], *types[2:] * 3))}
    inputs = operands(torch.device("cpu"), 5, dim, types)
    want = gradients(*inputs)
    assert not outside(rounded(want), want, 5)
    for kept in (0.0, 15 / 16):
        assert "h" in outside(rounded(gradients(*inputs, behind=kept)), want, 5)
        assert {"residual", "h"} & set(outside(rounded(gradients(*inputs, front=kept)), want, 5))
        if kept == 0.0:
            assert "residual" in outside(rounded(gradients(*inputs, front=kept)), want, 5)
