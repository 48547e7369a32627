"""The norms around a block with its gate and residual sum, and their gradients, against float64."""
import pytest
import torch

from torchtitan_amd import ops
from torchtitan_amd.modules import ResidualRMSNorm, residual_rms_norm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # float32 rounds by at most this, relative to the value
EPS = 1e-5
BF, F32 = torch.bfloat16, torch.float32
KINDS = [(True, True, True), (False, False, True), (True, False, True), (False, True, True), (True, True, False),
         (False, True, False), (True, False, False), (False, False, False)]  # post, gate, pre


def half(dtype):
    return 0.0 if dtype == F32 else torch.finfo(dtype).eps / 2


def reference(h, r, post, gate, pre, scale, dstream, dnormed):
    """Outputs and gradients from their formulas, and the same with every term's absolute value: what their float32
    errors are relative to.  Matrices in float64; the gate expanded to the rows, its gradient one row each."""
    dim = h.shape[1]
    one = torch.ones((), dtype=torch.float64, device=h.device)
    p, g, w = (one if t is None else t for t in (post, gate, pre))
    s1 = torch.rsqrt(h.square().mean(1, keepdim=True) + EPS) if post is not None else one
    n = h * s1 * p
    t = scale * r + g * n
    t_abs = (scale * r).abs() + (g * n).abs()
    s2 = torch.rsqrt(t.square().mean(1, keepdim=True) + EPS)
    # t is off by some U of t_abs, and the norm behind it by as much of its largest share
    spread = 1 + (t_abs * t.abs()).mean(1, keepdim=True) * s2.square()
    out = dict(stream=(t, t_abs), normed=(t * s2 * w, t_abs * s2 * w.abs() * spread))
    hat, hat_abs = t * s2, t_abs * s2 * spread
    e, e_abs = (torch.zeros_like(h) if dstream is None else dstream), torch.zeros_like(h) if dstream is None else dstream.abs()
    if pre is not None and dnormed is not None:
        u, u_abs = dnormed * w, (dnormed * w).abs()
        e = e + s2 * (u - hat * (u * hat).mean(1, keepdim=True))
        e_abs = e_abs + s2 * spread * (u_abs + hat_abs * (u_abs * hat_abs).mean(1, keepdim=True))
        out["pre"] = ((dnormed * hat), dnormed.abs() * hat_abs)
    elif pre is not None:
        out["pre"] = (torch.zeros_like(h), torch.zeros_like(h))
    out["residual"] = (scale * e, abs(scale) * e_abs)
    out["gate"] = (e * n, e_abs * n.abs())
    q, q_abs = e * g, e_abs * g.abs()
    if post is None:
        out["h"] = (q, q_abs)
        return out
    k, k_abs = h * s1, (h * s1).abs()
    out["post"] = (q * k, q_abs * k_abs)
    out["h"] = (s1 * (q * p - k * (q * p * k).mean(1, keepdim=True)),
                s1 * (q_abs * p.abs() + k_abs * (q_abs * p.abs() * k_abs).mean(1, keepdim=True)))
    return out


def close(got, want, absolute, terms, what):
    """`terms` float32 operations, each off by U of the absolute values that it works on, then the result's rounding."""
    got, bound = got.double(), want.abs() * half(got.dtype) + (terms * U) * absolute * 1.01 + 1e-38
    assert got.shape == want.shape
    assert ((got - want).abs() <= bound).all(), (what, float(((got - want).abs() / bound).max()))


def check(h, r, post, gate, pre, scale=1.0, use=(True, True), seed=0):
    g = torch.Generator(device=h.device).manual_seed(seed)
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (h, r, post, gate, pre)]
    stream, normed = residual_rms_norm(leaves[0], leaves[1], post_weight=leaves[2], gate=leaves[3], pre_weight=leaves[4],
                                       residual_scale=scale, eps=EPS)
    assert stream.dtype == r.dtype and stream.shape == h.shape and (normed is None) == (pre is None)
    ds = torch.randn(h.shape, generator=g, device=h.device).to(r.dtype) if use[0] else None
    dy = torch.randn(h.shape, generator=g, device=h.device).to(h.dtype) if use[1] and pre is not None else None
    results, into = [], []
    for t, d in ((stream, ds), (normed, dy)):
        if d is not None:
            assert t.dtype == d.dtype
            results.append(t), into.append(d)
    used = [t for t in leaves if t is not None]
    grads = dict(zip([n for n, t in zip(("h", "residual", "post", "gate", "pre"), leaves) if t is not None],
                     torch.autograd.grad(results, used, into, allow_unused=True)))
    dim = h.shape[-1]
    flat = lambda t: None if t is None else t.detach().double().reshape(-1, dim)
    rows = h.numel() // dim
    gate_rows = flat(gate)
    if gate is not None:
        groups = gate_rows.shape[0]
        gate_rows = gate_rows.repeat_interleave(rows // groups, 0)
    vec = lambda t: None if t is None else t.detach().double()
    want = reference(flat(h), flat(r), vec(post), gate_rows, vec(pre), scale, flat(ds), flat(dy))
    # a mean of `dim` terms in any order, and some twenty operations around each of at most four of them
    terms = 2 * dim + 80
    close(stream.detach().reshape(-1, dim), *want["stream"], dim + 20, "stream")
    if pre is not None:
        close(normed.detach().reshape(-1, dim), *want["normed"], terms, "normed")
    for name in ("h", "residual"):
        close(grads[name].reshape(-1, dim), *want[name], 2 * terms, name)
        assert grads[name].dtype == (h if name == "h" else r).dtype
    for name, w in (("post", post), ("pre", pre)):
        if w is not None and name in want:
            if grads[name] is None:
                assert name == "pre" and dy is None
                continue
            close(grads[name], want[name][0].sum(0), want[name][1].sum(0), 2 * terms + rows, name)
            assert grads[name].dtype == w.dtype
    if gate is not None:
        value, absolute = (t.view(groups, rows // groups, dim).sum(1) for t in want["gate"])
        close(grads["gate"].reshape(-1, dim), value, absolute, 2 * terms + rows // groups, "gate")
        assert grads["gate"].shape == gate.shape and grads["gate"].dtype == gate.dtype
    with torch.no_grad():
        plain = residual_rms_norm(h, r, post_weight=post, gate=gate, pre_weight=pre, residual_scale=scale, eps=EPS)
    assert torch.equal(plain[0], stream) and (normed is None or torch.equal(plain[1], normed))
    again = torch.autograd.grad(residual_rms_norm(leaves[0], leaves[1], post_weight=leaves[2], gate=leaves[3], pre_weight=leaves[4],
                                                  residual_scale=scale, eps=EPS)[:1 + (normed is not None)][slice(not use[0], None if dy is not None else 1)],
                                used, into, allow_unused=True)
    assert all(a is b or torch.equal(a, b) for a, b in zip(again, grads.values()))
    return stream, normed, grads


def make(device, rows, dim, kind, types=(BF, BF, BF), gate_shape=None, seed=0):
    h_type, r_type, w_type = types
    shape = rows if isinstance(rows, tuple) else (rows,)
    g = torch.Generator(device=device).manual_seed(seed + sum(shape) * 7 + dim)
    n = lambda shape, t: torch.randn(shape, generator=g, device=device).to(t)
    vec = lambda s=(dim,): (1 + 0.3 * torch.randn(s, generator=g, device=device)).to(w_type)
    post, gate, pre = kind
    return (n((*shape, dim), h_type) * 2, n((*shape, dim), r_type) * 3, vec() if post else None,
            vec(gate_shape or (dim,)) if gate else None, vec() if pre else None)


WIDTHS = [1, 2, 7, 8, 63, 64, 65, 128, 130, 255, 256, 257, 511, 512, 513, 1000, 1024, 1025, 2047, 2048, 2049, 4096, 4097, 5000,
          8192, 8193, 16384, 16385, 20000]


@pytest.mark.parametrize("types", [(BF, BF, BF), (F32, F32, F32), (BF, F32, F32)], ids=["bf16", "f32", "mixed"])
@pytest.mark.parametrize("dim", WIDTHS)
def test_widths(device, dim, types):
    check(*make(device, 5, dim, (True, True, True), types), scale=0.5)
    check(*make(device, 3, dim, (False, False, True), types))


@pytest.mark.parametrize("kind", KINDS, ids=lambda k: "".join("pgn"[i] if v else "-" for i, v in enumerate(k)))
@pytest.mark.parametrize("dim", [96, 640, 2048, 2304, 4608, 17000])
def test_kinds(device, dim, kind):
    """Every choice of the operands, and either output alone."""
    operands = make(device, 11, dim, kind)
    check(*operands, scale=-1.5)
    check(*operands, use=(True, False))
    if kind[2]:
        check(*operands, use=(False, True))


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 63, 257, 1025, 3001])
@pytest.mark.parametrize("dim", [64, 1536, 4096])
def test_rows(device, rows, dim):
    check(*make(device, rows, dim, (True, True, True)))
    check(*make(device, rows, dim, (True, False, True), (BF, F32, BF)))


@pytest.mark.parametrize("shape,gate", [((4, 6), (4, 1)), ((4, 6), (4, 6)), ((1, 9), (1, 1)), ((3, 5, 7), (3, 5, 1)),
                                        ((3, 5, 7), (3, 1, 1)), ((600, 3), (600, 1)), ((2, 700), (2, 1)), ((1500, 1), (1500, 1)),
                                        ((7, 301), (7, 1)), ((2, 5), (1, 1))])
@pytest.mark.parametrize("dim", [72, 2048, 2500, 16400])
def test_gates_of_sequences_and_rows(device, shape, gate, dim):
    check(*make(device, shape, dim, (True, True, True), gate_shape=(*gate, dim)))
    check(*make(device, shape, dim, (False, True, False), (BF, BF, F32), gate_shape=(*gate, dim)))


def test_many_rows_share_and_own_gates(device):
    check(*make(device, (70000, 1), 8, (True, True, True), gate_shape=(70000, 1, 8)))
    check(*make(device, (35000, 2), 8, (True, True, True), gate_shape=(35000, 1, 8)))


@pytest.mark.parametrize("dim", [20, 128, 190, 256, 300, 511])
@pytest.mark.parametrize("rows,gates", [(9000, 9000), (9000, 3000), (10000, 2000), (9003, 1), (4000, 4000), (16390, 8195)])
@pytest.mark.parametrize("post", [True, False])
def test_narrow_rows_with_gates_for_a_few_rows_each(device, rows, gates, dim, post):
    """Rows whose lanes work on their own, and those that share a strip, with all counts of rows left over."""
    h, r, p, g, w = make(device, rows, dim, (post, True, True), (BF, F32, F32), gate_shape=(gates, dim))
    gate = g if gates == rows else g.reshape(gates, 1, dim)
    shape = (rows, dim) if gates == rows else (gates, rows // gates, dim)
    check(h.reshape(shape), r.reshape(shape), p, gate, w, 0.9)


@pytest.mark.parametrize("dim", [513, 1000, 1024, 2050, 4096, 4100])
@pytest.mark.parametrize("rows,gates", [(2100, 2100), (2100, 1050), (2049, 683), (2048, 512)])
def test_wide_rows_with_gates_for_a_few_rows_each(device, rows, gates, dim):
    for types in ((BF, BF, BF), (BF, F32, F32)):
        h, r, p, g, w = make(device, (gates, rows // gates), dim, (True, True, True), types, gate_shape=(gates, 1, dim))
        check(h, r, p, g, w, 1.1)


@pytest.mark.parametrize("types", [(BF, BF, BF), (F32, F32, F32), (BF, F32, BF)], ids=["bf16", "f32", "mixed"])
@pytest.mark.parametrize("dim", [4104, 5119, 5120, 5121, 6143, 6144, 6150, 7168])
def test_rows_of_some_thousands(device, dim, types):
    check(*make(device, (2, 300), dim, (True, True, True), types, gate_shape=(2, 1, dim)), 0.7)
    check(*make(device, 515, dim, (False, False, True), types))


@pytest.mark.parametrize("shape,dim,kind", [((16, 3200), 2048, (True, True, True)), ((1, 51201), 2047, (True, True, True)),
                                            ((51200,), 2048, (False, False, True)), ((25603,), 4096, (True, False, True)),
                                            ((10, 10241), 1000, (True, True, True)), ((40, 5121), 512, (False, True, True)),
                                            ((400, 256), 1024, (True, True, True)), ((205000,), 505, (True, True, True)),
                                            ((51200, 1), 2048, (True, True, True))])
def test_matrices_that_no_cache_holds(device, shape, dim, kind):
    gate_shape = (shape[0], *[1] * (len(shape) - 1), dim) if len(shape) > 1 else None
    check(*make(device, shape, dim, kind, gate_shape=gate_shape), 0.8)
    torch.cuda.empty_cache()


def test_strides_and_alignment(device):
    g = torch.Generator(device=device).manual_seed(3)
    for dim, lo in ((512, 1), (2048, 3), (100, 5), (5000, 7)):
        wide = torch.randn((9, dim + 9), generator=g, device=device).to(BF)
        r = torch.randn((9, dim + 20), generator=g, device=device)[:, 11:11 + dim]
        vectors = (1 + 0.1 * torch.randn((3, dim + 1), generator=g, device=device)).to(BF)[:, 1:]
        check(wide[:, lo:lo + dim], r, *vectors)
        check(wide[:, lo:lo + dim], wide[:, :dim], *vectors.float())
        column = torch.randn((dim, 9), generator=g, device=device).to(BF).t()
        check(column, column, *vectors)                     # transposed; the block's output is the stream itself
        check(wide[:1, :dim].expand(9, dim), wide[:, :dim], None, None, vectors[0])


def test_the_same_tensor_twice(device):
    h, _, post, gate, pre = make(device, 6, 512, (True, True, True))
    x = h.clone().requires_grad_(True)
    stream, normed = residual_rms_norm(x, x, post_weight=post, gate=gate, pre_weight=pre)
    (both,) = torch.autograd.grad(normed.float().sum(), x)
    a, b = h.clone().requires_grad_(True), h.clone().requires_grad_(True)
    _, normed = residual_rms_norm(a, b, post_weight=post, gate=gate, pre_weight=pre)
    da, db = torch.autograd.grad(normed.float().sum(), (a, b))
    assert torch.equal(both, da + db)


def test_rows_of_zeros_and_what_is_not_finite(device):
    h, r, post, gate, pre = make(device, 6, 640, (True, True, True))
    h[0], r[0] = 0, 0
    h[2, 5], r[3, 7] = float("inf"), float("nan")
    stream, normed = residual_rms_norm(h, r, post_weight=post, gate=gate, pre_weight=pre)
    assert not stream[0].any() and not normed[0].any()
    for row in (2, 3):
        assert normed[row].isnan().any() and stream[row].isnan().any()
    fine = residual_rms_norm(h[[0, 1, 4, 5]], r[[0, 1, 4, 5]], post_weight=post, gate=gate, pre_weight=pre)
    assert torch.equal(stream[[0, 1, 4, 5]], fine[0]) and torch.equal(normed[[0, 1, 4, 5]], fine[1])
    leaves = [t.detach().requires_grad_(True) for t in (h, r)]
    out = residual_rms_norm(*leaves, post_weight=post, gate=gate, pre_weight=pre)
    dh, dr = torch.autograd.grad([t.sum() for t in out], leaves)
    assert dh[[0, 1, 4, 5]].isfinite().all() and dr[[0, 1, 4, 5]].isfinite().all()


@pytest.mark.parametrize("cols", [9, 20, 131, 250, 1030, 4099, 9001, 16390])
@pytest.mark.parametrize("from_end", [0, 3, 7, 8])
def test_an_infinity_leaves_the_rest_of_its_row_as_the_formula_does(device, cols, from_end):
    """An infinite element makes its row's norm infinite: the others are 0 behind the norm, itself NaN."""
    h, r, post, _, pre = make(device, 3, cols, (True, False, True))
    at = cols - 1 - from_end
    h[1, at] = float("inf")
    stream, _ = residual_rms_norm(h, r, post_weight=post)
    _, normed = residual_rms_norm(h, r, pre_weight=pre)
    others = torch.arange(cols, device=device) != at
    assert torch.equal(stream[1, others], r[1, others]) and stream[1, at].isnan()
    assert not normed[1, others].any() and normed[1, at].isnan()
    assert stream[[0, 2]].isfinite().all() and normed[[0, 2]].isfinite().all()


def test_only_some_gradients_are_wanted(device):
    operands = make(device, 7, 768, (True, True, True))
    every = [t.clone().requires_grad_(True) for t in operands]
    call = lambda t: residual_rms_norm(t[0], t[1], post_weight=t[2], gate=t[3], pre_weight=t[4], residual_scale=2.0)
    want = torch.autograd.grad([t.float().sum() for t in call(every)], every)
    for i in range(5):
        some = [t.clone().requires_grad_(k == i) for k, t in enumerate(operands)]
        (got,) = torch.autograd.grad([t.float().sum() for t in call(some)], [some[i]])
        assert torch.equal(got, want[i])


def test_plain_sum_gives_both_gradients_their_own_memory(device):
    """Without gate, norm behind the block and scale both gradients are equal: an optimizer may still change one of them."""
    h, r, _, _, pre = make(device, 6, 512, (False, False, True))
    h, r = (torch.nn.Parameter(t) for t in (h, r))
    stream, normed = residual_rms_norm(h, r, pre_weight=pre)
    (stream.float().sum() + normed.float().sum()).backward()
    assert torch.equal(h.grad, r.grad)
    before = r.grad.clone()
    h.grad.zero_()
    assert torch.equal(r.grad, before)


def test_a_side_stream_and_a_captured_graph(device):
    operands = make(device, (8, 300), 2048, (True, True, True), gate_shape=(8, 1, 2048))
    h, r, post, gate, pre = operands
    flat = (h.view(-1, 2048), r.view(-1, 2048), post, gate.view(8, 2048), pre)
    dstream, dnormed = torch.randn_like(flat[0]), torch.randn_like(flat[0])

    def both():
        stream, normed, rstd = ops.residual_norm(*flat, 0.5, EPS, want_rstd=True)
        return stream, normed, *ops.residual_norm_bwd(*flat, 0.5, rstd, dstream, dnormed)

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    for _ in range(4):
        for t in (*flat, dstream, dnormed):
            t.copy_(torch.randn_like(t))
        graph.replay()
        want = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(device):
    h, r, post, gate, pre = make(device, 6, 64, (True, True, True))
    with pytest.raises(ValueError):
        residual_rms_norm(h, r[:5])
    with pytest.raises(ValueError):
        residual_rms_norm(h, r, post_weight=post[:63])
    with pytest.raises(ValueError):
        residual_rms_norm(h, r, gate=torch.ones((5, 64), device=device))
    with pytest.raises(ValueError):
        residual_rms_norm(h, r, pre_weight=pre.cpu())
    with pytest.raises(TypeError):
        ops.residual_norm(h.half(), r.half(), None, None, None, 1.0, EPS)
    with pytest.raises(TypeError):
        ops.residual_norm(h.float(), r, None, None, None, 1.0, EPS)
    with pytest.raises(ValueError):
        ops.residual_norm(h, r, None, torch.ones((4, 64), device=device), None, 1.0, EPS)
    x = h.clone().requires_grad_(True)
    stream, _ = residual_rms_norm(x, r, post_weight=post)
    (grad,) = torch.autograd.grad(stream.float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.float().sum().backward()


def test_module(device):
    seam = ResidualRMSNorm.Config(post_norm=True, gate=True, gate_init=0.1, residual_scale=0.5).build(dim=96).to(device)
    h, r = torch.randn((2, 3, 96), device=device), torch.randn((2, 3, 96), device=device)
    stream, normed = seam(h, r)
    t = 0.5 * r.double() + 0.1 * torch.nn.functional.rms_norm(h.double(), (96,), eps=1e-5)
    assert (stream.double() - t).abs().max() <= 200 * U * t.abs().max()
    assert (normed.double() - torch.nn.functional.rms_norm(t, (96,), eps=1e-5)).abs().max() <= 400 * U * 10
    assert [n for n, _ in seam.named_parameters()] == ["post_weight", "gate", "pre_weight"]


def test_a_gate_without_dimensions_is_refused_as_others_are(device):
    h = torch.randn((3, 64), device=device)
    for gate in (torch.ones((), device=device), torch.ones((3, 1), device=device), torch.ones((2, 64), device=device)):
        with pytest.raises(ValueError, match="gate must be"):
            residual_rms_norm(h, h, gate=gate)
