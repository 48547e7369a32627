"""Embedding, norms around a block and gradient clipping without a GPU: their formulas in torch operations, gradients
against differences, and the refusals."""
import math
from ctypes import c_int32, c_void_p

import pytest
import torch
import torch.nn.functional as F

from torchtitan_amd import _lib, ops
from torchtitan_amd.gradients import clip_grad_norm_, get_total_norm
from torchtitan_amd.modules import Embedding, ResidualRMSNorm, residual_rms_norm, scaled_embedding

D = torch.float64


def test_embedding_formula():
    weight = torch.randn((7, 5))
    ids = torch.tensor([[0, 6, 3], [3, 7, -1]])
    out = scaled_embedding(ids, weight, 2.0)
    assert torch.equal(out[0], 2.0 * weight[[0, 6, 3]]) and torch.equal(out[1, 0], 2.0 * weight[3]) and not out[1, 1:].any()
    assert torch.equal(scaled_embedding(ids + 10, weight, 2.0, first_row=10), out)
    assert scaled_embedding(ids, weight, dtype=torch.bfloat16).dtype == torch.bfloat16
    inside = torch.tensor([1, 1, 4])
    mine, theirs = weight.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    scaled_embedding(inside, mine, padding_idx=4).square().sum().backward()
    F.embedding(inside, theirs, padding_idx=4).square().sum().backward()
    assert torch.equal(mine.grad, theirs.grad)
    w = torch.randn((4, 3), dtype=D, requires_grad=True)
    assert torch.autograd.gradcheck(lambda t: scaled_embedding(torch.tensor([3, 0, 3, 9]), t, 1.7), (w,))


@pytest.mark.parametrize("post,gate,pre", [(p, g, n) for p in (0, 1) for g in (0, 1, 2) for n in (0, 1)])
def test_norm_gradients_against_differences(post, gate, pre):
    torch.manual_seed(post + 2 * gate + 8 * pre)
    vec = lambda shape=(6,): torch.randn(shape, dtype=D, requires_grad=True)
    h, r = vec((3, 4, 6)), vec((3, 4, 6))
    weights = dict(post_weight=vec() if post else None, gate=[None, vec(), vec((3, 1, 6))][gate], pre_weight=vec() if pre else None)
    names = [k for k, v in weights.items() if v is not None]

    def call(h, r, *given):
        stream, normed = residual_rms_norm(h, r, residual_scale=0.7, eps=1e-3, **dict(zip(names, given)))
        return stream if normed is None else (stream, normed)

    assert torch.autograd.gradcheck(call, (h, r, *(weights[n] for n in names)))


def test_norm_formula():
    h, r, w, v = torch.randn((5, 32)), torch.randn((5, 32)), torch.rand(32) + 0.5, torch.rand(32) + 0.5
    stream, normed = residual_rms_norm(h, r, post_weight=w, pre_weight=v, residual_scale=0.5, eps=1e-6)
    want = 0.5 * r + F.rms_norm(h, (32,), w, 1e-6)
    assert torch.allclose(stream, want, rtol=1e-5, atol=1e-6)
    assert torch.allclose(normed, F.rms_norm(want, (32,), v, 1e-6), rtol=1e-5, atol=1e-6)
    assert residual_rms_norm(h, r)[1] is None
    empty = residual_rms_norm(h[:0], r[:0], pre_weight=v)
    assert empty[0].shape == (0, 32) and empty[1].shape == (0, 32)


def test_modules_are_built_from_their_configs():
    table = Embedding.Config(scale=3.0, padding_idx=1).build(num_embeddings=6, embedding_dim=4)
    table.init_weights(init_std=0.5)
    assert not table.weight[1].any() and torch.equal(table(torch.tensor([0])), 3.0 * table.weight[:1])
    seam = ResidualRMSNorm.Config(post_norm=True, gate=True, gate_init=0.0).build(dim=8)
    r = torch.randn((2, 8))
    assert torch.equal(seam(torch.randn((2, 8)), r)[0], r)
    last = ResidualRMSNorm.Config(pre_norm=False).build(dim=8)
    assert last(r, r)[1] is None and list(last.parameters()) == []


def test_clipping_runs_through_torch_off_the_gpu():
    mine, theirs = ([torch.nn.Parameter(torch.zeros(s)) for s in ((3, 4), (5,), (2,))] for _ in range(2))
    for p, q in zip(mine[:2], theirs[:2]):  # the last has no gradient
        p.grad = torch.randn(p.shape)
        q.grad = p.grad.clone()
    for kind in (2.0, 1.0, 3.0, math.inf):
        a, b = clip_grad_norm_(mine, 0.5, kind), torch.nn.utils.clip_grad_norm_(theirs, 0.5, kind)
        assert torch.equal(a, b) and all(torch.equal(p.grad, q.grad) for p, q in zip(mine[:2], theirs[:2]))
    assert float(get_total_norm([])) == 0.0
    mine[0].grad[0, 0] = math.inf
    with pytest.raises(RuntimeError):
        clip_grad_norm_(mine, 0.5, error_if_nonfinite=True)


def test_refusals():
    weight = torch.randn((4, 8))
    with pytest.raises(TypeError):
        scaled_embedding(torch.zeros(2), weight)
    with pytest.raises(ValueError):
        scaled_embedding(torch.zeros(2, dtype=torch.int64), weight[0])
    with pytest.raises(_lib.MXLibraryError):
        ops.embedding_fwd(torch.zeros(2, dtype=torch.int64), weight)
    h = torch.randn((2, 3, 8))
    for gate in (torch.ones(7), torch.ones((2, 8)), torch.ones((3, 1, 8)), torch.ones((1, 3, 8)), torch.ones(()),
                 torch.ones((2, 3, 1, 8))):
        with pytest.raises(ValueError):
            residual_rms_norm(h, h, gate=gate)
    with pytest.raises(ValueError):
        residual_rms_norm(h, h[0])
    with pytest.raises(ValueError):
        residual_rms_norm(h, h, pre_weight=torch.ones(4))
    with pytest.raises(TypeError):
        residual_rms_norm(h.long(), h.long())
    with pytest.raises(_lib.MXLibraryError):
        ops.residual_norm(h[0], h[0], None, None, None, 1.0, 1e-5)
    with pytest.raises(_lib.MXLibraryError):
        ops.grad_norm([weight])


def test_dense_tensors():
    t = torch.zeros((4, 6, 8))
    assert ops.is_dense(t) and ops.is_dense(t.permute(2, 0, 1)) and ops.is_dense(t[1:3]) and ops.is_dense(t[:, :, :0])
    assert not ops.is_dense(t[:, 1:]) and not ops.is_dense(t[:1].expand(4, 6, 8)) and not ops.is_dense(t[..., ::2])
    assert ops.is_dense(t[:1, :1, :1].transpose(0, 2)) and ops.is_dense(t[:, :1].squeeze(1)[:1])


def test_entry_points_check_their_arguments_before_any_launch():
    lib = _lib.load()
    P = c_void_p
    a, odd = P(0x1000), P(0x1002)
    # embedding: no tokens is no work, null pointers and rows that overlap are refused, so are misaligned elements
    assert lib.mx_embedding(None, 1, 0, None, 0, 10, 8, 8, 0, 1.0, None, 0, None) == 0
    assert lib.mx_embedding(None, 1, 4, a, 0, 10, 8, 8, 0, 1.0, a, 0, None) == 1
    assert lib.mx_embedding(a, 1, 4, a, 0, 10, 8, 7, 0, 1.0, a, 0, None) == 1
    assert lib.mx_embedding(a, 1, -1, a, 0, 10, 8, 8, 0, 1.0, a, 0, None) == 1
    assert lib.mx_embedding(a, 1, 4, odd, 1, 10, 8, 8, 0, 1.0, a, 0, None) == 2
    assert lib.mx_embedding(odd, 0, 4, a, 1, 10, 8, 8, 0, 1.0, a, 0, None) == 2
    assert lib.mx_embedding(a, 1, 4, a, 0, 1 << 31, 8, 8, 0, 1.0, a, 0, None) == 4
    assert lib.mx_embedding_grad(a, 1, 4, a, 0, 8, 0, 8, 0, -1, 1.0, None, 0, a, None) == 0
    assert lib.mx_embedding_grad(a, 1, 4, a, 0, 8, 9, 8, 0, -1, 1.0, a, 0, None, None) == 1
    assert lib.mx_embedding_grad(a, 1, 4, a, 0, 7, 9, 8, 0, -1, 1.0, a, 0, a, None) == 1
    assert lib.mx_embedding_grad(a, 1, 4, a, 0, 8, 9, 8, 0, -1, 1.0, odd, 1, a, None) == 2
    assert lib.mx_embedding_grad(a, 1, 1 << 31, a, 0, 8, 9, 8, 0, -1, 1.0, a, 0, a, None) == 4
    assert lib.mx_embedding_grad_workspace(0, 9, 8) == 0 < lib.mx_embedding_grad_workspace(5, 9, 8)
    # norms
    none = P(None)
    fwd = lambda h=a, hf=0, r=a, rf=0, rows=4, cols=8, ldh=8, ldr=8, post=none, gate=none, pre=none, fl=0, g=1, out=a, y=none: \
        lib.mx_residual_norm(h, hf, r, rf, rows, cols, ldh, ldr, post, gate, pre, fl, g, 1.0, 1e-5, out, y, None, None)
    assert fwd(rows=0, h=None, r=None, out=None) == 0
    for status, bad in ((1, dict(h=None)), (1, dict(ldh=7)), (1, dict(ldr=7)), (1, dict(hf=1)), (1, dict(g=0)), (1, dict(g=3)),
                        (1, dict(rows=-1)), (1, dict(out=None)), (1, dict(pre=a)), (2, dict(r=odd, rf=1)),
                        (2, dict(post=odd, fl=1)), (2, dict(gate=odd, fl=2)), (2, dict(pre=odd, fl=4, y=a)), (4, dict(rows=1 << 31))):
        assert fwd(**bad) == status, bad
    bwd = lambda post=none, gate=none, pre=none, rstd=a, ds=a, dy=none, dh=a, dr=a, dpost=none, dgate=none, dpre=none, ws=a, rows=4: \
        lib.mx_residual_norm_bwd(a, 0, a, 0, rows, 8, 8, 8, post, gate, pre, 0, 1, 1.0, rstd, ds, dy, dh, dr, dpost, dgate, dpre, ws, None)
    assert bwd(rows=0) == 0
    for bad in (dict(dpost=a), dict(dgate=a), dict(dpre=a), dict(dy=a), dict(rstd=None), dict(ws=None),
                dict(rows=0, pre=a, dpre=a)):
        assert bwd(**bad) == 1, bad
    assert bwd(ws=odd) == 2
    assert lib.mx_residual_norm_workspace(0, 8, 1) == 0 == lib.mx_residual_norm_workspace(4, 8, 3)
    # gradients
    ptrs, sizes, kinds = (c_void_p * 1)(0x1002), (_lib._I * 1)(5), (c_int32 * 1)(1)
    assert lib.mx_grad_norm(1, ptrs, sizes, kinds, 0, a, a, None) == 2
    kinds[0] = 0
    assert lib.mx_grad_norm(1, ptrs, sizes, kinds, 3, a, a, None) == 1 == lib.mx_grad_norm(1, ptrs, sizes, kinds, 0, None, a, None)
    assert lib.mx_grad_norm(1, None, sizes, kinds, 0, a, a, None) == 1 == lib.mx_grad_scale(1, ptrs, sizes, kinds, None, 1.0, None)
    sizes[0] = -1
    assert lib.mx_grad_scale(1, ptrs, sizes, kinds, a, 1.0, None) == 1
    sizes[0] = 1 << 60
    assert lib.mx_grad_scale(1, ptrs, sizes, kinds, a, 1.0, None) == 4
    assert lib.mx_grad_norm_workspace(0) == 0 and lib.mx_grad_norm_workspace(161) == 2 * lib.mx_grad_norm_workspace(160)


def test_entry_points_refuse_what_no_launch_holds():
    """A launch has fewer than 2^32 lanes, and rows are counted in 32 bits: status 4, before any launch."""
    lib, a = _lib.load(), c_void_p(0x1000)
    assert lib.mx_embedding(a, 1, 1 << 26, a, 0, 10, 8, 8, 0, 1.0, a, 0, None) == 4
    assert lib.mx_embedding(a, 1, 1 << 20, a, 0, 10, 1 << 17, 1 << 17, 0, 1.0, a, 0, None) == 4
    assert lib.mx_embedding(a, 1, 5, a, 0, 10, 1 << 40, 1 << 40, 0, 1.0, a, 0, None) == 4
    assert lib.mx_embedding_grad(a, 1, 4, a, 0, 1 << 28, 9, 1 << 28, 0, -1, 1.0, a, 0, a, None) == 4
    assert lib.mx_embedding_grad(a, 1, 4, a, 0, 4096, 1 << 24, 4096, 0, -1, 1.0, a, 0, a, None) == 4
    assert lib.mx_embedding_grad(a, 1, 1 << 30, a, 0, 8, 9, 8, 0, -1, 1.0, a, 0, a, None) == 4
    norm = lambda rows, cols: lib.mx_residual_norm(a, 0, a, 0, rows, cols, cols, cols, None, None, None, 0, 1, 1.0, 1e-5, a, None, None, None)
    assert norm(1 << 22, 5) == 4 and norm(1 << 22, 20000) == 4 and norm(1, 1 << 31) == 4
    ptrs, sizes, kinds = (c_void_p * 2)(0x1000, 0x2000), (_lib._I * 2)(1 << 36, 1 << 36), (c_int32 * 2)(1, 0)
    assert lib.mx_grad_norm(2, ptrs, sizes, kinds, 0, a, a, None) == 4
    assert lib.mx_grad_clip(2, ptrs, sizes, kinds, 0, a, 1.0, a, None) == 4


def test_embedding_and_norms_trace_without_a_break():
    """Off the GPU their formulas are traced, one graph; on it (fake tensors) one operator each."""
    class Two(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.tokens = Embedding.Config(scale=2.0).build(num_embeddings=9, embedding_dim=32)
            self.seam = ResidualRMSNorm.Config(post_norm=True, gate=True).build(dim=32)

        def forward(self, ids):
            x = self.tokens(ids)
            return self.seam(x, x)

    graphs = []
    module, ids = Two(), torch.zeros((2, 3), dtype=torch.int64)
    traced = torch.compile(module, backend=lambda graph, example: graphs.append(graph) or graph.forward, fullgraph=True)
    assert all(torch.equal(a, b) for a, b in zip(traced(ids), module(ids))) and len(graphs) == 1
    torch._dynamo.reset()
    import torchtitan_amd.compiled  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        w, ids = torch.empty((9, 32), dtype=torch.bfloat16, device="cuda"), torch.zeros((2, 3), dtype=torch.int64, device="cuda")
        out = torch.ops.torchtitan_amd.embedding_fwd(ids, w, 2.0, None, 0, torch.float32)
        assert out.shape == (2, 3, 32) and out.dtype == torch.float32
        grad = torch.ops.torchtitan_amd.embedding_bwd(ids, out, 9, 2.0, 0, None, torch.bfloat16)
        assert grad.shape == (9, 32) and grad.dtype == torch.bfloat16
        h, r = torch.empty((6, 32), dtype=torch.bfloat16, device="cuda"), torch.empty((6, 32), device="cuda")
        stream, normed, rstd = torch.ops.torchtitan_amd.residual_norm_fwd(h, r, w[0], None, w[1], 1.0, 1e-5)
        assert stream.dtype == torch.float32 and normed.dtype == torch.bfloat16 and rstd.shape == (2, 6)
        grads = torch.ops.torchtitan_amd.residual_norm_bwd(h, r, w[0], None, w[1], 1.0, rstd, stream, None,
                                                           [True, False, True, True, True])
        assert [tuple(g.shape) for g in grads] == [(6, 32), (0,), (32,), (0,), (32,)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gradients_of_equal_ids_are_added_up_in_float32(dtype):
    """In a table's own type the sum of ones ends where a one is less than half a step: at 256 in bf16, 2048 in fp16."""
    ids = torch.cat([torch.full((5001,), 2), torch.tensor([0, 9])])
    ones = torch.ones((5003, 8), dtype=dtype)
    want = torch.tensor([[1.0], [0.0], [5001.0], [0.0]]).to(dtype).expand(4, 8)
    weight = torch.randn((4, 8)).to(dtype)
    leaf = weight.clone().requires_grad_(True)
    scaled_embedding(ids, leaf).backward(ones)
    assert leaf.grad.dtype == dtype and torch.equal(leaf.grad, want)
    leaf = weight.clone().requires_grad_(True)
    scaled_embedding(ids, leaf, padding_idx=2).backward(ones)
    assert torch.equal(leaf.grad, torch.where(want > 1, 0, want))
    assert torch.equal(torch.func.grad(lambda t: (scaled_embedding(ids, t, dtype=torch.float32)).sum())(weight), want)
    module = Embedding.Config().build(num_embeddings=4, embedding_dim=8).to(dtype)
    torch._dynamo.reset()
    torch.compile(module, backend="aot_eager", fullgraph=True)(ids).backward(ones)
    torch._dynamo.reset()
    assert torch.equal(module.weight.grad, want)


def test_a_table_without_rows_has_a_gradient_without_rows():
    """A shard of no rows: zeros for every token, as part of the graph."""
    none = torch.empty((0, 6), dtype=torch.bfloat16, requires_grad=True)
    out = scaled_embedding(torch.arange(4).view(2, 2), none, dtype=torch.float32)
    assert out.shape == (2, 2, 6) and out.dtype == torch.float32 and not out.any()
    (grad,) = torch.autograd.grad(out.sum(), none)
    assert grad.shape == (0, 6) and grad.dtype == torch.bfloat16
    assert scaled_embedding(torch.zeros((0, 3), dtype=torch.int32), none).shape == (0, 3, 6)


@pytest.mark.skipif(torch.cuda.is_available(), reason="what is taken would be launched on addresses that are none")
def test_the_last_sizes_that_are_taken_and_the_first_that_are_refused():
    """Without a GPU a call that is taken ends at its launch, status 3; one that is refused never gets there, status 4."""
    lib, a = _lib.load(), c_void_p(0x1000)
    forward = lambda n, cols: lib.mx_embedding(a, 1, n, a, 0, 10, cols, cols, 0, 1.0, a, 0, None)
    for cols, most in ((8, 2 ** 26 - 4), (512, 2 ** 26 - 4), (1024, 2 ** 26 - 4), (1025, 2 ** 25 - 2), (2048, 2 ** 25 - 2), (4096, 2 ** 24 - 1)):
        assert (forward(most, cols), forward(most + 1, cols)) == (3, 4), cols
    gradient = lambda n, rows, cols: lib.mx_embedding_grad(a, 1, n, a, 0, cols, rows, cols, 0, -1, 1.0, a, 0, a, None)
    assert (gradient(2 ** 29 - 32, 9, 8), gradient(2 ** 29 - 31, 9, 8)) == (3, 4)
    assert (gradient(4, 9, 2 ** 27 - 2048), gradient(4, 9, 2 ** 27)) == (3, 4)  # slabs of 2048 columns
    assert (gradient(2 ** 29 - 32, 15 * 2 ** 18, 2 ** 13), gradient(4, 2 ** 22, 2 ** 13)) == (3, 4)  # 2^10 pieces a row
    assert (gradient(4, 2 ** 31 - 2, 1), gradient(4, 2 ** 31 - 1, 1)) == (3, 4)
    norm = lambda rows, cols: lib.mx_residual_norm(a, 0, a, 0, rows, cols, cols, cols, None, None, None, 0, 1, 1.0, 1e-5, a, None, None, None)
    back = lambda rows, cols: lib.mx_residual_norm_bwd(a, 0, a, 0, rows, cols, cols, cols, None, None, None, 0, 1, 1.0, a, a, None, a, a,
                                                       None, None, None, a, None)
    for call in (norm, back):
        for cols, most in ((1, 2 ** 22 - 1), (7, 2 ** 22 - 1), (8, 2 ** 31 - 1), (128, 2 ** 31 - 1), (16384, 2 ** 31 - 1), (16385, 2 ** 22 - 1)):
            assert (call(most, cols), call(most + 1, cols)) == (3, 4), cols
        assert (call(1, 2 ** 31 - 1), call(1, 2 ** 31)) == (3, 4)
    ptrs, sizes, kinds = (c_void_p * 2)(0x1000, 0x2000), (_lib._I * 2)(), (c_int32 * 2)(1, 0)
    for second, status in ((8192, 3), (8193, 4)):  # behind 2^24 - 2 chunks of float32 one of bf16, or two
        sizes[0], sizes[1] = (2 ** 24 - 2) * 4096, second
        assert lib.mx_grad_norm(2, ptrs, sizes, kinds, 0, a, a, None) == status
        assert lib.mx_grad_scale(2, ptrs, sizes, kinds, a, 1.0, None) == status
        assert lib.mx_grad_clip(2, ptrs, sizes, kinds, 0, a, 1.0, a, None) == status


@pytest.mark.parametrize("strict", [False, True])
def test_embedding_and_norms_export_as_operators(strict):
    """On the GPU (fake tensors, which torch.export's default way runs the module on) one operator each."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    class Two(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.tokens = Embedding.Config(scale=2.0).build(num_embeddings=9, embedding_dim=32)
            self.seam = ResidualRMSNorm.Config(post_norm=True, gate=True).build(dim=32)

        def forward(self, ids):
            x = self.tokens(ids)
            return self.seam(x, x)

    with FakeTensorMode(), torch.device("cuda"):
        module, ids = Two(), torch.zeros((2, 3), dtype=torch.int64)
    targets = [str(n.target) for n in torch.export.export(module, (ids,), strict=strict).graph.nodes if n.op == "call_function"]
    assert [t for t in targets if "torchtitan_amd" in t] == ["torchtitan_amd.embedding_fwd.default", "torchtitan_amd.residual_norm_fwd.default"]
    assert not any("rsqrt" in t or "index" in t for t in targets)
