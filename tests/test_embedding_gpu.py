"""The embedding's lookup and its gradient by sorted tokens against float64."""
import pytest
import torch

from torchtitan_amd import ops
from torchtitan_amd.modules import Embedding, scaled_embedding

pytestmark = pytest.mark.gpu

U = 2.0 ** -24  # float32 rounds by at most this, relative to the value
TYPES = [(torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32), (torch.float32, torch.bfloat16),
         (torch.bfloat16, torch.float32)]


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, bound):
    """Within `bound`, and not finite where and as `want` is not."""
    got = got.double()
    same = (got == want) | (got.isnan() & want.isnan())
    assert (same | ((got - want).abs() <= bound)).all(), float(((got - want).abs() - bound)[~same].max())


def reference(ids, weight, scale, padding, first, dout):
    """(out, grad, the sums of the absolute values that a row of the gradient adds up, how many they are)."""
    rows, cols = weight.shape
    table = torch.zeros((rows + 1, cols), dtype=torch.float64, device=weight.device)
    table[:rows] = weight.double() * scale
    row = ids.reshape(-1).long() - first
    row = torch.where((row >= 0) & (row < rows), row, rows)
    out = table[row].view(*ids.shape, cols)
    counted = row if padding is None else torch.where(ids.reshape(-1) == padding, rows, row)
    d = dout.reshape(-1, cols).double()
    total, absolute = torch.zeros_like(table), torch.zeros_like(table)
    total.index_add_(0, counted, d)
    absolute.index_add_(0, counted, d.abs())
    count = torch.bincount(counted, minlength=rows + 1)[:rows, None]
    return out, total[:rows] * scale, absolute[:rows] * abs(scale), count


def check(ids, weight, scale, padding, first, dtype, dout):
    weight = weight.detach().requires_grad_(True)
    out = scaled_embedding(ids, weight, scale, padding_idx=padding, first_row=first, dtype=dtype)
    assert out.dtype == dtype and out.shape == (*ids.shape, weight.shape[1])
    (grad,) = torch.autograd.grad(out, weight, dout)
    assert grad.dtype == weight.dtype and grad.shape == weight.shape
    want, gwant, absolute, count = reference(ids, weight.detach(), scale, padding, first, dout)
    # one product in float32, one rounding to the result's type
    close(out.detach(), want, want.abs() * (half(dtype) * (dtype != torch.float32) + 2 * U))
    # n terms added in any order are off by at most n U of their absolute values' sum; then the product and the rounding
    close(grad, gwant, gwant.abs() * half(weight.dtype) * (weight.dtype != torch.float32) + (count + 3) * U * absolute * 1.01)
    no_grad = scaled_embedding(ids, weight.detach(), scale, padding_idx=padding, first_row=first, dtype=dtype)
    assert torch.equal(no_grad, out)
    (again,) = torch.autograd.grad(scaled_embedding(ids, weight, scale, padding_idx=padding, first_row=first, dtype=dtype), weight, dout)
    assert torch.equal(again, grad)


def make(device, tokens, rows, cols, w_type, o_type, seed, vocab=None, skew=False):
    g = torch.Generator(device=device).manual_seed(seed)
    weight = torch.randn((rows, cols), generator=g, device=device).to(w_type)
    vocab = vocab or rows
    ids = torch.randint(0, vocab, (tokens,), generator=g, device=device)
    if skew:  # half of the tokens are the same one, an eighth another
        ids[::2], ids[1::8] = vocab // 2, vocab - 1
    dout = torch.randn((tokens, cols), generator=g, device=device).to(o_type)
    return ids, weight, dout


@pytest.mark.parametrize("w_type,o_type", TYPES)
@pytest.mark.parametrize("tokens,rows,cols", [(1, 1, 1), (1, 5, 8), (2, 1, 3), (7, 3, 64), (65, 11, 129), (64, 300, 512),
                                              (200, 40, 1000), (33, 1000, 2047), (129, 7, 4100)])
def test_small_sizes(device, tokens, rows, cols, w_type, o_type):
    ids, weight, dout = make(device, tokens, rows, cols, w_type, o_type, tokens + cols)
    check(ids, weight, 1.0, None, 0, o_type, dout)
    check(ids, weight, 45.25, int(ids[0]), 0, o_type, dout)


@pytest.mark.parametrize("skew", [False, True])
@pytest.mark.parametrize("tokens,rows,cols", [(1000, 50000, 24), (8192, 1000, 72), (8193, 513, 40), (20011, 151936, 16),
                                              (70001, 300, 20), (140003, 1200, 8), (16400, 3, 264)])
def test_many_tokens(device, tokens, rows, cols, skew):
    ids, weight, dout = make(device, tokens, rows, cols, torch.bfloat16, torch.bfloat16, tokens, skew=skew)
    check(ids, weight, 0.5, rows // 2 if skew else None, 0, torch.bfloat16, dout)
    check(ids.int(), weight.float(), 1.0, None, 0, torch.float32, dout.float())


@pytest.mark.parametrize("tokens", [127, 9000])
def test_a_single_id(device, tokens):
    """Every token the same, the first row and the last; and every token padding."""
    for row in (0, 36):
        _, weight, dout = make(device, tokens, 37, 96, torch.float32, torch.bfloat16, tokens)
        ids = torch.full((tokens,), row, device=device)
        check(ids, weight, 2.0, None, 0, torch.bfloat16, dout)
        check(ids, weight, 2.0, row, 0, torch.bfloat16, dout)


@pytest.mark.parametrize("tokens", [300, 12000])
def test_vocabulary_shards_add_up(device, tokens):
    ids, weight, dout = make(device, tokens, 1000, 80, torch.float32, torch.float32, 5)
    ids[3], ids[4], ids[5] = -1, 2 ** 40, -2 ** 62  # no shard has these
    whole = ops.embedding_fwd(ids, weight, 3.0)
    assert not whole[3:6].any()
    total = torch.zeros_like(whole)
    grads = []
    for first, last in ((0, 1), (1, 400), (400, 1000)):
        shard = weight[first:last]
        check(ids, shard, 3.0, 7, first, torch.float32, dout)
        total += ops.embedding_fwd(ids, shard, 3.0, first)
        grads.append(ops.embedding_bwd(ids, dout, last - first, 3.0, first, 7))
    assert torch.equal(total, whole)
    assert torch.equal(torch.cat(grads)[1:], ops.embedding_bwd(ids, dout, 1000, 3.0, 0, 7)[1:])


def test_no_tokens_and_no_rows(device):
    weight = torch.randn((9, 16), device=device, requires_grad=True)
    for shape in ((0,), (3, 0)):
        out = scaled_embedding(torch.zeros(shape, dtype=torch.int64, device=device), weight)
        assert out.shape == (*shape, 16)
        (grad,) = torch.autograd.grad(out.sum(), weight)
        assert not grad.any()
    none = torch.empty((0, 16), device=device, requires_grad=True)
    out = scaled_embedding(torch.arange(4, device=device), none)
    assert out.shape == (4, 16) and not out.any()
    assert torch.autograd.grad(out.sum(), none)[0].shape == (0, 16)


def test_strides_and_alignment(device):
    """Tables and gradients that are parts of wider ones, start at any element, or are expanded or transposed."""
    g = torch.Generator(device=device).manual_seed(1)
    for dtype in (torch.bfloat16, torch.float32):
        wide = torch.randn((50, 131), generator=g, device=device).to(dtype)
        ids = torch.randint(0, 50, (6, 4), generator=g, device=device)
        dwide = torch.randn((24, 140), generator=g, device=device).to(dtype)
        for lo, cols in ((0, 128), (1, 128), (3, 127), (5, 1)):
            weight = wide[:, lo:lo + cols]
            dout = dwide[:, lo:lo + cols].unflatten(0, (6, 4))
            assert not dout.is_contiguous()
            check(ids, weight, 1.5, None, 0, dtype, dout)
            check(ids.t(), weight, 1.5, None, 0, dtype, dout.transpose(0, 1))
        check(ids, wide.t()[:50, :40], 1.0, None, 0, dtype, dwide[:1, :40].expand(24, 40).unflatten(0, (6, 4)))
        check(ids, wide[:1].expand(50, 131), 1.0, None, 0, dtype, dwide[:, :131].unflatten(0, (6, 4)))


def test_values_that_are_not_finite(device):
    inf, nan = float("inf"), float("nan")
    weight = torch.tensor([[inf, 1.0], [nan, -inf], [-0.0, 3e38]], device=device)
    ids = torch.tensor([0, 1, 2, 5], device=device)
    out = ops.embedding_fwd(ids, weight, 2.0)
    assert out.tolist()[0] == [inf, 2.0] and out[1, 0].isnan() and out[1, 1] == -inf and out[2, 1] == inf
    assert not out[3].any()
    dout = torch.tensor([[inf, 1.0], [nan, 1.0], [1.0, nan], [nan, inf]], device=device)
    grad = ops.embedding_bwd(ids, dout, 3, 1.0, 0, 1)  # nan only where a counted token of the row has one
    assert grad[0].tolist() == [inf, 1.0] and not grad[1].any() and grad[2, 0] == 1 and grad[2, 1].isnan()


def test_gradient_accumulates_into_a_tied_weight(device):
    cfg = Embedding.Config(padding_idx=2, scale=4.0)
    module = cfg.build(num_embeddings=31, embedding_dim=48).to(device)
    module.init_weights()
    ids = torch.randint(0, 31, (3, 5), device=device)
    out = module(ids)
    logits = out @ module.weight.t()
    logits.square().sum().backward()
    w = module.weight.detach().double().requires_grad_(True)
    rows = w[ids] * 4.0
    rows = torch.where((ids == 2)[..., None], rows.detach(), rows)
    (rows @ w.t()).square().sum().backward()
    # (a product of 48 terms in float32 on either side, squares of up to 2^10, 15 tokens)
    assert (module.weight.grad.double() - w.grad).abs().max() <= 1e-4 * w.grad.abs().max()


def test_a_side_stream_and_a_captured_graph(device):
    ids, weight, dout = make(device, 9001, 400, 264, torch.bfloat16, torch.bfloat16, 3, skew=True)
    want = ops.embedding_fwd(ids, weight, 2.0), ops.embedding_bwd(ids, dout, 400, 2.0, 0, 5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.embedding_fwd(ids, weight, 2.0), ops.embedding_bwd(ids, dout, 400, 2.0, 0, 5)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grad = ops.embedding_fwd(ids, weight, 2.0), ops.embedding_bwd(ids, dout, 400, 2.0, 0, 5)
    for seed in range(4):
        new_ids, new_weight, new_dout = make(device, 9001, 400, 264, torch.bfloat16, torch.bfloat16, seed, skew=seed % 2 == 0)
        ids.copy_(new_ids), weight.copy_(new_weight), dout.copy_(new_dout)
        graph.replay()
        want = ops.embedding_fwd(ids, weight, 2.0), ops.embedding_bwd(ids, dout, 400, 2.0, 0, 5)
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(grad, want[1])


def test_refusals(device):
    weight = torch.randn((4, 8), device=device)
    ids = torch.zeros(3, dtype=torch.int64, device=device)
    with pytest.raises(TypeError):
        ops.embedding_fwd(ids.float(), weight)
    with pytest.raises(TypeError):
        ops.embedding_fwd(ids, weight.half())
    with pytest.raises(TypeError):
        ops.embedding_fwd(ids, weight, dtype=torch.float16)
    with pytest.raises(ValueError):
        ops.embedding_fwd(ids.cpu(), weight)
    with pytest.raises(ValueError):
        ops.embedding_bwd(ids, torch.zeros((2, 8), device=device), 4)
    out = scaled_embedding(ids, weight.requires_grad_(True))
    (grad,) = torch.autograd.grad(out.sum(), weight, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


@pytest.mark.parametrize("tokens", [100, 8191, 8200, 33000, 90000])
@pytest.mark.parametrize("cols", [5, 136, 2056])
def test_runs_of_every_length(device, tokens, cols):
    """Ids repeated 1 to 700 times, in any order: runs that begin and end anywhere in the pieces that are summed by one
    workgroup, several long ones next to each other."""
    if tokens * cols > 2 ** 26:
        tokens = 2 ** 26 // cols
    g = torch.Generator(device=device).manual_seed(tokens)
    lengths = torch.randint(1, 20, (tokens,), generator=g, device=device)
    lengths[::7] = 64
    lengths[1::29] = torch.randint(100, 700, lengths[1::29].shape, generator=g, device=device)
    ids = torch.arange(tokens, device=device).repeat_interleave(lengths)[:tokens] * 3
    rows = int(ids.max()) + 5
    ids = ids[torch.randperm(tokens, generator=g, device=device)]
    weight = torch.randn((rows, cols), generator=g, device=device)
    dout = torch.randn((tokens, cols), generator=g, device=device).to(torch.bfloat16)
    check(ids, weight, 1.0, None, 0, torch.bfloat16, dout)
    check(ids, weight[: rows // 2], 1.0, int(ids[0]), 0, torch.bfloat16, dout)  # half of the tokens have no row


@pytest.mark.parametrize("rows", [511, 512, 300000, 2 ** 18 - 1, 2 ** 18])
def test_tables_around_a_digit_of_the_sort(device, rows):
    ids, weight, dout = make(device, 10007, rows, 8, torch.bfloat16, torch.bfloat16, rows)
    ids[:3] = torch.tensor([0, rows - 1, rows], device=device)
    check(ids, weight, 1.0, None, 0, torch.bfloat16, dout)


@pytest.mark.parametrize("cols", [5, 63, 64, 65, 128, 200, 256, 257, 300, 511, 512, 513, 1024, 1030])
@pytest.mark.parametrize("w_type,o_type", TYPES)
def test_forward_of_every_width(device, cols, w_type, o_type):
    """Every result is one product in float32 and its rounding: equal bits.  The table's rows are apart, ids lie on both sides of it."""
    g = torch.Generator(device=device).manual_seed(cols)
    weight = torch.randn((40, cols + 3), generator=g, device=device).to(w_type)[:, 1:cols + 1]
    for n in (1, 3, 515):
        ids = torch.randint(95, 145, (n,), generator=g, device=device)
        out = scaled_embedding(ids, weight, 1.7, first_row=100, dtype=o_type)
        row = ids - 100
        inside = (row >= 0) & (row < 40)
        want = torch.where(inside[:, None], weight.float()[row.clamp(0, 39)] * torch.tensor(1.7, device=device), 0.0).to(o_type)
        assert torch.equal(out, want)
