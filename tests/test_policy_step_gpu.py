"""GPU: a policy step from logits to weights, every stage against 64 bits; what the losses write with offsets that are none."""
import ctypes

import pytest
import torch

from tests.sequence_losses import tokens_of
from tests.test_optimizers_cpu import step64, step_bounds
from torchtitan_amd import _lib, ops
from torchtitan_amd.gradients import get_total_norm
from torchtitan_amd.optimizers import AdamW
from torchtitan_amd.rl import policy_loss, token_log_probs

pytestmark = pytest.mark.gpu


def test_gradient_and_update_of_a_policy_step(device):
    """Log-probabilities, loss, gradient of the weights, its norm and the clipped update with 8-bit moments, three times."""
    torch.manual_seed(7)
    vocab, dim, tokens = 1003, 64, 700
    hidden = torch.randn(tokens, dim, device=device).bfloat16()
    target = torch.randint(0, vocab, (tokens,), device=device)
    weight = torch.nn.Parameter((torch.randn(vocab, dim, device=device) * 0.05).bfloat16())
    bounds, advantages = [0, 100, 100, 350, 690], [1.0, 2.0, -1.0, 0.5]
    hyper = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8)
    opt = AdamW([weight], **hyper, weight_decay=0.05, state_bits=8, master_weights=True, seed=2)
    with torch.no_grad():
        old = token_log_probs(hidden @ weight.t(), target)
    zero = torch.zeros(vocab, dim, device=device)
    m, v = zero, zero
    for step in range(1, 4):
        logits = (hidden @ weight.t()).detach()
        lp = token_log_probs(hidden @ weight.t(), target)
        loss, _ = policy_loss(lp, torch.tensor(advantages, device=device), old, old, offsets=torch.tensor(bounds, device=device), kl_coef=0.1,
                              average="sequence")
        loss.backward()
        # the loss of these log-probabilities, and their gradient
        lp64 = lp.detach().double().requires_grad_(True)
        terms = []
        for s, A in enumerate(advantages):
            x = (lp64 - old.double())[bounds[s]:bounds[s + 1]]
            if x.numel():
                r = x.exp()
                terms.append((-torch.minimum(r * A, r.clamp(0.8, 1.2) * A) + 0.1 * (torch.exp(-x) - 1 + x)).mean())
        want = torch.stack(terms).mean()
        assert abs(float(loss.detach()) - float(want.detach())) <= 2.0 ** -24 * abs(float(want.detach())) + 1e-12
        (dlp,) = torch.autograd.grad(want, lp64)
        # that of the weights: the logits' gradient is rounded to bf16 (2^-8 of every value), multiplied and added up in float32
        # (tokens + 1 roundings), and rounded to bf16; the softmax in it is off by the log-sum's float32 roundings (1e-5)
        dlogits = dlp[:, None] * (torch.nn.functional.one_hot(target, vocab) - torch.softmax(logits.double(), 1))
        want = dlogits.t().contiguous() @ hidden.double()
        parts = dlogits.t().abs().contiguous() @ hidden.double().abs()
        assert float(want.abs().max()) > 1e-4
        off = (weight.grad.double() - want).abs()
        assert (off <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 1e-5 + (tokens + 1) * 2.0 ** -24) * 1.01 * parts + 1e-30).all()
        # its norm, and the update of the master weights by it
        norm = get_total_norm([weight.grad])
        assert abs(float(norm) - float(weight.grad.double().norm())) <= 1e-5 * float(norm)
        limit = 0.5 * float(norm) if step > 1 else 2.0 * float(norm)
        factor = min(1.0, limit / (float(norm) + 1e-6))
        before = opt.state[weight]["master"].clone() if step > 1 else weight.detach().float()
        args = (before, weight.grad, m, v, step, *hyper.values(), 0.05, factor)
        want, bound = step64(*args), step_bounds(*args)
        opt.step(total_norm=norm, max_norm=limit)
        master = opt.state[weight]["master"]
        assert ((master.double().cpu() - want[0]).abs() <= bound[0]).all()
        assert torch.equal(weight.detach(), master.bfloat16())
        moved = (want[0] - before.double().cpu() * (1 - 1e-2 * 0.05)).abs()
        assert float((moved > 100 * bound[0]).double().mean()) > 0.9  # (an update that did not happen would be seen)
        ((m, v),) = opt.moments(torch.float32)
        for got, w, least in ((m, want[1], 2.0 ** -16), (v, want[2], 2.0 ** -32)):
            size = w.abs().view(-1, 32).amax(1, keepdim=True).expand(-1, 32).reshape(w.shape)
            assert ((got.double().cpu() - w).abs() <= w.abs() / 8 * 1.0001 + size * least).all()
        weight.grad = None


class Guarded:
    """`size` bytes in the middle of a buffer, whose other bytes must stay as they are."""

    def __init__(self, size: int, device):
        self.size, self.buffer = size, torch.full((8192 + size + 8192,), 0xA5, dtype=torch.uint8, device=device)

    @property
    def pointer(self):
        return ctypes.c_void_p(self.buffer.data_ptr() + 8192)

    def untouched(self) -> bool:
        return bool((self.buffer[:8192] == 0xA5).all()) and bool((self.buffer[8192 + self.size:] == 0xA5).all())


def falling(count: int, tokens: int, seed: int):
    """Offsets in no order, some outside of the array."""
    return torch.randint(-tokens, 3 * tokens, (count + 1,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("tokens", [2000, 40000])
@pytest.mark.parametrize("bad", [[0, 1500, 700], [-5, 700, 1 << 40], [1 << 40, -1, 5], [2000, 2000, 0], [1999, 3, 1], falling(64, 2000, 0),
                                 falling(4096, 2000, 1)], ids=["inside", "beyond", "before", "at the end", "down", "64", "4096"])
def test_offsets_that_are_none_write_nothing_outside(device, tokens, bad):
    """Some loss and gradient; the bytes around the gradient, the sums kept for it, the outputs and the workspace stay."""
    lib, sequences = _lib.load(), len(bad) - 1
    case = tokens_of((tokens,), device, offsets=[0, tokens])
    advantages, offsets = torch.ones(sequences, device=device), torch.tensor(bad, device=device)
    lp, dloss = case["log_probs"].detach(), torch.ones((), device=device)
    pointer = lambda t: t.data_ptr()
    shared = dict(log_probs=pointer(lp), ref_log_probs=pointer(case["ref"]), log_probs_f32=1, ref_f32=1, offsets=pointer(offsets),
                  sequences=sequences, tokens=tokens, offsets_i64=1)
    policy = ops.PolicyArgs(**shared, old_log_probs=pointer(case["old"]), old_f32=1, advantages=pointer(advantages), kl=2, ratio_low=0.8,
                            ratio_high=1.2, kl_coef=0.1)
    preference = ops.PreferenceArgs(**shared, kind=0, beta=0.1)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    for args, name, more, each in ((policy, "policy", 5, 2 * sequences + 2), (preference, "preference", sequences, sequences + 1)):
        loss, out, kept, work, grad = (Guarded(size, device) for size in (
            4, 4 * more, 8 * each, lib.mx_sequence_loss_workspace(tokens, sequences), 4 * tokens))
        fwd, bwd = getattr(lib, f"mx_{name}_loss"), getattr(lib, f"mx_{name}_loss_bwd")
        assert fwd(ctypes.byref(args), loss.pointer, out.pointer, kept.pointer, work.pointer, stream) == 0
        assert bwd(ctypes.byref(args), kept.pointer, ctypes.c_void_p(pointer(dloss)), grad.pointer, stream) == 0
        torch.cuda.synchronize()
        for what, guarded in (("loss", loss), ("outputs", out), ("sums", kept), ("workspace", work), ("gradient", grad)):
            assert guarded.untouched(), (name, what)
        assert not (grad.buffer[8192:8192 + 4 * tokens].view(torch.int32) == 0xA5A5A5A5 - (1 << 32)).any()  # (every token has one)
