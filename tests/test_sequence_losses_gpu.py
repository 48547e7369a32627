"""GPU: the policy and preference losses' kernels against 64 bits."""
import math

import pytest
import torch

from tests.sequence_losses import check_policy, check_preference, tokens_of
from tests.test_sequence_losses_cpu import overflowing_terms
from torchtitan_amd import ops
from torchtitan_amd.gradients import get_total_norm
from torchtitan_amd.optimizers import AdamW
from torchtitan_amd.rl import compute_policy_gradient_loss, policy_loss, preference_loss, token_log_probs

pytestmark = pytest.mark.gpu


def cuts(count, tokens, seed=0, behind=0, before=0):
    g = torch.Generator().manual_seed(seed)
    inner = torch.randint(before, tokens - behind + 1, (count - 1,), generator=g).sort().values.tolist()
    return [before, *inner, tokens - behind]


LAYOUTS = {
    "rows": dict(shape=(6, 9)), "one token": dict(shape=(2, 1)), "nothing": dict(shape=(4, 0)), "no sequences": dict(shape=(5,), offsets=[0]),
    "masked": dict(shape=(10, 77), mask=0.6), "all masked": dict(shape=(2, 70), mask=0.0), "long rows": dict(shape=(4, 5003), mask=0.9),
    "whole chunks": dict(shape=(4, 512)), "rows of 64": dict(shape=(40, 64), mask=0.5), "single tokens": dict(shape=(700, 1)),
    "short": dict(shape=(300, 3), mask=0.5), "packed": dict(shape=(5000,), offsets=cuts(14, 5000, 1, 7)),
    "empty ones": dict(shape=(600,), offsets=[0, 0, 0, 64, 64, 128, 128, 300, 512, 512, 513, 577, 600]),
    "many short": dict(shape=(3001,), offsets=cuts(1000, 3001, 2, 100, 50), mask=0.8),
    "one long": dict(shape=(40000,), offsets=[0, 1, 39990], mask=0.99), "many joined": dict(shape=(2600, 130)),
    "behind alone": dict(shape=(1500,), offsets=[0, 3, 5]), "before alone": dict(shape=(1500,), offsets=[1490, 1495, 1500]),
}


@pytest.mark.parametrize("name", LAYOUTS)
@pytest.mark.parametrize("ratio,average", [("token", "token"), ("token", "sequence"), ("sequence", "sequence"), ("sequence", "token")])
def test_policy_loss(device, name, ratio, average):
    layout, kinds = LAYOUTS[name], ("k1", "k2", "k3", "k3_swapped")
    kl = kinds[sum(map(ord, name + ratio + average)) % 4]
    check_policy(policy_loss, tokens_of(device=device, **layout), ratio=ratio, average=average, kl=kl, kl_coef=0.3, entropy_coef=0.1,
                 clip_eps=0.1, clip_eps_high=0.3)
    check_policy(policy_loss, tokens_of(device=device, dtype=torch.bfloat16, old=False, ref=False, **layout), ratio=ratio,
                 average=average)
    if ratio == "token":
        check_policy(policy_loss, tokens_of(device=device, per_token=True, dtype=torch.bfloat16, **layout), average=average)


@pytest.mark.parametrize("name", [n for n, x in LAYOUTS.items() if (x["shape"][0] if "offsets" not in x else len(x["offsets"]) - 1) % 2 == 0])
@pytest.mark.parametrize("kind,smoothing", [("sigmoid", 0.0), ("sigmoid", 0.2), ("hinge", 0.0), ("ipo", 0.0)])
def test_preference_loss(device, name, kind, smoothing):
    for mean, dtype in ((False, torch.float32), (True, torch.bfloat16)):
        check_preference(preference_loss, tokens_of(device=device, dtype=dtype, **LAYOUTS[name]), kind=kind, label_smoothing=smoothing,
                         average_log_probs=mean, beta=0.7)
    check_preference(preference_loss, tokens_of(device=device, ref=False, **LAYOUTS[name]), kind=kind, label_smoothing=smoothing)


@pytest.mark.parametrize("kl", ["k1", "k2", "k3", "k3_swapped"])
@pytest.mark.parametrize("outside", [math.nan, math.inf, -math.inf])
def test_estimators_and_what_masked_places_hold(device, kl, outside):
    case = tokens_of((12, 130), device, mask=0.5, outside=outside, per_token=True)
    check_policy(policy_loss, case, kl=kl, kl_coef=1.0)


def test_other_layouts_types_and_views(device):
    """int32 offsets, strided and shifted views, float16 beside float32, float64 advantages: the same numbers."""
    case = tokens_of((333,), device, offsets=[0, 100, 333])
    args = lambda c: (c["log_probs"], c["advantages"], c["old"], c["ref"])
    want = policy_loss(*args(case), offsets=case["offsets"], kl_coef=0.1)[0]
    assert torch.equal(policy_loss(*args(case), offsets=case["offsets"].int(), kl_coef=0.1)[0], want)
    for step, first in ((2, 0), (1, 3)):
        wide = torch.zeros(step * 333 + first, device=device)
        wide[first::step] = case["log_probs"].detach()
        lp = wide[first::step].requires_grad_(True)
        loss, _ = policy_loss(lp, case["advantages"].double(), case["old"], case["ref"], offsets=case["offsets"], kl_coef=0.1)
        assert torch.equal(loss, want)
        assert torch.equal(torch.autograd.grad(loss, lp)[0], torch.autograd.grad(policy_loss(*args(case), offsets=case["offsets"],
                                                                                             kl_coef=0.1)[0], case["log_probs"])[0])
    check_policy(policy_loss, tokens_of((6, 50), device, dtype=torch.float16))
    half = dict(case, old=case["old"].half())
    check_policy(policy_loss, half)


def test_bad_offsets_stay_inside(device):
    """Offsets that fall or leave the array give some loss, but nothing outside is touched: the gradient's neighbours stay."""
    case = tokens_of((2000,), device, offsets=[0, 700, 2000])
    for bad in ([0, 1500, 700], [-5, 700, 1 << 40], [1 << 40, -1, 5], [2000, 2000, 0], [1999, 3, 1]):
        loss, _ = policy_loss(case["log_probs"], case["advantages"], case["old"], offsets=torch.tensor(bad, device=device))
        grad = torch.autograd.grad(loss, case["log_probs"])[0]
        assert grad.shape == (2000,)
    torch.cuda.synchronize()
    check_policy(policy_loss, case)


def test_without_a_gradient_and_twice(device):
    case = tokens_of((16, 300), device, mask=0.7)
    args = (case["log_probs"], case["advantages"], case["old"], case["ref"])
    loss, metrics = policy_loss(*args, mask=case["mask"], kl_coef=0.1)
    with torch.no_grad():
        again, more = policy_loss(*args, mask=case["mask"], kl_coef=0.1)
    assert torch.equal(loss, again) and torch.equal(metrics, more) and not again.requires_grad
    a = torch.autograd.grad(loss, case["log_probs"], retain_graph=True)[0]
    b = torch.autograd.grad(loss * 1.0, case["log_probs"], retain_graph=True)[0]
    assert torch.equal(a, b)
    (g,) = torch.autograd.grad(loss, case["log_probs"], create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        g.sum().backward()


def test_saved_tensors_that_hooks_replace(device):
    """Packed to the host and back (checkpointing's offload): the same gradient; another type back is an error."""
    case = tokens_of((16, 300), device, mask=0.7)
    call = lambda: policy_loss(case["log_probs"], case["advantages"], case["old"], case["ref"], mask=case["mask"], kl_coef=0.1)[0]
    want = torch.autograd.grad(call(), case["log_probs"])[0]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.to(device)):
        loss = call()
    assert torch.equal(torch.autograd.grad(loss, case["log_probs"])[0], want)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.double()):
        loss = call()
    with pytest.raises(RuntimeError, match="saved tensor"):
        torch.autograd.grad(loss, case["log_probs"])
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t[:3] if t.shape == (16,) else t):  # (too few advantages)
        loss = call()
    with pytest.raises(RuntimeError, match="saved tensor"):
        torch.autograd.grad(loss, case["log_probs"])


def test_streams_and_a_captured_step(device):
    """Forward and backward captured into a graph and replayed on new values, with eager work between the replays."""
    case = tokens_of((64, 700), device, mask=0.7)
    pair = tokens_of((64, 700), device, mask=0.7, seed=3)
    dloss = torch.tensor(0.5, device=device)

    def step():
        loss, metrics = policy_loss(case["log_probs"], case["advantages"], case["old"], case["ref"], mask=case["mask"], kl_coef=0.1)
        other, rewards = preference_loss(pair["log_probs"], pair["ref"], mask=pair["mask"])
        return (loss.detach(), metrics, *torch.autograd.grad(loss, case["log_probs"], dloss), other.detach(), rewards,
                *torch.autograd.grad(other, pair["log_probs"], dloss))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(on_side, step()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        with torch.no_grad():
            for c in (case, pair):
                c["log_probs"].copy_(torch.where(c["mask"], -torch.rand(64, 700, device=device), -math.inf))
            case["advantages"].normal_()
            case["mask"].logical_xor_(torch.zeros((), dtype=torch.bool, device=device))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))


@pytest.mark.parametrize("dynamic", [False, True])
def test_traced_as_nodes_of_the_graph(device, dynamic):
    """Under torch.compile the losses are operators of the graph: the eager bits, without a break."""
    torch._dynamo.reset()
    try:
        for shape in ((8, 40), (6, 50)):
            case = tokens_of(shape, device, mask=0.7)

            def call(lp):
                loss, metrics = policy_loss(lp * 1.0, case["advantages"], case["old"], case["ref"], mask=case["mask"], kl_coef=0.1)
                other, rewards = preference_loss(lp * 1.0, case["ref"], mask=case["mask"], kind="ipo")
                return loss, metrics, other, rewards

            compiled = torch.compile(call, fullgraph=True, backend="aot_eager", dynamic=dynamic)
            got, want = compiled(case["log_probs"]), call(case["log_probs"])
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            a, b = (torch.autograd.grad(x[0] + x[2], case["log_probs"])[0] for x in (got, want))
            assert torch.equal(a, b)
            with torch.no_grad():
                assert torch.equal(compiled(case["log_probs"])[0], want[0])
        packed = tokens_of((300,), device, offsets=[0, 100, 100, 290], dtype=torch.bfloat16)
        call = lambda lp: policy_loss(lp, packed["advantages"].double(), packed["old"].float(), offsets=packed["offsets"])[0]
        got, want = torch.compile(call, fullgraph=True, backend="aot_eager")(packed["log_probs"]), call(packed["log_probs"])
        assert torch.equal(got, want)
        assert torch.equal(*(torch.autograd.grad(x, packed["log_probs"])[0] for x in (got, want)))
    finally:
        torch._dynamo.reset()


def test_under_a_timer_and_in_transforms(device):
    """The launches one by one under a kernel timer give the same bits; function transforms take the formula in torch operations."""
    case, pair = tokens_of((8, 40), device, mask=0.7), tokens_of((8, 40), device, mask=0.7, seed=2, dtype=torch.bfloat16)

    def call():
        loss, metrics = policy_loss(case["log_probs"], case["advantages"], case["old"], case["ref"], mask=case["mask"], kl_coef=0.1)
        other, rewards = preference_loss(pair["log_probs"], pair["ref"], mask=pair["mask"])
        return (loss, metrics, other, rewards, *torch.autograd.grad(loss, case["log_probs"], retain_graph=True),
                *torch.autograd.grad(other, pair["log_probs"], retain_graph=True))

    want, timer = call(), ops.KernelTimer()
    ops.set_kernel_timer(timer)
    try:
        got = call()
        with torch.no_grad():
            assert torch.equal(policy_loss(case["log_probs"], case["advantages"], case["old"], mask=case["mask"])[0].isnan(),
                               torch.tensor(False, device=device))
        (g,) = torch.autograd.grad(got[0], case["log_probs"], create_graph=True)
        with pytest.raises(RuntimeError, match="cannot be differentiated again"):
            g.sum().backward()
    finally:
        ops.set_kernel_timer(None)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert {"policy_loss", "policy_loss_bwd", "preference_loss", "preference_loss_bwd"} <= set(timer.summary())
    grad = torch.func.grad(lambda lp: policy_loss(lp, case["advantages"], case["old"], case["ref"], mask=case["mask"], kl_coef=0.1)[0])(
        case["log_probs"].detach())
    assert torch.allclose(grad, want[4], rtol=1e-6, atol=1e-12)  # (64 bits there too; one rounding)


class _TwoLayers(torch.nn.Module):
    def __init__(self, vocab=1000, dim=32):
        super().__init__()
        self.emb = torch.nn.Embedding(vocab, dim)
        self.out = torch.nn.Linear(dim, vocab, bias=False)

    def forward(self, tokens, attention_masks=None):
        h = self.emb(tokens)
        return self.out(h + h.cumsum(dim=1) * 0.1)


def test_the_sample_loss_runs_through_it(device):
    """compute_policy_gradient_loss over uneven samples: the loss and gradient of the samples one by one."""
    torch.manual_seed(5)
    model = _TwoLayers().to(device).bfloat16()
    rng = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, 1000, (n,), generator=rng).tolist()
    prompts, answers = [ids(n) for n in (5, 9, 3, 7)], [ids(n) for n in (12, 130, 1, 600)]
    advantages = torch.tensor([0.5, -0.2, 1.5, -1.0])
    ref = [torch.randn(len(a), generator=rng).to(device) * 0.1 - 7 for a in answers]
    seen = []
    hook = torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append(t.dtype), t)[1], lambda t: t)
    with hook:
        total, metrics, lps = compute_policy_gradient_loss(model, answers, prompts, advantages, ref)
    assert torch.float64 in seen and type(total.grad_fn).__name__ != "AddBackward0"  # (the one node)
    apart, apart_metrics, _ = compute_policy_gradient_loss(model, answers, prompts, advantages.double(), ref)  # (in torch operations)
    # float32 means there: some hundred roundings of values up to about 10
    assert abs(float(total) - float(apart)) <= 1e-4
    assert all(abs(metrics[k] - apart_metrics[k]) <= 1e-4 for k in metrics)
    total.backward()
    first = model.out.weight.grad.clone()
    model.zero_grad()
    apart.backward()
    # bf16 gradients of bf16 products: two of their roundings apart at most, summed over the samples in float32
    assert float((first.float() - model.out.weight.grad.float()).norm()) <= 2.0 ** -7 * float(first.float().norm())


def test_terms_without_a_coefficient_are_left_out(device):
    overflowing_terms(device)


def test_the_sample_loss_takes_what_it_took(device):
    """Fewer prompts than answers, a negative clipping width and coefficients that are tensors go through torch operations or
    the same tokens, as ever."""
    torch.manual_seed(5)
    model = _TwoLayers().to(device).bfloat16()
    rng = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, 1000, (n,), generator=rng).tolist()
    prompts, answers = [ids(n) for n in (5, 9)], [ids(n) for n in (12, 30)]
    ref = [torch.full((len(a),), -7.0, device=device) for a in answers]
    A = torch.tensor([0.5, -0.2])
    want = compute_policy_gradient_loss(model, answers, prompts, A, ref)[0].item()
    more = compute_policy_gradient_loss(model, answers + [ids(4)], prompts, A, ref)[0].item()
    assert more == want
    assert math.isfinite(compute_policy_gradient_loss(model, answers, prompts, A, ref, ppo_clip_eps=-0.1)[0].item())
    coefficient = torch.tensor(0.1, device=device, requires_grad=True)
    total, metrics, _ = compute_policy_gradient_loss(model, answers, prompts, A, ref, kl_coef=coefficient)
    (g,) = torch.autograd.grad(total, coefficient)
    assert abs(g.item() - metrics["kl_div"]) <= 1e-6 * abs(metrics["kl_div"]) and abs(total.item() - want) <= 1e-4


def test_a_training_step_from_logits_to_weights(device):
    """Log-probabilities, loss, gradient, its norm, the clipped update in 8 bits, twice, against the same step in 64 bits where each
    begins."""
    torch.manual_seed(7)
    vocab, dim, tokens = 1003, 64, 700
    hidden = torch.randn(tokens, dim, device=device).bfloat16()
    target = torch.randint(0, vocab, (tokens,), device=device)
    weight = torch.nn.Parameter((torch.randn(vocab, dim, device=device) * 0.05).bfloat16())
    offsets = torch.tensor([0, 100, 100, 350, 690], device=device)
    advantages = torch.tensor([1.0, 2.0, -1.0, 0.5], device=device)
    opt = AdamW([weight], lr=1e-2, state_bits=8, master_weights=True, seed=2)
    with torch.no_grad():
        old = token_log_probs(hidden @ weight.t(), target)
    for step in range(2):
        lp = token_log_probs(hidden @ weight.t(), target)
        loss, metrics = policy_loss(lp, advantages, old, old, offsets=offsets, kl_coef=0.1, average="sequence")
        loss.backward()
        norm = get_total_norm([weight.grad])
        before = opt.state[weight]["master"].clone() if step else weight.detach().float()
        assert torch.isfinite(norm) and float(norm) > 0
        # a first step's update is lr times the gradient's sign, whatever its size; afterwards at most a few lr
        opt.step(total_norm=norm, max_norm=0.1)
        moved = (opt.state[weight]["master"] - before * (1 - 1e-2 * 1e-2)).abs()
        assert float(moved.max()) <= 1e-2 * 1.0001 * (1 if step == 0 else 4)
        assert torch.equal(weight.detach(), opt.state[weight]["master"].bfloat16())
        lp64 = lp.detach().double().requires_grad_(True)
        # the gradient with respect to the log-probabilities, again from the formula
        r = torch.exp(lp64 - old.double())
        terms = []
        for s in (0, 2, 3):
            i = slice(int(offsets[s]), int(offsets[s + 1]))
            x = lp64[i] - old.double()[i]
            terms.append((-torch.minimum(r[i] * advantages[s], r[i].clamp(0.8, 1.2) * advantages[s]) + 0.1 * (torch.exp(-x) - 1 + x)).mean())
        want = torch.stack(terms).mean()
        assert abs(float(loss) - float(want)) <= 1e-6 * max(1.0, abs(float(want)))
        weight.grad = None


def test_a_policy_step_of_a_converted_model(device):
    """Linears in MXFP8, the sample loss, the gradients' norm, an update with 8-bit moments that clips as it reads, and the hand-over: the
    casts that were kept are made anew from the updated weights."""
    from torchtitan_amd.modules import Linear
    from torchtitan_amd.mx_tensor import MXFP8TrainingWeight
    from torchtitan_amd.protocols import ModelConvertersContainer
    from torchtitan_amd.quantization.mx import MXFP8Converter, export_mxfp8_state_dict

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            linear = lambda k, n: Linear.Config().build(in_features=k, out_features=n)
            self.emb = torch.nn.Embedding(512, 128)
            self.up, self.down, self.out = linear(128, 256), linear(256, 128), linear(128, 512)

        def forward(self, tokens, attention_masks=None):
            h = self.emb(tokens)
            return self.out(h + self.down(torch.nn.functional.silu(self.up(h))))

    torch.manual_seed(0)
    model = Model().to(device).bfloat16()
    box = ModelConvertersContainer.Config(converters=[MXFP8Converter.Config(fqns=["up", "down"], cache_weight_casts=True)]).build(
        parallel_dims=None, model_compile_enabled=False)
    box.convert(model)
    opt = AdamW(model.parameters(), lr=1e-2, state_bits=8, master_weights=True)
    rng = torch.Generator().manual_seed(1)
    ids = lambda n: torch.randint(0, 512, (n,), generator=rng).tolist()
    prompts, answers = [ids(n) for n in (5, 9)], [ids(n) for n in (27, 55)]
    ref = [torch.full((len(a),), -6.0, device=device) for a in answers]
    for step in range(2):
        total, metrics, _ = compute_policy_gradient_loss(model, answers, prompts, torch.tensor([1.0, -0.5]), ref)
        total.backward()
        before = {n: p.detach().as_subclass(torch.Tensor).clone() for n, p in model.named_parameters()}
        norm = get_total_norm([p.grad for p in model.parameters()])
        opt.step(total_norm=norm, max_norm=1.0)
        box.post_optimizer_hook(model)
        payload = export_mxfp8_state_dict(model)
        converted = 0
        for name, p in model.named_parameters():
            plain = p.detach().as_subclass(torch.Tensor)
            assert torch.isfinite(plain).all() and not torch.equal(plain, before[name])
            assert torch.equal(plain, opt.state[p]["master"].bfloat16())
            if isinstance(p, MXFP8TrainingWeight):
                converted += 1
                assert torch.equal(payload[name]["codes"], ops.to_mx_dim0(plain, "rceil").codes)
        assert converted == 2
        opt.zero_grad()


def test_the_launches_are_the_librarys(device):
    case = tokens_of((4, 4), device)
    loss, _ = policy_loss(case["log_probs"], case["advantages"])
    assert "LossNode" in type(loss.grad_fn).__name__ or "LossNode" in loss.grad_fn.name()
    assert ops.native_rows(case["log_probs"])


def test_more_tokens_than_31_bits_count(device):
    """Two sequences on either side of place 2^31 and one behind it: constant log-ratios, the loss in closed form."""
    tokens = (1 << 31) + 70001
    offsets = torch.tensor([5, (1 << 31) - 3, (1 << 31) + 1000, tokens - 7], device=device)
    lp = torch.full((tokens,), -1.0, dtype=torch.bfloat16, device=device).requires_grad_(True)
    old = torch.full((tokens,), -1.125, dtype=torch.bfloat16, device=device)
    advantages = torch.tensor([1.0, -2.0, 3.0], device=device)
    loss, metrics = policy_loss(lp, advantages, old, offsets=offsets, average="sequence", clip_eps=0.2)
    r = math.exp(0.125)
    assert abs(loss.item() + r * 2.0 / 3) <= 1e-6 and abs(metrics[3].item() - r) <= 1e-6
    (grad,) = torch.autograd.grad(loss, lp)
    ends = offsets.tolist()
    for s, A in enumerate(advantages.tolist()):
        want, n = -A * r / 3, ends[s + 1] - ends[s]
        for i in (ends[s], ends[s + 1] - 1):
            assert abs(grad[i].item() * n - want) <= abs(want) * 2.0 ** -8
    assert not grad[:5].any() and not grad[-7:].any()
