"""AdamW over all parameters of a model in a few launches, with moments in float32 or in 8 bits.

Counterpart of the optimizer that the reference's container builds (torchtitan/components/optimizer.py), with torch's own
signature.  bf16 and float32 parameters on a GPU, converted weights among them, run as HIP kernels; everything else runs
the same formula in torch operations.  The gradients' clipping (``gradients.py``) can be applied as they are read.
"""
from __future__ import annotations

import math

import torch

from . import _lib, ops
from .mx_tensor import MXFP8TrainingWeight, _capture, _unwrap

_TYPES = (torch.Tensor, torch.nn.Parameter, MXFP8TrainingWeight)
_MOMENTS = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_scale", "exp_avg_sq", "exp_avg_sq_scale")}


# ------------------------------------------------------------------------------ moments in 8 bits, in torch operations
# (exponent bias, largest code, its exponent, what carries a float32's mantissa above the largest code's, has a sign): the
# first moment in e4m3, the second in e5m3 without a sign; blocks of 32 values with an E8M0 scale.
_FIRST, _SECOND = (7, 0x7E, 8, 0x1FFFFF, True), (15, 0xFF, 16, 0x0FFFFF, False)


def _mixed(x):
    x = ((x ^ (x >> 16)) * 0x6A09E667) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0xBB67AE85) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_bits(n: int, seed: int, step: int, number: int, device) -> torch.Tensor:
    """16 random bits for each of n values, the kernel's."""
    key = 0
    for word in (seed & 0xFFFFFFFF, seed >> 32, step, number):
        key = _mixed((key + word + 0x9E3779B9) & 0xFFFFFFFF)
    pair = torch.arange(-(-n // 2), dtype=torch.int64, device=device)
    bits = _mixed((pair * 0x9E3779B9 + key) & 0xFFFFFFFF)
    return torch.stack((bits & 0xFFFF, bits >> 16), 1).reshape(-1)[:n]


def _blocks(x: torch.Tensor) -> torch.Tensor:
    x = x.reshape(-1)
    return torch.nn.functional.pad(x, (0, -x.numel() % ops.BLOCK)).view(-1, ops.BLOCK)


def _encode(x: torch.Tensor, form, random: torch.Tensor):
    """(codes [blocks, 32], scales [blocks]) of float32 values."""
    bias, most, top, up, signed = form
    x, random = _blocks(x), _blocks(random)
    bits = x.abs().view(torch.int32).long()
    amax = bits.amax(1) if bits.shape[0] else bits.new_zeros(0)
    scale = torch.where(amax > 0, ((amax + up) >> 23) - top, 0).clamp(0, 254)
    scale = torch.where(amax >= 0x7F800000, 255, scale)
    size = torch.ldexp(x.abs().double(), (bias - scale).double()[:, None]).float().view(torch.int32).long()
    code = torch.where(x == 0, 0, ((size + (random << 4) + 8) >> 20).clamp(max=most))
    if not signed:
        code = torch.where(x > 0, code.clamp(min=1), code)
    code = torch.where(scale[:, None] == 255, most, code)
    if signed:
        code = code | (x.signbit().long() << 7)
    return code.to(torch.uint8), scale.to(torch.uint8)


def _decode(codes: torch.Tensor, scales: torch.Tensor, form, n: int) -> torch.Tensor:
    """The n float32 values of codes."""
    bias, _, _, _, signed = form
    code, scale = codes.long(), scales.long()
    size = ((code & 127 if signed else code) << 20).to(torch.int32).view(torch.float32)
    value = torch.ldexp(size.double(), (scale - bias).double()[:, None]).float()
    value = torch.where(scale[:, None] == 255, math.nan, value)
    return (torch.where(code >= 128, -value, value) if signed else value).reshape(-1)[:n]


def _in_torch_ops(p, g, state, group, norm, limit, step, number):
    (b1, b2), lr, eps = group["betas"], float(group["lr"]), group["eps"]
    wide = torch.promote_types(p.dtype, torch.float32)
    g = g.to(wide)
    if norm is not None:
        g = g * (limit / (norm.to(g.device, torch.float32) + 1e-6)).clamp(max=1.0)
    if group["maximize"]:
        g = -g
    if group["state_bits"] == 8:
        m = _decode(state["exp_avg"], state["exp_avg_scale"], _FIRST, p.numel()).view(p.shape)
        v = _decode(state["exp_avg_sq"], state["exp_avg_sq_scale"], _SECOND, p.numel()).view(p.shape)
    else:
        m, v = state["exp_avg"], state["exp_avg_sq"]
    m_new, v_new = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
    below = v_new.sqrt() * (1 / math.sqrt(1 - b2 ** step)) + eps
    w = state.get("master", p)
    new = w.to(wide) * (1 - lr * group["weight_decay"]) - (m_new / below) * (lr / (1 - b1 ** step))
    if w is not p:
        w.copy_(new)
    p.copy_(new)
    if group["state_bits"] == 8:
        random = _random_bits(p.numel(), group["seed"], step, number, p.device)
        for name, x, form in (("exp_avg", m_new, _FIRST), ("exp_avg_sq", v_new, _SECOND)):
            codes, scales = _encode(x, form, random)
            state[name].copy_(codes)
            state[name + "_scale"].copy_(scales)
    else:
        m.copy_(m_new)
        v.copy_(v_new)


def _kernel_takes(p: torch.Tensor) -> bool:
    return (type(p) in _TYPES and p.is_cuda and p.dtype in ops.ROW_TYPES and p.layout == torch.strided and not p.is_neg()
            and ops.is_dense(p))


def _check_numbers(group) -> None:
    lr, betas, eps, weight_decay = (group[name] for name in ("lr", "betas", "eps", "weight_decay"))
    if isinstance(lr, torch.Tensor) and lr.numel() != 1:
        raise ValueError("a tensor lr must have one element")
    if not float(lr) >= 0:
        raise ValueError(f"lr must not be negative, got {lr}")
    if not all(0 <= b < 1 for b in betas):
        raise ValueError(f"betas must be in [0, 1), got {betas}")
    if not eps >= 0 or not weight_decay >= 0:
        raise ValueError(f"eps and weight_decay must not be negative, got {eps} and {weight_decay}")
    if group["state_bits"] not in _MOMENTS:
        raise ValueError(f"state_bits must be 32 or 8, got {group['state_bits']}")
    if not 0 <= group["seed"] < 1 << 64:
        raise ValueError("seed must fit 64 bits without a sign")


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` (without its amsgrad, foreach, fused and differentiable) with moments in `state_bits` bits whatever the
    parameters' type.

        g = f * gradient               (its sign turned with `maximize`)
        m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
        p = (1 - lr * weight_decay) p - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

    in float32, p rounded once to its type.  `master_weights`: parameters narrower than float32 keep a float32 weight in
    their state, which the step updates; the parameter is its rounding (a value that is written into the parameter from outside
    wants a new state).

    ``state_bits=8``: the first moment is held in e4m3, the second in e5m3 without a sign, 32 values in the order of memory with a
    power of two between them (``exp_avg`` uint8 [blocks, 32] and ``exp_avg_scale`` [blocks]; likewise ``exp_avg_sq``), rounded
    up or down by chance so that their mean is the exact one; `seed` decides about that chance, the same seed gives the same
    bits.  A block whose gradients hold an infinity or a NaN becomes NaN.  Such parameters must be contiguous.  (On the GPU, with
    eps of 1e-9 or more, the root of such an update is within an ulp and the quotient within two, else rounded right as all others;
    whatever else is in the list, a value has the same bits, but for its parameter's number there, by which the chance goes too.)

    ``step(total_norm=..., max_norm=...)`` scales the gradients by min(1, max_norm / (total_norm + 1e-6)) as they are read:
    ``clip_grads_with_norm_`` without its pass over memory (the gradients stay as they are, and of bf16 ones no scaled rounding).

    Gradients are read in float32 (float32 ones of bf16 parameters as they are).

    With `capturable` the step counters are on the device and `lr` may be a float32 tensor there: a step can be captured into a
    graph once a step has run outside of one.  A graph goes on with the tensors that it was captured with: a state that is loaded
    afterwards wants a new one."""

    def __init__(self, params, lr: float | torch.Tensor = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, state_bits: int = 32, master_weights: bool = False, maximize: bool = False,
                 capturable: bool = False, seed: int = 0):
        self._counters = {}  # group -> (float32 step counters by the parameters' numbers, what follows from them)
        defaults = dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                        master_weights=master_weights, maximize=maximize, capturable=capturable, seed=seed)
        _check_numbers(defaults)
        super().__init__(params, defaults)

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        try:
            group = self.param_groups[-1]
            _check_numbers(group)
            if len(set(group["params"])) != len(group["params"]):
                raise ValueError("a parameter is listed twice")
        except Exception:
            self.param_groups.pop()
            raise

    def __setstate__(self, state):
        super().__setstate__(state)
        self._counters = {}

    # -------------------------------------------------------------------------------- state
    def _new_state(self, p: torch.Tensor, group) -> None:
        if p.is_cuda and type(p) in _TYPES and _capture(p):
            raise RuntimeError("AdamW: the state of a parameter is made by its first step, which cannot be captured into a "
                               "graph: run one step outside")
        plain, state = _unwrap(p.detach()), {}
        if plain.is_complex():
            raise TypeError(f"AdamW: complex parameters are not supported, got {p.dtype}")
        wide = torch.promote_types(p.dtype, torch.float32)
        if group["state_bits"] == 8:
            if hasattr(type(p), "__tensor_flatten__") or not p.is_contiguous() or wide != torch.float32:
                raise ValueError(f"AdamW: moments in 8 bits want plain contiguous parameters of up to 32 bits, got "
                                 f"{type(p).__name__} {p.dtype} {tuple(p.shape)} with strides {p.stride()}")
            blocks = -(-p.numel() // ops.BLOCK)
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros((blocks, ops.BLOCK), dtype=torch.uint8, device=p.device)
                state[name + "_scale"] = torch.zeros(blocks, dtype=torch.uint8, device=p.device)
        else:
            for name in ("exp_avg", "exp_avg_sq"):
                state[name] = torch.zeros_like(plain, dtype=wide, memory_format=torch.preserve_format)
        if group["master_weights"] and p.dtype != wide:
            state["master"] = plain.to(wide, copy=True)
        state["step"] = 0
        self.state[p] = state

    def load_state_dict(self, state_dict) -> None:
        """As torch's, but moments keep their own types, and `state_bits`, `master_weights` and `capturable` stay this
        optimizer's: a state that ``torch.optim.AdamW`` or this optimizer with others of them has saved is converted.  Hooks in front of
        the loading give the state that is converted, those behind it see the converted one."""
        held = [{key: group[key] for key in ("state_bits", "master_weights", "capturable")} for group in self.param_groups]
        saved, ids, before = {}, [], (self.state, self.param_groups, self._counters)

        def take(_, hooked):
            if any(group.get("amsgrad") for group in hooked["param_groups"]):
                raise ValueError("AdamW: a state with amsgrad cannot be gone on with here")
            # (torch would round the moments to their parameters' types)
            ids.extend(i for group in hooked["param_groups"] for i in group["params"])
            parameters = set(ids)
            saved.update(hooked["state"])
            return {**hooked, "state": {i: one for i, one in saved.items() if i not in parameters}}

        def convert(_):
            self._counters = {}
            for group, own in zip(self.param_groups, held):
                group.update(own)
                for key, value in self.defaults.items():
                    group.setdefault(key, value)
            number = -1
            try:
                for group in self.param_groups:
                    for p in group["params"]:
                        number += 1
                        if saved.get(ids[number]):
                            self._load_one(p, group, saved[ids[number]], number)
            except Exception:  # (a state that does not fit is not loaded by half)
                self.state, self.param_groups, self._counters = before
                raise

        # behind the caller's hooks in front of it, before those behind it
        own_hooks = (self.register_load_state_dict_pre_hook(take), self.register_load_state_dict_post_hook(convert, prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in own_hooks:
                hook.remove()

    @torch.no_grad()
    def _load_one(self, p, group, saved, number: int) -> None:
        self._new_state(p, group)
        state = self.state[p]
        state["step"] = int(saved["step"])
        wide = torch.promote_types(p.dtype, torch.float32)
        eight = saved["exp_avg"].dtype == torch.uint8
        if eight and group["state_bits"] == 8:
            moves = {name: saved[name] for name in _MOMENTS[8]}
        elif eight:
            blocks = -(-p.numel() // ops.BLOCK)
            if any(saved[name].shape[0] != blocks for name in _MOMENTS[8]):
                raise ValueError(f"AdamW: a saved exp_avg has shape {tuple(saved['exp_avg'].shape)}, its parameter {tuple(p.shape)}")
            moves = {name: _decode(saved[name].to(p.device), saved[name + "_scale"].to(p.device), form, p.numel()).view(p.shape)
                     for name, form in (("exp_avg", _FIRST), ("exp_avg_sq", _SECOND))}
        elif group["state_bits"] == 8:
            moves, random = {}, _random_bits(p.numel(), group["seed"], state["step"], number, p.device)
            for name, form in (("exp_avg", _FIRST), ("exp_avg_sq", _SECOND)):
                values = saved[name].to(p.device, torch.float32)
                if values.shape != p.shape:
                    raise ValueError(f"AdamW: a saved {name} has shape {tuple(values.shape)}, its parameter {tuple(p.shape)}")
                moves[name], moves[name + "_scale"] = _encode(values, form, random)
        else:
            moves = {name: saved[name] for name in _MOMENTS[32]}
        if "master" in state and "master" in saved:
            moves["master"] = saved["master"]
        for name, value in moves.items():
            if value.shape != state[name].shape:
                raise ValueError(f"AdamW: a saved {name} has shape {tuple(value.shape)}, expected {tuple(state[name].shape)}")
            state[name].copy_(value.to(state[name].dtype) if state[name].dtype == wide else value)

    def _counter(self, index: int, first: int):
        """The device's step counters of a group whose parameters have the numbers from `first` on, and their corrections; the
        states' steps are its elements."""
        group = self.param_groups[index]
        device = next((p.device for p in group["params"] if p.is_cuda), None)
        if device is None:
            raise RuntimeError("AdamW: capturable wants parameters on a GPU")
        steps, corrections = self._counters.get(index) or (None, None)
        here = [(first + i, self.state[p]) for i, p in enumerate(group["params"]) if self.state.get(p)]
        if steps is None or any(not isinstance(s["step"], torch.Tensor) or s["step"].data_ptr() != steps.data_ptr() + 4 * i
                                for i, s in here):
            if _capture(torch.empty(0, device=device)):
                raise RuntimeError("AdamW: step counters are laid out by a step outside of a capture")
            values = [float(s["step"]) for _, s in here]
            if steps is None or steps.device != device:
                size = first + len(group["params"])
                steps = torch.zeros(size, dtype=torch.float32, device=device)
                corrections = torch.zeros((size, 4), dtype=torch.float32, device=device)
                self._counters[index] = (steps, corrections)
            for value, (i, state) in zip(values, here):
                steps[i] = value
                state["step"] = steps[i]
        return steps, corrections

    # -------------------------------------------------------------------------------- step
    def step(self, closure=None, *, total_norm: torch.Tensor | None = None, max_norm: float | None = None):
        """One update of every parameter with a gradient; the closure's value, if there is one."""
        if (total_norm is None) != (max_norm is None):
            raise ValueError("total_norm and max_norm come together")
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        first = 0
        with torch.no_grad():
            for index, group in enumerate(self.param_groups):
                self._step_group(index, group, first, total_norm, 0.0 if max_norm is None else float(max_norm))
                first += len(group["params"])
        return loss

    def _step_group(self, index: int, group, first: int, norm, limit: float) -> None:
        params = group["params"]
        if not group["capturable"] and all(type(p) in _TYPES for p in params) and params and ops.native_rows(_unwrap(params[0])):
            states = [self.state.get(p) for p in params]
            b1, b2 = group["betas"]
            if _lib.blocks().adamw(params, states, first, group["state_bits"] == 8, float(group["lr"]), b1, b2, group["eps"],
                                   group["weight_decay"], group["maximize"], norm, limit, group["seed"]):
                return
        with_grad = [(first + i, p) for i, p in enumerate(params) if p.grad is not None]
        for _, p in with_grad:
            if p.grad.is_sparse:
                raise RuntimeError("AdamW: sparse gradients are not supported")
            if not self.state.get(p):
                self._new_state(p, group)
        if norm is not None:
            norm = (norm.full_tensor() if hasattr(norm, "full_tensor") else norm).detach().reshape(())
        work = [_Work(number, p, self.state[p]) for number, p in with_grad]
        if group["capturable"] and work:
            if not all(w.kernel and w.p.device == work[0].p.device for w in work):
                raise RuntimeError("AdamW: capturable wants bf16 or float32 parameters on one GPU")
            self._launch(work, group, norm, limit, *self._counter(index, first))
            return
        if any(_capture(w.p) for w in work):
            raise RuntimeError("AdamW: a step that is captured into a graph wants capturable=True")
        by_device: dict = {}
        for w in work:
            if w.kernel:
                by_device.setdefault(w.p.device, []).append(w)
                continue
            step = int(w.state["step"]) + 1
            _in_torch_ops(w.p, w.g, w.held, group, norm, limit, step, w.number)
            w.state["step"] = step
        for some in by_device.values():
            self._launch(some, group, norm, limit)

    def _launch(self, work, group, norm, limit: float, counters=None, corrections=None) -> None:
        eight = group["state_bits"] == 8
        operands = []
        for w in work:
            p, g = w.p, w.g
            if g.device != p.device or g.shape != p.shape:
                raise ValueError(f"AdamW: a gradient of shape {tuple(g.shape)} on {g.device} for a parameter of {tuple(p.shape)} on {p.device}")
            kept = p.dtype if g.dtype == p.dtype else torch.float32  # (wider gradients keep float32's bits)
            if g.dtype != kept or g.is_neg() or type(g) is not torch.Tensor or not _same_order(g, p):
                g = torch.empty_like(p, dtype=kept).copy_(g)
            moments = [w.held[name] for name in _MOMENTS[group["state_bits"]]]
            master = w.held.get("master")
            _check_state(p, moments, master, eight)
            operands.append((p, g, moments, master, 0 if counters is not None else int(w.state["step"]) + 1, w.number))
        on_device = counters is not None and isinstance(group["lr"], torch.Tensor) and group["lr"].is_cuda
        ops.adamw_(operands, eight, 0.0 if on_device else float(group["lr"]), group["betas"], group["eps"], group["weight_decay"],
                   group["maximize"], norm, limit, group["seed"], counters, group["lr"] if on_device else None, corrections)
        if counters is None:  # (a refused step has not been one)
            for w in work:
                w.state["step"] = int(w.state["step"]) + 1

    @torch.no_grad()
    def moments(self, dtype: torch.dtype = torch.bfloat16) -> list:
        """(first moment, second moment) of every parameter in order, None for one without a state.  Moments in 32 bits are the state's own
        tensors; those in 8 bits are written out in `dtype`, bfloat16 or float32, of which the first holds their codes as they
        are (but for values below its range)."""
        if dtype not in ops.ROW_TYPES:
            raise TypeError(f"moments are written in bfloat16 or float32, got {dtype}")
        out, asked = [], []
        for group in self.param_groups:
            params = group["params"]
            if group["state_bits"] == 8 and params and all(type(p) in _TYPES for p in params) and ops.native_rows(_unwrap(params[0])):
                pairs = _lib.blocks().adamw_moments(params, [self.state.get(p) for p in params], dtype == torch.float32)
                if pairs is not None:
                    out += pairs
                    continue
            for p in params:
                state = self.state.get(p)
                if not state:
                    out.append(None)
                elif group["state_bits"] == 32:
                    out.append((state["exp_avg"], state["exp_avg_sq"]))
                else:
                    pair = tuple(torch.empty(p.shape, dtype=dtype, device=p.device) for _ in range(2))
                    if p.is_cuda:
                        for second, (name, t) in enumerate(zip(("exp_avg", "exp_avg_sq"), pair)):
                            asked.append((state[name], state[name + "_scale"], second, t))
                    else:
                        for name, form, t in zip(("exp_avg", "exp_avg_sq"), (_FIRST, _SECOND), pair):
                            t.copy_(_decode(state[name], state[name + "_scale"], form, p.numel()).view(p.shape))
                    out.append(pair)
        for device in {t.device for *_, t in asked}:
            ops.adamw_moments([a for a in asked if a[3].device == device])
        return out


def _local(t: torch.Tensor) -> torch.Tensor:
    """A plain tensor: of a converted weight its values, of a distributed tensor this rank's shard."""
    t = _unwrap(t)
    return t.to_local() if hasattr(t, "to_local") else t


class _Work:
    """What a step reads and writes of one parameter: plain tensors (every value is updated by itself, so that a distributed
    parameter is updated shard by shard)."""

    __slots__ = ("number", "p", "g", "held", "state", "kernel")

    def __init__(self, number: int, p: torch.Tensor, state: dict):
        g = p.grad
        if hasattr(p, "placements") and hasattr(g, "placements") and g.placements != p.placements:
            g = g.redistribute(placements=p.placements)
        self.number, self.p, self.g, self.state = number, _local(p.detach()), _local(g), state
        self.held = {name: _local(t) for name, t in state.items() if name != "step"}
        self.kernel = _kernel_takes(self.p)


def _same_order(t: torch.Tensor, p: torch.Tensor) -> bool:
    """t's elements lie in memory as p's do."""
    return (t.is_contiguous() and p.is_contiguous()) or (t.shape == p.shape and t.stride() == p.stride())


def _check_state(p, moments, master, eight: bool) -> None:
    blocks = -(-p.numel() // ops.BLOCK)
    want = [(blocks * ops.BLOCK, torch.uint8), (blocks, torch.uint8)] * 2 if eight else [(p.numel(), torch.float32)] * 2
    want.append((p.numel(), torch.float32))
    for t, (n, dtype) in zip((*moments, master), want):
        if t is None:
            continue
        fits = t.is_contiguous() if dtype == torch.uint8 else _same_order(t, p)
        if t.numel() != n or t.dtype != dtype or t.device != p.device or not fits:
            raise ValueError(f"AdamW: a state of {tuple(t.shape)} {t.dtype} on {t.device} with strides {t.stride()} does not fit a "
                             f"parameter of {tuple(p.shape)} on {p.device} with strides {p.stride()}: {n} x {dtype} wanted")
