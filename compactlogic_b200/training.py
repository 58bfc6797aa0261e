"""Operators of a training step that stand before, between and after the logic layers, on hand-written sm_100a kernels:

* ``layer_norm`` / ``LogicLayerNorm``: real-valued observations or activations, normalised over their features;
* ``dropout`` / ``LogicDropout``: a mask from a counter-based generator, drawn again in the backward pass, never stored;
* ``action_log_probs``: log-probability of one chosen class per row, differentiable;
* ``policy_loss``: the clipped policy loss with a KL term, whose logit gradient is made in the same pass.

All four take the layers' own storage (``[batch, features]`` views of feature-major memory) and ordinary row-major tensors
alike, without copies, and run on the current stream.  A strided tensor that is neither is copied first.

First derivatives are complete.  Of second ones (create_graph) only dropout's exist; the others raise when they are asked for.
"""
from collections import deque
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple, Union
from weakref import WeakValueDictionary

import torch

from . import _lib as L
from .functional import GradSlot, _incoming_grad, first_order

__all__ = ["LogicDropout", "LogicLayerNorm", "PolicyLoss", "action_log_probs", "dropout", "layer_norm", "policy_loss"]

_LOW = (torch.bfloat16, torch.float16)
_ACC = {torch.float32: torch.float32, torch.bfloat16: torch.float32, torch.float16: torch.float32,
        torch.float64: torch.float64}
_BYTES = {torch.float32: 4, torch.float64: 8}

# The small calls of a training step are bound by the host, so the paths below keep to one allocation where several buffers
# live and die together, and look up the current stream by its device index.  A launch goes to the current GPU: where a public
# call's input is on another one, the call starts over with that one current (autograd's backward passes have it so).
_stream = torch._C._cuda_getCurrentRawStream
_device = torch._C._cuda_getDevice


# ------------------------------------------------------------------------------------------------------------ layouts
def _matrix(x: torch.Tensor) -> Tuple[torch.Tensor, int, int]:
    """A [n, d] tensor with one contiguous axis (a copy when ``x`` has none), whether that axis is n, and the other's
    stride.  A tensor that is both (one row, one column) counts as rows."""
    n, d = x.shape
    sn, sd = x.stride()
    if (sd == 1 or d <= 1) and (sn >= d or n <= 1):
        return x, 0, sn if n > 1 else d
    if (sn == 1 or n <= 1) and (sd >= n or d <= 1):
        return x, 1, sd if d > 1 else n
    return x.contiguous(), 0, d


def _dense(x: torch.Tensor) -> torch.Tensor:
    """``x``, or the copy that ``_matrix`` makes of it, within the graph."""
    return x if x.is_contiguous() else _matrix(x)[0]


def _like(x: torch.Tensor, inner: int) -> torch.Tensor:
    """A new dense [n, d] tensor with the contiguous axis of ``_matrix``."""
    n, d = x.shape
    return torch.empty_strided((n, d), (1, n) if inner else (d, 1), dtype=x.dtype, device=x.device)


def _check(what: str, x: torch.Tensor) -> int:
    """The dtype code of an input that has to be on a GPU."""
    if not x.is_cuda:
        raise RuntimeError("compactlogic_b200 kernels need CUDA tensors (there is no CPU fallback)")
    return L.dtype_code(x.dtype)


def _same_device(what: str, x: torch.Tensor, name: str, t: torch.Tensor) -> None:
    if t.get_device() != x.get_device():
        raise RuntimeError(f"{what}: {name} is on {t.device}, the input on {x.device}")


# ------------------------------------------------------------------------------------------------------------ dropout
def _drop(x: torch.Tensor, p: float, rescale: bool, seed: int, offset: int, rng: Optional[torch.Tensor]) -> torch.Tensor:
    x, inner, ld = _matrix(x)
    y = _like(x, inner)
    n, d = x.shape
    if inner:
        n, d = d, n
    status = L.lib().clb_dropout(L.dtype_code(x.dtype), x.data_ptr(), ld, n, d, inner, p, rescale, seed, offset,
                                 rng.data_ptr() if rng is not None else 0, y.data_ptr(), d, _stream(x.get_device()))
    if status:
        L.check(status, "clb_dropout")
    return y


class _DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rescale, seed, offset, rng, in_slot, out_slot):
        ctx.args = (p, rescale, seed, offset, rng)
        ctx.in_slot, ctx.out_slot, ctx.dtype, ctx.shape = in_slot, out_slot, x.dtype, x.shape
        return _drop(x, *ctx.args)

    @staticmethod
    def backward(ctx, gy):
        slot = ctx.out_slot
        if slot is not None and slot.grad is not None:
            gy = _incoming_grad(gy.t(), slot, torch.float32).t()
        if gy.requires_grad and torch.is_grad_enabled():  # create_graph: linear in gy
            gx = _DropoutFn.apply(gy, *ctx.args, None, None)
        else:
            gx = _drop(gy, *ctx.args)
        if ctx.in_slot is not None:
            ctx.in_slot.add(gx.float().t())
            gx = torch.zeros((), dtype=ctx.dtype, device=gx.device).expand(ctx.shape)
        return gx, None, None, None, None, None, None, None


def _dropout(x, p, rescale, seed, offset, rng):
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p must be in [0, 1], got {p}")
    _check("dropout", x)
    if x.get_device() != _device():
        with torch.cuda.device(x.device):
            return _dropout(x, p, rescale, seed, offset, rng)
    flat = x if x.dim() == 2 else x.reshape(x.shape[0], -1) if x.dim() > 2 and x.shape[0] else x.reshape(1, -1)
    out_slot = None
    if x.requires_grad and torch.is_grad_enabled():
        # between logic layers (conv layers' outputs have four axes) with 16-bit activations the gradient is handed over in
        # fp32, past autograd's rounding
        in_slot = None
        if x.dim() > 1 and x.dtype in _LOW:
            in_slot, out_slot = getattr(x, "_clb_slot", None), GradSlot()
        y = _DropoutFn.apply(flat, p, rescale, seed, offset, rng, in_slot, out_slot)
    else:
        y = _drop(flat, p, rescale, seed, offset, rng)
    if x.dim() != 2:
        y = y.reshape(x.shape)
    if out_slot is not None:
        y._clb_slot = out_slot
    return y


def dropout(x: torch.Tensor, p: float = 0.5, *, seed: int, offset: int = 0, rescale: bool = True) -> torch.Tensor:
    """Zero each entry of ``x`` with probability ``p`` (in steps of 2^-32) and scale the others by 1 / (1 - p), or leave them
    as they are with ``rescale=False`` (soft bits then stay in [0, 1]).

    Entry (i, j) of ``x`` taken as [first axis, all others] (a tensor of one axis as a single row [1, all]) is kept when its
    word of Philox4x32-10 under the key ``seed`` and the counter (j / 2, i / 2, ``offset``) is at least p 2^32, rounded: the
    mask depends on seed, offset and place alone, not on layout, strides or type, and is not stored.  Use another ``offset``
    for each pass.  A dropped entry is 0 whatever it held."""
    if not (0 <= seed < 1 << 64 and 0 <= offset < 1 << 64):
        raise ValueError("dropout: seed and offset are unsigned 64-bit numbers")
    return _dropout(x, p, rescale, seed, offset, None)


def _generator_place(index: int):
    """Where torch's generator of a GPU stands, which moves on by one draw; None while a graph is captured."""
    if torch.cuda.is_current_stream_capturing():
        return None
    generator = torch.cuda.default_generators[index]
    at = generator.get_offset()
    generator.set_offset(at + 4)
    return index, generator.initial_seed(), at


class LogicDropout(torch.nn.Module):
    """``dropout`` between logic layers, a new mask for each training pass; the identity in eval mode.

    The buffer ``rng_state`` (int64 {seed, offset}) advances on the device, so a captured training step
    (``compactlogic_b200.graph``) draws a new mask at each replay, and a loaded checkpoint continues the sequence.  ``seed``
    defaults to a draw from torch's generator.  Passes of one module on several streams at once are not ordered.  Data-parallel
    ranks with equal states mask their samples alike: after buffers were broadcast or loaded, give each rank a seed of its own
    (``m.rng_state[0] += rank``).

    A pass that activation checkpointing (``torch.utils.checkpoint``, either form) computes again draws the mask of the pass
    that it repeats.  The two are matched by where torch's CUDA generator stands, which checkpointing puts back
    (``preserve_rng_state``); passes that may be repeated, those without gradients or under saved-tensor hooks, move it on as
    torch's dropout does.  A forward pass inside a backward pass that matches none, or two, raises."""

    def __init__(self, p: float = 0.5, rescale: bool = True, seed: Optional[int] = None):
        super().__init__()
        if not 0.0 <= p <= 1.0:
            raise ValueError(f"LogicDropout: p must be in [0, 1], got {p}")
        if seed is None:
            seed = int(torch.randint(0, 1 << 62, ()).item())
        if not 0 <= seed < 1 << 63:
            raise ValueError("LogicDropout: seed must be in [0, 2^63)")
        self.p, self.rescale = float(p), bool(rescale)
        self.register_buffer("rng_state", torch.tensor([seed, 0], dtype=torch.int64))
        self._forget()

    def _forget(self):
        # {generator place: {seed, offset}} of passes that may be repeated.  The pass's autograd node keeps the entry; of those
        # without a node the newest are kept.
        self._passes = WeakValueDictionary()
        self._loose = deque(maxlen=1024)

    def __getstate__(self):
        return {k: v for k, v in self.__dict__.items() if k not in ("_passes", "_loose")}

    def __setstate__(self, state):
        super().__setstate__(state)
        self._forget()

    def _draw(self, x):
        """The generator state {seed, offset} of one pass, on the device."""
        again = torch._C._current_graph_task_id() != -1  # a forward pass inside a backward pass
        node = x.requires_grad and torch.is_grad_enabled()
        place = None
        if again or not node or torch._C._autograd._top_saved_tensors_default_hooks(True) is not None:
            place = _generator_place(x.get_device())
        if again:
            used = self._passes.get(place)
            if used is None or used.shared_place:
                raise RuntimeError("LogicDropout: a pass inside a backward pass has to recompute one earlier pass, which torch's "
                                   "CUDA generator tells; checkpoint with preserve_rng_state=True, and do not seed the "
                                   "generator alike for two passes in flight")
            return used
        used = torch.empty(2, dtype=torch.int64, device=x.device)
        status = L.lib().clb_dropout_advance(self.rng_state.data_ptr(), used.data_ptr(), _stream(x.get_device()))
        if status:
            L.check(status, "clb_dropout_advance")
        if place is not None:
            used.shared_place = place in self._passes
            self._passes[place] = used
            if not node:
                self._loose.append(used)
        return used

    def forward(self, x):
        if not self.training or self.p == 0.0:
            return x
        _check("LogicDropout", x)
        _same_device("LogicDropout", x, "rng_state", self.rng_state)
        if x.get_device() != _device():
            with torch.cuda.device(x.device):
                return self.forward(x)
        return _dropout(x, self.p, self.rescale, 0, 0, self._draw(x))

    def extra_repr(self):
        return f"p={self.p}, rescale={self.rescale}"


# --------------------------------------------------------------------------------------------------------- layer norm
@lru_cache(maxsize=256)
def _norm_bytes(code, n, d, inner, backward):
    return L.lib().clb_layer_norm_workspace_bytes(code, n, d, inner, backward)


def _norm_workspace(code, n, d, inner, backward, device):
    nbytes = _norm_bytes(code, n, d, inner, backward)
    return nbytes, torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _norm_forward(x, weight, bias, eps, keep):
    """(y, x as laid out, statistics [2 n] or None)"""
    x, inner, ld = _matrix(x)
    n, d = x.shape
    y = _like(x, inner)
    code = L.dtype_code(x.dtype)
    acc = _ACC[x.dtype]
    stats = torch.empty(2 * n, dtype=acc, device=x.device) if keep else None
    at = stats.data_ptr() if keep else 0
    nbytes, ws = _norm_workspace(code, n, d, inner, 0, x.device)
    status = L.lib().clb_layer_norm_forward(code, x.data_ptr(), ld, n, d, inner, L.ptr(weight), L.ptr(bias), eps,
                                            y.data_ptr(), n if inner else d, at, at + n * _BYTES[acc] if keep else 0,
                                            L.ptr(ws), nbytes, _stream(x.get_device()))
    if status:
        L.check(status, "clb_layer_norm_forward")
    return y, x, stats


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, x, ctx.stats = _norm_forward(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight)
        return y

    @staticmethod
    def backward(ctx, gy):
        x, weight = ctx.saved_tensors
        stats, given = ctx.stats, gy
        n, d = x.shape
        x, inner, ld = _matrix(x)
        gy, g_inner, ldg = _matrix(gy)
        if g_inner != inner:
            gy, ldg = (gy.t().contiguous().t(), n) if inner else (gy.contiguous(), d)
        acc = _ACC[x.dtype]
        need = ctx.needs_input_grad
        gx = _like(x, inner) if need[0] else None
        gw = torch.empty(d, dtype=acc, device=x.device) if need[1] else None
        gb = torch.empty(d, dtype=acc, device=x.device) if need[2] else None
        code = L.dtype_code(x.dtype)
        nbytes, ws = _norm_workspace(code, n, d, inner, 1, x.device)
        at = stats.data_ptr()
        status = L.lib().clb_layer_norm_backward(code, x.data_ptr(), ld, gy.data_ptr(), ldg, n, d, inner, L.ptr(weight), at,
                                                 at + n * _BYTES[acc], L.ptr(gx), n if inner else d, L.ptr(gw), L.ptr(gb),
                                                 L.ptr(ws), nbytes, _stream(x.get_device()))
        if status:
            L.check(status, "clb_layer_norm_backward")
        if torch.is_grad_enabled():
            gx, gw, gb = (first_order("layer_norm", gx, x, weight, given), first_order("layer_norm", gw, x, given),
                          first_order("layer_norm", gb, given))
        return gx, gw, gb, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (the features); the output has the layout of ``x``.

    ``weight`` and ``bias`` (optional, [features]) are fp32 for fp32, bf16 and fp16 activations and fp64 for fp64, as the
    layers' parameters are; statistics and the parameters' gradients are summed in that type, in a fixed order."""
    _check("layer_norm", x)
    if x.get_device() != _device():
        with torch.cuda.device(x.device):
            return layer_norm(x, weight, bias, eps)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise RuntimeError(f"layer_norm: expected [..., features], got shape {tuple(x.shape)}")
    acc = _ACC[x.dtype]
    grad = x.requires_grad
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _same_device("layer_norm", x, name, t)
            if t.dtype != acc or t.shape != x.shape[-1:]:
                raise RuntimeError(f"layer_norm: {name} must be {acc} [{x.shape[-1]}], got {t.dtype} {tuple(t.shape)}")
            grad = grad or t.requires_grad
    if not eps >= 0.0:
        raise ValueError(f"layer_norm: eps must not be negative, got {eps}")
    weight = weight if weight is None or weight.is_contiguous() else weight.contiguous()
    bias = bias if bias is None or bias.is_contiguous() else bias.contiguous()
    flat = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if grad and torch.is_grad_enabled():
        y = _LayerNormFn.apply(_dense(flat), weight, bias, eps)
    else:
        y = _norm_forward(flat, weight, bias, eps, False)[0]
    return y if x.dim() == 2 else y.reshape(x.shape)


class LogicLayerNorm(torch.nn.Module):
    """``layer_norm`` with learned fp32 weight and bias (``affine=False``: none)."""

    def __init__(self, features: int, eps: float = 1e-5, affine: bool = True):
        super().__init__()
        self.features, self.eps = features, eps
        self.weight = torch.nn.Parameter(torch.ones(features)) if affine else None
        self.bias = torch.nn.Parameter(torch.zeros(features)) if affine else None

    def forward(self, x):
        if x.shape[-1:] != (self.features,):
            raise RuntimeError(f"LogicLayerNorm({self.features}): got shape {tuple(x.shape)}")
        w, b = self.weight, self.bias
        if x.dtype == torch.float64 and w is not None:
            w, b = w.double(), b.double()
        return layer_norm(x, w, b, self.eps)

    def extra_repr(self):
        return f"{self.features}, eps={self.eps}, affine={self.weight is not None}"


# ------------------------------------------------------------------------------------------------------------- losses
def _per_row(what, name, t, z, lead):
    """A per-row argument as a contiguous [n] tensor on the logits' device."""
    if t.get_device() != z.get_device():
        _same_device(what, z, name, t)
    if t.shape != lead:
        raise RuntimeError(f"{what}: {name} must have shape {tuple(lead)}, got {tuple(t.shape)}")
    return t if t.dim() == 1 and t.is_contiguous() else t.reshape(-1).contiguous()


def _rows_of(what, logits, actions, mask):
    """Logits as [n, v] and the per-row arguments flattened to match."""
    _check(what, logits)
    if logits.dim() == 2 and actions.dtype is torch.int64 and mask is None:  # the common call, in few steps
        n, v = logits.shape
        if v and actions.dim() == 1 and actions.shape[0] == n and actions.is_contiguous() and actions.is_cuda and \
                actions.get_device() == logits.get_device():
            return logits, actions, None, (n,)
    lead = logits.shape[:-1]
    if logits.dim() < 1 or logits.shape[-1] < 1:
        raise RuntimeError(f"{what}: expected logits [..., classes], got shape {tuple(logits.shape)}")
    if actions.dtype != torch.int64:
        if actions.is_floating_point() or actions.is_complex() or actions.dtype == torch.bool:
            raise RuntimeError(f"{what}: actions must be integers, got {actions.dtype}")
        actions = actions.long()
    actions = _per_row(what, "actions", actions, logits, lead)
    if mask is not None:
        if mask.dtype != torch.bool and mask.dtype != torch.uint8:
            raise RuntimeError(f"{what}: mask must be bool {tuple(lead)}, got {mask.dtype} {tuple(mask.shape)}")
        mask = _per_row(what, "mask", mask, logits, lead)
    z = logits if logits.dim() == 2 else logits.reshape(-1, logits.shape[-1])
    return z, actions, mask, lead


def _logit_grad(z, actions, mask, temperature, stats, slope, scale, upstream, up_stride, gz=None):
    """gz for one upstream gradient; a given ``gz`` already holds the gradient for an upstream of 1.  stats, slope and
    scale are addresses (0: none)."""
    z, inner, ld = _matrix(z)
    n, v = z.shape
    fresh = gz is None
    if fresh:
        gz = _like(z, inner)
    status = L.lib().clb_logit_grad(L.dtype_code(z.dtype), z.data_ptr(), ld, n, v, inner, actions.data_ptr(), L.ptr(mask),
                                    temperature, stats, slope, scale, upstream.data_ptr(), up_stride, not fresh,
                                    gz.data_ptr(), n if inner else v, _stream(z.get_device()))
    if status:
        L.check(status, "clb_logit_grad")
    return gz


def _logp_forward(z, actions, mask, temperature, keep):
    z, inner, ld = _matrix(z)
    n, v = z.shape
    acc = _ACC[z.dtype]
    logp = torch.empty(n, dtype=acc, device=z.device)
    stats = torch.empty(2 * n, dtype=acc, device=z.device) if keep else None
    status = L.lib().clb_action_logp(L.dtype_code(z.dtype), z.data_ptr(), ld, n, v, inner, actions.data_ptr(), L.ptr(mask),
                                     temperature, logp.data_ptr(), L.ptr(stats), _stream(z.get_device()))
    if status:
        L.check(status, "clb_action_logp")
    return logp, z, stats


class _LogProbFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, actions, mask, temperature):
        logp, z, ctx.stats = _logp_forward(z, actions, mask, temperature, True)
        ctx.save_for_backward(z, actions, mask)
        ctx.temperature = temperature
        return logp

    @staticmethod
    def backward(ctx, g):
        z, actions, mask = ctx.saved_tensors
        gz = _logit_grad(z, actions, mask, ctx.temperature, ctx.stats.data_ptr(), 0, 0, g, g.stride(0))
        return first_order("action_log_probs", gz, z, g), None, None, None


def _check_temperature(what, temperature):
    if not temperature > 0.0:
        raise ValueError(f"{what}: temperature must be positive, got {temperature}")


def action_log_probs(logits: torch.Tensor, actions: torch.Tensor, *, mask: Optional[torch.Tensor] = None,
                     temperature: float = 1.0) -> torch.Tensor:
    """log softmax(logits / temperature)[..., actions], in the arithmetic type (fp32; fp64 for fp64 logits), differentiable
    with respect to the logits.

    ``logits`` [..., classes] in row-major or class-major storage (as GroupSum returns it), ``actions`` integers [...].
    Rows where ``mask`` (bool [...]) is False are not read: their value and gradient are 0 and their action may be
    anything.  In other rows an action outside [0, classes) gives NaN."""
    z, act, m, lead = _rows_of("action_log_probs", logits, actions, mask)
    if z.get_device() != _device():
        with torch.cuda.device(z.device):
            return action_log_probs(logits, actions, mask=mask, temperature=temperature)
    _check_temperature("action_log_probs", temperature)
    if z.requires_grad and torch.is_grad_enabled():
        logp = _LogProbFn.apply(_dense(z), act, m, temperature)
    else:
        logp = _logp_forward(z, act, m, temperature, False)[0]
    return logp if len(lead) == 1 else logp.reshape(lead)


class PolicyLoss(NamedTuple):
    """What ``policy_loss`` returns: the loss (differentiable), and per row, without gradients, the chosen actions'
    log-probabilities, the ratios to the old policy, and the KL term (None without ``ref_log_probs``)."""
    loss: torch.Tensor
    log_probs: torch.Tensor
    ratio: torch.Tensor
    kl: Optional[torch.Tensor]


def _policy(z, actions, mask, adv, old, ref, low, high, kl_coef, temperature, reduction, grad):
    """The loss, the per-row results, the logit gradient (None where it is not made in this pass), and what the gradient of
    another pass needs: one buffer of slope [n], stats [2 n], scale [1] (and the rows' losses [n])."""
    z, inner, ld = _matrix(z)
    n, v = z.shape
    acc = _ACC[z.dtype]
    dev = z.device
    per_row = reduction == "none"
    logp, ratio = torch.empty(n, dtype=acc, device=dev), torch.empty(n, dtype=acc, device=dev)
    kl = torch.empty(n, dtype=acc, device=dev) if ref is not None else None
    loss = torch.empty((n,) if per_row else (), dtype=acc, device=dev)
    kept = torch.empty(4 * n + 1, dtype=acc, device=dev)
    at, size = kept.data_ptr(), _BYTES[acc]
    # the mean's and the sum's gradient is made in the same pass, for an upstream gradient of 1
    gz = _like(z, inner) if grad and not per_row else None
    status = L.lib().clb_policy_loss(
        L.dtype_code(z.dtype), z.data_ptr(), ld, n, v, inner, actions.data_ptr(), L.ptr(mask), adv.data_ptr(), old.data_ptr(),
        L.ptr(ref), low, high, kl_coef, temperature, reduction == "mean", 0 if per_row else loss.data_ptr(),
        at + 3 * n * size, loss.data_ptr() if per_row else at + (3 * n + 1) * size, logp.data_ptr(), ratio.data_ptr(),
        L.ptr(kl), at if grad else 0, at + n * size if grad else 0, L.ptr(gz), n if inner else v, _stream(z.get_device()))
    if status:
        L.check(status, "clb_policy_loss")
    return loss, logp, ratio, kl, z, gz, kept


class _PolicyLossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, z, actions, mask, adv, old, ref, low, high, kl_coef, temperature, reduction):
        loss, logp, ratio, kl, z, ctx.gz, ctx.kept = _policy(z, actions, mask, adv, old, ref, low, high, kl_coef, temperature,
                                                             reduction, True)
        ctx.save_for_backward(z, actions, mask)
        ctx.temperature, ctx.per_row = temperature, reduction == "none"
        ctx.set_materialize_grads(False)
        if kl is None:
            ctx.mark_non_differentiable(logp, ratio)
        else:
            ctx.mark_non_differentiable(logp, ratio, kl)
        return loss, logp, ratio, kl

    @staticmethod
    def backward(ctx, g, *unused):
        if g is None:
            return (None,) * 11
        z, actions, mask = ctx.saved_tensors
        at, size, n = ctx.kept.data_ptr(), ctx.kept.element_size(), z.shape[0]
        # The gradient made in the forward pass is handed out once; a later call (a retained graph) makes another.
        gz, ctx.gz = ctx.gz, None
        gz = _logit_grad(z, actions, mask, ctx.temperature, at + n * size, at, at + 3 * n * size, g,
                         g.stride(0) if ctx.per_row else 0, gz)
        return (first_order("policy_loss", gz, z, g),) + (None,) * 10


def policy_loss(logits: torch.Tensor, actions: torch.Tensor, advantages: torch.Tensor, old_log_probs: torch.Tensor, *,
                ref_log_probs: Optional[torch.Tensor] = None, mask: Optional[torch.Tensor] = None,
                clip: Union[float, Tuple[float, float]] = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                reduction: str = "mean") -> PolicyLoss:
    """The clipped policy loss with a KL term, over the rows where ``mask`` is True (all without a mask):

        lp = action_log_probs(logits, actions, temperature),  ratio = exp(lp - old_log_probs)
        row = -min(ratio * advantages, clamp(ratio, 1 - clip_low, 1 + clip_high) * advantages) + kl_coef * kl
        kl = exp(ref_log_probs - lp) - (ref_log_probs - lp) - 1

    ``reduction``: "mean" over the counted rows (0 when none counts), "sum", or "none" (per row).  ``clip`` is one bound or
    (clip_low, clip_high).  The gradient goes to ``logits`` alone; the other arguments are data.  Rows that do not count
    are not read, give zeros, and get a zero gradient; a counted row whose action is outside [0, classes) gives NaN.

    With "mean" and "sum" the logit gradient is computed in the forward pass, for an upstream gradient of 1; ``backward``
    hands it over, or computes it anew where the upstream gradient is another (a scaled loss).  Between the two passes the
    call holds that gradient, as large as the logits, outside the saved tensors that offloading hooks see."""
    z, act, m, lead = _rows_of("policy_loss", logits, actions, mask)
    if z.get_device() != _device():
        with torch.cuda.device(z.device):
            return policy_loss(logits, actions, advantages, old_log_probs, ref_log_probs=ref_log_probs, mask=mask, clip=clip,
                               kl_coef=kl_coef, temperature=temperature, reduction=reduction)
    _check_temperature("policy_loss", temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError(f"policy_loss: reduction must be mean, sum or none, got {reduction!r}")
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    if not (low >= 0.0 and high >= 0.0):
        raise ValueError(f"policy_loss: clip must not be negative, got {clip}")
    acc = _ACC[z.dtype]
    given = []
    n, dev = z.shape[0], z.get_device()
    for name, t in (("advantages", advantages), ("old_log_probs", old_log_probs), ("ref_log_probs", ref_log_probs)):
        if t is not None and not (t.dtype is acc and t.dim() == 1 and t.shape[0] == n and len(lead) == 1 and
                                  t.is_contiguous() and t.get_device() == dev):
            t = _per_row("policy_loss", name, t if t.dtype is acc else t.to(acc), z, lead)
        given.append(t)
    args = (act, m, *given, low, high, kl_coef, temperature, reduction)
    if z.requires_grad and torch.is_grad_enabled():
        out = _PolicyLossFn.apply(_dense(z), *args)
    else:
        with torch.no_grad():
            out = _policy(z, *args, False)[:4]
    if len(lead) != 1:
        out = tuple(t if t is None or (i == 0 and reduction != "none") else t.reshape(lead) for i, t in enumerate(out))
    return PolicyLoss(*out)
