"""Operators around a language model's output layer: layer norm, token log probabilities, distillation.

GPU tensors run the HIP kernels of csrc/kernels/layer_norm.hip and csrc/kernels/vocab_rows.hip, CPU
tensors the formulas below (both f32 inside, f32 or bf16 outside).  Matrices may be slices of wider
ones (any row stride); only elements of a row that are not next to each other cost a copy.

``layer_norm``          y = gamma (x - mean) / sqrt(var + eps) + beta over the last dimension
``token_log_probs``     log p of given tokens under softmax(logits / T), the entropy of that
                        distribution and its top alternatives; differentiable in the logits
``distillation_loss``   T^2 KL(teacher || student) from the teacher's top logits; differentiable in the
                        student's logits

Gradients are of first order and in reverse mode: create_graph=True is refused (on the CPU, what differentiates
them again), and so is a tensor that carries a forward-mode tangent.

The lists of top alternatives that ``token_log_probs`` returns (id -1 where nothing is left) are the
teacher's lists that ``distillation_loss`` takes.
"""
from __future__ import annotations

import math
import weakref
from typing import NamedTuple, Optional

import torch
from torch.autograd.function import once_differentiable

from . import _native
from .nn import _grad_ready
from ..variables import Variable

MAX_TOP = 64              # top alternatives of one position
MAX_TEACHER_TOP = 1024    # entries of a teacher's list
MAX_WIDTH = 1 << 24       # vocabulary entries / features
_FLOATS = (torch.float32, torch.bfloat16)
_WHOLE = (torch.int64, torch.int32)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as [rows, width], its own memory wherever the elements of a row are next to each other."""
    if x.stride(-1) != 1 and x.shape[-1] != 1:
        x = x.contiguous()
    return x if x.dim() == 2 else x.reshape(math.prod(x.shape[:-1]), x.shape[-1])


def _check_matrix(x: torch.Tensor, what: str) -> None:
    if x.dtype not in _FLOATS:
        raise TypeError("%s: float32 or bfloat16 expected, got %s" % (what, x.dtype))
    if x.dim() < 2 or not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError("%s: at least two dimensions, the last between 1 and %d, expected; got %s"
                         % (what, MAX_WIDTH, tuple(x.shape)))


def _check_side(t: torch.Tensor, x: torch.Tensor, shape, dtypes, what: str) -> None:
    if t.dtype not in dtypes:
        raise TypeError("%s: %s expected, got %s" % (what, " or ".join(str(d)[6:] for d in dtypes), t.dtype))
    if t.device != x.device:
        raise ValueError("%s: on %s, the matrix is on %s" % (what, t.device, x.device))
    if t.shape != shape:
        raise ValueError("%s: shape %s expected, got %s" % (what, tuple(shape), tuple(t.shape)))


def _check_temperature(t: float) -> None:
    if not 1e-6 <= t <= 1e6:
        raise ValueError("temperature: a number between 1e-6 and 1e6 expected, got %r" % t)


# ====================================================================== layer norm
def _ln_ref(x, gamma, beta, eps):
    xf = x.float()
    mean = xf.mean(1, keepdim=True)
    xc = xf - mean
    rstd = torch.rsqrt((xc * xc).mean(1, keepdim=True) + eps)
    y = xc * rstd
    if gamma is not None:
        y = y * gamma
    if beta is not None:
        y = y + beta
    return y.to(x.dtype), torch.cat([mean, rstd], 1)


def _ln_bwd_ref(x, dy, stats, gamma, dgamma, dbeta, want_dx):
    dy = dy.float()
    xhat = (x.float() - stats[:, :1]) * stats[:, 1:]
    if dgamma is not None:
        dgamma.add_((dy * xhat).sum(0))
    if dbeta is not None:
        dbeta.add_(dy.sum(0))
    if not want_dx:
        return None
    g = dy if gamma is None else dy * gamma
    dx = stats[:, 1:] * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
    return dx.to(x.dtype)


class _Watcher:
    """Keeps the GPU's nodes informed of a store: where its gradients are, and whether it has a hook, as of the
    backward pass (csrc/torch_ops/lm_ops.cpp).  A copy of the store gets one of its own."""
    stores: "weakref.WeakValueDictionary[int, object]" = weakref.WeakValueDictionary()

    def __init__(self, store):
        self.number = torch.ops.tfx.store_new()
        weakref.finalize(self, torch.ops.tfx.store_free, self.number).atexit = False
        _Watcher.stores[self.number] = store
        self.update(store)

    def update(self, store) -> None:
        torch.ops.tfx.store_set(self.number, store.grad, store.grad_ready_hook is not None)

    def __deepcopy__(self, memo):
        return None

    def __reduce__(self):
        return type(None), ()


def _store_number(store) -> int:
    if store.watcher is None:
        store.watcher = _Watcher(store)
    return store.watcher.number


def _ready(number: int, at: int) -> None:
    """The variable at element ``at`` of that store has its gradient (called by the GPU's nodes)."""
    store = _Watcher.stores.get(number)
    if store is not None:
        _grad_ready(next(v for v in store.vars if v.offset == at and v.numel))


_library = torch.library.Library("tfx", "FRAGMENT")
_library.define("grad_ready(int store, int at) -> ()")
_library.impl("grad_ready", _ready, "CompositeExplicitAutograd")


class _LayerNorm(torch.autograd.Function):
    """The CPU's node, and the GPU's where a gradient hook has to run after the backward pass."""

    @staticmethod
    def forward(ctx, x, anchor, gamma: Optional[Variable], beta: Optional[Variable], eps):
        ctx.vars, ctx.native = (gamma, beta), _native.use_native(x)
        g = gamma.master if gamma is not None else None
        b = beta.master if beta is not None else None
        if ctx.native:
            y, stats = torch.ops.tfx.layer_norm_fwd(x, g, b, eps)
        else:
            y, stats = _ln_ref(_rows(x), g, b, eps)
        ctx.save_for_backward(x, stats)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, stats = ctx.saved_tensors
        gamma, beta = ctx.vars
        g = gamma.master if gamma is not None else None
        dg = gamma.grad if gamma is not None and gamma.trainable else None
        db = beta.grad if beta is not None and beta.trainable else None
        need = ctx.needs_input_grad[0]
        if ctx.native:
            dx = torch.ops.tfx.layer_norm_bwd(x, gy, stats, g, dg, db, need)
        else:
            dx = _ln_bwd_ref(_rows(x), _rows(gy), stats, g, dg, db, need)
        _grad_ready(gamma if dg is not None else None, beta if db is not None else None)
        return (dx.view(gy.shape) if need else None), None, None, None, None


def layer_norm(x: torch.Tensor, gamma: Optional[Variable] = None, beta: Optional[Variable] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm of ``x`` [..., C] (f32 or bf16) over its last dimension, with the biased variance:
    ``gamma * (x - mean) / sqrt(var + eps) + beta``.  ``gamma`` / ``beta``: variables of shape [C], or
    None for 1 / 0 (not one variable as both); their gradients accumulate into ``var.grad``, summed in one
    order (equal inputs give equal gradients).  The result has ``x``'s type and is contiguous.  Statistics,
    sums and products are f32; the forward and each input gradient are rounded once."""
    width = x.shape[-1] if x.dim() else 0
    anchor = None
    hook = False
    if gamma is not None and gamma is beta:
        raise ValueError("layer_norm: gamma and beta are the same variable")
    for v, what in ((gamma, "gamma"), (beta, "beta")):
        if v is not None:
            if v.shape != (width,):
                raise ValueError("layer_norm: %s of shape %s for an input of %s" % (what, v.shape, tuple(x.shape)))
            if v.store is None or v.store.master is None:
                raise ValueError("layer_norm: the store of %s is not finalized" % what)
            if v.store.master.device != x.device:
                raise ValueError("layer_norm: %s is on %s, the input on %s" % (what, v.store.master.device, x.device))
            if v.trainable:
                hook |= v.store.grad_ready_hook is not None
                if not x.requires_grad:  # the store's leaf records the call only where nothing else does
                    anchor = v.store.anchor
    native = _native.use_native(x)
    if native and not hook:
        gs, bs = gamma and gamma.store, beta and beta.store
        return torch.ops.tfx.layer_norm(
            x, anchor, gs and gs.master, gamma.offset if gs else 0, bs and bs.master, beta.offset if bs else 0,
            _store_number(gs) if gs and gamma.trainable else -1, _store_number(bs) if bs and beta.trainable else -1, eps)
    _check_matrix(x, "layer_norm")
    if not (eps >= 1e-30 and math.isfinite(eps)):
        raise ValueError("layer_norm: eps of at least 1e-30 expected, got %r" % eps)
    return _LayerNorm.apply(x, anchor, gamma, beta, eps)


# ====================================================================== token log probabilities
class TokenLogProbs(NamedTuple):
    """What :func:`token_log_probs` returns: ``logp`` and ``entropy`` [...] f32 (``entropy`` None unless asked
    for), ``top_logp`` [..., K] f32 and ``top_ids`` [..., K] int64 (None for ``top_k=0``)."""
    logp: torch.Tensor
    entropy: Optional[torch.Tensor]
    top_logp: Optional[torch.Tensor]
    top_ids: Optional[torch.Tensor]


def _log_softmax_ref(x, temperature):
    """(z, logs, empty) of rows: z = (x - their maximum) / T, log p = z - logs; ``empty`` where nothing but -inf is left (logs
    is 0 there).  The maximum is taken off first: of a row of the type's lowest value, or far from 0, z would round away."""
    x = x.float()
    m = x.amax(1, keepdim=True)
    z = (x - torch.where(m == -math.inf, torch.zeros_like(m), m)) / temperature
    s = torch.exp(z).sum(1, keepdim=True)
    empty = s == 0
    return z, torch.log(torch.where(empty, torch.ones_like(s), s)), empty


def _dist_ref(z, logs):
    """(p, log p with 0 where p is 0)"""
    p = torch.exp(z - logs)
    return p, torch.where(p == 0, torch.zeros_like(p), z - logs)


def _tokens_ref(x, tokens, top_k, temperature):
    z, logs, empty = _log_softmax_ref(x, temperature)
    p, logq = _dist_ref(z, logs)
    V = x.shape[1]
    t = tokens.long()[:, None]
    real = t >= 0
    logp = z.gather(1, t.clamp(0, V - 1)) - logs
    logp = torch.where(empty, torch.full_like(logp, -math.inf), logp)
    logp = torch.where(t >= V, torch.full_like(logp, math.nan), logp)
    zero = torch.zeros_like(logp)
    ent = -(p * logq).sum(1, keepdim=True)
    top = ids = None
    if top_k:
        v = x.float() + 0.0
        some = (v > -math.inf) & real  # neither NaN nor -inf
        v = torch.where(some, v, torch.full_like(v, -math.inf))
        # stable: equal values in the order of their ids
        order = torch.sort(v, dim=1, descending=True, stable=True)[1][:, :top_k]
        there = some.gather(1, order)
        top = torch.where(there, z.gather(1, order) - logs, torch.full_like(zero, -math.inf))
        ids = torch.where(there, order, torch.full_like(order, -1))
        if ids.shape[1] < top_k:
            pad = (0, top_k - ids.shape[1])
            top = torch.nn.functional.pad(top, pad, value=-math.inf)
            ids = torch.nn.functional.pad(ids, pad, value=-1)
    return torch.where(real, logp, zero)[:, 0], torch.where(real, ent, zero)[:, 0], top, ids


def _tokens_bwd_ref(x, tokens, g, h, temperature):
    z, logs, empty = _log_softmax_ref(x, temperature)
    p, logq = _dist_ref(z, logs)
    t = tokens.long()[:, None]
    dz = torch.zeros_like(p)
    if g is not None:
        dz = -p * g[:, None]
        left = torch.where(empty | (t < 0) | (t >= x.shape[1]), torch.zeros_like(g[:, None]), g[:, None])
        dz.scatter_add_(1, t.clamp(0, x.shape[1] - 1), left)
    if h is not None:
        ent = -(p * logq).sum(1, keepdim=True)
        dz = dz - p * (logq + ent) * h[:, None]
    dz = torch.where(t >= x.shape[1], torch.full_like(dz, math.nan), dz / temperature)
    return torch.where(t < 0, torch.zeros_like(dz), dz).to(x.dtype)


class _TokenLogProbs(torch.autograd.Function):
    """The CPU's node (the GPU's: csrc/torch_ops/lm_ops.cpp)"""

    @staticmethod
    def forward(ctx, logits, tokens, top_k, temperature):
        x = _rows(logits)
        ctx.temperature, ctx.shape = temperature, logits.shape
        ctx.set_materialize_grads(False)
        logp, ent, top, ids = _tokens_ref(x, tokens, top_k, temperature)
        ctx.save_for_backward(x, tokens)
        if top is not None:
            ctx.mark_non_differentiable(top, ids)
        return logp, ent, top, ids

    @staticmethod
    @once_differentiable
    def backward(ctx, g, h, *unused):
        if g is None and h is None:
            return None, None, None, None
        x, tokens = ctx.saved_tensors
        return _tokens_bwd_ref(x, tokens, g, h, ctx.temperature).view(ctx.shape), None, None, None


def token_log_probs(logits: torch.Tensor, tokens: torch.Tensor, top_k: int = 0, entropy: bool = False,
                    temperature: float = 1.0) -> TokenLogProbs:
    """Log probabilities of ``tokens`` under ``softmax(logits / temperature)``, in one pass over the logits.

    ``logits`` [..., V] f32 or bf16, ``tokens`` [...] int64 or int32.  ``entropy=True`` adds the entropy of
    each position's distribution (in nats), ``top_k`` (up to 64) its most likely tokens and their log
    probabilities, best first; equal logits are ordered by their id.  Gradients flow to the logits from
    ``logp`` and ``entropy``, none from the alternatives.  Sums are f32: both are off by some 1e-6, and by f32's rounding
    of their own size.

    * a negative token marks padding: logp 0, entropy 0, no alternatives, gradient 0, whatever its logits hold;
    * a logit of -inf is a masked token: probability 0, never an alternative.  With fewer than ``top_k``
      tokens left the rest of the list has id -1 and log probability -inf.  A position with no token left has
      logp -inf, entropy 0, gradient 0;
    * a token outside the vocabulary gives a logp of NaN and a gradient of NaN;
    * a NaN or +inf among the logits makes the position's values and gradient NaN (NaN is never an
      alternative)."""
    if _native.use_native(logits):
        return TokenLogProbs(*torch.ops.tfx.token_log_probs(logits, tokens, top_k, bool(entropy), temperature))
    _check_matrix(logits, "logits")
    lead = logits.shape[:-1]
    _check_side(tokens, logits, lead, _WHOLE, "tokens")
    if not 0 <= top_k <= MAX_TOP:
        raise ValueError("top_k between 0 and %d expected, got %r" % (MAX_TOP, top_k))
    _check_temperature(temperature)
    logp, ent, top, ids = _TokenLogProbs.apply(logits, tokens.reshape(-1), int(top_k), float(temperature))
    return TokenLogProbs(logp.view(lead), ent.view(lead) if entropy else None,
                         top.view(*lead, top_k) if top_k else None, ids.view(*lead, top_k) if top_k else None)


# ====================================================================== distillation
def _teacher_ref(x, teacher, ids, weight, temperature):
    """(teacher's q, log q, rows that learn, rows with an id outside the vocabulary, per-row factor)"""
    there = ids >= 0
    t, logs, empty = _log_softmax_ref(torch.where(there, teacher.float(), torch.full_like(teacher.float(), -math.inf)),
                                      temperature)
    bad = (ids >= x.shape[1]).any(1, keepdim=True)
    w = weight[:, None] if weight is not None else torch.full_like(logs, 1.0 / max(1, x.shape[0]))
    bad = bad & (w != 0)
    real = there.any(1, keepdim=True) & ~empty & (w != 0) & ~bad
    return torch.exp(t - logs), t - logs, real, bad, w


def _distill_ref(x, teacher, ids, weight, temperature):
    q, logq, real, bad, w = _teacher_ref(x, teacher, ids, weight, temperature)
    z, logs, empty = _log_softmax_ref(x, temperature)
    logp = z.gather(1, ids.long().clamp(0, x.shape[1] - 1)) - logs
    logp = torch.where(empty, torch.full_like(logp, -math.inf), logp)
    kl = torch.where((q == 0) | ~real, torch.zeros_like(q), q * (logq - logp)).sum(1, keepdim=True)
    rows = torch.where(real, temperature * temperature * w * kl, torch.zeros_like(kl))
    rows = torch.where(bad, torch.full_like(kl, math.nan), rows)
    return rows.double().sum().float()


def _distill_bwd_ref(x, teacher, ids, weight, g, temperature):
    q, _, real, bad, w = _teacher_ref(x, teacher, ids, weight, temperature)
    z, logs, empty = _log_softmax_ref(x, temperature)
    dz = torch.exp(z - logs).scatter_add(1, ids.long().clamp(0, x.shape[1] - 1), torch.where(ids >= 0, -q, torch.zeros_like(q)))
    dz = torch.where(real & ~empty, dz * (g * w * temperature), torch.zeros_like(dz))
    return torch.where(bad, torch.full_like(dz, math.nan), dz).to(x.dtype)


class _Distillation(torch.autograd.Function):
    """The CPU's node (the GPU's: csrc/torch_ops/lm_ops.cpp)"""

    @staticmethod
    def forward(ctx, logits, teacher, ids, weight, temperature):
        x = _rows(logits)
        ctx.temperature, ctx.shape = temperature, logits.shape
        ctx.save_for_backward(x, teacher, ids, weight)
        return _distill_ref(x, teacher, ids, weight, temperature)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        x, teacher, ids, weight = ctx.saved_tensors
        dx = _distill_bwd_ref(x, teacher, ids, weight, g, ctx.temperature)
        return dx.view(ctx.shape), None, None, None, None


def distillation_loss(logits: torch.Tensor, teacher_logits: torch.Tensor, teacher_ids: torch.Tensor,
                      temperature: float = 1.0, row_weight: Optional[torch.Tensor] = None,
                      unit_seed: bool = False) -> torch.Tensor:
    """``sum_r w_r T^2 KL(q_r || softmax(logits_r / T))``, a scalar, where ``q_r`` is the softmax of
    ``teacher_logits_r / T`` over the teacher's list of row r: K top logits (or log probabilities: a constant
    does not matter) ``teacher_logits`` [..., K], f32 or bf16, at the vocabulary entries ``teacher_ids``
    [..., K], int64 or int32, K up to 1024.  ``logits`` [..., V] f32 or bf16.  ``row_weight`` [...] f32:
    the w_r; 1 / rows if None (the mean).  The teacher and the weights are constants: gradients flow to
    ``logits`` alone.

    * an id below 0 is no entry (lists may be ragged); a row with none, with only -inf logits, or of
      weight 0 adds nothing: loss 0 and gradient 0, whatever its logits hold;
    * an id that occurs twice counts with both its entries;
    * an id outside the vocabulary makes the loss and the row's gradient NaN;
    * a student's logit of -inf where the teacher has some probability makes the loss +inf; a row whose
      logits are all -inf has no gradient.

    ``unit_seed=True`` says that the loss is the root of ``backward()`` (seed 1): where the rows fit a
    block's registers (V up to 131072 in bf16, 65536 in f32) the gradient is then formed by the forward pass,
    which reads the logits once for both.  Another seed is applied all the same, in a pass of its own that rounds
    once more; the gradient can be taken once."""
    if _native.use_native(logits):
        return torch.ops.tfx.distillation_loss(logits, teacher_logits, teacher_ids, temperature, row_weight,
                                               bool(unit_seed))
    _check_matrix(logits, "logits")
    lead = logits.shape[:-1]
    if teacher_ids.dim() != logits.dim() or not 1 <= teacher_ids.shape[-1] <= MAX_TEACHER_TOP:
        raise ValueError("teacher_ids [..., K] with K between 1 and %d expected, got %s"
                         % (MAX_TEACHER_TOP, tuple(teacher_ids.shape)))
    k = teacher_ids.shape[-1]
    _check_side(teacher_ids, logits, (*lead, k), _WHOLE, "teacher_ids")
    _check_side(teacher_logits, logits, (*lead, k), _FLOATS, "teacher_logits")
    if row_weight is not None:
        _check_side(row_weight, logits, lead, (torch.float32,), "row_weight")
        row_weight = row_weight.detach().reshape(-1)
    _check_temperature(temperature)
    return _Distillation.apply(logits, teacher_logits.detach().reshape(-1, k), teacher_ids.reshape(-1, k), row_weight,
                               float(temperature))


__all__ = ["layer_norm", "token_log_probs", "TokenLogProbs", "distillation_loss"]
