"""Losses that fine-tune a trained latent diffusion model, beside p_losses (`train.EpsLossFn`): from preferences - pairs of a preferred and
a rejected latent against a frozen reference network - and from rewards - denoising transitions with advantages.

    out = preference_loss(model_out, ref_out, x_t, noise, sqrt_1mac, beta=2000.0)
    out.loss.backward()

Both take the network outputs of the mixed prediction (get_mixed_prediction, diffusion/ddpm.py:469-477) and differentiate through it, to
the output and to `mixing_logit`; every value is computed in libddmi_hip (include/ddmi_hip.h "Fine-tuning"), autograd only sequences
forward and backward.  `train.LDMTrainStep.preference_step` / `.policy_step` are the training steps made of them.

Tensors live on one GPU, samples along the first axis, channels along the second, anything behind them ([B, C, H, W] latents, [B, C, L]
clips).  model_out and ref_out are both fp32 or both bf16, everything else is fp32; strides are free (a strided tensor is copied).
Gradients are those of first order in reverse mode: a second order, or a forward-mode tangent, raises.

The calls enqueue work on the tensors' device's current stream and nothing else: no synchronisation, and a forward + backward can be captured
in a hipGraph (the workspace is a torch tensor of the call, so graphs share none).  A capture is refused while an eager loss lives that was built
on the default stream over leaves that the captured one differentiates too (a network's parameters among them); other graphs on such leaves
are the caller's to drop.  A backward that is captured apart from its forward needs the forward on a side stream.
"""
from __future__ import annotations

import contextlib
import ctypes as C
import functools
import math
import weakref
from typing import NamedTuple, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_HERE = contextlib.nullcontext()
_OUT_TYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


class PreferenceLoss(NamedTuple):
    """loss: scalar, differentiable.  margin [pairs]: beta times the implicit reward of the preferred sample over the rejected one's
    (> 0: ranked as preferred).  mse [2 pairs]: mean((prediction - noise)^2).  Both 0 where a pair is left out."""
    loss: torch.Tensor
    margin: torch.Tensor
    mse: torch.Tensor


class PolicyLoss(NamedTuple):
    """loss: scalar, differentiable.  logp, ratio, kl [B]: per transition, 0 where it is left out."""
    loss: torch.Tensor
    logp: torch.Tensor
    ratio: torch.Tensor
    kl: torch.Tensor


def _p(t: Optional[torch.Tensor]):
    return None if t is None else t.data_ptr()


def _expect(who, name, t, shape, dtype=torch.float32):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{who}: {name} is a tensor, got {type(t).__name__}")
    if t.shape != shape:
        raise ValueError(f"{who}: {name} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != dtype:
        raise ValueError(f"{who}: {name} is {t.dtype}, expected {dtype}")


def _check_outputs(who, model_out, ref_out, x_t, sqrt_1mac, mixing_logit, ref_mixing_logit):
    if not isinstance(model_out, torch.Tensor) or model_out.dim() < 2 or model_out.numel() == 0:
        raise ValueError(f"{who}: model_out is a non-empty [B, C, ...] tensor")
    if model_out.dtype not in _OUT_TYPES:
        raise ValueError(f"{who}: model_out is fp32 or bf16, got {model_out.dtype}")
    shape = model_out.shape
    if ref_out is not None:
        _expect(who, "ref_out", ref_out, shape, model_out.dtype)
    _expect(who, "x_t", x_t, shape)
    _expect(who, "sqrt_1mac", sqrt_1mac, shape[:1])
    if mixing_logit is None:
        if ref_mixing_logit is not None:
            raise ValueError(f"{who}: ref_mixing_logit without mixing_logit")
    else:
        if ref_mixing_logit is None and ref_out is not None:
            raise ValueError(f"{who}: mixing_logit needs ref_mixing_logit, the reference network's own (frozen) one")
        for name, t in (("mixing_logit", mixing_logit), ("ref_mixing_logit", ref_mixing_logit)):
            if t is not None and (t.dtype != torch.float32 or t.numel() != shape[1]):
                raise ValueError(f"{who}: {name} holds {shape[1]} fp32 values, one a channel, got {tuple(t.shape)} {t.dtype}")


def _check_constants(who, **tensors):
    for name, t in tensors.items():
        if t is not None and t.requires_grad:
            raise ValueError(f"{who}: {name} requires a gradient, but only model_out and mixing_logit get one: detach it")


def _check_device(who, *tensors) -> int:
    index = tensors[0].get_device()
    if index < 0 or not tensors[0].is_cuda:
        raise ValueError(f"{who}: tensors live on a GPU, got {tensors[0].device}")
    for t in tensors:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{who}: all tensors live on one device, got {tensors[0].device} and {t.device}")
    return index


@functools.lru_cache(maxsize=256)
def _workspace_bytes(B: int, Cc: int, HW: int, mixed: bool) -> int:
    n = C.c_size_t(0)
    _lib.check(_lib.lib().ddmi_train_loss_workspace_bytes(B, Cc, HW, int(mixed), C.byref(n)))
    return n.value


def _flat(t):
    return None if t is None else (t.detach() if t.requires_grad else t).contiguous()


def _launch(entry, tensors, extra, args, stats, g, grads, mixed):
    """One call of a loss's C entry point: ((loss, *statistics), (d_model_out, d_logit, what it takes to ask for them again)).  tensors:
    model_out, ref_out, x_t, noise / x_prev, sqrt_1mac, mixing_logit, ref_mixing_logit, weight - contiguous; extra: the tensors, args: the
    numbers behind them; stats: rows of each statistic; g: the upstream gradient (None: 1); grads, mixed: whether the output's / the logit's
    gradient is wanted."""
    out, logit = tensors[0], tensors[5]
    B, Cc, dev = out.shape[0], out.shape[1], out.device
    HW = out.numel() // (B * Cc)
    d_out = torch.empty_like(out) if grads else None
    d_logit = torch.empty_like(logit) if mixed else None
    results = [torch.empty((), dtype=torch.float32, device=dev)] + [torch.empty((n,), dtype=torch.float32, device=dev) for n in stats]
    ws = torch.empty(_workspace_bytes(B, Cc, HW, logit is not None), dtype=torch.uint8, device=dev)
    given = _lib.LossIn(*map(_p, tensors), HW, Cc, _OUT_TYPES[out.dtype])
    at, workspace, outputs = list(map(_p, extra)), (ws.data_ptr(), ws.numel()), (_p(d_out), _p(d_logit))
    _lib.check(entry(C.byref(given), *args[0], *at, *args[1], _p(g), *workspace, *map(_p, results), *outputs, _lib.raw_stream(out.get_device())))
    again = None
    if grads and out.dtype != torch.float32:      # (the noise's rows are the preference loss's, the transition is the policy loss's)
        again = (C.byref(given), B, tensors[3].shape[0], at[0] if at else None), workspace, outputs, ws
    return results, (d_out, d_logit, again)


class LossFn(torch.autograd.Function):
    """A loss that is computed already, its gradients for an upstream gradient of 1 along with it.  The first backward hands those out.  Where
    the upstream gradient, which only the device knows, is another, fp32 gradients are multiplied in place, and bf16 ones are computed again from
    the inputs and the sums in the forward's workspace: multiplied, they would be rounded to bf16 twice.  A later backward (retain_graph) is a
    call of its own from the saved inputs, as is one that is captured apart from its forward: each replay of it would multiply once more."""

    @staticmethod
    def forward(ctx, model_out, mixing_logit, loss, grads, again, capture):      # loss, grads in lists: they are no inputs
        entry, tensors, extra, *rest = again
        saved = tensors + extra
        ctx.beside = {i: t for i, t in enumerate(saved) if t is not None and t.is_inference()}      # autograd does not save these itself
        ctx.save_for_backward(*(saved if not ctx.beside else [None if i in ctx.beside else t for i, t in enumerate(saved)]))
        ctx.grads, ctx.again, ctx.index, ctx.capture = grads, (entry, rest), model_out.get_device(), capture
        if grads and grads[2] and torch._C._autograd._top_saved_tensors_default_hooks(False):
            ctx.grads = None      # a hook moves the inputs that these would be computed again from: as for a later backward then
        return loss[0]

    @staticmethod
    def backward(ctx, g):
        return LossFn._with_graph(ctx, g) if torch.is_grad_enabled() else LossFn._gradients(ctx, g)

    @staticmethod
    def _gradients(ctx, g):
        with _lib.on_device(ctx.index) if torch._C._cuda_getDevice() != ctx.index else _HERE:
            stream = torch._C._cuda_getCurrentRawStream(ctx.index)
            capture = _lib.capture_id(stream) if stream else 0
            if capture and capture != ctx.capture:      # a backward alone is captured: of a graph that was not looked at when it was built
                _check_graphs([n for n, _ in ctx.next_functions])
            if not g.is_contiguous():
                g = g.contiguous()
            if ctx.grads is not None and capture == ctx.capture:
                (d_out, d_logit, again), ctx.grads = ctx.grads, None
                if again is None:
                    _lib.check(_lib.lib().ddmi_train_loss_scale(g.data_ptr(), d_out.data_ptr(), _lib.DTYPE_F32, d_out.numel(), _p(d_logit),
                                                                0 if d_logit is None else d_logit.numel(), stream))
                else:
                    ctx.saved_tensors      # the inputs are read where the forward had them: raises where one was changed since
                    inputs, workspace, outputs, _ = again
                    _lib.check(_lib.lib().ddmi_train_loss_again(*inputs, g.data_ptr(), *workspace, *outputs, stream))
            else:
                saved, (entry, (args, stats, mixed)) = ctx.saved_tensors, ctx.again
                saved = tuple(ctx.beside.get(i, t) for i, t in enumerate(saved))
                d_out, d_logit, _ = _launch(entry, saved[:8], saved[8:], args, stats, g, True, mixed)[1]
        return d_out, d_logit, None, None, None, None

    _with_graph = staticmethod(once_differentiable(_gradients.__func__))      # create_graph: a second derivative through here raises


# A leaf's gradient is added on the stream that was current when the first graph on that leaf was built, as long as such a graph lives.  If that
# is the default stream, a captured backward of the leaf would draw it into the capture, which ends the process.  Python cannot ask a node for
# its stream, so what these losses see is kept: a leaf that is given to a loss has the first loss's stream noted on its node (gone with the
# node), and the losses built on the default stream are known while they live, and a capture walks their graphs for the leaves behind a network.  A
# capture that finds one of its own leaves there is refused before anything is recorded.  Graphs that no loss of this module ends are not seen.
_FIRST_STREAM = "ddmi: stream of the first loss"
_DEFAULT = 0


class _Living:
    """Objects for as long as something else holds them; adding one costs an append, the dead are swept out now and then."""

    def __init__(self):
        self.refs, self.sweep = [], 64

    def add(self, node):
        self.refs.append(weakref.ref(node))
        if len(self.refs) > self.sweep:
            self.refs = [r for r in self.refs if r() is not None]
            self.sweep = max(64, 2 * len(self.refs))

    def __iter__(self):
        return iter([n for n in (r() for r in self.refs) if n is not None])

    def __len__(self):
        return len(list(iter(self)))


_on_default_stream = _Living()
_REFUSED = ("fine-tuning loss: captured while the graph of an eager loss of the same tensors, built on the default stream, lives (or another graph "
            "that keeps their accumulation nodes since): drop it first, or build it on a side stream")


def _mark_leaves(loss, *inputs, stream=_DEFAULT):
    for t, (node, _) in zip(inputs, loss.grad_fn.next_functions):
        if node is not None and t.is_leaf:
            node.metadata.setdefault(_FIRST_STREAM, stream)


def _check_leaves(*inputs):
    if any(torch.autograd.graph.get_gradient_edge(t).node.metadata.get(_FIRST_STREAM) == _DEFAULT
           for t in inputs if t is not None and t.requires_grad and t.is_leaf):
        raise RuntimeError(_REFUSED)


def _accumulation_nodes(starts):
    """The accumulation nodes behind some nodes of a graph, by identity (a node's Python object is one as long as it is held)."""
    seen, found, todo = {}, {}, [n for n in starts if n is not None]
    while todo:
        node = todo.pop()
        if id(node) in seen:
            continue
        seen[id(node)] = node
        if not node.next_functions and hasattr(node, "variable"):
            found[id(node)] = node
        todo += [n for n, _ in node.next_functions if n is not None]
    return found


def _meets_default_stream(nodes) -> bool:
    """Whether the graph behind `nodes` meets one of a living loss on the default stream."""
    losses = list(_on_default_stream)
    if not losses:
        return False
    old = {k: n for k, n in _accumulation_nodes(losses).items() if n.metadata.get(_FIRST_STREAM, _DEFAULT) == _DEFAULT}
    return bool(old.keys() & _accumulation_nodes(nodes).keys())


def _check_graphs(nodes):
    if _meets_default_stream(nodes):
        nodes.clear()      # the error's traceback keeps none of them alive
        raise RuntimeError(_REFUSED)


def may_be_captured(leaves) -> bool:
    """Whether a backward that ends in these leaves may be captured now: not while an eager loss on the default stream reaches one of them."""
    return not _meets_default_stream([torch.autograd.graph.get_gradient_edge(t).node for t in leaves if t.requires_grad])


def _loss(entry, model_out, mixing_logit, others, extra, args, stats):
    """(loss, *statistics), the loss differentiable in model_out and mixing_logit where they ask for it."""
    ref_out, x_t, second, sqrt_1mac, ref_mixing_logit, weight = others
    tensors = tuple(map(_flat, (model_out, ref_out, x_t, second, sqrt_1mac, mixing_logit, ref_mixing_logit, weight)))
    extra = tuple(map(_flat, extra))
    mixed = mixing_logit is not None and mixing_logit.requires_grad
    if not (torch.is_grad_enabled() and (model_out.requires_grad or mixed)):
        return _launch(entry, tensors, extra, args, stats, None, False, False)[0]
    stream = _lib.raw_stream(model_out.get_device())
    capture = _lib.capture_id(stream)
    if capture:
        _check_leaves(model_out, mixing_logit)
        _check_graphs([torch.autograd.graph.get_gradient_edge(t).node for t in (model_out, mixing_logit) if t is not None and t.requires_grad])
    results, grads = _launch(entry, tensors, extra, args, stats, None, True, mixed)
    loss = LossFn.apply(model_out, mixing_logit, results[:1], grads, (entry, tensors, extra, args, stats, mixed), capture)
    _mark_leaves(loss, model_out, mixing_logit, stream=stream)
    if stream == _DEFAULT:
        _on_default_stream.add(loss.grad_fn)
    return [loss] + results[1:]


def preference_loss(model_out, ref_out, x_t, noise, sqrt_1mac, beta, mixing_logit=None, ref_mixing_logit=None, weight=None,
                    label_smoothing=0.0) -> PreferenceLoss:
    """The preference loss of `pairs` pairs: rows [0, pairs) of model_out, ref_out, x_t [2 pairs, C, ...] and sqrt_1mac [2 pairs] belong to
    the preferred latents, rows [pairs, 2 pairs) to the rejected ones.

        e      = mean((prediction - noise)^2) a sample
        margin = -beta / 2 ((e - e_ref) of the preferred - (e - e_ref) of the rejected)
        loss   = the weighted mean over the pairs of -(1 - label_smoothing) log sigma(margin) - label_smoothing log sigma(-margin)

    noise: [2 pairs, C, ...], or [pairs, C, ...] where both samples of a pair got the same noise.  weight [pairs]: a pair whose weight is not
    > 0 is left out - nothing of it is read (it may hold NaN), its gradient is zero.  Differentiable in model_out and mixing_logit."""
    who = "preference_loss"
    _check_outputs(who, model_out, ref_out, x_t, sqrt_1mac, mixing_logit, ref_mixing_logit)
    if ref_out is None:
        raise ValueError(f"{who}: ref_out is the reference network's output")
    if model_out.shape[0] % 2:
        raise ValueError(f"{who}: model_out holds pairs, got {model_out.shape[0]} samples")
    pairs = model_out.shape[0] // 2
    if not isinstance(noise, torch.Tensor) or noise.dim() < 1 or noise.shape[0] not in (pairs, 2 * pairs):
        raise ValueError(f"{who}: noise has {pairs} (shared by a pair) or {2 * pairs} rows")
    _expect(who, "noise", noise, (noise.shape[0],) + model_out.shape[1:])
    if weight is not None:
        _expect(who, "weight", weight, (pairs,))
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not math.isfinite(beta) or not 0.0 <= label_smoothing <= 1.0:
        raise ValueError(f"{who}: beta is finite and label_smoothing in [0, 1], got {beta}, {label_smoothing}")
    _check_constants(who, ref_out=ref_out, x_t=x_t, noise=noise, sqrt_1mac=sqrt_1mac, ref_mixing_logit=ref_mixing_logit, weight=weight)
    if forward_ad._current_level >= 0:
        _lib.refuse_tangents(who, model_out, ref_out, x_t, noise, sqrt_1mac, mixing_logit, ref_mixing_logit, weight)
    dev = _check_device(who, model_out, ref_out, x_t, noise, sqrt_1mac, mixing_logit, ref_mixing_logit, weight)
    with _lib.on_device(dev):
        _lib.init_device(dev)
        return PreferenceLoss(*_loss(_lib.lib().ddmi_train_pref_loss, model_out, mixing_logit, (ref_out, x_t, noise, sqrt_1mac, ref_mixing_logit, weight),
                                     (), ((pairs, noise.shape[0]), (beta, label_smoothing)), (pairs, 2 * pairs)))


def _check_transition(who, model_out, x_prev, transition, weight, **rows):
    B = model_out.shape[0]
    _expect(who, "x_prev", x_prev, model_out.shape)
    _expect(who, "transition", transition, (B, 3))
    for name, t in dict(rows, weight=weight).items():
        if t is not None or name != "weight":
            _expect(who, name, t, (B,))


def policy_loss(model_out, x_t, x_prev, transition, sqrt_1mac, logp_old, advantage, clip_range, ref_out=None, kl_coef=0.0, mixing_logit=None,
                ref_mixing_logit=None, weight=None) -> PolicyLoss:
    """The clipped policy loss of B denoising transitions x_t -> x_prev (both [B, C, ...]) that an earlier state of the network sampled.

        mu    = A x_t + E prediction, deviation s, with transition [B, 3] = (A, E, s) (DDPM.transition_coefs)
        logp  = mean over the values of log N(x_prev; mu, s^2),   ratio = exp(logp - logp_old)
        kl    = mean((mu - mu_ref)^2) / (2 s^2)                   (0 without ref_out)
        loss  = the weighted mean of max(-advantage ratio, -advantage clip(ratio, 1 - clip_range, 1 + clip_range)) + kl_coef kl

    logp_old [B] is what `transition_log_prob` gave when the transition was sampled.  A transition with s = 0 (a chain's last step) has no
    density and is left out, as is one whose weight [B] is not > 0; a negative or NaN deviation shows as NaN.  Differentiable in model_out and mixing_logit."""
    who = "policy_loss"
    _check_outputs(who, model_out, ref_out, x_t, sqrt_1mac, mixing_logit, ref_mixing_logit)
    _check_transition(who, model_out, x_prev, transition, weight, logp_old=logp_old, advantage=advantage)
    clip_range, kl_coef = float(clip_range), float(kl_coef)
    if not clip_range >= 0.0 or not math.isfinite(kl_coef):
        raise ValueError(f"{who}: clip_range >= 0 and kl_coef finite, got {clip_range}, {kl_coef}")
    if kl_coef != 0.0 and ref_out is None:
        raise ValueError(f"{who}: kl_coef without ref_out, the reference network's output")
    _check_constants(who, ref_out=ref_out, x_t=x_t, x_prev=x_prev, transition=transition, sqrt_1mac=sqrt_1mac, logp_old=logp_old, advantage=advantage,
                     ref_mixing_logit=ref_mixing_logit, weight=weight)
    if forward_ad._current_level >= 0:
        _lib.refuse_tangents(who, model_out, ref_out, x_t, x_prev, transition, sqrt_1mac, logp_old, advantage, mixing_logit, ref_mixing_logit, weight)
    dev = _check_device(who, model_out, ref_out, x_t, x_prev, transition, sqrt_1mac, logp_old, advantage, mixing_logit, ref_mixing_logit, weight)
    with _lib.on_device(dev):
        _lib.init_device(dev)
        B = model_out.shape[0]
        return PolicyLoss(*_loss(_lib.lib().ddmi_train_policy_loss, model_out, mixing_logit,
                                 (ref_out, x_t, x_prev, sqrt_1mac, ref_mixing_logit, weight), (transition, logp_old, advantage),
                                 ((B,), (clip_range, kl_coef)), (B, B, B)))


def transition_log_prob(model_out, x_t, x_prev, transition, sqrt_1mac, mixing_logit=None, weight=None) -> torch.Tensor:
    """logp [B] of `policy_loss` alone (no gradient): what a rollout records as `logp_old`."""
    who = "transition_log_prob"
    _check_outputs(who, model_out, None, x_t, sqrt_1mac, mixing_logit, None)
    _check_transition(who, model_out, x_prev, transition, weight)
    if forward_ad._current_level >= 0:
        _lib.refuse_tangents(who, model_out, x_t, x_prev, transition, sqrt_1mac, mixing_logit, weight)
    dev = _check_device(who, model_out, x_t, x_prev, transition, sqrt_1mac, mixing_logit, weight)
    with _lib.on_device(dev):
        _lib.init_device(dev)
        B, Cc = model_out.shape[:2]
        HW = model_out.numel() // (B * Cc)
        tensors = tuple(map(_flat, (model_out, None, x_t, x_prev, sqrt_1mac, mixing_logit, None, weight)))
        transition = _flat(transition)
        logp = torch.empty((B,), dtype=torch.float32, device=model_out.device)
        ws = torch.empty(_workspace_bytes(B, Cc, HW, mixing_logit is not None), dtype=torch.uint8, device=model_out.device)
        given = _lib.LossIn(*map(_p, tensors), HW, Cc, _OUT_TYPES[model_out.dtype])
        _lib.check(_lib.lib().ddmi_train_policy_loss(C.byref(given), B, transition.data_ptr(), None, None, 0.0, 0.0, None, ws.data_ptr(), ws.numel(), None,
                                                     logp.data_ptr(), None, None, None, None, _lib.raw_stream(dev)))
        return logp
