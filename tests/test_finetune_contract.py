"""Calls of the fine-tuning operators that are refused, and rules of their plans, without a GPU."""
import ctypes as C
import gc
import math
import types

import numpy as np
import pytest
import torch
import torch.utils.checkpoint
from torch.autograd import forward_ad

import finetune_ref as R
from ddmi_amd import _lib, finetune, train
from ddmi_amd.finetune import policy_loss, preference_loss, transition_log_prob
from ddmi_amd.optim import _ENTRY, AdamW, adamw_step
from ddmi_amd.train import FlatParams, LDMTrainStep


# ---- forward-mode derivatives -------------------------------------------------------------------------------------------------------
def loss_call(op):
    """The loss and its arguments; `logp`: transition_log_prob, the policy loss's forward alone."""
    d = R.make("pref" if op == "pref" else "policy", 4, 3, 5)
    if op == "logp":
        return transition_log_prob, {k: d[k] for k in ("model_out", "x_t", "x_prev", "transition", "sqrt_1mac", "mixing_logit", "weight")}
    return (preference_loss if op == "pref" else policy_loss), d


@pytest.mark.parametrize("op,name", [(op, name) for op in ("pref", "policy", "logp") for name, t in loss_call(op)[1].items() if isinstance(t, torch.Tensor)])
def test_forward_mode_tangents_are_refused(op, name, monkeypatch):
    """A dual tensor requires no gradient: going by its pointer would give a loss without a tangent, a derivative of zero."""
    monkeypatch.setattr(finetune, "_check_device", lambda who, *tensors: pytest.fail("the tangent was not looked at"))
    loss, d = loss_call(op)
    with forward_ad.dual_level():
        d[name] = forward_ad.make_dual(d[name], torch.ones_like(d[name]))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            loss(**d)


@pytest.mark.parametrize("which", range(4))
def test_adamw_step_refuses_tangents(which):
    lists = [[torch.zeros(5)] for _ in range(4)]
    with forward_ad.dual_level():
        lists[which][0] = forward_ad.make_dual(lists[which][0], torch.ones(5))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            adamw_step(*lists, 1, lr=1e-3)


def test_no_tangent_is_no_refusal():
    """Inside a level, tensors without a tangent go on (here: to the refusal of CPU tensors)."""
    with forward_ad.dual_level():
        for op in ("pref", "policy", "logp"):
            loss, d = loss_call(op)
            with pytest.raises(ValueError, match="live on a GPU"):
                loss(**d)


# ---- numbers and pointers that no formula has ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan])
def test_factors_are_finite(value):
    """An infinite beta times the zero of a pair that is left out would put NaN into the logit's gradient."""
    loss, d = loss_call("pref")
    with pytest.raises(ValueError, match="beta is finite"):
        loss(**dict(d, beta=value))
    loss, d = loss_call("policy")
    with pytest.raises(ValueError, match="kl_coef finite"):
        loss(**dict(d, kl_coef=value))
    c = CLoss()
    assert c.pref(beta=value, size=0) == INVALID and b"beta finite" in c.error()
    assert c.policy(kl_coef=value, size=0) == INVALID and b"kl_coef finite" in c.error()


INVALID = 1


class CLoss:
    """Calls of the losses' C entries that are refused before a pointer is followed."""
    names = ("model_out", "ref_out", "x_t", "second", "sqrt_1mac", "mixing_logit", "ref_mixing_logit", "weight")

    def __init__(self, out_dtype=0):
        self.lib = _lib.lib()
        self.fields = dict({n: 64 for n in self.names}, HW=5, C=3, out_dtype=out_dtype)

    def error(self):
        return _lib.lib().ddmi_last_error()

    def pref(self, beta=1.0, dloss=64, ws=64, size=1 << 20, loss=64, margin=64, mse=64, d_out=64, d_logit=64, **fields):
        s = _lib.LossIn(**dict(self.fields, **fields))
        return self.lib.ddmi_train_pref_loss(C.byref(s), 2, 2, beta, 0.0, dloss, ws, size, loss, margin, mse, d_out, d_logit, None)

    def policy(self, transition=64, old=64, adv=64, kl_coef=0.5, dloss=64, ws=64, size=1 << 20, loss=64, logp=64, ratio=64, kl=64, d_out=64, d_logit=64,
               **fields):
        s = _lib.LossIn(**dict(self.fields, **fields))
        return self.lib.ddmi_train_policy_loss(C.byref(s), 4, transition, old, adv, 0.1, kl_coef, dloss, ws, size, loss, logp, ratio, kl, d_out, d_logit,
                                               None)


@pytest.mark.parametrize("out_dtype", [0, 1])
def test_c_losses_refuse_unaligned_pointers(out_dtype):
    """A size of zero for the workspace ends a call that gets past the pointers, so that no kernel is launched on made-up ones."""
    c = CLoss(out_dtype)
    assert c.pref(size=0) == INVALID and b"workspace" in c.error()
    assert c.policy(size=0) == INVALID and b"workspace" in c.error()
    for call, outputs in ((c.pref, ("dloss", "loss", "margin", "mse", "d_logit")),
                          (c.policy, ("transition", "old", "adv", "dloss", "loss", "logp", "ratio", "kl", "d_logit"))):
        for name in c.names + outputs + ("d_out",):
            of_output = name in ("model_out", "ref_out", "d_out")
            for at in (65,) if of_output and out_dtype == 1 else (65, 66):
                assert call(**{name: at, "size": 0}) == INVALID and b"aligned to their values" in c.error(), name
            if of_output and out_dtype == 1:                     # two bytes a value
                assert call(**{name: 66, "size": 0}) == INVALID and b"workspace" in c.error(), name


def test_c_scale_refuses_unaligned_pointers():
    scale = lambda up=64, out=64, dt=0, logit=64: _lib.lib().ddmi_train_loss_scale(up, out, dt, 4, logit, 3, None)      # noqa: E731
    for kw in (dict(up=66), dict(out=66), dict(logit=65), dict(out=65, dt=1)):
        assert scale(**kw) == INVALID and b"aligned" in _lib.lib().ddmi_last_error(), kw


def entries(n):
    e = np.zeros(n, dtype=_ENTRY)
    for k in ("param", "grad", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
        e[k] = 64
    e["numel"], e["step"], e["lr"] = 4, 1, 1e-3
    return e


def adamw_multi(e, bits=32):
    return _lib.lib().ddmi_train_adamw_multi(e.ctypes.data, len(e), 0.9, 0.999, 1e-8, 1.0, 0, 0, 0, bits, None), _lib.lib().ddmi_last_error()


@pytest.mark.parametrize("bits,names", [(32, ("param", "grad", "exp_avg", "exp_avg_sq")), (8, ("param", "grad", "exp_avg_scale", "exp_avg_sq_scale"))])
def test_c_adamw_refuses_unaligned_pointers(bits, names):
    for name in names:
        e = entries(2)
        e[name][1] = 66
        rc, text = adamw_multi(e, bits)
        assert rc == INVALID and b"aligned to their values" in text, name


def test_c_adamw_refuses_a_tensor_too_large_before_it_launches():
    """The 60th of a list whose first 48 would be a launch of their own (which no card here could run)."""
    e = entries(60)
    e["numel"][59] = 1 << 37
    rc, text = adamw_multi(e)
    assert rc == INVALID and b"more than 2^36" in text


# ---- grids -----------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("mixed", [0, 1])
def test_loss_grids_stay_below_2_to_32_threads(mixed):
    """The gradient's launch has a workgroup of 256 threads for each span, one for each channel and one for the loss: at most 2^24 - 1."""
    size = C.c_size_t(0)
    ask = lambda B, channels: _lib.lib().ddmi_train_loss_workspace_bytes(B, channels, 1, mixed, C.byref(size))      # noqa: E731
    most = 2 ** 24 - 1
    for channels in (1, 3):
        assert ask(most - 1 - channels, channels) == 0 and size.value > 0
        assert ask(most - channels, channels) == INVALID and b"too many values" in _lib.lib().ddmi_last_error()


# ---- optimizer states ------------------------------------------------------------------------------------------------------------------
def stepped(cls=torch.optim.AdamW, **kw):
    """Two groups of CPU parameters, and torch's state dict after a step over them."""
    ps = [torch.nn.Parameter(torch.full((k + 2,), 1.0)) for k in range(3)]
    opt = cls([{"params": ps[:2], "weight_decay": 0.1}, {"params": ps[2:]}], **dict(dict(lr=1e-3, betas=(0.8, 0.9), eps=1e-6), **kw))
    for p in ps:
        p.grad = torch.full_like(p, 0.5)
    opt.step()
    return ps, opt.state_dict()


def snapshot(opt):
    bits = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t      # noqa: E731
    slabs = [opt.exp_avg, opt.exp_avg_sq] + ([opt.exp_avg_scale, opt.exp_avg_sq_scale] if opt.state_bits == 8 else [])
    return [bits(t).clone() for ts in slabs for t in ts], [dict(g) for g in opt.param_groups], opt.betas, opt.eps, list(opt.steps)


def of_group(k, **kw):
    return lambda sd: sd["param_groups"][k].update(kw)


def of_state(i, **kw):
    return lambda sd: sd["state"].__setitem__(i, {k: v for k, v in dict(sd["state"].get(i, {}), **kw).items() if v is not None})


@pytest.mark.parametrize("change,message", [
    (of_group(1, amsgrad=True), "amsgrad"),
    (of_group(0, maximize=True), "maximize"),
    (of_group(0, decoupled_weight_decay=False), "part of the gradient"),
    (of_group(1, betas=(0.7, 0.9)), "same betas and eps"),
    (of_group(1, eps=1e-3), "same betas and eps"),
    (lambda sd: [g.update(betas=(1.0, 0.9)) for g in sd["param_groups"]], r"betas in \[0, 1\)"),
    (of_group(0, params=[0]), "other parameter groups"),
    (of_state(9, step=1.0, exp_avg=torch.zeros(2), exp_avg_sq=torch.zeros(2)), "state for parameters"),
    (of_state(2, exp_avg=None), "has no"),
    (of_state(1, exp_avg_sq=torch.zeros(9)), "exp_avg_sq of parameter 1 has shape"),
    (of_state(0, step=-1.0), "steps"),
])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dicts_of_other_optimizers_are_refused_and_change_nothing(change, message, bits):
    ps, sd = stepped()
    opt = AdamW([{"params": ps[:2], "weight_decay": 0.2}, {"params": ps[2:]}], lr=5e-4, state_bits=bits)
    opt.set_moments(0, torch.ones(2), torch.ones(2), 3)
    before = snapshot(opt)
    sd["param_groups"][0]["lr"] = 9.0
    change(sd)
    with pytest.raises(ValueError, match=message):
        opt.load_state_dict(sd)
    after = snapshot(opt)
    assert all(map(torch.equal, before[0], after[0])) and before[1:] == after[1:]


def test_state_dict_of_torch_loads():
    ps, sd = stepped()
    opt = AdamW([{"params": ps[:2], "weight_decay": 0.2}, {"params": ps[2:]}], lr=5e-4)
    opt.load_state_dict(sd)
    assert [g["lr"] for g in opt.param_groups] == [1e-3] * 2 and [g["weight_decay"] for g in opt.param_groups] == [0.1, 0.01]
    assert opt.betas == (0.8, 0.9) and opt.eps == 1e-6 and opt.steps == [1, 1, 1]
    for i in range(3):
        assert all(torch.equal(a, sd["state"][i][k]) for a, k in zip(opt.moments(i), ("exp_avg", "exp_avg_sq")))
    with pytest.raises(ValueError, match="part of the gradient"):
        opt.load_state_dict(stepped(torch.optim.Adam)[1])


def test_set_moments_checks_both_before_either_is_set():
    opt = AdamW([torch.zeros(4)])
    with pytest.raises(ValueError, match="exp_avg_sq"):
        opt.set_moments(0, torch.ones(4), torch.ones(5), 1)
    assert not opt.exp_avg[0].any() and opt.steps == [0]


# ---- the training step -----------------------------------------------------------------------------------------------------------------
def test_rollout_of_a_clipping_sampler_is_refused():
    """The ancestral sampler clips x_0 where the configuration says so, and then its steps have no mean A x_t + E eps."""
    host = types.SimpleNamespace(_ddpmconfig={"clip_denoised": True, "channels": 2}, num_timesteps=12, mixing_logit=None, video=False, channels=2, image_size=4,
                                 device=torch.device("cpu"), model=lambda *a: pytest.fail("the chain was begun"))
    with pytest.raises(ValueError, match="clip_denoised"):
        LDMTrainStep.rollout(host, 2)


@pytest.mark.parametrize("change,message", [(lambda r: r.pop("b"), "'b' .* is missing"), (lambda r: r.update(b=torch.ones(1)), r"'b' \(3,\) is \(1,\) there")])
def test_a_reference_of_another_model_is_refused(change, message):
    """A missing parameter used to leave a reference half filled, one of a single value to be spread over the parameter."""
    named = [("a", torch.nn.Parameter(torch.zeros(2))), ("b", torch.nn.Parameter(torch.zeros(3)))]
    kept = torch.zeros(5)
    host = types.SimpleNamespace(flat=FlatParams([p for _, p in named], "cpu"), named_parameters=lambda: named, device=torch.device("cpu"), reference=kept)
    reference = {"a": torch.ones(2), "b": torch.ones(3)}
    change(reference)
    with pytest.raises(ValueError, match=message):
        LDMTrainStep.load_training_state(host, {"reference": reference})
    assert host.reference is kept and not kept.any()


# ---- gradients asked again -------------------------------------------------------------------------------------------------------------
def test_c_loss_again_refuses():
    """A workspace of no bytes ends a call that gets past its arguments."""
    c = CLoss(1)

    def again(B=4, noise_rows=2, transition=None, dloss=64, size=0, d_out=64, d_logit=64, **fields):
        s = _lib.LossIn(**dict(c.fields, **fields))
        return c.lib.ddmi_train_loss_again(C.byref(s), B, noise_rows, transition, dloss, 64, size, d_out, d_logit, None)

    for kw in (dict(), dict(noise_rows=4), dict(transition=64, noise_rows=0), dict(transition=64, ref_out=None, ref_mixing_logit=None)):
        assert again(**kw) == INVALID and b"workspace" in c.error(), kw
    for kw, text in ((dict(dloss=None), b"null"), (dict(d_out=None), b"null"), (dict(B=3), b"neither"), (dict(noise_rows=3), b"neither"),
                     (dict(ref_out=None), b"neither"), (dict(transition=64, x_t=None), b"neither"),
                     (dict(mixing_logit=None, ref_mixing_logit=None), b"d_logit goes"), (dict(dloss=66), b"aligned"), (dict(d_logit=66), b"aligned"),
                     (dict(d_out=65), b"aligned"), (dict(transition=65), b"aligned"), (dict(x_t=66), b"aligned"), (dict(B=0, noise_rows=0), b"empty batch")):
        assert again(**kw) == INVALID and text in c.error(), (kw, c.error())


# ---- captures and the graphs that live beside them -------------------------------------------------------------------------------------
def eager_loss(model_out, mixing_logit=None, stream=0):
    """A loss's graph node as a call leaves it behind, without a launch."""
    tensors = tuple(t if t is None else t.detach() for t in (model_out, None, None, None, None, mixing_logit, None, None))
    loss = finetune.LossFn.apply(model_out, mixing_logit, [torch.zeros(())], None, (None, tensors, (), (), (), False), 0)
    finetune._mark_leaves(loss, model_out, mixing_logit, stream=stream)
    if not stream:
        finetune._on_default_stream.add(loss.grad_fn)
    return loss


def captured(model_out, mixing_logit=None):
    finetune._check_leaves(model_out, mixing_logit)
    finetune._check_graphs([torch.autograd.graph.get_gradient_edge(t).node for t in (model_out, mixing_logit) if t is not None and t.requires_grad])


def leaf():
    return torch.ones(2, 3, requires_grad=True)


@pytest.mark.parametrize("behind", [lambda w, b: (w * 2 + b) @ torch.ones(3, 3), lambda w, b: torch.utils.checkpoint.checkpoint(torch.mul, w, b, use_reentrant=False)],
                         ids=["network", "checkpointed"])
def test_a_capture_sees_the_parameters_behind_a_network(behind):
    w, b, other = leaf(), leaf(), leaf()
    loss = eager_loss(behind(w, b))                   # without a mixing logit: no leaf is an input of the loss
    with pytest.raises(RuntimeError, match="captured while"):
        captured(w.exp())
    with pytest.raises(RuntimeError, match="captured while"):
        captured(other * 2, b)
    captured(other * 2)
    captured(w.detach(), other)
    held = loss * 3                                   # whatever keeps its graph keeps the loss
    del loss
    gc.collect()
    with pytest.raises(RuntimeError, match="captured while"):
        captured(w)
    del held
    gc.collect()
    captured(w.exp() + b)


def test_a_leaf_that_a_side_stream_saw_first_may_be_captured():
    """The node is that of the first graph: a loss on the default stream that joins it later does not move it, also once it is gone."""
    w = leaf()
    first = eager_loss(w, stream=7)
    second = eager_loss(w)
    captured(w)
    del second
    gc.collect()
    captured(w)
    del first
    gc.collect()
    last = eager_loss(w)
    with pytest.raises(RuntimeError, match="captured while"):
        captured(w)
    del last
    gc.collect()
    captured(w)


def test_a_leaf_that_the_default_stream_saw_first_stays_refused_while_its_node_lives():
    w = leaf()
    first, second = eager_loss(w), eager_loss(w, stream=7)
    del first
    gc.collect()
    with pytest.raises(RuntimeError, match="captured while"):
        captured(w)
    del second
    gc.collect()
    captured(w)


def test_a_refusal_that_is_kept_keeps_no_node():
    w = leaf()
    loss = eager_loss(w * 2)
    with pytest.raises(RuntimeError) as kept:
        finetune._check_graphs([torch.autograd.graph.get_gradient_edge(w).node])
    torch.autograd.graph.get_gradient_edge(w).node.metadata["alive"] = True
    del loss
    gc.collect()
    assert not torch.autograd.graph.get_gradient_edge(w).node.metadata and "captured while" in str(kept.value)


def test_losses_on_the_default_stream_are_not_kept_alive():
    before = len(finetune._on_default_stream)
    w = leaf()
    losses = [eager_loss(w * k) for k in range(3)]
    assert len(finetune._on_default_stream) == before + 3
    del losses
    gc.collect()
    assert len(finetune._on_default_stream) == before


# ---- the one-pass form and the card ----------------------------------------------------------------------------------------------------
def plan(B, channels, hw, mixed, policy, has_ref, units):
    one, spans = C.c_int(-1), C.c_int(-1)
    assert _lib.lib().ddmi_debug_loss_plan(B, channels, hw, mixed, policy, has_ref, units, C.byref(one), C.byref(spans)) == 0
    return one.value, spans.value


@pytest.mark.parametrize("policy,has_ref", [(0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("mixed", [0, 1])
def test_workgroups_that_wait_for_each_other_fit_the_card(policy, has_ref, mixed):
    """On a card of any number of compute units: those of a sample (a pair) are no more than the units, which hold two workgroups each, and
    the launch has one and a half for each."""
    rows_of = 1 if policy else 2
    taken = {}
    for units in (0, 1, 8, 32, 64, 128, 256, 304):
        taken[units] = 0
        for B in (2, 8, 48, 140, 512, 4096):
            for channels in (1, 3, 64, 190, 1100):
                for hw in (1, 77, 1295, 2048, 4096, 33001, 1 << 20, 1 << 24):
                    if B * channels * hw > 1 << 36:           # more than any card holds: refused
                        continue
                    one, spans = plan(B, channels, hw, mixed, policy, has_ref, units)
                    taken[units] += one
                    if one:
                        assert spans * rows_of <= units and spans * B >= 1.5 * units, (units, B, channels, hw)
    assert taken[0] == 0 and all(taken[u] > 0 for u in (8, 32, 64, 128, 256)), taken


def test_smaller_cards_take_smaller_batches_in_one_pass():
    """64 x 64 x 64 latents, 16 (with KL: 32) spans a sample: 12 pairs fill the whole card, a few fill an eighth of it; 32 spans of a pair do
    not fit sixteen units."""
    assert plan(24, 64, 4096, 1, 0, 1, 256) == (1, 16) and plan(16, 64, 4096, 1, 0, 1, 256)[0] == 0
    assert plan(4, 64, 4096, 1, 0, 1, 32) == (1, 16) and plan(2, 64, 4096, 1, 0, 1, 32)[0] == 0
    assert plan(512, 64, 4096, 1, 0, 1, 16)[0] == 0 and plan(512, 64, 4096, 1, 1, 1, 32) == (1, 32)


def test_workspace_covers_every_card():
    """What a call needs does not depend on the card: a plan of one pass on some card has its room."""
    size = C.c_size_t(0)
    for B, channels, hw in ((48, 64, 2048), (4, 64, 4096), (2, 64, 4096)):
        assert _lib.lib().ddmi_train_loss_workspace_bytes(B, channels, hw, 1, C.byref(size)) == 0
        most = max(plan(B, channels, hw, 1, 0, 1, u)[1] for u in (0, 8, 32, 256))
        assert size.value >= 256 + B * most * (16 + 4)


def test_many_losses_leave_no_long_list_behind():
    w = leaf()
    kept = [eager_loss(w * k) for k in range(10)]
    for k in range(1000):
        eager_loss(w * k)
    gc.collect()
    assert len(finetune._on_default_stream.refs) <= 2 * 64 + 1 and all(n.grad_fn in list(finetune._on_default_stream) for n in kept)


def test_a_training_step_asks_before_it_captures(monkeypatch):
    """With an eager loss of the caller's alive on its parameters, a step that would record its graph runs as it is, and records later."""
    p, q = leaf(), leaf()
    assert finetune.may_be_captured([p, q])
    loss = eager_loss(p.exp())
    assert not finetune.may_be_captured([q, p]) and finetune.may_be_captured([q, p.detach()])
    monkeypatch.setattr(train._lib, "check", lambda rc: None)
    monkeypatch.setattr(train._lib, "lib", lambda: types.SimpleNamespace(ddmi_train_arena_generation=lambda *a: 0))
    monkeypatch.setattr(torch.cuda, "CUDAGraph", lambda: pytest.fail("a capture was begun"))
    z = torch.zeros(2, 3)
    host = types.SimpleNamespace(model=types.SimpleNamespace(tc=types.SimpleNamespace(h=0)), _graph_generation=0, _graphs={(2, 3): "warm"},
                                 flat=types.SimpleNamespace(params=[p, q]), _micro_body=lambda *a: "eager")
    assert LDMTrainStep._graphed_micro(host, z, z, z) == "eager" and host._graphs == {(2, 3): "warm"}
    del loss
    gc.collect()
    assert finetune.may_be_captured([p, q])
