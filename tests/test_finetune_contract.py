"""Calls of the fine-tuning operators that are refused, and rules of their plans, without a GPU."""
import ctypes as C
import math

import pytest
import torch
from torch.autograd import forward_ad

import finetune_ref as R
from ddmi_amd import _lib, finetune
from ddmi_amd.finetune import policy_loss, preference_loss, transition_log_prob
from ddmi_amd.optim import adamw_step


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
