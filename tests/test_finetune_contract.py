"""Calls of the fine-tuning operators that are refused, and rules of their plans, without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

import finetune_ref as R
from ddmi_amd import finetune
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
