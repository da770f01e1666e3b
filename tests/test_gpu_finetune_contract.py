"""What the fine-tuning operators promise at the edges of their arguments, on the GPU."""
import math

import pytest
import torch

import finetune_ref as R
from ddmi_amd.finetune import transition_log_prob
from test_gpu_finetune import DEV, call

pytestmark = pytest.mark.gpu
# two passes; one pass
BOTH = [(6, 4, 9), (140, 3, 33001)]


@pytest.mark.parametrize("s", [math.nan, -0.1])
@pytest.mark.parametrize("B,C,T", BOTH)
def test_a_deviation_that_is_none_shows(s, B, C, T):
    """Only a deviation of zero leaves a transition out; a broken one is not averaged away."""
    d = R.make("policy", B, C, T, seed=5, device=DEV)
    d["transition"][2, 2] = s
    got = call("policy", d)
    assert math.isnan(got["loss"].item()) and math.isnan(float(got["logp"][2]))
    assert torch.isnan(got["d_model_out"][2]).all() and torch.isnan(got["d_logit"]).all()
    other = torch.arange(B, device=DEV) != 2
    assert torch.isfinite(got["logp"][other]).all() and torch.isfinite(got["d_model_out"][other]).all()
    logp = transition_log_prob(d["model_out"], d["x_t"], d["x_prev"], d["transition"], d["sqrt_1mac"], d["mixing_logit"])
    assert torch.isnan(logp).tolist() == (~other).tolist()
    d["weight"] = other.float()                       # left out by its weight, it does not show
    got = call("policy", d)
    assert torch.isfinite(got["loss"]) and not got["d_model_out"][2].any() and float(got["logp"][2]) == 0.0
