"""The fine-tuning operators without a GPU: what they refuse, the 8-bit moments' format, transition coefficients."""
import ctypes as C
import gc
import math

import numpy as np
import pytest
import torch

import finetune_ref as R
from ddmi_amd import _lib, finetune
from ddmi_amd.ddpm import DDPM, ddim_time_pairs
from ddmi_amd.finetune import policy_loss, preference_loss, transition_log_prob
from ddmi_amd.optim import AdamW, adamw_step, blocks_of, decode_moment, encode_moment


def pref_args(**kw):
    d = R.make("pref", 4, 3, 5)
    d.update(kw)
    return d


def policy_args(**kw):
    d = R.make("policy", 4, 3, 5)
    d.update(kw)
    return d


@pytest.mark.parametrize("change,message", [
    (dict(model_out=torch.zeros(4)), r"non-empty \[B, C"),
    (dict(model_out=torch.zeros(0, 3, 5)), "non-empty"),
    (dict(model_out=torch.zeros(4, 3, 5, dtype=torch.float16)), "fp32 or bf16"),
    (dict(ref_out=torch.zeros(4, 3, 5, dtype=torch.bfloat16)), "ref_out is torch.bfloat16"),
    (dict(ref_out=torch.zeros(4, 3, 4)), "ref_out has shape"),
    (dict(ref_out=None), "reference network's output"),
    (dict(x_t=torch.zeros(4, 3, 5, dtype=torch.bfloat16)), "x_t is"),
    (dict(noise=torch.zeros(3, 3, 5)), "noise has 2 .* or 4 rows"),
    (dict(noise=torch.zeros(2, 3, 4)), "noise has shape"),
    (dict(sqrt_1mac=torch.zeros(2)), "sqrt_1mac has shape"),
    (dict(ref_mixing_logit=None), "needs ref_mixing_logit"),
    (dict(mixing_logit=None), "ref_mixing_logit without"),
    (dict(mixing_logit=torch.zeros(4)), "mixing_logit holds 3"),
    (dict(weight=torch.ones(4)), "weight has shape"),
    (dict(beta=float("nan")), "beta"),
    (dict(label_smoothing=1.5), "label_smoothing"),
    (dict(ref_out=torch.zeros(4, 3, 5, requires_grad=True)), "ref_out requires a gradient"),
    (dict(), "live on a GPU"),
])
def test_preference_loss_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        preference_loss(**pref_args(**change))


def test_preference_loss_refuses_an_odd_batch():
    d = R.make("pref", 4, 3, 5)
    d = {k: (t[:3] if isinstance(t, torch.Tensor) and t.shape[:1] == (4,) else t) for k, t in d.items()}
    with pytest.raises(ValueError, match="holds pairs, got 3"):
        preference_loss(**d)


@pytest.mark.parametrize("change,message", [
    (dict(x_prev=torch.zeros(4, 3, 4)), "x_prev has shape"),
    (dict(transition=torch.zeros(4, 2)), "transition has shape"),
    (dict(transition=torch.zeros(4, 3, dtype=torch.float64)), "transition is"),
    (dict(logp_old=torch.zeros(3)), "logp_old has shape"),
    (dict(advantage=None), "advantage is a tensor"),
    (dict(clip_range=-0.1), "clip_range"),
    (dict(clip_range=float("nan")), "clip_range"),
    (dict(ref_out=None), "kl_coef without ref_out"),
    (dict(weight=torch.ones(4, dtype=torch.bool)), "weight is"),
    (dict(advantage=torch.zeros(4, requires_grad=True)), "advantage requires a gradient"),
    (dict(), "live on a GPU"),
])
def test_policy_loss_refuses(change, message):
    with pytest.raises(ValueError, match=message):
        policy_loss(**policy_args(**change))


def test_transition_log_prob_refuses():
    d = policy_args()
    with pytest.raises(ValueError, match="live on a GPU"):
        transition_log_prob(d["model_out"], d["x_t"], d["x_prev"], d["transition"], d["sqrt_1mac"], d["mixing_logit"])
    with pytest.raises(ValueError, match="weight has shape"):
        transition_log_prob(d["model_out"], d["x_t"], d["x_prev"], d["transition"], d["sqrt_1mac"], d["mixing_logit"], torch.ones(3))


def adam_args(n=5, bits=32, **kw):
    z = lambda: torch.zeros(n)      # noqa: E731
    d = dict(params=[z()], grads=[z()], exp_avgs=[z()], exp_avg_sqs=[z()], step=1, lr=1e-3)
    if bits == 8:
        e = lambda: torch.zeros(n, dtype=torch.uint8).view(torch.float8_e4m3fn)      # noqa: E731
        d.update(exp_avgs=[e()], exp_avg_sqs=[e()], exp_avg_scales=[torch.ones(blocks_of(n))], exp_avg_sq_scales=[torch.ones(blocks_of(n))])
    d.update(kw)
    return d


@pytest.mark.parametrize("args,message", [
    (adam_args(grads=[]), "have"),
    (adam_args(params=[torch.zeros(5, dtype=torch.float64)]), "fp32 or bf16"),
    (adam_args(grads=[torch.zeros(5, dtype=torch.float16)]), "fp32 or bf16"),
    (adam_args(grads=[torch.zeros(4)]), "gradient has another number"),
    (adam_args(grads=[torch.zeros(1, 5)]), "another shape"),
    (adam_args(exp_avgs=[torch.zeros(6)]), "exp_avg has another number"),
    (adam_args(exp_avgs=[torch.zeros(5, dtype=torch.bfloat16)]), "all fp32 or all float8"),
    (adam_args(params=[torch.zeros(10)[::2]]), "contiguous"),
    (adam_args(step=0), "step counts from 1"),
    (adam_args(betas=(1.0, 0.9)), "betas"),
    (adam_args(exp_avg_scales=[torch.ones(1)]), "fp32 moments have no scales"),
    (adam_args(bits=8, exp_avg_scales=None), "need exp_avg_scales"),
    (adam_args(300, bits=8, exp_avg_scales=[torch.ones(1)]), "one for each 256"),
    (adam_args(), "live on one GPU"),
])
def test_adamw_step_refuses(args, message):
    with pytest.raises(ValueError, match=message):
        adamw_step(**args)


def test_adamw_step_of_nothing():
    adamw_step([], [], [], [], 1, lr=1e-3)


def test_adamw_refuses():
    p = torch.nn.Parameter(torch.zeros(4))
    for kw, message in ((dict(params=[p], state_bits=16), "32 or 8"), (dict(params=[]), "no parameters"), (dict(params=[p, p]), "given twice"),
                        (dict(params=[{"params": [p], "momentum": 1}]), "momentum"), (dict(params=[torch.zeros(4, dtype=torch.float16)]), "fp32 or bf16")):
        with pytest.raises(ValueError, match=message):
            AdamW(**kw)


def test_c_entries_refuse():
    L, ws = _lib.lib(), C.c_size_t(0)
    one = C.c_void_p(64)
    for args in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 1)):
        assert L.ddmi_train_loss_workspace_bytes(*args, C.byref(ws)) == 1
    assert L.ddmi_train_loss_workspace_bytes(4, 3, 5, 1, C.byref(ws)) == 0 and ws.value > 0
    s = _lib.LossIn(64, 64, 64, 64, 64, 64, 64, None, 5, 3, 0)

    def pref(pairs=2, rows=2, a=0.0, at=64, size=None, d_out=one, d_logit=one):
        return L.ddmi_train_pref_loss(C.byref(s), pairs, rows, 1.0, a, None, C.c_void_p(at), ws.value if size is None else size, one, one, one, d_out,
                                      d_logit, None)

    assert pref(size=ws.value - 1) == 1 and pref(at=65) == 1 and pref(rows=3) == 1 and pref(a=2.0) == 1 and pref(pairs=0) == 1 and pref(d_out=None) == 1
    s.out_dtype = 7
    assert pref() == 1
    s.out_dtype, s.ref_mixing_logit = 0, None
    assert pref() == 1
    s.ref_mixing_logit, s.ref_out = 64, None
    assert pref() == 1

    def policy(old=one, adv=one, kl=0.0, clip=0.1, loss=one, d_out=None, d_logit=None):
        return L.ddmi_train_policy_loss(C.byref(s), 4, one, old, adv, clip, kl, None, one, ws.value, loss, one, one, one, d_out, d_logit, None)

    assert policy(kl=0.5) == 1 and policy(adv=None) == 1 and policy(clip=-1.0) == 1 and policy(loss=None) == 1       # KL without a reference first
    assert policy(old=None, adv=None, d_out=one) == 1 and policy(d_logit=one) == 1
    s.mixing_logit = s.ref_mixing_logit = None
    assert policy(d_out=one, d_logit=one) == 1
    assert L.ddmi_train_loss_scale(None, one, 0, 4, None, 0, None) == 1 and L.ddmi_train_loss_scale(one, one, 0, 0, None, 0, None) == 1
    assert L.ddmi_debug_loss_polls(-1) == 1
    e = np.zeros(1, dtype=[("p", "u8", 6), ("n", "i8", 2), ("f", "f8", 2), ("i", "i8")])
    assert e.itemsize == 88
    e["p"], e["n"] = 64, [4, 1]
    adam = lambda bits=32, pd=0, b1=0.9, n=1: L.ddmi_train_adamw_multi(e.ctypes.data, n, b1, 0.9, 1e-8, 1.0, 0, pd, 0, bits, None)      # noqa: E731
    assert adam(bits=16) == 1 and adam(pd=2) == 1 and adam(b1=1.0) == 1 and adam(n=-1) == 1
    e["p"][0, 4] = 0
    assert adam(bits=8) == 1
    e["p"][0, 0] = 66
    assert adam() == 1
    e["p"][0, 0], e["n"][0, 1] = 64, 0
    assert adam() == 1


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import shutil
    import subprocess
    from ddmi_amd import optim
    fields = lambda name, names: "".join(f'_Static_assert(offsetof({name}, {f}) == {o}, "{f}");\n' for f, o in names)      # noqa: E731
    text = '#include "ddmi_hip.h"\n' + f"_Static_assert(sizeof(ddmi_loss_in) == {C.sizeof(_lib.LossIn)}, \"\");\n" + \
        f"_Static_assert(sizeof(ddmi_adamw_tensor) == {optim._ENTRY.itemsize}, \"\");\n" + \
        fields("ddmi_loss_in", [(n, getattr(_lib.LossIn, n).offset) for n, _ in _lib.LossIn._fields_]) + \
        fields("ddmi_adamw_tensor", [(n, optim._ENTRY.fields[n][1]) for n in optim._ENTRY.names])
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no gcc")
    src = tmp_path / "h.c"
    src.write_text(text)
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([gcc, "-std=c11", "-fsyntax-only", "-I", os.path.join(root, "include"), str(src)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


@pytest.mark.parametrize("n", [1, 255, 256, 257, 1000])
@pytest.mark.parametrize("root", [False, True])
def test_moments_round_trip(n, root):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g) * torch.exp2(torch.randint(-8, 8, (n,), generator=g).float())
    x = x * x if root else x
    x[::7] = 0.0
    codes, scales = encode_moment(x, root)
    assert codes.dtype == torch.float8_e4m3fn and codes.shape == (n,) and scales.shape == (blocks_of(n),)
    assert torch.equal(scales, R.block_scales((x.sqrt() if root else x).double()).float())
    y = decode_moment(codes, scales, root)
    s = scales.repeat_interleave(256)[:n].double()
    a, b = (x.double().sqrt(), y.double().sqrt()) if root else (x.double(), y.double())
    # half a step of the code (2^-4 of a value, 2^-10 of the scale below the least normal one), what a root is raised to the least code by,
    # and the roots' own roundings
    assert ((a - b).abs() <= a.abs() * 2.0 ** -4 + s * (2.0 ** -9 if root else 2.0 ** -10) + 2 * R.U * a.abs()).all()
    assert ((y > 0) == (x > 0)).all() if root else (y[x == 0] == 0).all()
    again, scales2 = encode_moment(y, root)
    # a value that came out of the 8-bit state goes back into it unchanged
    assert torch.equal(decode_moment(again, scales2, root), y)


def test_transition_coefs_give_the_samplers_mean():
    """x_prev of a sampler's step without noise, written out (ddpm.py:248-255, 353-369), against A x_t + E eps."""
    d = DDPM(model=None, timesteps=40, sampling_timesteps=10, ddim_sampling_eta=0.7, channels=2)
    x, eps = 0.37, -1.21
    for t in (39, 17, 1, 0):
        A, E, s = d.transition_coefs(t)
        x0 = float(d.sqrt_recip_alphas_cumprod[t]) * x - float(d.sqrt_recipm1_alphas_cumprod[t]) * eps
        mean = float(d.posterior_mean_coef1[t]) * x0 + float(d.posterior_mean_coef2[t]) * x
        assert abs(A * x + E * eps - mean) <= 1e-6 * (abs(x0) + abs(x)) and (s == 0.0) == (t == 0)
    for t, t_next in ddim_time_pairs(40, 10):
        A, E, s = d.transition_coefs(t, t_next)
        k = d._base_coefs(t) if t_next < 0 else d.ddim_coefs(t, t_next)
        x0 = k.sqrt_recip_ac * x - k.sqrt_recipm1_ac * eps
        mean = x0 if t_next < 0 else k.sqrt_ac_next * x0 + k.c_dir * eps
        assert abs(A * x + E * eps - mean) <= 1e-6 * (abs(x0) + abs(x)) and math.isclose(s, 0.0 if t_next < 0 else k.sigma)
    with pytest.raises(ValueError, match="clip"):
        DDPM(model=None, timesteps=40, sampling_timesteps=40, clip_denoised=True, channels=2).transition_coefs(3)


def test_leaves_are_marked_as_long_as_their_graph_lives():
    a, b = torch.zeros(3, requires_grad=True), torch.zeros(3, requires_grad=True)
    inner = a * 2
    loss = torch.mul(inner, b)                       # a graph node with an inner and a leaf input, as a loss has them
    finetune._check_leaves(a, b)
    finetune._mark_leaves(loss, inner, b)
    finetune._check_leaves(a, None)
    finetune._check_leaves(inner, None)
    with pytest.raises(RuntimeError, match="captured while"):
        finetune._check_leaves(inner, b)
    del loss
    gc.collect()
    finetune._check_leaves(inner, b)
