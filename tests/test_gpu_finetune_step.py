"""The fine-tuning operators together, as a training step uses them: reference network, loss, backward through the UNet, AdamW."""
import math
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import finetune_ref as R
from ddmi_amd import initweights as iw
from ddmi_amd.train import LDMTrainStep
from helpers import TOL_FP32, named_state, rel_err

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
UNET = dict(image_size=8, in_channels=64, model_channels=32, out_channels=64, attention_resolutions=[2], num_res_blocks=1, channel_mult=[1, 2],
            num_head_channels=32)


def trainer(numerics="fp32", **kw):
    tr = LDMTrainStep(UNET, dict(timesteps=1000, channels=64, image_size=8), numerics=numerics, lr=1e-3, device=DEV, **kw)
    st = {"model." + k: v for k, v in named_state("ft.unet", [(k, tuple(p.shape)) for k, p in tr.model.state_dict().items()]).items()}
    st["mixing_logit"] = iw.normal("ft", "mixing_logit", (1, 64, 1, 1), 0.0, 0.5)
    return tr.load_state_dict(st).finalize()


def pairs(P=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn((P, 64, 8, 8), generator=g) for _ in range(3)] + [torch.randint(0, 1000, (P,), generator=g)]


def test_preference_step_gradients():
    """The slab's gradients against autograd of the formula on the same network outputs (fp32 network, torch's own loss ops)."""
    a, b = trainer(), trainer()
    for tr in (a, b):
        tr.set_reference()
        with torch.no_grad():                    # the trained network has moved from the reference
            tr.flat.data += 1e-2 * torch.randn(tr.flat.n, generator=torch.Generator().manual_seed(1)).to(DEV)
    zw, zl, noise, t = (v.to(DEV) for v in pairs())
    out = a.preference_loss_and_backward(zw, zl, beta=5.0, t=t, noise=noise, label_smoothing=0.1)
    ac, s1 = b.sqrt_ac[t].view(-1, 1, 1, 1), b.sqrt_1mac[t].view(-1, 1, 1, 1)
    x, t2, n2 = torch.cat([ac * zw + s1 * noise, ac * zl + s1 * noise]), torch.cat([t, t]), torch.cat([noise, noise])
    m = torch.cat([s1, s1]) * x
    mix = lambda o, logit: m + torch.sigmoid(logit) * (o - m)      # noqa: E731
    with b._as_reference() as logit:
        e_ref = (mix(b.model(x, t2), logit) - n2).double().square().mean((1, 2, 3))
    e = (mix(b.model(x, t2), b.mixing_logit) - n2).double().square().mean((1, 2, 3))
    h = -2.5 * ((e - e_ref)[:3] - (e - e_ref)[3:])
    loss = -(0.9 * torch.nn.functional.logsigmoid(h) + 0.1 * torch.nn.functional.logsigmoid(-h)).mean()
    loss.backward()
    loss = loss.detach()
    assert abs(float(out.loss) - float(loss)) < TOL_FP32 * float(loss)
    assert rel_err(out.margin.cpu(), h.detach().cpu()) < TOL_FP32 and rel_err(out.mse.cpu(), e.detach().cpu()) < TOL_FP32
    floor = 1e-6 * float(b.flat.grad.abs().max())
    for (k, p), (_, q) in zip(a.named_parameters(), b.named_parameters()):
        assert float((p.grad - q.grad).abs().max()) < TOL_FP32 * float(q.grad.abs().max()) + floor, k


@pytest.mark.parametrize("numerics", ["fp32", "bf16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_preference_steps_leave_the_reference_alone(numerics, bits):
    tr = trainer(numerics, optimizer_state_bits=bits)
    with pytest.raises(ValueError, match="set_reference"):
        tr.preference_step(*[v.to(DEV) for v in pairs()[:2]], beta=5.0)
    assert not tr.flat.grad.any()
    tr.set_reference()
    before, pointers = tr.flat.data.clone(), [p.data_ptr() for p in tr.flat.params]
    zw, zl, noise, t = (v.to(DEV) for v in pairs())
    out = tr.preference_step(zw, zl, beta=500.0, t=t, noise=noise)
    # the first step starts at the reference: the same network gives the same outputs, no margin, loss log 2
    assert not out.margin.any() and float(out.loss) == pytest.approx(math.log(2.0), rel=2 * R.U)
    for _ in range(3):
        out = tr.preference_step(zw, zl, beta=500.0, t=t, noise=noise)
    assert torch.equal(tr.reference, before) and [p.data_ptr() for p in tr.flat.params] == pointers
    assert torch.isfinite(out.loss) and torch.isfinite(tr.flat.data).all() and out.margin.any() and tr.opt_step == 4
    assert not torch.equal(tr.flat.data, before)
    tr.train_step(zw, t, noise)                       # ordinary training goes on with the same optimizer
    assert tr.opt_step == 5


def test_8_bit_moments_with_a_captured_micro_step():
    """use_graph: the captured micro-step fills the slab, the optimizer runs behind it; the same states as without a graph."""
    runs = []
    for graph in (False, True):
        tr = trainer(optimizer_state_bits=8, use_graph=graph)
        for k in range(4):
            zw, _, noise, t = (v.to(DEV) for v in pairs(seed=k))
            tr.train_step(zw, t, noise)
        runs.append(tr)
    assert torch.equal(runs[0].flat.data, runs[1].flat.data)
    tr = runs[1].set_reference()
    zw, zl, noise, t = (v.to(DEV) for v in pairs(seed=9))
    tr.preference_step(zw, zl, beta=10.0, t=t, noise=noise)        # twice the batch: the arena may move, graphs are made again
    tr.train_step(zw, t, noise)
    tr.train_step(zw, t, noise)
    assert torch.isfinite(tr.flat.data).all() and tr.opt_step == 7


def test_first_step_of_8_bit_moments_is_that_of_32():
    """From zero moments the parameters move by the unrounded moments: the same step up to fp32 rounding (a change of at most lr = 1e-3
    within 16 roundings, and the parameter's own two on either side)."""
    a, b = trainer(), trainer(optimizer_state_bits=8)
    zw, zl, noise, t = (v.to(DEV) for v in pairs())
    for tr in (a, b):
        tr.train_step(zw, t, noise)
    assert ((a.flat.data - b.flat.data).abs() <= 32 * R.U * 1e-3 + 4 * R.U * a.flat.data.abs()).all()
    for tr in (a, b):
        for _ in range(3):
            tr.train_step(zw, t, noise)
    assert torch.isfinite(b.flat.data).all()


def test_checkpoint_of_8_bit_moments_resumes_bit_for_bit(tmp_path):
    from ddmi_amd import checkpoint as CK
    zw, zl, noise, t = (v.to(DEV) for v in pairs())
    a = trainer(optimizer_state_bits=8)
    for _ in range(3):
        a.train_step(zw, t, noise)
    path = os.path.join(tmp_path, "ldm-last.pt")
    a.save(path)
    b = trainer(optimizer_state_bits=8)
    ck = CK.read_checkpoint(path)
    b.load_state_dict({k: v for k, v in ck["diffusion"].items() if k.startswith("model.") or k == "mixing_logit"}).finalize()
    b.load_training_state(ck)
    assert b.opt_step == 3
    for tr in (a, b):
        tr.train_step(zl, t, noise)
    assert torch.equal(a.flat.data, b.flat.data)
    for x, y in ((a.opt8.exp_avg, b.opt8.exp_avg), (a.opt8.exp_avg_sq, b.opt8.exp_avg_sq)):
        assert all(torch.equal(u.view(torch.uint8), v.view(torch.uint8)) for u, v in zip(x, y))
    c = trainer()                                     # the same file into 32-bit moments
    c.load_state_dict({k: v for k, v in ck["diffusion"].items() if k.startswith("model.") or k == "mixing_logit"}).finalize()
    c.load_training_state(ck)
    assert c.opt_step == 3 and torch.isfinite(c.flat.exp_avg).all() and c.flat.exp_avg.any()


@pytest.mark.parametrize("numerics", ["fp32", "bf16"])
@pytest.mark.parametrize("steps", [None, 6])
def test_rollout_and_policy_step(numerics, steps):
    cfg = dict(timesteps=12, channels=64, image_size=8)
    tr = LDMTrainStep(UNET, cfg, numerics=numerics, lr=1e-4, device=DEV, optimizer_state_bits=8)
    st = {"model." + k: v for k, v in named_state("ft.unet", [(k, tuple(p.shape)) for k, p in tr.model.state_dict().items()]).items()}
    tr.load_state_dict(st, strict=False).finalize().set_reference()
    r = tr.rollout(4, sampling_timesteps=steps, eta=0.8, generator=torch.Generator(DEV).manual_seed(3))
    S = steps or 12
    assert r.x_t.shape == (S, 4, 64, 8, 8) and r.logp.shape == (S, 4) and torch.isfinite(r.x_0).all()
    assert torch.equal(r.x_t[1:], r.x_prev[:-1]) and torch.equal(r.x_prev[-1], r.x_0)
    last = r.transition[:, 2] == 0
    assert last.tolist() == [False] * (S - 1) + [True] and not r.logp[last].any() and r.logp[~last].all()
    # the sampler's noise is what the log-density says it is: (x_prev - mean) / s of unit variance over 4 x 4096 values (five deviations)
    want = -0.5 - r.transition[:-1, 2].double().log() - 0.5 * math.log(2 * math.pi)
    assert ((r.logp[:-1].double().mean(1) - want).abs() < 5 * math.sqrt(0.5 / (4 * 4096))).all()
    adv = torch.tensor([1.0, -1.0, 0.5, -0.5], device=DEV)
    k = [S - 1, 0, 1, 2]                              # one step of each chain; the first row has no density
    pick = lambda v: torch.stack([v[i, b] for b, i in enumerate(k)])      # noqa: E731
    args = (pick(r.x_t), pick(r.x_prev), r.t[k], r.transition[k], pick(r.logp), adv)
    out = tr.policy_step(*args, clip_range=0.2, kl_coef=0.1)
    # nothing has moved: every ratio is one (two evaluations of one network, logp rounded to fp32 in between), no KL
    assert float(out.ratio[0]) == 0.0 and ((out.ratio[1:] - 1).abs() <= 4 * R.U * (1 + pick(r.logp)[1:].abs())).all() and not out.kl.any()
    for _ in range(2):
        out = tr.policy_step(*args, clip_range=0.2, kl_coef=0.1)
    assert torch.isfinite(out.loss) and out.kl[1:].all() and torch.isfinite(tr.flat.data).all() and tr.opt_step == 3


def test_video_latents_fine_tune_too():
    """The tri-plane network on [B, C, L] latents with a mixing logit [1, C, 1]: preference step, rollout, policy step."""
    unet = dict(size1=8, size2=8, size3=4, in_channels=64, model_channels=32, out_channels=64, attention_resolutions=[2], num_res_blocks=1,
                channel_mult=[1, 2], num_head_channels=32)
    tr = LDMTrainStep(unet, dict(timesteps=10, channels=64, domain="video"), numerics="fp32", lr=1e-4, device=DEV)
    st = {"model." + k: v for k, v in named_state("ft.unet3", [(k, tuple(p.shape)) for k, p in tr.model.state_dict().items()]).items()}
    tr.load_state_dict(st, strict=False).finalize().set_reference()
    L = 8 * 8 + 2 * 8 * 4
    g = torch.Generator(DEV).manual_seed(1)
    zw, zl = (torch.randn((2, 64, L), device=DEV, generator=g) for _ in range(2))
    out = tr.preference_step(zw, zl, beta=100.0, t=torch.tensor([3, 7]))
    assert float(out.loss) == pytest.approx(math.log(2.0), rel=2 * R.U) and tr.opt_step == 1
    r = tr.rollout(2, generator=g)
    assert r.x_0.shape == (2, 64, L) and r.logp.shape == (10, 2) and r.logp[:-1].all()
    k, b = torch.tensor([2, 5], device=DEV), torch.arange(2, device=DEV)
    out = tr.policy_step(r.x_t[k, b], r.x_prev[k, b], r.t[k], r.transition[k], r.logp[k, b], torch.tensor([1.0, -1.0]), clip_range=0.1, kl_coef=0.1)
    assert ((out.ratio - 1).abs() <= 4 * R.U * (1 + r.logp[k, b].abs())).all() and out.kl.all() and torch.isfinite(tr.flat.data).all()


def test_main_fine_tunes_from_preferences(golden, tmp_path):
    """`main.py` with lossconfig.objective preference: pairs of latents from a file, 8-bit moments, a checkpoint that resumes."""
    import yaml
    cfgs = golden.json("configs.json")
    save = str(tmp_path)
    np.save(os.path.join(save, "pairs.npy"), np.random.default_rng(0).standard_normal((6, 2, 64, 8, 8)).astype(np.float32))
    cfg = {"model": {"embed_dim": cfgs["TOY_EMBED"], "lr": 1e-4, "pretrained": False, "resume": False,
                     "params": {"unetconfig": cfgs["TOY_UNET"], "ddconfig": cfgs["TOY_DD"], "mlpconfig": cfgs["MLP_CFG"],
                                "ddpmconfig": {"timesteps": 1000, "sampling_timesteps": 5, "ddim_sampling_eta": 0.0, "image_size": 8, "channels": 64},
                                "lossconfig": {"gradient_accumulate_every": 2, "ema_update_every": 1, "objective": "preference", "beta": 100.0,
                                               "optimizer_state_bits": 8}}},
           "data": {"domain": "image", "mode": "train", "save_pth": save, "test_batch_size": 2, "batch_size": 4, "test_resolution": 32, "train_steps": 4,
                    "latents": os.path.join(save, "pairs.npy")}}

    def run(name, **model):
        path = os.path.join(save, name)
        with open(path, "w") as f:
            yaml.safe_dump(dict(cfg, model=dict(cfg["model"], **model)), f)
        out = subprocess.run([sys.executable, os.path.join(ROOT, "main.py"), "--exp", "ldm", "--configs", path, "--numerics", "fp32"],
                             capture_output=True, text=True, timeout=900)
        assert out.returncode == 0, out.stdout[-2000:] + out.stderr[-2000:]
        return out.stdout

    log = run("a.yaml")
    assert "iter 0: Dae loss : 0.6931" in log and "after 2 optimizer steps" in log
    import shutil
    shutil.copy(os.path.join(save, "ldm-last.pt"), os.path.join(save, "first.pt"))
    log = run("b.yaml", resume=True)
    assert "AdamW state, optimizer step 2" in log and "after 4 optimizer steps" in log
    first, second = (torch.load(p, map_location="cpu", weights_only=True) for p in (os.path.join(save, "first.pt"), os.path.join(save, "ldm-last.pt")))
    assert second["reference"].keys() == first["reference"].keys()
    for k, v in first["reference"].items():           # resumed against the network that the first run started from
        assert torch.equal(v, second["reference"][k]), k
    assert any(not torch.equal(v, first["diffusion"][k]) for k, v in first["reference"].items())
