"""What the fine-tuning operators promise at the edges of their arguments, on the GPU."""
import gc
import math

import pytest
import torch

import finetune_ref as R
from ddmi_amd import _lib
from ddmi_amd.finetune import policy_loss, preference_loss, transition_log_prob
from ddmi_amd.optim import adamw_step
from test_gpu_finetune import DEV, SHAPES, call, reference
from test_gpu_finetune_step import pairs, trainer

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


# ---- sums in 64 bits: the bounds without what sums in 32 would add -------------------------------------------------------------------
D = 2.0 ** -53


def sum_64(t, e):
    """A sum of n terms in 64 bits, in whatever order: n - 1 additions, each off by half a step of a partial sum (and the products' own)."""
    return t.sum((1, 2)), (e + (t[0].numel() + 64) * D * t.abs()).sum((1, 2))


def gradients_64(general):
    """The logit's gradient as a 64-bit sum over batch and values of the terms' errors alone; the rest as it was."""
    def gradients(out, d, row, c, part, e_part, res, e_res, k, e_k, far=None, e_far=None, q=None, e_q=None):
        done = general(out, d, row, c, part, e_part, res, e_res, k, e_k, far, e_far, q, e_q)
        if c is None:
            return done
        chan, bound = 0.0, 0.0
        for f, e_f, r, e_r in ((k, e_k, res, e_res), (q, e_q, far, e_far)):
            if f is None:
                continue
            s = r * part
            chan = chan + (row(f) * s).sum((0, 2))
            each = e_r * part.abs() + r.abs() * e_part + e_r * e_part + (len(s) * s.shape[2] + 64) * D * s.abs()
            bound = bound + (row(e_f) * (s.abs() + each) + row(f.abs()) * each).sum((0, 2))
        slope = (c * (1 - c)).reshape(-1)
        want = chan * slope
        done["d_logit"] = (want, bound * slope + 1.01 * R.U * (want.abs() + bound * slope) + 2.0 ** -149)
        return done
    return gradients


@pytest.mark.parametrize("B,C,T", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("op,kl", [("pref", True), ("policy", True), ("policy", False)])
def test_sums_are_held_in_64_bits(op, kl, B, C, T, dtype, monkeypatch):
    monkeypatch.setattr(R, "_gradients", gradients_64(R._gradients))
    monkeypatch.setattr(R, "_sum", sum_64)
    d = R.make(op, B, C, T, dtype, kl=kl, seed=B + C + T + 1, device=DEV)
    R.check(call(op, d), reference(op, d), (B, C, T))


def test_gradients_of_many_small_transitions():
    """100 000 transitions of three values, weights among them, and a clip too wide to have a border nearby: every output."""
    d = R.make("policy", 100000, 3, 1, seed=12, device=DEV)
    d["weight"] = (torch.arange(100000, device=DEV) % 7).float()
    d["clip_range"] = 1e9
    R.check(call("policy", d), reference("policy", d))


# ---- upstream gradients ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("op,kl", [("pref", True), ("policy", True), ("policy", False)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,C,T", BOTH)
@pytest.mark.parametrize("mixed,weight", [(True, None), (False, "some")])
@pytest.mark.parametrize("up", [3.0, -1.0 / 3.0])
def test_an_upstream_gradient_costs_no_second_rounding_to_bf16(op, kl, dtype, B, C, T, mixed, weight, up):
    """The first backward's gradients are `up` times the formula's within the formula's own bound: one rounding to the output's type, and the
    fp32 factor's and product's own.  A second backward gives the same (in bf16 the same bits)."""
    d = R.make(op, B, C, T, dtype, mixed, kl=kl, weight=weight, seed=31, device=DEV)
    want = reference(op, d)
    leaves = [d["model_out"].requires_grad_()] + ([d["mixing_logit"].requires_grad_()] if mixed else [])
    loss = (preference_loss if op == "pref" else policy_loss)(**d).loss
    up = torch.tensor(up, device=DEV)
    first, second = (torch.autograd.grad(loss, leaves, up, retain_graph=True) for _ in range(2))
    for grads in (first, second):
        for g, name in zip(grads, ("d_model_out", "d_logit")):
            w, bound = (t.to(DEV) for t in want[name])
            w, scale = w * up.double(), float(up.double().abs())
            # the bound holds what is rounded last relative to the value: it scales with it; two more roundings in fp32; the least numbers
            over = (g.double().reshape(w.shape) - w).abs() - (bound * scale + 2.02 * R.U * (w.abs() + bound * scale) + 2.0 ** -133)
            assert float(over.max()) <= 0, (name, float(over.max()))
    if dtype == torch.bfloat16:
        assert all(map(torch.equal, first, second))


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("B,C,T", BOTH)
def test_upstream_gradients_of_bf16_in_a_graph(op, B, C, T):
    """Forward and backward captured together, replayed with upstream gradients that are 1 and are not, and with other inputs."""
    sets = [R.make(op, B, C, T, torch.bfloat16, seed=s, device=DEV) for s in (1, 2)]
    loss_of = preference_loss if op == "pref" else policy_loss

    def grads(d, up):
        d = dict(d, model_out=d["model_out"].detach().requires_grad_(), mixing_logit=d["mixing_logit"].detach().requires_grad_())
        return torch.autograd.grad(loss_of(**d).loss, [d["model_out"], d["mixing_logit"]], up)

    values = (1.0, 3.0, -0.7)
    want = {(i, v): grads(d, torch.tensor(v, device=DEV)) for i, d in enumerate(sets) for v in values}
    static = {k: t.clone() if isinstance(t, torch.Tensor) else t for k, t in sets[0].items()}
    up, graph, side = torch.ones((), device=DEV), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        grads(static, up)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = grads(static, up)
    for i, v in ((0, 1.0), (0, 3.0), (1, 3.0), (1, 3.0), (0, -0.7), (1, 1.0), (1, -0.7)):
        for k, t in static.items():
            if isinstance(t, torch.Tensor):
                t.copy_(sets[i][k])
        up.fill_(v)
        graph.replay()
        grads(sets[1 - i], up)                        # eager work between the replays
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want[i, v])), (i, v)


def test_inputs_changed_before_a_backward_that_reads_them():
    """bf16 gradients are computed again from the inputs where the upstream gradient is not 1: changed in place, they are refused."""
    d = R.make("pref", 6, 4, 9, torch.bfloat16, seed=5, device=DEV)
    loss = preference_loss(**dict(d, model_out=d["model_out"].requires_grad_())).loss
    d["x_t"].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


# ---- captures ------------------------------------------------------------------------------------------------------------------------------
def test_capture_refused_over_parameters_of_a_living_eager_loss():
    """The parameters lie behind the network's output and there is no mixing logit; once the eager loss is gone, the capture runs."""
    d = R.make("pref", 6, 7, 131, mixed=False, device=DEV)
    w = torch.full((7, 1), 0.5, device=DEV, requires_grad=True)
    base = d["model_out"]

    def grad():
        return torch.autograd.grad(preference_loss(**dict(d, model_out=base * w)).loss, w)[0]

    eager = preference_loss(**dict(d, model_out=base * w))
    refused, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    other = torch.zeros(1, device=DEV)
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="captured while the graph of an eager loss"):
            preference_loss(**dict(d, model_out=base * w))
        other.add_(1)
    del eager
    gc.collect()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = grad()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = grad()
    for _ in range(3):
        graph.replay()
        eager = preference_loss(**dict(d, model_out=base.clone().requires_grad_())).loss      # eager work of other leaves
        torch.cuda.synchronize()
        assert torch.equal(got, want)


# ---- waits that end early ------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("polls", [1, 3, 20])
@pytest.mark.parametrize("B,C,T", [(48, 64, 2048), (140, 3, 33001)])
def test_workgroups_that_stop_waiting_leave_the_same_bits(op, polls, B, C, T):
    """Some find their neighbours' sums, one does not, and those after it look once: whoever computes a span, it is the same."""
    d = R.make(op, B, C, T, seed=8, device=DEV)
    want = call(op, d)
    try:
        _lib.check(_lib.lib().ddmi_debug_loss_polls(polls))
        got = [call(op, d) for _ in range(3)]
    finally:
        _lib.check(_lib.lib().ddmi_debug_loss_polls(4096))
    got.append(call(op, d))                           # the next call waits again: the mark is that of a call
    for g in got:
        for k in want:
            assert torch.equal(want[k], g[k]), k


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_that_a_hook_moves(op, dtype):
    """Inputs packed to the host and back: handed-out gradients and computed ones are those without a hook."""
    d = R.make(op, 6, 7, 131, dtype, device=DEV)
    leaves = [d["model_out"].requires_grad_(), d["mixing_logit"].requires_grad_()]
    loss_of = preference_loss if op == "pref" else policy_loss
    up = torch.tensor(3.0, device=DEV)
    loss = loss_of(**d).loss
    want = [torch.autograd.grad(loss, leaves, up, retain_graph=True) for _ in range(2)]
    with torch.autograd.graph.save_on_cpu():
        loss = loss_of(**{k: t.clone() if k in ("x_t", "noise", "x_prev", "ref_out") else t for k, t in d.items()}).loss
    junk = [torch.full_like(d["x_t"], math.nan) for _ in range(8)]      # what was freed is used again
    for w in want:
        assert all(map(torch.equal, torch.autograd.grad(loss, leaves, up, retain_graph=True), w))
    del junk


# ---- AdamW's quotient ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("g_type", [torch.float32, torch.bfloat16])
def test_adamw_divides(g_type):
    """With betas of zero and no eps the change is lr g / |g|: the root of a rounded square is the number itself, and a number divided by itself
    is one, so the parameters are lr exactly."""
    n = 100003
    g = torch.randn(n, generator=torch.Generator().manual_seed(3)).to(g_type).to(DEV)
    g[g == 0] = 1.0
    p, m, v = (torch.zeros(n, device=DEV) for _ in range(3))
    adamw_step([p], [g], [m], [v], 1, lr=0.5, betas=(0.0, 0.0), eps=0.0)
    assert torch.equal(p, -0.5 * g.float().sign())


def test_a_graphed_training_step_beside_a_living_loss():
    """use_graph records on the second step of a shape; while the caller holds an eager loss on the parameters it runs eagerly instead, with
    the same numbers, and records once the loss is gone."""
    def eager_loss(tr, z, noise, t):
        x = torch.cat([z, z])
        out = tr.model(x, torch.cat([t, t]))
        return preference_loss(out, out.detach(), x, noise, torch.full((6,), 0.5, device=DEV), 1.0)

    nodes = lambda tr: [torch.autograd.graph.get_gradient_edge(p).node for p in tr.flat.params]      # noqa: E731
    runs = []
    for hold in (False, True):
        tr = trainer(use_graph=True).set_reference()
        held = []
        for k in range(4):
            zw, _, noise, t = (v.to(DEV) for v in pairs(seed=k))
            if hold and k == 1:
                held.append(eager_loss(tr, zw, noise, t))
                assert not any(n.metadata.update(held=True) for n in nodes(tr))
            if k == 3:
                held.clear()
                gc.collect()
                assert not any(n.metadata for n in nodes(tr))           # nothing of it is left before anything is recorded
            tr.train_step(zw, t, noise)
            assert isinstance(tr._graphs[tuple(zw.shape)], tuple) == (k >= (3 if hold else 1))
        runs.append(tr.flat.data.clone())
    assert torch.equal(*runs)


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("which", ["output", "logit"])
@pytest.mark.parametrize("B,C,T", BOTH)
def test_gradients_of_one_leaf_alone(op, dtype, which, B, C, T):
    """The output's without the logit's and the other way round, for an upstream gradient that is not 1: what both together give."""
    d = R.make(op, B, C, T, dtype, seed=11, device=DEV)
    loss_of = preference_loss if op == "pref" else policy_loss
    up = torch.tensor(-1.7, device=DEV)
    names = ["model_out", "mixing_logit"]
    both = {n: d[n].clone().requires_grad_() for n in names}
    want = dict(zip(names, torch.autograd.grad(loss_of(**dict(d, **both)).loss, both.values(), up)))
    name = names[which == "logit"]
    w, bound = (t.to(DEV).reshape(d[name].shape) for t in reference(op, d)["d_logit" if which == "logit" else "d_model_out"])
    w, scale = w * up.double(), float(up.double().abs())
    one = d[name].clone().requires_grad_()
    loss = loss_of(**dict(d, **{name: one})).loss
    assert torch.equal(torch.autograd.grad(loss, one, up, retain_graph=True)[0], want[name])
    again = torch.autograd.grad(loss, one, up)[0]
    # Computed anew, an fp32 gradient is not the multiplied one to the last bits, and where the residual's and the KL term's parts cancel a
    # rounding of a part is many of their sum (k up rounded before the sum, against the sum times up): both are within the formula's bound,
    # which counts the parts' roundings, and two more of the value's.
    assert ((again.double() - w).abs() <= bound * scale + 2.02 * R.U * (w.abs() + bound * scale) + 2.0 ** -133).all()
    if dtype == torch.bfloat16:
        assert torch.equal(again, want[name])


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_upstream_gradients_of_more_than_2_to_31_values(op):
    """bf16 gradients computed again behind offsets of 2^31: times four is exact, so they are four times the handed-out ones."""
    C, T, B = 64, 65536, 514
    small = R.make(op, 2 if op == "pref" else 1, C, T, torch.bfloat16, seed=3, device=DEV)
    d = {}
    for k, t in small.items():
        if not isinstance(t, torch.Tensor) or "logit" in k:
            d[k] = t
        elif op == "pref":
            d[k] = torch.cat([h.expand((B // 2,) + h.shape[1:]) for h in t.split(1)]).contiguous()
        else:
            d[k] = t.expand((B,) + t.shape[1:]).contiguous()
    d["model_out"].requires_grad_()
    loss_of = preference_loss if op == "pref" else policy_loss
    one = torch.autograd.grad(loss_of(**d).loss, d["model_out"], torch.ones((), device=DEV))[0]
    four = torch.autograd.grad(loss_of(**d).loss, d["model_out"], torch.full((), 4.0, device=DEV))[0]
    normal = one.abs() >= 2.0 ** -126
    assert torch.equal(torch.where(normal, one * 4, one), torch.where(normal, four, one)) and bool(normal[[0, -1]].any())
