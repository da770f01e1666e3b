"""The fine-tuning losses and AdamW over many tensors on the GPU, against 64-bit formulas with derived bounds (finetune_ref)."""
import gc
import math

import pytest
import torch

import finetune_ref as R
from ddmi_amd import _lib
from ddmi_amd.finetune import policy_loss, preference_loss, transition_log_prob
from ddmi_amd.optim import AdamW, adamw_step, blocks_of

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# (B, C, T): one value; odd planes; more rows than a workgroup holds; rows of one value; several segments a row; rows shared by four waves;
# enough values for the largest workgroups
SHAPES = [(2, 1, 1), (2, 64, 64), (6, 5, 7), (4, 3, 1), (2, 1100, 3), (2, 2, 20001), (6, 48, 1295), (4, 7, 4096), (2, 64, 65536)]
# the residuals kept in registers (from 384 workgroups on): whole turns; odd planes; short rows; segments of long odd rows
LARGE = [(48, 64, 2048), (80, 33, 2501), (500, 190, 77), (140, 3, 33001), (36, 64, 4100)]
SHAPES += LARGE


def call(op, d, up=None):
    d = dict(d)
    out = d["model_out"] = d["model_out"].detach().clone().requires_grad_()
    logit = d["mixing_logit"]
    if logit is not None:
        logit = d["mixing_logit"] = logit.detach().clone().requires_grad_()
    r = (preference_loss if op == "pref" else policy_loss)(**d)
    leaves = [out] + ([logit] if logit is not None else [])
    g = torch.autograd.grad(r.loss if up is None else r.loss * up, leaves)
    return dict(r._asdict(), d_model_out=g[0], d_logit=g[1].reshape(-1) if len(g) > 1 else None)


def reference(op, d):
    cpu = {k: t.cpu() if isinstance(t, torch.Tensor) else t for k, t in d.items()}
    big = cpu["model_out"].numel() > 1 << 21
    return (R.preference if op == "pref" else R.policy)(d if big else cpu)


@pytest.mark.parametrize("B,C,T", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mixed", [True, False])
def test_preference_loss(B, C, T, dtype, mixed):
    d = R.make("pref", B, C, T, dtype, mixed, shared=T % 2 == 1, seed=B + C + T, device=DEV)
    R.check(call("pref", d), reference("pref", d), (B, C, T))


@pytest.mark.parametrize("B,C,T", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mixed,kl", [(True, True), (True, False), (False, True), (False, False)])
def test_policy_loss(B, C, T, dtype, mixed, kl):
    d = R.make("policy", B, C, T, dtype, mixed, kl=kl, seed=B + C + T, device=DEV)
    R.check(call("policy", d), reference("policy", d), (B, C, T))
    logp = transition_log_prob(d["model_out"], d["x_t"], d["x_prev"], d["transition"], d["sqrt_1mac"], d["mixing_logit"])
    assert torch.equal(logp, call("policy", d)["logp"])


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("weight", ["some", "none_left"])
@pytest.mark.parametrize("mixed", [True, False])
@pytest.mark.parametrize("B,C,T", [(14, 5, 33), (80, 50, 1701)])
def test_rows_left_out(op, weight, mixed, B, C, T):
    """Rows of weight 0 hold NaN and infinities: none of it may show, their gradients are zeros, and the mean is over the others."""
    d = R.make(op, B, C, T, weight=weight, mixed=mixed, seed=3, device=DEV)
    got = call(op, d)
    R.check(got, reference(op, d), weight)
    gone = d["weight"] == 0
    gone = torch.cat([gone, gone]) if op == "pref" else gone
    assert not got["d_model_out"][gone].any()
    if weight == "none_left":
        assert float(got["loss"]) == 0.0


def test_transition_without_noise_is_left_out():
    d = R.make("policy", 6, 4, 9, seed=5, device=DEV)
    d["transition"][2, 2] = 0.0
    got = call("policy", d)
    R.check(got, reference("policy", d))
    assert float(got["logp"][2]) == 0.0 and not got["d_model_out"][2].any()


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_nan_in_a_row_that_takes_part_shows(op):
    d = R.make(op, 6, 4, 9, seed=5, device=DEV)
    d["model_out"][1, 2, 3] = float("nan")
    got = call(op, d)
    assert math.isnan(float(got["loss"]))
    assert torch.isfinite(got["d_model_out"][[2, 5]]).all()           # rows of other pairs keep theirs


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("B,C,T", LARGE)
def test_one_pass_that_does_not_wait_gives_the_same_bits(op, B, C, T):
    """With a single look at the neighbours' sums most workgroups leave their part to the backward call: same loss, same gradients."""
    d = R.make(op, B, C, T, seed=8, device=DEV)
    want = call(op, d)
    try:
        _lib.check(_lib.lib().ddmi_debug_loss_polls(0))
        got = call(op, d)
    finally:
        _lib.check(_lib.lib().ddmi_debug_loss_polls(4096))
    for k in want:
        assert torch.equal(want[k], got[k]), k


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_strided_and_offset_inputs(op):
    d = R.make(op, 6, 5, 31, torch.bfloat16, seed=9, device=DEV)
    want = call(op, d)
    odd = {}
    for k, t in d.items():
        if isinstance(t, torch.Tensor) and t.dim() == 3:
            t = t.transpose(1, 2).contiguous().transpose(1, 2) if k == "x_t" else torch.cat([t.reshape(-1)[:1], t.reshape(-1)])[1:].view(t.shape)
        elif isinstance(t, torch.Tensor) and t.dim() == 1:
            t = torch.stack([t, t], 1)[:, 0]
        odd[k] = t
    got = call(op, odd)
    for k in want:
        assert torch.equal(want[k], got[k]), k


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_image_shaped_and_plain_vectors(op):
    """[B, C, H, W] is [B, C, H W]; [B, C] is [B, C, 1]."""
    d = R.make(op, 4, 6, 12, seed=2, device=DEV)
    shaped = {k: (t.reshape(t.shape[0], 6, 3, 4) if isinstance(t, torch.Tensor) and t.dim() == 3 and "logit" not in k else t) for k, t in d.items()}
    a, b = call(op, d), call(op, shaped)
    assert torch.equal(a["loss"], b["loss"]) and torch.equal(a["d_model_out"].reshape(-1), b["d_model_out"].reshape(-1))
    d = R.make(op, 4, 6, 1, seed=2, device=DEV)
    flat = {k: (t.reshape(t.shape[0], 6) if isinstance(t, torch.Tensor) and t.dim() == 3 and "logit" not in k else t) for k, t in d.items()}
    assert torch.equal(call(op, d)["loss"], call(op, flat)["loss"])


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_gradient_against_differences(op):
    """(loss(x + s v) - loss(x - s v)) / 2 s along a random direction v.  The losses carry rounding errors within their own bounds; the
    difference's curvature is measured by halving s (its error is of second order: a third of the change)."""
    d = R.make(op, 4, 5, 37, seed=21, device=DEV)
    got = call(op, d)
    v = torch.randn(d["model_out"].shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    vl = torch.randn(d["mixing_logit"].shape, generator=torch.Generator().manual_seed(2)).to(DEV)
    want = float((got["d_model_out"].double() * v).sum() + (got["d_logit"].double() * vl.reshape(-1)).sum())

    def loss(s):
        e = dict(d, model_out=d["model_out"] + s * v, mixing_logit=d["mixing_logit"] + s * vl)
        return float((preference_loss if op == "pref" else policy_loss)(**e).loss)

    s = 2.0 ** -9
    wide, near = (loss(2 * s) - loss(-2 * s)) / (4 * s), (loss(s) - loss(-s)) / (2 * s)
    e_loss = float(reference(op, d)["loss"][1]) * 4 / s + abs(float(got["loss"])) * 4 * R.U / s
    # the shifted inputs are rounded too: half a step of values up to 8, along the gradient
    e_in = float(got["d_model_out"].double().abs().sum()) * 8 * R.U * 2 / s
    assert abs(near - want) <= abs(wide - near) + e_loss + e_in, (near, want)


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("B,C,T", [(6, 5, 33), (50, 64, 2051)])
def test_upstream_gradient_and_second_backward(op, B, C, T):
    d = R.make(op, B, C, T, seed=4, device=DEV)
    one, three = call(op, d), call(op, d, 4.0)
    assert torch.equal(one["d_model_out"] * 4, three["d_model_out"]) and torch.equal(one["d_logit"] * 4, three["d_logit"])
    out = d["model_out"].clone().requires_grad_()
    r = (preference_loss if op == "pref" else policy_loss)(**dict(d, model_out=out))
    first = torch.autograd.grad(r.loss, out, retain_graph=True)[0].clone()
    first.mul_(0)                                                       # what a caller does with its gradient does not reach the next one
    assert torch.equal(torch.autograd.grad(r.loss, out)[0], one["d_model_out"])
    with torch.no_grad():                                               # without a gradient: two sums of other lengths in a large batch
        alone = (preference_loss if op == "pref" else policy_loss)(**d).loss
    assert abs(float(alone) - float(one["loss"])) <= 2 * R.U * abs(float(alone))


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_second_order_gradients_are_refused(op):
    d = R.make(op, 4, 3, 5, seed=4, device=DEV)
    out = d["model_out"].clone().requires_grad_()
    loss = (preference_loss if op == "pref" else policy_loss)(**dict(d, model_out=out)).loss
    scale = torch.ones((), device=DEV, requires_grad=True)
    g = torch.autograd.grad(loss * scale, out, create_graph=True)[0]
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_many_small_rows(op):
    """More rows than one turn of any workgroup: 100 000 of three values each, weights among them."""
    d = R.make(op, 100000, 3, 1, seed=12, device=DEV)
    rows = 50000 if op == "pref" else 100000
    d["weight"] = (torch.arange(rows, device=DEV) % 7).float()
    if op == "policy":        # far from the clip's borders
        d["clip_range"] = 1e-30
    got = call(op, d)
    assert torch.isfinite(got["loss"]) and torch.isfinite(got["d_model_out"]).all()
    if op == "pref":
        R.check(got, reference(op, d))
    else:
        want = R.policy(dict(d, clip_range=1e9))      # nothing clipped, for the statistics
        R.check({k: got[k] for k in ("logp", "ratio", "kl")}, {k: want[k] for k in ("logp", "ratio", "kl")})


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("B,C,T", [(8, 16, 1025), (80, 33, 2501)])
def test_same_bits_on_every_run_and_stream(op, B, C, T):
    d = R.make(op, B, C, T, seed=6, device=DEV)
    a = call(op, d)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        b = call(op, d)
    c = call(op, d)
    torch.cuda.synchronize()
    for k in a:
        assert torch.equal(a[k], b[k]) and torch.equal(a[k], c[k]), k


def test_two_streams_at_once():
    """Large calls of both losses on two streams, each waiting for its own workgroups: the results are those of either alone."""
    sets = [(op, R.make(op, B, C, T, seed=B, device=DEV)) for op, (B, C, T) in (("pref", LARGE[0]), ("policy", LARGE[1]), ("policy", LARGE[4]), ("pref", LARGE[1]))]
    want = [call(op, d) for op, d in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for rep in range(4):
        for i, (op, d) in enumerate(sets):
            with torch.cuda.stream(streams[(i + rep) % 2]):
                got.append((i, call(op, d)))
    torch.cuda.synchronize()
    for i, g in got:
        for k in g:
            assert torch.equal(g[k], want[i][k]), (i, k)


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("B,C,T", [(6, 7, 131), (80, 33, 2501)])
def test_captured_and_replayed(op, B, C, T):
    """Two captured forwards + backwards of different inputs, replayed by turns with eager work between: each replay is the eager result."""
    sets = [R.make(op, B, C, T, seed=s, device=DEV) for s in (1, 2, 3, 4)]
    want = [call(op, d) for d in sets]
    static = [{k: t.clone() if isinstance(t, torch.Tensor) else t for k, t in sets[i].items()} for i in (0, 1)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for d in static:
            call(op, d)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs = []
    for d in static:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(op, d)
        graphs.append((g, out))
    for i in (0, 1, 2, 3, 1, 0):
        for j in (0, 1):
            src = sets[(i + j) % 4]
            for k, t in static[j].items():
                if isinstance(t, torch.Tensor):
                    t.copy_(src[k])
            graphs[j][0].replay()
        call(op, sets[(i + 2) % 4])
        torch.cuda.synchronize()
        for j in (0, 1):
            for k in want[0]:
                assert torch.equal(graphs[j][1][k], want[(i + j) % 4][k]), (i, j, k)


def test_capture_refused_while_an_eager_loss_of_the_leaves_lives():
    """An eager loss that was built on the default stream ties its leaves' gradients to that stream; gone, the capture runs."""
    d = R.make("pref", 6, 7, 131, device=DEV)
    d["model_out"].requires_grad_()
    d["mixing_logit"].requires_grad_()
    leaves = [d["model_out"], d["mixing_logit"]]
    eager = preference_loss(**d)
    want = torch.autograd.grad(eager.loss, leaves)
    refused, graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    other = torch.zeros(1, device=DEV)
    with torch.cuda.graph(refused):
        with pytest.raises(RuntimeError, match="captured while the graph of an eager loss"):
            preference_loss(**d)
        other.add_(1)
    del eager
    gc.collect()
    assert not any(torch.autograd.graph.get_gradient_edge(t).node.metadata for t in leaves)
    with torch.cuda.graph(graph):
        got = torch.autograd.grad(preference_loss(**d).loss, leaves)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want))


@pytest.mark.parametrize("op", ["pref", "policy"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_backward_captured_apart_from_its_forward(op, dtype):
    """Replayed several times with an upstream gradient that is not 1: each replay is the eager backward, nothing is multiplied twice."""
    d = R.make(op, 6, 7, 131, dtype, device=DEV)
    leaves = [d["model_out"].requires_grad_(), d["mixing_logit"].requires_grad_()]
    up = torch.tensor(3.0, device=DEV)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        loss = (preference_loss if op == "pref" else policy_loss)(**d).loss
        torch.autograd.grad(loss, leaves, up, retain_graph=True)                # handed out; those after it are computed from the inputs
        want = {v: torch.autograd.grad(loss, leaves, torch.tensor(v, device=DEV), retain_graph=True) for v in (3.0, -0.7)}
        loss = (preference_loss if op == "pref" else policy_loss)(**d).loss
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(loss, leaves, up, retain_graph=True)
    for v in (3.0, 3.0, -0.7, -0.7, 3.0):
        up.fill_(v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(map(torch.equal, got, want[v])), v


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_reference_output_made_in_inference_mode(op):
    d = R.make(op, 6, 7, 131, device=DEV)
    leaves = [d["model_out"].requires_grad_(), d["mixing_logit"].requires_grad_()]
    loss_of = preference_loss if op == "pref" else policy_loss
    want = loss_of(**d).loss
    with torch.inference_mode():
        d = {k: t.clone() if k in ("ref_out", "x_t") else t for k, t in d.items()}
    loss = loss_of(**d).loss
    assert d["ref_out"].is_inference() and torch.equal(loss, want)
    for _ in range(2):      # handed out, computed again
        assert all(map(torch.equal, torch.autograd.grad(loss, leaves, retain_graph=True), torch.autograd.grad(want, leaves, retain_graph=True)))


def test_graphed_callable():
    """Forward and backward in two graphs, the backward taken twice."""
    d = R.make("pref", 6, 7, 131, device=DEV)
    leaves = [d.pop("model_out").requires_grad_(), d.pop("mixing_logit").requires_grad_()]

    def loss_of(model_out, mixing_logit):
        return preference_loss(model_out=model_out, mixing_logit=mixing_logit, **d).loss

    graphed = torch.cuda.make_graphed_callables(loss_of, tuple(t.detach().clone().requires_grad_() for t in leaves))
    for _ in range(2):
        first = loss_of(*leaves)
        torch.autograd.grad(3.0 * first, leaves, retain_graph=True)
        want = torch.autograd.grad(3.0 * first, leaves)
        loss = 3.0 * graphed(*leaves)
        assert torch.equal(loss, 3.0 * first)
        for _ in range(3):
            got = torch.autograd.grad(loss, leaves, retain_graph=True)
            torch.cuda.synchronize()
            assert all(map(torch.equal, got, want))
        del first


# ---------------------------------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------------------------------
def lists(shapes, p_type, g_type, bits, seed, offset=0):
    """Parameters, gradients and moments; `offset`: places that their storage starts off an aligned address."""
    g = torch.Generator().manual_seed(seed)

    def place(t):
        return torch.cat([t.reshape(-1)[:1]] * offset + [t.reshape(-1)])[offset:].view(t.shape).to(DEV) if not offset else \
            torch.cat([torch.zeros(offset, dtype=t.dtype), t.reshape(-1)]).to(DEV)[offset:].view(t.shape)

    p = [place(torch.randn(s, generator=g).to(p_type)) for s in shapes]
    gr = [place((0.1 * torch.randn(s, generator=g)).to(g_type)) for s in shapes]
    if bits == 32:
        return p, gr, [place(0.02 * torch.randn(s, generator=g)) for s in shapes], [place((0.1 * torch.randn(s, generator=g)) ** 2) for s in shapes], {}
    sizes = [math.prod(s) for s in shapes]
    codes = lambda lo, hi, n: torch.randint(lo, hi, (n,), generator=g, dtype=torch.uint8)      # noqa: E731
    m = [place(codes(0, 0x70, n) | (codes(0, 2, n) << 7)).view(torch.float8_e4m3fn) for n in sizes]
    v = [place(codes(0x20, 0x70, n)).view(torch.float8_e4m3fn) for n in sizes]
    scale = lambda n: torch.exp2(torch.randint(-16, -12, (blocks_of(n),), generator=g).float()).to(DEV)      # noqa: E731
    return p, gr, m, v, {"exp_avg_scales": [scale(n) for n in sizes], "exp_avg_sq_scales": [scale(n) for n in sizes]}


ADAM_SHAPES = [[(1,)], [(255,), (256,), (257,)], [(3, 5, 7), (1025,), (4096,), (4097,), (2, 3)], [(k % 37 + 1,) for k in range(130)], [(3, 70001)]]


def bits_of(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("shapes", ADAM_SHAPES, ids=["one", "ends", "mixed", "many", "long"])
@pytest.mark.parametrize("p_type,g_type", [(torch.float32, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32),
                                           (torch.bfloat16, torch.bfloat16)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_adamw_step(shapes, p_type, g_type, bits, offset):
    p, g, m, v, scales = lists(shapes, p_type, g_type, bits, 7, offset)
    hyper = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1, grad_scale=0.5)
    step, seed = 3, 1234
    before = [[t.detach().clone() for t in ts] for ts in (p, g, m, v)]
    old = {k: [t.clone() for t in ts] for k, ts in scales.items()}
    adamw_step(p, g, m, v, step, seed=seed, **hyper, **scales)
    for i in range(len(shapes)):
        n = p[i].numel()
        pb, gb, mb, vb = (ts[i].reshape(-1).cpu() for ts in before)
        assert torch.equal(g[i].cpu().reshape(-1), gb)
        mb, vb = mb.float().double(), vb.float().double()
        if bits == 8:
            mb = mb * old["exp_avg_scales"][i].cpu().double().repeat_interleave(256)[:n]
            vb = (vb * old["exp_avg_sq_scales"][i].cpu().double().repeat_interleave(256)[:n]) ** 2
        want = R.adamw(pb.double(), gb.double(), mb, vb, step, **hyper)
        rnd = R.random_bits(n, seed, step, i)
        p1, e_p = want["p"]
        got = p[i].cpu().double().reshape(-1)
        if p_type == torch.float32:
            assert ((got - p1).abs() <= e_p + R.U * p1.abs()).all()
        else:                                     # up with the probability of what is cut off: 16 random bits
            unit = torch.exp2(torch.frexp(p1)[1].double() - 8)
            cut = (R.mix32(rnd ^ 0x68E31DA4) & 0xFFFF).double() * 2.0 ** -16 * unit
            lo, hi = ((p1.abs() + s * e_p).div(unit).add(cut / unit).floor() * unit for s in (-1, 1))
            # a value whose error reaches into the next binade has another unit there: within that error of either rounding
            assert ((got.abs() >= lo - e_p) & (got.abs() <= hi + e_p) & (got.sign() * p1.sign() >= 0)).all()
        if bits == 32:
            for k, t in (("m", m), ("v", v)):
                w, e = want[k]
                assert ((t[i].cpu().double().reshape(-1) - w).abs() <= e + R.U * w.abs()).all(), k
            continue
        for k, t, name, r, root in (("m", m, "exp_avg_scales", ((rnd & 0xFFF) << 8) | 0x80, False), ("root", v, "exp_avg_sq_scales", rnd >> 12, True)):
            w, e = want[k]
            s = scales[name][i].cpu().double()
            # the block's largest value, in 32 bits, is within its error of the one in 64: next to a power of two it may lie on the other
            # side (sqrt(0.01 (0.5 * 0.3125)^2 + 1e-11) is 2^-6 (1 + 2.6e-8), less than half a step of fp32 above 2^-6)
            assert ((s >= R.block_scales((w.abs() - e).clamp_min(0))) & (s <= R.block_scales(w.abs() + e))).all(), name
            lo, hi = R.codes_allowed(w, e, s, r, root)
            code = t[i].cpu().float().double().reshape(-1)
            assert ((code.abs() >= lo) & (code.abs() <= hi)).all(), k
            assert float((lo != hi).double().mean()) < 0.01          # the allowance is the exception
            assert ((code * w >= 0) | (code == 0)).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_is_reproducible_and_independent_of_the_list(bits):
    """Twice the same bits, on another stream too; a tensor's result depends on its own place in the list, not on its neighbours."""
    shapes = [(40, 70), (9,), (1000,)]
    results = []
    for k in range(3):
        p, g, m, v, scales = lists(shapes, torch.bfloat16, torch.float32, bits, 5)
        st = torch.cuda.Stream() if k == 1 else torch.cuda.current_stream()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            if k == 2:        # the same places, other neighbours
                p[1], g[1] = p[1] * 3, g[1] * 5
            adamw_step(p, g, m, v, [2, 2, 9], lr=[1e-3, 1e-2, 1e-4], weight_decay=[0.0, 0.1, 0.2], seed=3, **scales)
        torch.cuda.synchronize()
        results.append((p, m, v, *scales.values()))
    for ts in zip(*results):
        for i in range(3):
            assert torch.equal(bits_of(ts[0][i]), bits_of(ts[1][i]))
            if i != 1:
                assert torch.equal(bits_of(ts[0][i]), bits_of(ts[2][i]))


def test_adamw_writes_nothing_behind_a_tensor():
    n = 300
    slab = {k: torch.full((4096,), 77, dtype=torch.uint8, device=DEV) for k in ("p", "m", "v")}
    sc = [torch.full((8,), 3.0, device=DEV) for _ in range(2)]
    p = slab["p"][:4 * n].view(torch.float32)
    p.fill_(1.0)
    m, v = (slab[k][:n].view(torch.float8_e4m3fn) for k in "mv")
    adamw_step([p], [torch.ones(n, device=DEV)], [m], [v], 1, lr=0.1, exp_avg_scales=[sc[0][:2]], exp_avg_sq_scales=[sc[1][:2]])
    assert (slab["p"][4 * n:] == 77).all() and (slab["m"][n:] == 77).all() and (slab["v"][n:] == 77).all()
    assert (sc[0][2:] == 3).all() and (sc[1][2:] == 3).all() and (sc[0][:2] != 3).all()


def test_adamw_refuses_shared_memory_and_captures():
    p = [torch.zeros(8, device=DEV)]
    s = lambda: [torch.zeros(8, device=DEV), torch.zeros(8, device=DEV)]      # noqa: E731
    with pytest.raises(ValueError, match="shares memory"):
        adamw_step(p * 2, s(), s(), s(), 1, lr=0.1)
    big = torch.zeros(12, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        adamw_step([big[:8], big[4:]], s(), s(), s(), 1, lr=0.1)
    with pytest.raises(ValueError, match="shares memory"):
        adamw_step(p, [big[:8]], [big[4:]], s()[:1], 1, lr=0.1)
    same = torch.ones(8, device=DEV)                      # one gradient for two parameters is only read
    adamw_step(s(), [same, same], s(), s(), 1, lr=0.1)
    g, a, b = s()[:1], s()[:1], s()[:1]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="graph capture"):
            adamw_step(p, g, a, b, 1, lr=0.1)
        big.add_(1)
    graph.replay()
    torch.cuda.synchronize()
    assert not p[0].any()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_nan_gradient_stays_with_its_value(bits):
    p, g, m, v, scales = lists([(600,)], torch.float32, torch.float32, bits, 5)
    clean = lists([(600,)], torch.float32, torch.float32, bits, 5)
    g[0][300], g[0][301] = float("nan"), float("inf")
    adamw_step(p, g, m, v, 2, lr=1e-3, **scales)
    adamw_step(*clean[:4], 2, lr=1e-3, **clean[4])
    other = torch.ones(600, dtype=torch.bool, device=DEV)
    other[300:302] = False
    assert torch.isnan(p[0][~other]).all() and torch.equal(p[0][other], clean[0][0][other])
    assert torch.isnan(m[0].float()[300]) and not torch.isfinite(m[0].float()[301])
    if bits == 32:
        assert torch.equal(m[0][other], clean[2][0][other])
    else:                # the block's scale is that of its finite values; the outliers were not its largest before
        far = other.clone()
        far[256:512] = False
        assert torch.equal(bits_of(m[0])[far], bits_of(clean[2][0])[far])
        assert torch.isfinite(m[0].float()[other]).all()


def test_rounding_of_8_bit_moments_is_unbiased():
    """Over 4096 equal values the mean of a moment is its exact value within six standard deviations of a rounding (of at most a step's
    half each, independent): round-to-nearest would leave every one where it is."""
    n = 4096
    p, g = [torch.zeros(n, device=DEV)], [torch.full((n,), 1.0, device=DEV)]
    m, v = ([torch.full((n,), c, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)] for c in (0x70, 0x70))      # 128
    scales = [[torch.full((16,), 2.0 ** -7, device=DEV)] for _ in range(2)]                                                  # the value is 1
    g[0].fill_(1.1)
    adamw_step(p, g, m, v, 5, lr=1e-3, betas=(0.9, 0.999), exp_avg_scales=scales[0], exp_avg_sq_scales=scales[1])
    for codes, scale, want in ((m, scales[0], 0.9 + 0.1 * 1.1), (v, scales[1], math.sqrt(0.999 + 0.001 * 1.21))):
        val = codes[0].float() * scale[0].repeat_interleave(256)
        step = 2.0 ** -3
        assert len(set(val.tolist())) == 2
        assert abs(float(val.double().mean()) - want) <= 6 * 0.5 * step / math.sqrt(n) + step * 2.0 ** -12, (float(val.mean()), want)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_class_steps_groups_and_checkpoints(bits):
    g = torch.Generator().manual_seed(2)
    make = lambda: [torch.nn.Parameter(torch.randn(s, generator=g.manual_seed(2)).to(DEV)) for s in ((33, 9), (300,), (5,))]      # noqa: E731
    ps, qs = make(), make()
    groups = lambda v: [{"params": v[:2], "weight_decay": 0.1}, {"params": v[2:], "lr": 1e-2}]      # noqa: E731
    a, b = AdamW(groups(ps), lr=1e-3, state_bits=bits, seed=9), AdamW(groups(qs), lr=1e-3, state_bits=bits, seed=9)
    t = torch.optim.AdamW([{"params": [p.detach().clone().requires_grad_() for p in v["params"]], **{k: x for k, x in v.items() if k != "params"}}
                           for v in groups(ps)], lr=1e-3, weight_decay=0.0)
    tp = [p for gr in t.param_groups for p in gr["params"]]
    for k in range(4):
        if k == 3:                                # a schedule
            for opt in (a, b, t):
                opt.param_groups[0]["lr"] = 5e-4
        for p, q in zip(ps, tp):
            grad = torch.randn(p.shape, generator=g).to(DEV)
            p.grad, q.grad = grad, grad.clone()
        if k == 2:
            ps[1].grad = tp[1].grad = None        # sits this step out
        a.step()
        t.step()
        if k == 1:
            sd = a.state_dict()
            for p, q in zip(ps, qs):
                q.data.copy_(p.data)
            b.load_state_dict(sd)
        elif k > 1:
            for p, q in zip(ps, qs):
                q.grad = p.grad
            b.step()
    assert a.steps == [4, 3, 4] == b.steps
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)                  # resumed from the state dict: the same bits
    if bits == 32:
        t2 = torch.optim.AdamW([{"params": [x]} for x in tp])
        for p, q in zip(ps, tp):                  # four steps of at most lr each; both in 32 bits
            assert float((p - q).abs().max()) <= 4 * (1e-2 * 40 + 8) * R.U * float(1 + p.abs().max())
        del t2
        for i, st in a.state_dict()["state"].items():
            ref = t.state[tp[i]]
            assert float(st["step"]) == float(ref["step"])
            assert torch.allclose(st["exp_avg"], ref["exp_avg"], rtol=32 * R.U, atol=32 * R.U)
            assert torch.allclose(st["exp_avg_sq"], ref["exp_avg_sq"], rtol=64 * R.U, atol=0)
    a.zero_grad(set_to_none=True)
    assert all(p.grad is None for p in ps)
    before = [p.detach().clone() for p in ps]
    a.step()
    assert all(torch.equal(x, p) for x, p in zip(before, ps)) and a.steps == [4, 3, 4]


def test_adamw_of_a_tensor_of_more_than_2_to_32_values():
    """Offsets that pass 32 bits: places around 2^32 and the end, against the formula with their own random bits."""
    n = 2 ** 32 + 777
    g = torch.Generator().manual_seed(5)
    base = [torch.randn(1 << 20, generator=g).to(DEV, torch.bfloat16) for _ in range(2)]
    tile = lambda b: b.repeat(-(-n // b.numel()))[:n]      # noqa: E731
    p, grad = tile(base[0]), tile(base[1])
    m, v = (torch.zeros(n, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2))
    scales = [torch.ones(blocks_of(n), device=DEV) for _ in range(2)]
    hyper = dict(lr=2e-3, betas=(0.9, 0.99), eps=1e-7, weight_decay=0.1)
    adamw_step([p], [grad], [m], [v], 1, seed=3, exp_avg_scales=[scales[0]], exp_avg_sq_scales=[scales[1]], **hyper)
    for first, count in ((0, 1024), (2 ** 31 - 512, 1024), (2 ** 32 - 512, 1024), (2 ** 32 + 512, 265)):
        here = slice(first, first + count)
        old = [tile_of.repeat(2)[first % (1 << 20):][:count].cpu().double() for tile_of in base]
        want = R.adamw(old[0], old[1], torch.zeros(count, dtype=torch.float64), torch.zeros(count, dtype=torch.float64), 1, **hyper)
        rnd = R.random_bits(count, 3, 1, 0, first)
        p1, e_p = want["p"]
        unit = torch.exp2(torch.frexp(p1)[1].double() - 8)
        cut = (R.mix32(rnd ^ 0x68E31DA4) & 0xFFFF).double() * 2.0 ** -16
        lo, hi = (((p1.abs() + s * e_p) / unit + cut).floor() * unit for s in (-1, 1))
        got = p[here].cpu().double()
        assert ((got.abs() >= lo - e_p) & (got.abs() <= hi + e_p)).all(), first
        blk = slice(first // 256, -(-(first + count) // 256))
        for k, t, scale, r, root in (("m", m, scales[0], ((rnd & 0xFFF) << 8) | 0x80, False), ("root", v, scales[1], rnd >> 12, True)):
            w, e = want[k]
            s = scale[blk].cpu().double()
            assert ((s >= R.block_scales((w.abs() - e).clamp_min(0))) & (s <= R.block_scales(w.abs() + e))).all(), (first, k)
            lo, hi = R.codes_allowed(w, e, s, r, root)
            code = t[here].cpu().float().double()
            assert ((code.abs() >= lo) & (code.abs() <= hi)).all(), (first, k)


@pytest.mark.parametrize("op", ["pref", "policy"])
def test_losses_of_more_than_2_to_31_values(op):
    """The last pair / transition of a batch whose offsets pass 2^31, against the same one alone (the mean over n rows divides by n)."""
    C, T, B = 64, 65536, 514
    rows = B // 2 if op == "pref" else B
    small = R.make(op, 2 if op == "pref" else 1, C, T, torch.bfloat16, seed=3, device=DEV)
    d = {}
    for k, t in small.items():
        if not isinstance(t, torch.Tensor) or "logit" in k:
            d[k] = t
        elif op == "pref":        # preferred rows, then rejected ones
            d[k] = torch.cat([h.expand((rows,) + h.shape[1:]) for h in t.split(1)]).contiguous()
        else:
            d[k] = t.expand((B,) + t.shape[1:]).contiguous()
    alone, got = call(op, small), call(op, d)
    for k in ("margin",) if op == "pref" else ("logp", "ratio", "kl"):
        assert torch.allclose(got[k].double(), alone[k].double().expand(rows), rtol=4 * R.U, atol=1e-9), k
    # The gradient times n is that of the row alone, and within the same bound of the formula: every rounding is relative to what it rounds (a
    # bare multiple of bf16's half step is not enough where the residual's and the KL term's parts of a gradient cancel: they are rounded
    # before they are added), but for the least numbers, which grow with n.
    w, bound = reference(op, small)["d_model_out"]
    for i in ([0, rows - 1, rows, B - 1] if op == "pref" else [0, 256, B - 1]):
        j = i // rows if op == "pref" else 0
        assert ((got["d_model_out"][i].double() * rows - w[j].to(DEV)).abs() <= bound[j].to(DEV) + rows * 2.0 ** -133).all(), i
    assert torch.allclose(got["d_logit"], alone["d_logit"], rtol=1e-4, atol=1e-4 * float(alone["d_logit"].abs().max()))


def test_adamw_of_mixed_types_in_one_list():
    """fp32 and bf16 parameters and gradients side by side: each is what it is in a list of its own kind at the same place."""
    kinds = [(torch.float32, torch.float32), (torch.bfloat16, torch.float32), (torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16)]
    shapes = [(300,), (1000,), (77,), (513,)]
    for bits in (32, 8):
        made = [lists(shapes, p, g, bits, 5) for p, g in kinds]
        pick = [[made[i][j][i] for i in range(4)] for j in range(4)]
        scales = {k: [made[i][4][k][i].clone() for i in range(4)] for k in made[0][4]}
        p, g, m, v = [[t.clone() for t in ts] for ts in pick]
        adamw_step(p, g, m, v, 2, lr=1e-3, seed=7, **scales)
        for i, (a, b, c, d, sc) in enumerate(made):
            adamw_step(a, b, c, d, 2, lr=1e-3, seed=7, **sc)
            assert torch.equal(a[i], p[i]) and torch.equal(bits_of(c[i]), bits_of(m[i])) and torch.equal(bits_of(d[i]), bits_of(v[i])), (bits, i)


def test_adamw_skips_empty_tensors_and_steps_nothing_else():
    z = lambda *s: torch.zeros(s, device=DEV)      # noqa: E731
    a = AdamW([z(0), torch.ones(3, device=DEV), z(4, 0)], lr=0.1, state_bits=8)
    for p in a.params:
        p.grad = torch.ones_like(p)
    a.step()
    assert a.steps == [1, 1, 1] and (a.params[1] < 1).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_step_counts_as_a_change_of_the_parameters(bits):
    """A graph that saved the values before the step refuses its backward."""
    p = torch.nn.Parameter(torch.ones(300, device=DEV))
    opt = AdamW([p], lr=0.1, state_bits=bits)
    loss, before = (p * p).sum(), p._version
    p.grad = torch.ones_like(p)
    opt.step()
    assert p._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()
    (p * p).sum().backward()
