"""Timed cases of the fine-tuning operators: the preference loss and the clipped policy loss of a latent diffusion model with
their gradients, and the AdamW step over many tensors with its moments in 32 or in 8 bits.

`run` computes them in elementary torch operations (`own = False`) or through ddmi_amd's entry points (`own = True`).
Latents are [B, C, H W] (an image's plane, a shape's three planes stacked as channels, or a clip's plane tokens)."""
import math

import torch

own = False

DEV = "cuda:0"
BLOCK = 256           # values of a tensor that share one scale in the 8-bit moments
MASK = 0xFFFFFFFF


def listed():
    return [
        # one preferred and one rejected latent of the small test network: the smallest call, all latency
        {"name": "pref_smallest", "op": "pref", "pairs": 1, "channels": 64, "tokens": 64, "type": "fp32", "mixed": True, "shared_noise": True, "masked": False},
        # image latents 64 x 64 of the AFHQ configuration, 16 pairs a step as with gradient accumulation
        {"name": "pref_image", "op": "pref", "pairs": 16, "channels": 64, "tokens": 4096, "type": "fp32", "mixed": True, "shared_noise": True, "masked": False},
        # a padded last batch of latents with odd planes (35 x 37), network outputs kept in bf16, two of the pairs left out
        {"name": "pref_ragged", "op": "pref", "pairs": 23, "channels": 48, "tokens": 1295, "type": "bf16", "mixed": True, "shared_noise": False, "masked": True},
        # 256 pairs of image latents: the 512 samples a card trains on in the training benchmark
        {"name": "pref_largest", "op": "pref", "pairs": 256, "channels": 64, "tokens": 4096, "type": "fp32", "mixed": True, "shared_noise": True, "masked": False},
        # one denoising transition of the small test network: the smallest policy step
        {"name": "policy_smallest", "op": "policy", "batch": 1, "channels": 64, "tokens": 64, "type": "fp32", "mixed": True, "kl": True, "masked": False},
        # transitions of tri-plane shape latents (192 x 16 x 16), no reference network
        {"name": "policy_shape", "op": "policy", "batch": 64, "channels": 192, "tokens": 256, "type": "fp32", "mixed": True, "kl": False, "masked": False},
        # transitions of video latents (2048 plane tokens) with the KL term, network outputs in bf16, finished chains left out
        {"name": "policy_video", "op": "policy", "batch": 96, "channels": 64, "tokens": 2048, "type": "bf16", "mixed": True, "kl": True, "masked": True},
        # 512 transitions of image latents with the KL term: the largest batch of the training benchmark
        {"name": "policy_largest", "op": "policy", "batch": 512, "channels": 64, "tokens": 4096, "type": "fp32", "mixed": True, "kl": True, "masked": False},
        # a small network's 128 parameters (most of a few dozen values) in bf16, moments in 32 bits: all latency
        {"name": "adamw32_small", "op": "adamw", "bits": 32, "type": "bf16", "width": 48, "mult": "1,2", "blocks": 1},
        # the AFHQ network's parameters (half a billion values in 368 tensors), moments in 32 bits
        {"name": "adamw32_largest", "op": "adamw", "bits": 32, "type": "fp32", "width": 224, "mult": "1,2,4,6", "blocks": 2},
        # a network of odd width, moments in 8 bits: blocks that end inside a tensor everywhere
        {"name": "adamw8_odd", "op": "adamw", "bits": 8, "type": "bf16", "width": 67, "mult": "1,3", "blocks": 1},
        # the AFHQ network's parameters with the moments in 8 bits
        {"name": "adamw8_largest", "op": "adamw", "bits": 8, "type": "fp32", "width": 224, "mult": "1,2,4,6", "blocks": 2},
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["pref", "policy", "adamw"])
    if op == "adamw":
        return {"op": op, "bits": rng.choice([8, 32]), "type": rng.choice(["fp32", "bf16"]), "width": spread(8, 160),
                "mult": rng.choice(["1", "1,2", "1,3", "1,2,2", "1,2,4"]), "blocks": rng.choice([1, 2])}
    channels, tokens = spread(1, 256), spread(1, 8192)
    most = 2 ** 26 // (channels * tokens)        # half of the largest listed batch
    batch = min(spread(1, 512), max(1, most))
    c = {"op": op, "channels": channels, "tokens": tokens, "type": rng.choice(["fp32", "bf16"]), "mixed": rng.random() < 0.75, "masked": rng.random() < 0.5}
    return dict(c, pairs=max(1, batch // 2), shared_noise=rng.random() < 0.5) if op == "pref" else dict(c, batch=batch, kl=rng.random() < 0.5)


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _network_shapes(width, mult, blocks):
    """The parameter shapes of a denoising U-Net: residual blocks, attention below the first level, skip connections."""
    mult, emb = [int(m) for m in mult.split(",")], 4 * width
    shapes = [(emb, width), (emb,), (emb, emb), (emb,), (width, 64, 3, 3), (width,)]

    def res(cin, cout):
        s = [(cin,), (cin,), (cout, cin, 3, 3), (cout,), (cout, emb), (cout,), (cout,), (cout,), (cout, cout, 3, 3), (cout,)]
        return s + ([(cout, cin, 1, 1), (cout,)] if cin != cout else [])

    def attention(c):
        return [(c,), (c,), (3 * c, c, 1), (3 * c,), (c, c, 1), (c,)]

    ch, skips = width, [width]
    for level, m in enumerate(mult):
        for _ in range(blocks):
            shapes += res(ch, m * width) + (attention(m * width) if level else [])
            ch = m * width
            skips.append(ch)
        if level < len(mult) - 1:
            shapes += [(ch, ch, 3, 3), (ch,)]
            skips.append(ch)
    shapes += res(ch, ch) + attention(ch) + res(ch, ch)
    for level, m in reversed(list(enumerate(mult))):
        for i in range(blocks + 1):
            shapes += res(ch + skips.pop(), m * width) + (attention(m * width) if level else [])
            ch = m * width
            if level and i == blocks:
                shapes += [(ch, ch, 3, 3), (ch,)]
    return shapes + [(ch,), (ch,), (64, ch, 3, 3), (64,)]


def _type(case):
    return torch.float32 if case["type"] == "fp32" else torch.bfloat16


def _sizes(case):
    return [math.prod(s) for s in _network_shapes(case["width"], case["mult"], case["blocks"])]


def _views(slab, shapes, sizes, pitch):
    out, at = [], 0
    for shape, n in zip(shapes, sizes):
        out.append(slab[at:at + n].view(shape))
        at += pitch(n)
    return out


def _blocks(n):
    return -(-n // BLOCK)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(*shape):
        return torch.randn(shape, device=DEV, generator=g)

    def rand(*shape):
        return torch.rand(shape, device=DEV, generator=g)

    if case["op"] == "adamw":
        shapes, sizes = _network_shapes(case["width"], case["mult"], case["blocks"]), _sizes(case)
        n, rows = sum(sizes), sum(_blocks(k) for k in sizes)
        s = {"case": case, "step": 400, "seed": seed % 65521, "lr": 1e-4, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01, "grad_scale": 0.5}
        # parameters and gradients are views of one slab each, one behind the other, as a training step lays them out
        s["p"], s["g"] = (0.05 * randn(n)).to(_type(case)), (0.002 * randn(n)).to(_type(case))
        s["params"], s["grads"] = (_views(s[k], shapes, sizes, lambda k: k) for k in "pg")
        if case["bits"] == 32:
            s["m"], s["v"] = 3e-4 * randn(n), (1e-3 * randn(n)) ** 2
            s["exp_avg"], s["exp_avg_sq"] = (_views(s[k], shapes, sizes, lambda k: k) for k in "mv")
            s["m_scale"] = s["v_scale"] = s["exp_avg_scale"] = s["exp_avg_sq_scale"] = None
        else:
            # codes of the first moment and of the second one's root, whole blocks a tensor; scales are powers of two
            flat = [(k,) for k in sizes]
            s["m"] = (randn(rows * BLOCK) * 64).clamp_(-256, 256).to(torch.float8_e4m3fn)
            s["v"] = (rand(rows * BLOCK) * 200 + 2).to(torch.float8_e4m3fn)
            s["m_scale"], s["v_scale"] = (torch.exp2(torch.randint(-20, -16, (rows,), device=DEV, generator=g).float()) for _ in range(2))
            s["exp_avg"], s["exp_avg_sq"] = (_views(s[k], flat, sizes, lambda k: _blocks(k) * BLOCK) for k in "mv")
            s["exp_avg_scale"], s["exp_avg_sq_scale"] = (_views(s[k], [(_blocks(k),) for k in sizes], [_blocks(k) for k in sizes], lambda k: k)
                                                         for k in ("m_scale", "v_scale"))
        return s
    B = 2 * case["pairs"] if case["op"] == "pref" else case["batch"]
    C, T, dt = case["channels"], case["tokens"], _type(case)
    s = {"case": case, "x_t": randn(B, C, T), "sqrt_1mac": 0.15 + 0.8 * rand(B)}
    s["logit"] = (randn(1, C, 1) - 1.0).requires_grad_() if case["mixed"] else None
    s["ref_logit"] = s["logit"].detach() + 0.01 * randn(1, C, 1) if case["mixed"] else None
    s["weight"] = None
    if case["op"] == "pref":
        half = B // 2
        s["sqrt_1mac"][half:] = s["sqrt_1mac"][:half]                        # both of a pair at one time step
        s["noise"] = randn(half if case["shared_noise"] else B, C, T)
        near = s["noise"].repeat(B // s["noise"].shape[0], 1, 1)
        out = near + 0.4 * randn(B, C, T)
        s["beta"], s["label_smoothing"] = 2000.0, 0.1 if case["masked"] else 0.0
        rows = half
    else:
        out = randn(B, C, T)
        sigma = 0.05 + 0.09 * rand(B)
        s["transition"] = torch.stack([1.0 + 0.01 * rand(B), -(0.02 + 0.1 * rand(B)), sigma], dim=1)
        s["advantage"], s["clip_range"], s["kl_coef"] = randn(B), 1e-4, 0.05 if case["kl"] else 0.0
        rows = B
    s["ref_out"] = (out + 0.02 * randn(B, C, T)).to(dt) if case["op"] == "pref" or case["kl"] else None
    s["model_out"] = out.to(dt)
    if case["op"] == "policy":
        # a chain's own step under the sampling network, which the trained one has moved a little from
        mu = _mean64(s, s["model_out"], s["logit"]) if B * C * T <= 2 ** 24 else torch.cat(
            [_mean64(s, s["model_out"], s["logit"], slice(b, b + 64)).float() for b in range(0, B, 64)])
        s["x_prev"] = (mu + sigma[:, None, None] * randn(B, C, T)).float()
        z = s["x_prev"] - mu.float()
        logp = -(z * z).mean((1, 2), dtype=torch.float64) / (2 * sigma.double() ** 2) - sigma.double().log() - 0.5 * math.log(2 * math.pi)
        s["logp_old"] = (logp + 3e-4 * randn(B)).float()
        del mu, z
    if case["masked"]:                       # rows that a batch was filled up with hold anything at all
        s["weight"] = 0.5 + rand(rows)
        s["weight"][max(1, rows // 2)::5] = 0.0
        gone = s["weight"] == 0
        gone = torch.cat([gone, gone]) if case["op"] == "pref" else gone
        s["model_out"][gone] = float("nan")
        s["x_t"][gone] = float("inf")
    s["model_out"].requires_grad_()
    return s


def work(case):
    if case["op"] == "adamw":
        n, t = sum(_sizes(case)), 4 if case["type"] == "fp32" else 2
        rows = sum(_blocks(k) for k in _sizes(case))
        state = 16 * n if case["bits"] == 32 else 4 * n + 16 * rows      # both moments in and out (and their scales)
        return {"bytes": 3 * t * n + state, "flops": 18 * n}
    C, T, t = case["channels"], case["tokens"], 4 if case["type"] == "fp32" else 2
    B = 2 * case["pairs"] if case["op"] == "pref" else case["batch"]
    n = B * C * T
    second = n // 2 if case["op"] == "pref" and case["shared_noise"] else n        # the noise, or the chain's next state
    ref = n if case["op"] == "pref" or case["kl"] else 0
    return {"bytes": t * (2 * n + ref) + 4 * (n + second), "flops": 20 * n}


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        state["step"] += 1
        if own:
            from ddmi_amd.optim import adamw_step
            adamw_step(state["params"], state["grads"], state["exp_avg"], state["exp_avg_sq"], state["step"], lr=state["lr"], betas=state["betas"],
                       eps=state["eps"], weight_decay=state["weight_decay"], grad_scale=state["grad_scale"],
                       exp_avg_scales=state["exp_avg_scale"], exp_avg_sq_scales=state["exp_avg_sq_scale"], seed=state["seed"])
        else:
            _adamw(state)
        return {k: state[k] for k in ("p", "m", "v", "m_scale", "v_scale")}
    if not own:
        with torch.no_grad():
            return _preference(state) if op == "pref" else _policy(state)
    from ddmi_amd.finetune import policy_loss, preference_loss
    mixing = {"mixing_logit": state["logit"], "ref_mixing_logit": state["ref_logit"], "weight": state["weight"]}
    if op == "pref":
        r = preference_loss(state["model_out"], state["ref_out"], state["x_t"], state["noise"], state["sqrt_1mac"], beta=state["beta"],
                            label_smoothing=state["label_smoothing"], **mixing)
        stats = {"margin": r.margin, "mse": r.mse}
    else:
        r = policy_loss(state["model_out"], state["x_t"], state["x_prev"], state["transition"], state["sqrt_1mac"], state["logp_old"],
                        state["advantage"], clip_range=state["clip_range"], ref_out=state["ref_out"], kl_coef=state["kl_coef"], **mixing)
        stats = {"logp": r.logp, "ratio": r.ratio, "kl": r.kl}
    leaves = [state["model_out"]] + ([state["logit"]] if state["logit"] is not None else [])
    grads = torch.autograd.grad(r.loss, leaves)
    return {"loss": r.loss, **stats, "d_model_out": grads[0], "d_logit": grads[1] if len(grads) > 1 else None}


def _mixed(out, m, logit):
    """The network's prediction: its output mixed, per channel, with the linear one `m`."""
    return out if logit is None else m + torch.sigmoid(logit) * (out - m)


def _moved(out, ref, m, logit, ref_logit):
    """The network's prediction less the reference's, from the difference of the outputs: both predictions alone would cancel."""
    if logit is None:
        return out - ref
    c, c_ref = torch.sigmoid(logit.double()), torch.sigmoid(ref_logit.double())
    return c.float() * (out - ref) + (c - c_ref).float() * (ref - m)


def _row(v):
    return v[:, None, None]


def _preference(s):
    """Per sample e = mean((prediction - noise)^2); margin h = -beta/2 ((e - e_ref) of the preferred - that of the rejected);
    loss = the weighted mean of -(1 - a) log sigma(h) - a log sigma(-h)."""
    half, out = s["case"]["pairs"], s["model_out"].float()
    n = out[0].numel()
    noise = s["noise"].repeat(2 * half // s["noise"].shape[0], 1, 1)
    m = _row(s["sqrt_1mac"]) * s["x_t"]
    d = _mixed(out, m, s["logit"]) - noise
    far = _moved(out, s["ref_out"].float(), m, s["logit"], s["ref_logit"])
    part = out - m
    w = torch.ones(half, device=DEV) if s["weight"] is None else s["weight"]
    if s["weight"] is not None:
        used = _row(torch.cat([w, w]) > 0)
        d, far, part = (torch.where(used, t, 0.0) for t in (d, far, part))
    more = (far * (2 * d - far)).sum((1, 2), dtype=torch.float64) / n
    mse = (d * d).sum((1, 2), dtype=torch.float64) / n
    h = -0.5 * s["beta"] * (more[:half] - more[half:])
    a, total = s["label_smoothing"], w.double().sum().clamp_min(1e-300)
    lsig = -torch.log1p(torch.exp(-h.abs()))
    loss = (w * -((1 - a) * (lsig + h.clamp_max(0)) + a * (lsig - h.clamp_min(0)))).sum() / total
    dh = w * (a * torch.sigmoid(h) - (1 - a) * torch.sigmoid(-h)) / total
    k = torch.cat([-dh, dh]) * (s["beta"] / n)
    g = _row(k.float()) * d
    c = None if s["logit"] is None else torch.sigmoid(s["logit"])
    return {"loss": loss.float(), "margin": torch.where(w > 0, h, 0.0).float(), "mse": mse.float(),
            "d_model_out": (g if c is None else g * c).to(s["model_out"].dtype),
            "d_logit": None if c is None else ((g * part).sum((0, 2), dtype=torch.float64)[None, :, None] * c * (1 - c)).float()}


def _policy(s):
    """mu = A x_t + E prediction; logp = the mean over the values of log N(x_prev; mu, sigma^2); ratio = exp(logp - logp_old);
    loss = the weighted mean of max(-adv ratio, -adv clip(ratio)) + kl_coef mean((mu - mu_ref)^2) / (2 sigma^2)."""
    out, logit = s["model_out"].float(), s["logit"]
    n = out[0].numel()
    A, E, sigma = (_row(v) for v in s["transition"].unbind(1))
    m = _row(s["sqrt_1mac"]) * s["x_t"]
    z, part = (s["x_prev"] - A * s["x_t"]) - E * _mixed(out, m, logit), out - m
    w = torch.ones(len(out), device=DEV) if s["weight"] is None else s["weight"]
    far = None if s["ref_out"] is None else E * _moved(out, s["ref_out"].float(), m, logit, s["ref_logit"])
    if s["weight"] is not None:
        used = _row(w > 0)
        z, part = torch.where(used, z, 0.0), torch.where(used, part, 0.0)
        far = None if far is None else torch.where(used, far, 0.0)
    var = s["transition"][:, 2].double() ** 2
    logp = -(z * z).sum((1, 2), dtype=torch.float64) / n / (2 * var) - 0.5 * var.log() - 0.5 * math.log(2 * math.pi)
    ratio = torch.exp(logp - s["logp_old"])
    kl = torch.zeros_like(ratio) if far is None else (far * far).sum((1, 2), dtype=torch.float64) / n / (2 * var)
    adv, eps, total = s["advantage"].double(), s["clip_range"], w.double().sum().clamp_min(1e-300)
    free, bound = -adv * ratio, -adv * ratio.clamp(1 - eps, 1 + eps)
    used = w > 0
    loss = torch.where(used, w * (torch.maximum(free, bound) + s["kl_coef"] * kl), 0.0).sum() / total
    k = torch.where(used & (free >= bound), -adv * ratio * w / total, 0.0) / (var * n)
    g = _row(k.float()) * z
    if far is not None:
        g = g + _row((w / total * s["kl_coef"] / (var * n)).float()) * far
    g = E * g
    c = None if logit is None else torch.sigmoid(logit)
    return {"loss": loss.float(), **{k: torch.where(used, v, 0.0).float() for k, v in (("logp", logp), ("ratio", ratio), ("kl", kl))},
            "d_model_out": (g if c is None else g * c).to(s["model_out"].dtype),
            "d_logit": None if c is None else ((g * part).sum((0, 2), dtype=torch.float64)[None, :, None] * c * (1 - c)).float()}


def _scalars(s):
    """What the step number gives: decay of the parameter, step size, the second moment's correction; each rounded to 32 bits in use."""
    b1, b2 = s["betas"]
    return 1.0 - s["lr"] * s["weight_decay"], s["lr"] / (1.0 - b1 ** s["step"]), 1.0 / math.sqrt(1.0 - b2 ** s["step"])


def _adamw(s):
    """m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, p = p (1 - lr wd) - lr / bc1 m / (sqrt(v) / bc2 + eps)."""
    b1, b2 = s["betas"]
    decay, size, inv_bc2 = _scalars(s)
    if s["case"]["bits"] == 32 and s["case"]["type"] == "fp32":
        # lists of tensors, one operation over all of them at a time
        grads = torch._foreach_mul(s["grads"], s["grad_scale"])
        torch._foreach_mul_(s["exp_avg"], b1)
        torch._foreach_add_(s["exp_avg"], grads, alpha=1.0 - b1)
        torch._foreach_mul_(s["exp_avg_sq"], b2)
        torch._foreach_mul_(grads, grads)
        torch._foreach_add_(s["exp_avg_sq"], grads, alpha=1.0 - b2)
        denom = torch._foreach_sqrt(s["exp_avg_sq"])
        torch._foreach_mul_(denom, inv_bc2)
        torch._foreach_add_(denom, s["eps"])
        change = torch._foreach_div(s["exp_avg"], denom)
        torch._foreach_mul_(s["params"], decay)
        torch._foreach_add_(s["params"], change, alpha=-size)
        return
    # one row for each block of 256 values of a tensor: the unit of the scales and of the random numbers
    sizes = _sizes(s["case"])
    p, g = (_rows(s[k], sizes) for k in ("params", "grads"))
    bits32 = s["case"]["bits"] == 32
    rnd, used = _random_rows(s, sizes)
    if bits32:
        m, v = (_rows(s[k], sizes) for k in ("exp_avg", "exp_avg_sq"))
    else:
        m, root = (s[k].view(-1, BLOCK).float() * s[k + "_scale"][:, None] for k in "mv")
        v = root * root
    g = g * s["grad_scale"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * (1.0 - b2)) * g
    root = v.sqrt()
    p = p * decay - (m / (root * inv_bc2 + s["eps"])) * size
    if s["case"]["type"] == "bf16":
        # round up with the probability of what is cut off (a parameter this coarse would stand still under nearest rounding)
        more = _mix32(rnd ^ _i32(0x68E31DA4)) & 0xFFFF
        p = ((p.view(torch.int32) + more) & _i32(0xFFFF0000)).view(torch.float32)
    _unrows(s["params"], p, sizes)
    if bits32:
        _unrows(s["exp_avg"], m, sizes)
        _unrows(s["exp_avg_sq"], v, sizes)
        return
    for name, x, r, positive in (("m", m, ((rnd & 0xFFF) << 8) | 0x80, False), ("v", root, (rnd >> 12) & 0xFFFFF, True)):
        x = torch.where(used, x, 0.0)
        scale = _block_scale(x.abs().amax(1))
        code = _encoded(x / scale[:, None], r, positive)
        s[name].view(-1, BLOCK).copy_(torch.where(used, code, s[name].view(torch.uint8).view(-1, BLOCK)).view(torch.float8_e4m3fn))
        s[name + "_scale"].copy_(scale)


def _rows(tensors, sizes):
    rows = torch.zeros(sum(_blocks(n) for n in sizes), BLOCK, device=DEV)
    places = rows.view(-1).split([_blocks(n) * BLOCK for n in sizes])
    torch._foreach_copy_([f[:n] for f, n in zip(places, sizes)], [t.reshape(-1) for t in tensors])
    return rows


def _unrows(tensors, rows, sizes):
    flat = rows.reshape(-1).split([_blocks(n) * BLOCK for n in sizes])
    torch._foreach_copy_([t.view(-1) for t in tensors], [f[:n] for f, n in zip(flat, sizes)])


def _i32(v):
    return v - (1 << 32) if v >= 1 << 31 else v


def _mix32(x):
    """A 32-bit integer mix (two multiplications, three shifts), on int32 tensors."""
    x = x ^ ((x >> 16) & 0xFFFF)
    x = x * _i32(0x85EBCA6B)
    x = x ^ ((x >> 13) & 0x7FFFF)
    x = x * _i32(0xC2B2AE35)
    return x ^ ((x >> 16) & 0xFFFF)


def _mix32_int(x):
    x ^= x >> 16
    x = x * 0x85EBCA6B & MASK
    x ^= x >> 13
    x = x * 0xC2B2AE35 & MASK
    return x ^ x >> 16


def _tensor_keys(s, count):
    """One key for each tensor of a step, from the seed, the step's number and the tensor's place in the list."""
    key = _mix32_int((_mix32_int(s["seed"] & MASK) + s["step"] * 0x9E3779B9) & MASK)
    return [_mix32_int((key + (i + 1) * 0x85EBCA77) & MASK) for i in range(count)]


def _random_rows(s, sizes):
    """32 random bits for each value: of its tensor's key, its block and its place in the block, int32 [blocks, 256]; and where there
    is a value (a tensor's last block is not full)."""
    size = torch.tensor(sizes, device=DEV)
    count = (size + BLOCK - 1) // BLOCK
    key = torch.tensor([_i32(k) for k in _tensor_keys(s, len(sizes))], device=DEV, dtype=torch.int32).repeat_interleave(count)
    first = (count.cumsum(0) - count).repeat_interleave(count)
    block = (torch.arange(len(key), device=DEV) - first).to(torch.int32)
    lane = torch.arange(BLOCK, device=DEV, dtype=torch.int32)[None]
    left = (size.repeat_interleave(count) - BLOCK * block).clamp_max(BLOCK)
    return _mix32(_mix32(key + block * _i32(0x9E3779B9))[:, None] + lane * _i32(0x9E3779B9)), lane < left[:, None]


def _block_scale(most):
    """2^k with most / 2^k in (128, 256], k between -120 and 120 (the smallest k where nothing is left)."""
    bits = most.view(torch.int32)
    k = (bits >> 23) - 127 + ((bits & 0x7FFFFF) != 0).int() - 8
    return ((k.clamp(-120, 120) + 127) << 23).view(torch.float32)


def _encoded(x, r, positive):
    """The 8-bit float (4 exponent and 3 fraction bits, bias 7) next above |x| with the probability of the part cut off, else the
    next below: `r` holds 20 random bits. `positive`: no sign, and only a zero becomes zero."""
    a = x.abs()
    bits = a.view(torch.int32)
    normal = ((bits + r) >> 20) - (120 << 3)
    small = (a * 512.0 + r.float() * 2.0 ** -20).floor().to(torch.int32)
    code = torch.where(a < 2.0 ** -6, small, normal)
    if positive:
        code = torch.where(a > 0, code.clamp_min(1), code)
    else:
        code = code | ((x.view(torch.int32) >> 24) & 0x80)
    return code.to(torch.uint8)


# ---------------------------------------------------------------------------------------------------------------------
# the same in 64 bits: losses differentiated by autograd, moments one tensor at a time on the table of the 8-bit values
# ---------------------------------------------------------------------------------------------------------------------
def _mean64(s, out, logit, at=slice(None)):
    A, E, _ = (v[:, None, None] for v in s["transition"][at].double().unbind(1))
    x, o = s["x_t"][at].double(), out[at].detach().double()
    eps = o
    if logit is not None:
        c = 1.0 / (1.0 + torch.exp(-logit.detach().double()))
        eps = (1 - c) * s["sqrt_1mac"][at].double()[:, None, None] * x + c * o
    return A * x + E * eps


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_adamw(s) if case["op"] == "adamw" else _exact_loss(s, case["op"])


def _exact_loss(s, op):
    leaf = s["logit"].detach().double().requires_grad_() if s["logit"] is not None else None
    B, half = len(s["model_out"]), len(s["model_out"]) // 2
    rows = half if op == "pref" else B
    weight = torch.ones(rows, device=DEV, dtype=torch.float64) if s["weight"] is None else s["weight"].double()
    total = weight.sum()
    keep = [i for i, w in enumerate(weight.tolist()) if w > 0]
    names = ("margin",) if op == "pref" else ("logp", "ratio", "kl")
    stats = {k: torch.zeros(rows, device=DEV, dtype=torch.float64) for k in names}
    if op == "pref":
        stats["mse"] = torch.zeros(B, device=DEV, dtype=torch.float64)
    d_out, loss = torch.zeros(s["model_out"].shape, device=DEV, dtype=torch.float64), 0.0
    step = max(1, 2 ** 23 // s["x_t"][0].numel())
    for at in range(0, len(keep), step):       # rows do not meet but in the sums
        i = torch.tensor(keep[at:at + step], device=DEV)
        j = torch.cat([i, i + half]) if op == "pref" else i
        out = s["model_out"].detach()[j].double().requires_grad_()
        x, sd = s["x_t"][j].double(), s["sqrt_1mac"][j].double()[:, None, None]

        def prediction(o, logit):
            if logit is None:
                return o
            c = 1.0 / (1.0 + torch.exp(-logit.double()))
            return (1 - c) * sd * x + c * o

        eps = prediction(out, leaf)
        if op == "pref":
            noise = s["noise"][j if len(s["noise"]) == B else torch.cat([i, i])].double()
            e = (eps - noise).square().mean((1, 2))
            e_ref = (prediction(s["ref_out"][j].double(), s["ref_logit"]) - noise).square().mean((1, 2))
            gap = (e - e_ref).view(2, -1)
            h = -s["beta"] / 2 * (gap[0] - gap[1])
            a = s["label_smoothing"]
            each = -(1 - a) * torch.nn.functional.logsigmoid(h) - a * torch.nn.functional.logsigmoid(-h)
            stats["margin"][i], stats["mse"][j] = h.detach(), e.detach()
        else:
            A, E, sigma = (v[:, None, None] for v in s["transition"][j].double().unbind(1))
            mu = A * x + E * eps
            logp = (-(s["x_prev"][j].double() - mu).square() / (2 * sigma ** 2) - sigma.log() - 0.5 * math.log(2 * math.pi)).mean((1, 2))
            ratio = (logp - s["logp_old"][j].double()).exp()
            kl = torch.zeros_like(ratio)
            if s["ref_out"] is not None:
                kl = ((mu - A * x - E * prediction(s["ref_out"][j].double(), s["ref_logit"])).square() / (2 * sigma ** 2)).mean((1, 2))
            adv = s["advantage"][j].double()
            each = torch.maximum(-adv * ratio, -adv * ratio.clamp(1 - s["clip_range"], 1 + s["clip_range"])) + s["kl_coef"] * kl
            for k, v in (("logp", logp), ("ratio", ratio), ("kl", kl)):
                stats[k][j] = v.detach()
        part = (weight[i] * each).sum() / total
        part.backward()
        loss = loss + part.detach()
        d_out[j] = out.grad
    return {"loss": loss, **stats, "d_model_out": d_out, "d_logit": None if leaf is None else leaf.grad}


def _exact_adamw(s):
    s["step"] += 1
    decay, size, inv_bc2 = _scalars(s)
    b1, b2 = s["betas"]
    sizes, bits8 = _sizes(s["case"]), s["case"]["bits"] == 8
    p = s["p"].double()
    keys = _tensor_keys(s, len(sizes))
    grid = torch.arange(127, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    m, v = s["m"].double() if not bits8 else s["m"].float().double(), s["v"].double() if not bits8 else s["v"].float().double()
    scales = [None, None] if not bits8 else [s["m_scale"].double(), s["v_scale"].double()]
    at = row = 0
    for n, key in zip(sizes, keys):
        nb = _blocks(n)
        here = slice(at, at + n)
        kept = slice(row * BLOCK, row * BLOCK + n) if bits8 else here
        index = torch.arange(n, device=DEV)
        block, lane = index // BLOCK, index % BLOCK
        g = s["g"][here].double() * s["grad_scale"]
        mi, vi = m[kept], v[kept]
        if bits8:
            mi, vi = mi * scales[0][row + block], (vi * scales[1][row + block]) ** 2
        mi, vi = b1 * mi + (1 - b1) * g, b2 * vi + (1 - b2) * g * g
        pi = p[here] * decay - size * mi / (vi.sqrt() * inv_bc2 + s["eps"])
        r = None
        if bits8 or s["case"]["type"] == "bf16":
            r = _mix64(_mix64((key + block * 0x9E3779B9) & MASK) + lane * 0x9E3779B9 & MASK)
        if s["case"]["type"] == "bf16":
            step = torch.exp2(torch.frexp(pi)[1].double() - 8)       # from one bf16 value of this binade to the next
            pi = torch.trunc(pi / step + pi.sign() * (_mix64(r ^ 0x68E31DA4) & 0xFFFF).double() / 65536) * step
        p[here] = pi
        if not bits8:
            m[kept], v[kept] = mi, vi
        else:
            for k, (x, bits) in enumerate(((mi, ((r & 0xFFF) << 8) | 0x80), (vi.sqrt(), r >> 12))):
                most = torch.zeros(nb, device=DEV, dtype=torch.float64).scatter_reduce(0, block, x.abs(), "amax")
                scale = torch.exp2((torch.ceil(torch.log2(most)) - 8).clamp(-120, 120))
                a = x.abs() / scale[block]
                below = (torch.searchsorted(grid, a, right=True) - 1).clamp(0, 125)
                up = (a - grid[below]) / (grid[below + 1] - grid[below]) + bits.double() / 2 ** 20 >= 1
                q = grid[below + up.long()]
                if k == 1:
                    q = torch.where(a > 0, q.clamp_min(grid[1]), q)
                (m, v)[k][kept] = q * x.sign() if k == 0 else q
                scales[k][row:row + nb] = scale
        at, row = at + n, row + nb
    return {"p": p, "m": m, "v": v, "m_scale": scales[0], "v_scale": scales[1]}


def _mix64(x):
    """The same 32-bit mix, on int64 tensors of 32-bit values."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & MASK
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & MASK
    return x ^ (x >> 16)
