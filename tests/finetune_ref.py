"""The fine-tuning operators in 64 bits, with the error that 32-bit arithmetic may make: every value comes as (value, bound).

Rules behind the bounds (u = 2^-24, half a step of fp32 relative to the value): a product or a sum of two rounded numbers adds u of its own
result; sums over values are held in 64 bits but for four neighbours added in 32 (3 u of the sum of magnitudes); a sum's error is at most
the sum of its terms' errors.  Bounds are worst cases, not statistics, so no case needs a factor on top."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(op, B, C, T, dtype=torch.float32, mixed=True, shared=False, weight=None, kl=True, seed=0, device="cpu", beta=50.0):
    """Inputs of a loss; for `pref` B is the number of samples (twice the pairs)."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g)      # noqa: E731
    d = {"x_t": r(B, C, T), "sqrt_1mac": 0.2 + 0.7 * torch.rand(B, generator=g)}
    rows = B // 2 if op == "pref" else B
    d["mixing_logit"] = r(1, C, 1) - 1 if mixed else None
    d["ref_mixing_logit"] = d["mixing_logit"] + 0.05 * r(1, C, 1) if mixed else None
    d["model_out"] = r(B, C, T).to(dtype)
    d["ref_out"] = (d["model_out"].float() + 0.1 * r(B, C, T)).to(dtype)
    if op == "pref":
        d["noise"] = r(rows if shared else B, C, T)
        d["beta"], d["label_smoothing"] = beta, 0.1
    else:
        sig = 0.1 + 0.2 * torch.rand(B, generator=g)
        A, E = 1 + 0.02 * torch.rand(B, generator=g), -0.05 - 0.1 * torch.rand(B, generator=g)
        d["transition"] = torch.stack([A, E, sig], 1)
        v = lambda t: t.double()[:, None, None]      # noqa: E731
        c = torch.sigmoid(d["mixing_logit"].double()) if mixed else 1.0
        m = v(d["sqrt_1mac"]) * d["x_t"] if mixed else 0.0
        mu = v(A) * d["x_t"] + v(E) * (m + c * (d["model_out"].double() - m))
        d["x_prev"] = (mu + v(sig) * r(B, C, T)).float()
        z = d["x_prev"].double() - mu
        logp = -(z * z).mean((1, 2)) / (2 * sig.double() ** 2) - sig.double().log() - 0.5 * math.log(2 * math.pi)
        d["logp_old"] = (logp + 0.2 * r(B)).float()
        d["advantage"], d["clip_range"] = r(B), 0.1
        d["kl_coef"] = 0.3 if kl else 0.0
        if not kl:
            d["ref_out"] = None
    if weight == "some":
        w = 0.5 + torch.rand(rows, generator=g)
        w[::3] = 0.0
        d["weight"] = w
        gone = torch.cat([w, w]) == 0 if op == "pref" else w == 0
        d["model_out"][gone] = float("nan")
        d["x_t"][gone] = float("inf")
    elif weight == "none_left":
        d["weight"] = torch.zeros(rows)
        d["model_out"][:] = float("nan")
    else:
        d["weight"] = None
    return {k: t.to(device) if isinstance(t, torch.Tensor) else t for k, t in d.items()}


def _common(d, used):
    keep = lambda t: torch.where(used, t, torch.zeros_like(t))      # noqa: E731
    row = lambda t: t.double()[:, None, None]      # noqa: E731
    o = keep(d["model_out"].double())
    x = keep(d["x_t"].double())
    r = keep(d["ref_out"].double()) if d["ref_out"] is not None else None
    if d["mixing_logit"] is None:
        part, eps, e_eps = torch.zeros_like(o), o, torch.zeros_like(o)
        far = o - r if r is not None else torch.zeros_like(o)
        e_far = U * far.abs()
        c = None
        e_part = torch.zeros_like(o)
    else:
        c, cr = (torch.sigmoid(d[k].double().reshape(1, -1, 1)) if d[k] is not None else None for k in ("mixing_logit", "ref_mixing_logit"))
        m = row(d["sqrt_1mac"]) * x
        e_m = U * m.abs()
        part = o - m
        e_part = e_m + U * part.abs()
        eps = m + c * part
        e_eps = c * e_part + U * (c * part).abs() + e_m + U * eps.abs()            # c itself is rounded
        if r is None:
            far, e_far = torch.zeros_like(o), torch.zeros_like(o)
        else:
            dc = c - cr
            far = c * (o - r) + dc * (r - m)
            e_far = 2 * U * (c * (o - r)).abs() + 2 * U * (dc * (r - m)).abs() + dc.abs() * (e_m + U * (r - m).abs()) + U * far.abs()
    return keep, row, o, x, part, e_part, eps, e_eps, far, e_far, c


def _sum(t, e):
    """A sum over the values: terms' errors, and four neighbours added in 32 bits (a product is rounded once, or not, as it is added)."""
    return t.sum((1, 2)), (e + 5 * U * t.abs()).sum((1, 2))


def preference(d):
    rows = d["model_out"].shape[0] // 2
    dev = d["model_out"].device
    w = torch.ones(rows, dtype=torch.float64, device=dev) if d["weight"] is None else d["weight"].double()
    w = torch.where(w > 0, w, torch.zeros_like(w))
    used = (torch.cat([w, w]) > 0)[:, None, None]
    keep, row, o, x, part, e_part, eps, e_eps, far, e_far, c = _common(d, used)
    n = o[0].numel()
    noise = keep(d["noise"].double().repeat(2 * rows // d["noise"].shape[0], 1, 1))
    res = keep(eps - noise)
    e_res = e_eps + U * res.abs()
    q = 2 * res - far
    e_q = 2 * e_res + e_far + U * q.abs()
    more, e_more = _sum(far * q, e_far * q.abs() + far.abs() * e_q + e_far * e_q)
    sq, e_sq = _sum(res * res, 2 * res.abs() * e_res + e_res ** 2)
    h = -0.5 * d["beta"] * (more[:rows] - more[rows:]) / n
    e_h = 0.5 * abs(d["beta"]) * (e_more[:rows] + e_more[rows:]) / n
    a, total = d["label_smoothing"], w.sum().clamp_min(1e-300)
    sp = torch.nn.functional.softplus
    each = (1 - a) * sp(-h) + a * sp(h)
    dh = (w / total) * (a * torch.sigmoid(h) - (1 - a) * torch.sigmoid(-h))
    e_dh = (w / total) * 0.25 * e_h                                    # sigma' <= 1/4
    k = torch.cat([-dh, dh]) * d["beta"] / n
    e_k = torch.cat([e_dh, e_dh]) * abs(d["beta"]) / n + U * k.abs()
    out = {"loss": ((w * each).sum() / total, (w * e_h).sum() / total), "margin": (torch.where(w > 0, h, 0 * h), e_h), "mse": (sq / n, e_sq / n)}
    return _gradients(out, d, row, c, part, e_part, res, e_res, k, e_k)


def _gradients(out, d, row, c, part, e_part, res, e_res, k, e_k, far=None, e_far=None, q=None, e_q=None):
    cc = 1.0 if c is None else c
    g = row(k) * res * cc
    e_g = (row(e_k) * res.abs() + row(k.abs()) * e_res) * cc + 4 * U * g.abs()
    s = res * part
    chan = (row(k) * s).sum((0, 2))
    e_chan = (row(e_k) * s.abs() + row(k.abs()) * (e_res * part.abs() + res.abs() * e_part + e_res * e_part + 7 * U * s.abs())).sum((0, 2))
    if far is not None:
        g2 = row(q) * far * cc
        g = g + g2
        e_g = e_g + (row(e_q) * far.abs() + row(q.abs()) * e_far) * cc + 4 * U * g2.abs() + U * g.abs()
        s = far * part
        chan = chan + (row(q) * s).sum((0, 2))
        e_chan = e_chan + (row(e_q) * s.abs() + row(q.abs()) * (e_far * part.abs() + far.abs() * e_part + e_far * e_part + 7 * U * s.abs())).sum((0, 2))
    out["d_model_out"] = (g, e_g)
    if c is not None:
        f = (c * (1 - c)).reshape(-1)
        out["d_logit"] = (chan * f, e_chan * f)
    else:
        out["d_logit"] = None
    return _stored(out, d)


def _stored(out, d):
    """What is stored is rounded once more: fp32, the output's gradient to its type."""
    done = {}
    for name, v in out.items():
        if v is None:
            done[name] = None
            continue
        step = half_step(d["model_out"].dtype) if name == "d_model_out" else U
        least = 2.0 ** -133 if name == "d_model_out" and d["model_out"].dtype == torch.bfloat16 else 2.0 ** -149
        done[name] = (v[0], v[1] + 1.01 * step * (v[0].abs() + v[1]) + least)
    return done


def policy(d):
    B = d["model_out"].shape[0]
    dev = d["model_out"].device
    w = torch.ones(B, dtype=torch.float64, device=dev) if d["weight"] is None else d["weight"].double()
    A, E, sig = d["transition"].double().unbind(1)
    w = torch.where((w > 0) & (sig > 0), w, torch.zeros_like(w))
    used = (w > 0)[:, None, None]
    keep, row, o, x, part, e_part, eps, e_eps, far, e_far, c = _common(d, used)
    n = o[0].numel()
    y = keep(d["x_prev"].double())
    first = y - row(A) * x                                             # one fused operation, then another
    z = keep(first - row(E) * eps)
    e_z = U * first.abs() + row(E.abs()) * e_eps + U * z.abs()
    var = torch.where(w > 0, sig, torch.ones_like(sig)) ** 2
    sq, e_sq = _sum(z * z, 2 * z.abs() * e_z + e_z ** 2)
    ff, e_ff = _sum(far * far, 2 * far.abs() * e_far + e_far ** 2)
    logp = -sq / n / (2 * var) - 0.5 * var.log() - 0.5 * math.log(2 * math.pi)
    e_logp = e_sq / n / (2 * var)
    out = {"logp": (torch.where(w > 0, logp, 0 * logp), e_logp)}
    if d.get("logp_old") is None:
        return _stored(out, d)
    ratio = torch.exp(logp - d["logp_old"].double())
    e_ratio = ratio * torch.expm1(e_logp)
    kl, e_kl = E ** 2 * ff / n / (2 * var), E ** 2 * e_ff / n / (2 * var)
    adv, ep, total = d["advantage"].double(), d["clip_range"], w.sum().clamp_min(1e-300)
    free, bound = -adv * ratio, -adv * ratio.clamp(1 - ep, 1 + ep)
    each = torch.maximum(free, bound) + d["kl_coef"] * kl
    live = (free >= bound) & (w > 0)
    near = ((ratio - (1 - ep)).abs() <= e_ratio) | ((ratio - (1 + ep)).abs() <= e_ratio)
    assert not bool((near & (w > 0)).any()), "a ratio too near to the clip's border to say which side 32 bits take"
    k = torch.where(live, -adv * ratio * w / total, torch.zeros_like(adv)) / (var * n) * E
    e_k = torch.where(live, adv.abs() * e_ratio * w / total, torch.zeros_like(adv)) / (var * n) * E.abs() + U * k.abs()
    q = w / total * d["kl_coef"] / (var * n) * E ** 2                  # the step from the reference is kept before E
    out.update(loss=((w * each).sum() / total, (w * (adv.abs() * e_ratio + d["kl_coef"] * e_kl)).sum() / total),
               ratio=(torch.where(w > 0, ratio, 0 * ratio), e_ratio), kl=(torch.where(w > 0, kl, 0 * kl), e_kl))
    return _gradients(out, d, row, c, part, e_part, z, e_z, k, e_k, *((far, e_far, q, U * q.abs()) if d["ref_out"] is not None else ()))


def check(got, want, what=""):
    for name, v in want.items():
        if v is None:
            assert got[name] is None, name
            continue
        g, (w, bound) = got[name].detach().double().cpu(), (t.cpu() for t in v)
        g = g.reshape(w.shape)
        assert torch.isfinite(g).all(), (what, name)
        over = (g - w).abs() - bound
        assert float(over.max()) <= 0, (what, name, float((g - w).abs().max()), float(bound[over == over.max()][0] if bound.dim() else bound))


# ---------------------------------------------------------------------------------------------------------------------
# AdamW
# ---------------------------------------------------------------------------------------------------------------------
MASK = 0xFFFFFFFF


def mix32(x):
    """The integer mix of the rounding's random bits, on int64 tensors (or ints) of 32-bit values."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & MASK
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & MASK
    return x ^ (x >> 16)


def random_bits(n, seed, step, index, first=0):
    """32 bits for each of n values of tensor `index` of the list, from value `first` on."""
    key = mix32((mix32(mix32(seed & MASK) + step * 0x9E3779B9 & MASK) + (index + 1) * 0x85EBCA77) & MASK)
    i = torch.arange(first, first + n, dtype=torch.int64)
    return mix32((mix32((key + ((i // 256) & MASK) * 0x9E3779B9) & MASK) + (i % 256) * 0x9E3779B9) & MASK)


GRID = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()      # the code's values that are not negative


def adamw(p, g, m, v, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.0, grad_scale=1.0):
    """One step in 64 bits on 64-bit tensors: {name: (value, bound)} before anything is rounded to be stored.  `root`: of the new v."""
    b1, b2 = betas
    gs = g * grad_scale
    m1, v1 = b1 * m + (1 - b1) * gs, b2 * v + (1 - b2) * gs * gs
    e_m = 4 * U * ((b1 * m).abs() + ((1 - b1) * gs).abs()) + 2.0 ** -140         # constants, products and the sum; the gradient's scaling
    e_v = 6 * U * v1 + 2.0 ** -140                                               # the same of terms that are not negative
    root = v1.sqrt()
    e_root = (v1 + e_v).sqrt() - root + U * root
    denom = root / math.sqrt(1 - b2 ** step) + eps
    change = lr / (1 - b1 ** step) * m1 / denom
    e_denom = e_root / math.sqrt(1 - b2 ** step) + 4 * U * denom
    low = (denom - e_denom).clamp_min(1e-300)
    # the quotient is m times the hardware's reciprocal (within one ulp: 2 U), rounded (U), times the step size (itself rounded: U), rounded (U)
    e_change = lr / (1 - b1 ** step) * (e_m / low + m1.abs() * e_denom / (denom * low)) + 5.01 * U * change.abs()
    p1 = p * (1 - lr * weight_decay) - change
    e_p = e_change + 2 * U * p.abs() + 2 * U * (p1.abs() + e_change)
    return {"p": (p1, e_p), "m": (m1, e_m), "v": (v1, e_v), "root": (root, e_root)}


def block_scales(x):
    """2^k with the block's largest |x| / 2^k in (128, 256]."""
    n = x.numel()
    rows = torch.zeros(-(-n // 256) * 256, dtype=torch.float64)
    rows[:n] = torch.where(x.isfinite(), x.abs(), torch.zeros_like(x))
    most = rows.view(-1, 256).amax(1)
    k = torch.where(most > 0, torch.ceil(torch.log2(most.clamp_min(1e-300))) - 8, torch.full_like(most, -120.0)).clamp(-120, 120)
    return torch.exp2(k)


def codes_allowed(x, err, scale, bits20, root):
    """(lowest, highest) value of the code that |x| +- err may be rounded to with the random bits."""
    s = scale.repeat_interleave(256)[:x.numel()]
    out = []
    for side in (-1, 1):
        a = ((x.abs() + side * err).clamp_min(0) / s).clamp_max(float(GRID[-1]))
        below = (torch.searchsorted(GRID, a, right=True) - 1).clamp(0, 125)
        frac = (a - GRID[below]) / (GRID[below + 1] - GRID[below])
        up = frac + bits20.double() * 2.0 ** -20 + side * 2.0 ** -20 >= 1
        q = GRID[below + up.long()]
        if root:
            q = torch.where(x > 0, q.clamp_min(float(GRID[1])), q)
        out.append(q)
    return out
