"""The measured calls of three operators that make up a training step: group normalisation with an activation on channels-last
maps, log probabilities / entropy / top alternatives of labels, and an AdamW step over many tensors with states in 32 or 8 bits.

`run` computes each either in its plain form (elementary torch operations in fp32) or, with `own` set, through this package.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
LR, BETAS, EPS, DECAY = 5e-4, (0.9, 0.999), 1e-8, 1e-4
BLOCK = 256                                    # elements that share one scale of an 8-bit state
GN_EPS = 1e-5


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one image of 128 x 256 after the encoder, normalised once in a forward pass: launch latency
        {"name": "gn_fwd_small", "op": "gn", "n": 1, "c": 128, "h": 16, "w": 32, "groups": 8, "dtype": "bf16", "act": "relu", "train": False},
        # the 128-channel encoder stage of the training recipe: 6 images of 512 x 1024 at 1/8 resolution
        {"name": "gn_train_encoder", "op": "gn", "n": 6, "c": 128, "h": 64, "w": 128, "groups": 32, "dtype": "bf16", "act": "relu", "train": True},
        # odd maps and 5 channels per group: nothing fits a 16-byte chunk
        {"name": "gn_train_odd", "op": "gn", "n": 3, "c": 30, "h": 61, "w": 93, "groups": 6, "dtype": "fp32", "act": "silu", "train": True},
        # the 16-channel decoder stage of 8 images of 1024 x 2048
        {"name": "gn_train_large", "op": "gn", "n": 8, "c": 16, "h": 512, "w": 1024, "groups": 4, "dtype": "bf16", "act": "silu", "train": True},
        # one answered token over a large vocabulary, with its alternatives
        {"name": "lp_single", "op": "lp", "rows": 1, "c": 131072, "inner": 1, "dtype": "bf16", "top": 8, "train": False, "ignored": 0.0},
        # a batch of the 1000-class classifier, top 5
        {"name": "lp_classifier", "op": "lp", "rows": 32, "c": 1000, "inner": 1, "dtype": "fp32", "top": 5, "train": False, "ignored": 0.0},
        # a training batch of tokens over an odd vocabulary: loss and entropy bonus
        {"name": "lp_tokens_train", "op": "lp", "rows": 4096, "c": 32001, "inner": 1, "dtype": "bf16", "top": 0, "train": True, "ignored": 0.1},
        # label maps of the training recipe: 6 images of 20 classes at 512 x 1024
        {"name": "lp_pixels_train", "op": "lp", "rows": 6, "c": 20, "inner": 512 * 1024, "dtype": "fp32", "top": 2, "train": True, "ignored": 0.05},
        # a linear head fine-tuned alone: a few small tensors
        {"name": "adamw_head", "op": "adamw", "sizes": "2560,20,1280,20,128,128,16", "dtype": "fp32", "bits": 32, "step": 3},
        # every parameter of the 20-class network in its own tensor
        {"name": "adamw_network", "op": "adamw", "sizes": "network", "dtype": "fp32", "bits": 32, "step": 1000},
        {"name": "adamw_network_8bit", "op": "adamw", "sizes": "network", "dtype": "fp32", "bits": 8, "step": 1000},
        # large matrices and ragged vectors in bf16
        {"name": "adamw_large_8bit", "op": "adamw", "sizes": "33554432,16777216,16777216,16777217,8388608,4194304,4096,4096,4095,1000", "dtype": "bf16", "bits": 8, "step": 20000},
    ]


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["gn", "lp_rows", "lp_pixels", "adamw"])
    dtype = rng.choice(["fp32", "bf16"])
    if op == "gn":
        groups = rng.choice([1, 2, 4, 8, 16, 32])
        c = groups * rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
        n = _log_uniform(rng, 1, 16)
        h = _log_uniform(rng, 4, 512)               # below about 16 values a group is all rounding: its gradient cancels to nothing
        w = max(4, min(_log_uniform(rng, 4, 1024), (8 * 16 * 512 * 512) // (n * c * h)))
        return {"op": "gn", "n": n, "c": c, "h": h, "w": w, "groups": groups, "dtype": dtype, "act": rng.choice(["none", "relu", "silu"]),
                "train": rng.random() < 0.6}
    if op == "lp_rows":
        c = _log_uniform(rng, 2, 200000)
        rows = _log_uniform(rng, 1, max(1, min(8192, 60_000_000 // c)))
        return {"op": "lp", "rows": rows, "c": c, "inner": 1, "dtype": dtype, "top": min(c, rng.choice([0, 0, 1, 3, 5, 20])),
                "train": rng.random() < 0.5, "ignored": rng.choice([0.0, 0.1])}
    if op == "lp_pixels":
        c = rng.choice([2, 6, 14, 19, 20, 33, 150])
        inner = _log_uniform(rng, 1, 400_000)
        rows = max(1, min(_log_uniform(rng, 1, 16), 60_000_000 // (c * inner)))
        return {"op": "lp", "rows": rows, "c": c, "inner": inner, "dtype": dtype, "top": min(c, rng.choice([0, 0, 1, 2, 5])),
                "train": rng.random() < 0.5, "ignored": rng.choice([0.0, 0.1])}
    sizes, left = [], 28_000_000
    for _ in range(rng.randint(1, 24)):
        sizes.append(_log_uniform(rng, 1, max(1, min(8_000_000, left))))
        left -= sizes[-1]
    return {"op": "adamw", "sizes": ",".join(map(str, sizes)), "dtype": dtype, "bits": rng.choice([8, 32]), "step": rng.choice([0, 1, 50, 5000])}


def _network_sizes():
    """Parameter sizes of the 20-class network (encoder, its 1x1 head, decoder) in registration order."""
    def down(i, o):
        return [(o - i) * i * 9, o - i, o, o]

    def block(c):
        return [3 * c * c, c, 3 * c * c, c, c, c] * 2

    def up(i, o):
        return [i * o * 9, o, o, o]

    return (down(3, 16) + down(16, 64) + block(64) * 5 + down(64, 128) + block(128) * 8 + [128 * 20, 20]
            + up(128, 64) + block(64) * 2 + up(64, 16) + block(16) * 2 + [16 * 20 * 4, 20])


def _sizes(case):
    return _network_sizes() if case["sizes"] == "network" else [int(s) for s in case["sizes"].split(",")]


def work(case):
    item = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "gn":
        e = case["n"] * case["c"] * case["h"] * case["w"]
        cost = {"none": 6, "relu": 7, "silu": 11}[case["act"]]
        return {"bytes": e * item * (5 if case["train"] else 2), "flops": e * cost * (3 if case["train"] else 1)}
    if case["op"] == "lp":
        rows = case["rows"] * case["inner"]
        e, k = rows * case["c"], case["top"]
        out = rows * (8 + 4 + 4 + k * 12)                       # target, log probability, entropy, the alternatives
        if not case["train"]:
            return {"bytes": e * item + out, "flops": e * 6}
        return {"bytes": 3 * e * item + out + rows * (8 + 8 + k * 12), "flops": e * 14}
    e = sum(_sizes(case))
    state = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
    return {"bytes": e * (3 * item + state), "flops": e * (16 if case["bits"] == 32 else 40)}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    return {"gn": _prepare_gn, "lp": _prepare_lp, "adamw": _prepare_adamw}[case["op"]](case, gen)


def _randn(gen, *shape):
    return torch.randn(*shape, device=DEV, generator=gen)


def _prepare_gn(case, gen):
    n, c, h, w = case["n"], case["c"], case["h"], case["w"]
    dt = TYPES[case["dtype"]]
    # what a convolution leaves behind: channels of different offsets and sizes
    x = _randn(gen, n, h, w, c) * (0.5 + torch.rand(c, device=DEV, generator=gen)) + 0.5 * _randn(gen, c)
    s = {"case": case, "x": x.to(dt).permute(0, 3, 1, 2), "weight": 1 + 0.1 * _randn(gen, c), "bias": 0.1 * _randn(gen, c)}
    if case["train"]:
        s["dy"] = _randn(gen, n, h, w, c).to(dt).permute(0, 3, 1, 2)
        for k in ("x", "weight", "bias"):
            s[k].requires_grad_()
    return s


def _prepare_lp(case, gen):
    n, c, inner, k = case["rows"], case["c"], case["inner"], case["top"]
    shape = (n, inner) if inner > 1 else (n,)
    # logits of a model that is fairly sure: a spread of 2, and the target raised
    z = 2 * _randn(gen, n, c, *shape[1:])
    t = torch.randint(0, c, shape, device=DEV, generator=gen)
    z.scatter_add_(1, t.unsqueeze(1), 3 + _randn(gen, *shape).unsqueeze(1))
    if case["ignored"]:
        t[torch.rand(shape, device=DEV, generator=gen) < case["ignored"]] = -100
    s = {"case": case, "logits": z.to(TYPES[case["dtype"]]), "target": t}
    if case["train"]:
        count = n * inner
        s["g_log_prob"] = (-1.0 + 0.1 * _randn(gen, *shape)) / count         # a mean log loss, weighted from row to row
        s["g_entropy"] = (-0.01 + 0.001 * _randn(gen, *shape)) / count       # and an entropy bonus
        if k:
            s["g_top"] = 0.1 * _randn(gen, n, k, *shape[1:]) / count
        s["logits"].requires_grad_()
    return s


def _prepare_adamw(case, gen):
    sizes, dt = _sizes(case), TYPES[case["dtype"]]
    starts, total = [], 0
    for e in sizes:                                                         # every tensor starts a block of its own
        starts.append(total)
        total += -(-e // BLOCK) * BLOCK
    live = torch.zeros(total, device=DEV)
    for a, e in zip(starts, sizes):
        live[a:a + e] = 1
    blocks = total // BLOCK
    spread = torch.exp(1.5 * _randn(gen, blocks, 1)) * torch.exp(0.5 * _randn(gen, blocks, BLOCK))     # gradients' sizes differ
    flat = lambda t: (t.reshape(-1) * live)                                                           # noqa: E731
    s = {"case": case, "p": flat(0.1 * _randn(gen, total)).to(dt), "g": flat(1e-3 * spread * _randn(gen, blocks, BLOCK)).to(dt)}
    m = flat(3e-4 * spread * _randn(gen, blocks, BLOCK)) if case["step"] else torch.zeros(total, device=DEV)
    r = flat(1e-3 * spread * (0.5 + torch.rand(blocks, BLOCK, device=DEV, generator=gen))) if case["step"] else torch.zeros(total, device=DEV)
    if case["bits"] == 32:
        s["m"], s["v"] = m, r * r
    else:
        for name, t in (("m", m), ("r", r)):
            t = t.view(blocks, BLOCK)
            scale = _scale_of(t.abs().amax(1, keepdim=True))
            s[name] = (t / scale).to(torch.float8_e4m3fn).view(-1)
            s[name + "_scale"] = scale.view(-1)
    s["step"] = case["step"]
    if own:
        from erfnet_pytorch_amd.optim import AdamW
        params = []
        for a, e in zip(starts, sizes):
            p = torch.nn.Parameter(s["p"][a:a + e])
            p.grad = s["g"][a:a + e]
            params.append(p)
        opt = AdamW(params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"])
        for p, a, e in zip(params, starts, sizes):
            st = {"step": torch.tensor(float(case["step"]))}
            if case["bits"] == 32:
                st["exp_avg"], st["exp_avg_sq"] = s["m"][a:a + e], s["v"][a:a + e]
            else:
                b, nb = a // BLOCK, -(-e // BLOCK)
                st["exp_avg"], st["exp_avg_scale"] = s["m"][a:a + e], s["m_scale"][b:b + nb]
                st["exp_avg_sq_root"], st["exp_avg_sq_root_scale"] = s["r"][a:a + e], s["r_scale"][b:b + nb]
            opt.state[p] = st
        s["opt"] = opt
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    return {"gn": _run_gn, "lp": _run_lp, "adamw": _run_adamw}[state["case"]["op"]](state)


def _run_gn(s):
    case = s["case"]
    if own:
        from erfnet_pytorch_amd.norm import group_norm_act
        if not case["train"]:
            with torch.no_grad():
                return {"y": group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], GN_EPS, case["act"])}
        y = group_norm_act(s["x"], case["groups"], s["weight"], s["bias"], GN_EPS, case["act"])
        dx, dw, db = torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])
        return {"y": y.detach(), "dx": dx, "dweight": dw, "dbias": db}
    with torch.no_grad():
        return _group_norm(s)


def _group_norm(s):
    """The definition, on [N, groups, channels of a group, H, W]; rounded once at the end."""
    case, x = s["case"], s["x"]
    n, c, h, w = x.shape
    g = case["groups"]
    split = (n, g, c // g, h, w)
    t = x.float().reshape(split)
    gamma, beta = (s[k].view(1, g, c // g, 1, 1) for k in ("weight", "bias"))
    dims = (2, 3, 4)
    centred = t - t.mean(dims, keepdim=True)
    rstd = (centred.square().mean(dims, keepdim=True) + GN_EPS).rsqrt()
    xhat = centred * rstd
    u = xhat * gamma + beta
    sig = 1 / (1 + torch.exp(-u)) if case["act"] == "silu" else None
    y = {"none": lambda: u, "relu": lambda: u.clamp_min(0), "silu": lambda: u * sig}[case["act"]]()
    last = lambda a: a.reshape(n, c, h, w).to(x.dtype).contiguous(memory_format=torch.channels_last)  # noqa: E731
    if not case["train"]:
        return {"y": last(y)}
    du = s["dy"].float().reshape(split)
    if case["act"] == "relu":
        du = du * (u > 0)
    elif case["act"] == "silu":
        du = du * (sig * (1 + u * (1 - sig)))
    dgamma, dbeta = (du * xhat).sum((0, 3, 4)).reshape(c), du.sum((0, 3, 4)).reshape(c)
    du = du * gamma
    dx = rstd * (du - du.mean(dims, keepdim=True) - xhat * (du * xhat).mean(dims, keepdim=True))
    return {"y": last(y), "dx": last(dx), "dweight": dgamma, "dbias": dbeta}


def _run_lp(s):
    case = s["case"]
    k = case["top"]
    if not own:
        with torch.no_grad():
            return _log_probs(s)
    from erfnet_pytorch_amd.loss import class_log_probs
    if not case["train"]:
        with torch.no_grad():
            out = class_log_probs(s["logits"], s["target"], top_k=k)
        got = {"log_prob": out.log_prob, "entropy": out.entropy}
        if k:
            got["top"], got["top_index"] = out.top_log_probs, out.top_indices
        return got
    out = class_log_probs(s["logits"], s["target"], top_k=k)
    got = {"log_prob": out.log_prob.detach(), "entropy": out.entropy.detach()}
    heads, grads = [out.log_prob, out.entropy], [s["g_log_prob"], s["g_entropy"]]
    if k:
        got["top"], got["top_index"] = out.top_log_probs.detach(), out.top_indices
        heads.append(out.top_log_probs)
        grads.append(s["g_top"])
    got["dlogits"], = torch.autograd.grad(heads, s["logits"], grads)
    return got


def _log_probs(s):
    case, k = s["case"], s["case"]["top"]
    z = s["logits"].float()
    valid = s["target"] != -100
    t = s["target"].clamp_min(0).unsqueeze(1)
    top = z.amax(1, keepdim=True)
    lse = top + torch.log(torch.exp(z - top).sum(1, keepdim=True))
    logp = z - lse
    del z
    p = torch.exp(logp)
    entropy = -(p * logp).sum(1)
    got = {"log_prob": logp.gather(1, t).squeeze(1) * valid, "entropy": entropy}
    if k:
        # equal values in the order of their index
        index = s["logits"].detach().sort(dim=1, descending=True, stable=True)[1].narrow(1, 0, k).contiguous()
        got["top"], got["top_index"] = logp.gather(1, index), index
    if case["train"]:
        gl, ge = (s["g_log_prob"] * valid).unsqueeze(1), s["g_entropy"].unsqueeze(1)
        total = gl + s["g_top"].sum(1, keepdim=True) if k else gl
        dz = -p * (total + ge * (logp + entropy.unsqueeze(1)))
        dz.scatter_add_(1, t, gl)
        if k:
            dz.scatter_add_(1, index, s["g_top"])
        got["dlogits"] = dz.to(s["logits"].dtype)
    return got


def _run_adamw(s):
    case = s["case"]
    if own:
        s["opt"].step()
    else:
        s["step"] += 1
        new = _adamw(s, s["step"])
        for k, v in new.items():
            s[k].copy_(v)
    return {k: s[k] for k in ("p", "m", "v", "r", "m_scale", "r_scale") if k in s}


def _scale_of(most):
    """The power of two that brings the largest value of a block to 448, the largest e4m3 value, or less."""
    f, e = torch.frexp(most)
    e = torch.where(most > 0, (e - 9 + (f > 0.875).to(e.dtype)).clamp(-126, 120), -126)
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _rounding_bits(count, step):
    """32 random bits per element, from its position and the step alone: the low half for m, the high half for sqrt(v)."""
    word = 0xFFFFFFFF
    h = torch.arange(count, device=DEV, dtype=torch.int64)
    h = (h ^ ((step * 0x9E3779B9) & word)) & word
    h = ((h ^ (h >> 16)) * 0x7FEB352D) & word
    h = ((h ^ (h >> 15)) * 0x846CA68B) & word
    h = h ^ (h >> 16)
    return h & 0xFFFF, h >> 16


def _to_e4m3(t, bits, least=False):
    """|t| <= 448 to an e4m3 value, up or down at random in proportion to the distance; with `least`, nothing but 0 becomes 0."""
    a = t.abs()
    low = a < 2.0 ** -6                                          # the spacing stays 2^-9 below 2^-6
    a = torch.where(low, a + 2.0 ** -6, a)
    a = ((a.view(torch.int32) + (bits << 4).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    a = torch.where(low, a - 2.0 ** -6, a)
    if least:
        a = torch.where(t > 0, a.clamp_min(2.0 ** -9), a)
    return torch.where(t < 0, -a, a).to(torch.float8_e4m3fn)


def _adamw(s, step):
    case = s["case"]
    (b1, b2), eight = BETAS, case["bits"] == 8
    g, p = s["g"].float(), s["p"].float()
    rows = lambda t: t.view(-1, BLOCK)                                                                # noqa: E731
    if eight:
        m = (rows(s["m"].float()) * s["m_scale"][:, None]).view(-1)
        v = (rows(s["r"].float()) * s["r_scale"][:, None]).view(-1).square()
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    r = v.sqrt()
    denom = r * (1 / math.sqrt(1 - b2 ** step)) + EPS
    p = p * (1 - LR * DECAY) - m / denom * (LR / (1 - b1 ** step))
    if not eight:
        return {"p": p, "m": m, "v": v}
    new = {"p": p}
    for name, t, bits in zip(("m", "r"), (m, r), _rounding_bits(p.numel(), step)):
        t = rows(t)
        scale = _scale_of(t.abs().amax(1, keepdim=True))
        new[name] = _to_e4m3(t / scale, rows(bits), least=name == "r").view(-1)
        new[name + "_scale"] = scale.view(-1)
    return new


# ------------------------------------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    with torch.no_grad():
        s = prepare(case, seed)
        d = torch.float64
        if case["op"] == "gn":
            return _exact_gn(s, d)
        if case["op"] == "lp":
            return _exact_lp(s, d)
        return _exact_adamw(s, d)


def _exact_gn(s, d):
    """Through per-channel sums: sum x and sum x^2 of a group about the mean of its first pixel's channels, gradients by the quotient rule."""
    case = s["case"]
    n, c, h, w = s["x"].shape
    g, m = case["groups"], (c // case["groups"]) * h * w
    x = s["x"].permute(0, 2, 3, 1).reshape(n, h * w, c).to(d)
    gamma, beta = s["weight"].to(d), s["bias"].to(d)
    expand = lambda t: t.repeat_interleave(c // g, dim=1).unsqueeze(1)                                # noqa: E731
    by_group = lambda t: t.sum(1).view(n, g, c // g).sum(2)                                           # noqa: E731
    mean = by_group(x) / m
    x = x - expand(mean)
    std = torch.sqrt(by_group(x * x) / m + GN_EPS)
    x = x / expand(std)
    u = x * gamma + beta
    if case["act"] == "relu":
        y, slope = torch.where(u > 0, u, 0.0), (u > 0).to(d)
    elif case["act"] == "silu":
        y = u * torch.sigmoid(u)
        slope = torch.sigmoid(u) + y * (1 - torch.sigmoid(u))
    else:
        y, slope = u, torch.ones_like(u)
    shape = lambda t: t.view(n, h, w, c).permute(0, 3, 1, 2)                                          # noqa: E731
    if not case["train"]:
        return {"y": shape(y)}
    e = s["dy"].permute(0, 2, 3, 1).reshape(n, h * w, c).to(d) * slope
    dw, db = (e * x).sum((0, 1)), e.sum((0, 1))
    e = e * gamma
    dx = (m * e - expand(by_group(e)) - x * expand(by_group(e * x))) / (m * expand(std))
    return {"y": shape(y), "dx": shape(dx), "dweight": dw, "dbias": db}


def _exact_lp(s, d):
    """Through the normalised probabilities; the alternatives' order is decided on the values given."""
    case, k = s["case"], s["case"]["top"]
    z = s["logits"].detach().to(d)
    z -= z.amax(1, keepdim=True)
    e = z.exp()
    total = e.sum(1, keepdim=True)
    p = e / total
    logp = z - total.log()
    live = (s["target"] >= 0).to(d)
    t = torch.where(s["target"] >= 0, s["target"], 0).unsqueeze(1)
    entropy = torch.special.entr(p).sum(1)
    got = {"log_prob": logp.gather(1, t)[:, 0] * live, "entropy": entropy}
    if k:
        index = s["logits"].detach().to(d).sort(dim=1, descending=True, stable=True)[1][:, :k]
        got["top"], got["top_index"] = logp.gather(1, index), index
    if case["train"]:
        gl, ge = s["g_log_prob"].to(d) * live, s["g_entropy"].to(d)
        dz = torch.zeros_like(p).scatter_add_(1, t, gl[:, None])
        pull = gl
        if k:
            gk = s["g_top"].to(d)
            dz.scatter_add_(1, index, gk)
            pull = pull + gk.sum(1)
        dz -= p * pull[:, None]
        dz -= ge[:, None] * (p * logp + p * entropy[:, None])
        got["dlogits"] = dz
    return got


def _exact_adamw(s, d):
    """The update in 64 bits from the values that the states stand for.  New 8-bit codes have no value in 64 bits: which way a
    number near a border goes is decided in 32."""
    case, step = s["case"], s["case"]["step"] + 1
    b1, b2 = BETAS
    g, p = s["g"].to(d), s["p"].to(d)
    if case["bits"] == 8:
        each = lambda t: t.to(d).repeat_interleave(BLOCK)                                             # noqa: E731
        m, v = s["m"].to(d) * each(s["m_scale"]), (s["r"].to(d) * each(s["r_scale"])) ** 2
    else:
        m, v = s["m"].to(d), s["v"].to(d)
    m = m + (1 - b1) * (g - m)
    v = v + (1 - b2) * (g * g - v)
    mhat, vhat = m / (1 - b1 ** step), v / (1 - b2 ** step)
    p = p - LR * (DECAY * p + mhat / (vhat.sqrt() + EPS))
    if case["bits"] == 8:
        return {"p": p, "m": None, "r": None, "m_scale": None, "r_scale": None}
    return {"p": p, "m": m, "v": v}
