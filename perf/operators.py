"""Cases that measure the discriminator's group-norm and 8-bit activation-checkpoint operators.

Where `own` is false every operator runs in its plain form (elementary torch operations); where it is true, through the
calls a user of esr_amd makes.  Four operators:

  norm     group norm + LeakyReLU of channels-last activations, a training step's forward and backward
  penalty  the same layer under the gradient penalty: forward, backward, and the backward's own backward
  pack     an activation kept in 8 bits (a power-of-two step per 32 channels of a pixel) and read back
  weights  a convolution's weight gradient from an input kept in 8 bits

The values next to LeakyReLU's kink decide between a slope of 1 and one of 0.2, so the statistics and the pre-activation
are held in 64 bits by the plain form; the elementwise rest is in 32 bits, long sums in 64.
"""
import math
import os
import sys

import torch

own = False

EPS, SLOPE = 1e-5, 0.2
# the most that one case costs: elements of a norm / penalty / pack case, and of the weights case's tap matrix
NORM_MAX, PACK_MAX, TAPS_MAX = 16 * 152 * 152 * 128, 16 * 304 * 304 * 64, 16 * 152 * 152 * 16 * 64


def listed():
    return [
        # first norm layer of a small patch (80 x 72 crops, three of them): the latency of one call
        {"name": "norm_small", "op": "norm", "n": 3, "c": 64, "h": 40, "w": 36, "groups": 32, "affine": True, "bits8": False},
        # the classifier's 8x8 layer: 100 channels in 4 groups of 25, an odd 31 x 31 map
        {"name": "norm_head", "op": "norm", "n": 16, "c": 100, "h": 31, "w": 31, "groups": 4, "affine": True, "bits8": False},
        # the widest map of the training step, 128 channels
        {"name": "norm_wide", "op": "norm", "n": 16, "c": 128, "h": 152, "w": 152, "groups": 32, "affine": True, "bits8": False},
        # instance norm (a group per channel, no affine) in the middle of the network
        {"name": "norm_instance", "op": "norm", "n": 16, "c": 256, "h": 76, "w": 76, "groups": 256, "affine": False, "bits8": False},
        # the first norm layer of the training step with its input kept in 8 bits
        {"name": "norm_8bit", "op": "norm", "n": 16, "c": 64, "h": 152, "w": 152, "groups": 32, "affine": True, "bits8": True},
        # gradient penalty through a middle layer
        {"name": "penalty", "op": "penalty", "n": 16, "c": 128, "h": 76, "w": 76, "groups": 32, "affine": True, "bits8": False},
        # the same on a small patch, with the 8-bit input
        {"name": "penalty_small_8bit", "op": "penalty", "n": 3, "c": 128, "h": 20, "w": 18, "groups": 32, "affine": True, "bits8": True},
        # checkpoint of an odd channel count on a small map
        {"name": "pack_small", "op": "pack", "n": 3, "c": 100, "h": 31, "w": 31},
        # checkpoint of the first convolution's output, the largest activation of the training step
        {"name": "pack_large", "op": "pack", "n": 16, "c": 64, "h": 304, "w": 304},
        # weight gradient of a 3x3 layer on a small patch
        {"name": "weights_small", "op": "weights", "n": 3, "ci": 64, "co": 128, "h": 40, "w": 36, "k": 3, "s": 1, "p": 1},
        # the training step's strided 4x4 layer, 304 -> 152
        {"name": "weights_4x4", "op": "weights", "n": 16, "ci": 64, "co": 64, "h": 304, "w": 304, "k": 4, "s": 2, "p": 1},
        # the training step's widest 3x3 layer
        {"name": "weights_3x3", "op": "weights", "n": 16, "ci": 64, "co": 128, "h": 152, "w": 152, "k": 3, "s": 1, "p": 1},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _channels(rng):
    return rng.choice([64, 100, 128, 256, 512, _log(rng, 1, 512), _log(rng, 1, 512)])


def draw(rng):
    op = rng.choice(["norm", "norm", "penalty", "pack", "weights", "weights"])
    n = _log(rng, 1, 32)
    if op == "weights":
        k, s, p = rng.choice([(3, 1, 1), (4, 2, 1), (4, 1, 1), (8, 1, 0), (1, 1, 0)])
        ci, co = _channels(rng), _channels(rng)
        outs = max(1, TAPS_MAX // (n * k * k * max(ci, co, 64)))  # output pixels of one image
        area = _log(rng, 1, min(outs, 152 * 152))
        ho = max(1, min(area, _log(rng, 1, 152)))
        wo = max(1, area // ho)
        return {"op": op, "n": n, "ci": ci, "co": co, "h": (ho - 1) * s + k - 2 * p + (0 if ho == 1 else rng.randrange(s)),
                "w": (wo - 1) * s + k - 2 * p, "k": k, "s": s, "p": p}
    most = PACK_MAX if op == "pack" else NORM_MAX if op == "norm" else NORM_MAX // 4
    c = _channels(rng)
    side = 304 if op == "pack" else 152
    groups = rng.choice([math.gcd(c, 32), math.gcd(c, 32), c, 1])
    # a group of few values leaves nothing of its gradient but rounding
    least = 1 if op == "pack" else -(-64 * groups // c)
    area = _log(rng, least, max(least, min(side * side, most // (n * c)) - side))
    h = max(1, min(area, _log(rng, 1, side)))
    case = {"op": op, "n": n, "c": c, "h": h, "w": -(-area // h)}
    if op != "pack":
        case.update(groups=groups, affine=rng.random() < 0.8, bits8=rng.random() < 0.4)
    return case


def _out_hw(c):
    return (c["h"] + 2 * c["p"] - c["k"]) // c["s"] + 1, (c["w"] + 2 * c["p"] - c["k"]) // c["s"] + 1


def work(case):
    if case["op"] == "weights":
        ho, wo = _out_hw(case)
        px = case["n"] * ho * wo
        return {"bytes": 4 * (case["n"] * case["h"] * case["w"] * case["ci"] + px * case["co"]
                              + case["k"] ** 2 * case["ci"] * case["co"]),
                "flops": 2 * px * case["k"] ** 2 * case["ci"] * case["co"]}
    e = case["n"] * case["c"] * case["h"] * case["w"]
    # tensors in and out: norm x, gy -> y, gx; penalty x, gy, u -> y, gx, g_x, g_gy; pack x -> x
    return {"bytes": 4 * e * {"norm": 4, "penalty": 7, "pack": 2}[case["op"]],
            "flops": e * {"norm": 20, "penalty": 45, "pack": 4}[case["op"]]}


def _nhwc(g, n, h, w, c, scale=1.0, shift=0.0):
    """What a convolution leaves: channels-last, each channel with a scale and an offset of its own."""
    t = torch.randn(n, h, w, c, generator=g, device="cuda")
    t *= scale * (0.5 + torch.rand(c, generator=g, device="cuda"))
    return t.add_(shift * torch.randn(c, generator=g, device="cuda"))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if case["op"] == "weights":
        ho, wo = _out_hw(case)
        x = torch.nn.functional.leaky_relu(_nhwc(g, case["n"], case["h"], case["w"], case["ci"], 1.0, 0.3), SLOPE)
        return {"case": dict(case), "x": x, "gy": _nhwc(g, case["n"], ho, wo, case["co"], 1e-3)}
    n, c, h, w = case["n"], case["c"], case["h"], case["w"]
    x = _nhwc(g, n, h, w, c, 2.0, 0.5)
    if case["op"] == "pack":
        return {"case": dict(case), "x": x}
    s = {"case": dict(case), "x": x.permute(0, 3, 1, 2).requires_grad_(), "weight": None, "bias": None}
    if case["affine"]:
        s["weight"] = (1 + 0.2 * torch.randn(c, generator=g, device="cuda")).requires_grad_()
        s["bias"] = (0.2 * torch.randn(c, generator=g, device="cuda")).requires_grad_()
    s["gy"] = _nhwc(g, n, h, w, c, 1e-3).permute(0, 3, 1, 2)
    if case["op"] == "penalty":
        s["gy"].requires_grad_()
        s["u"] = _nhwc(g, n, h, w, c).permute(0, 3, 1, 2)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _blocks(x):
    """[..., C] -> [..., ceil(C/32), 32], zeros behind the last channel."""
    c = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, -c % 32))
    return x.view(*x.shape[:-1], x.shape[-1] // 32, 32)


def _eight_bits(x, pre=None):
    """The values that x [..., C] stands for in 8 bits: code * step, step the smallest power of two with 127 * step >=
    the block's largest magnitude; a code that rounding took over the threshold of `pre` (pre-activation > 0) goes one
    step back.  pre: values [..., C] -> pre-activations in 64 bits; None: the values themselves."""
    c, pre = x.shape[-1], pre or (lambda v: v)
    xb = _blocks(x)
    m, e = torch.frexp(xb.abs().amax(-1, keepdim=True))
    step = ((torch.where(m > 127 / 128, e - 6, e - 7).clamp(min=-126) + 127) << 23).view(torch.float32)  # 2^k, exactly
    flat = lambda t: t.flatten(-2)[..., :c]  # noqa: E731
    step = flat(step.expand(xb.shape))
    code = torch.round(x / step)
    v = code * step
    want = pre(x) > 0
    return torch.where((pre(v) > 0) != want, (code + torch.where(v > x, -1.0, 1.0)) * step, v)


def _plain_norm(s):
    """Forward and backward on rows [N, HW, G, Cg]; returns what the penalty's second pass needs as well."""
    c, n = s["case"], s["case"]["n"]
    shape = (n, c["h"] * c["w"], c["groups"], c["c"] // c["groups"])
    rows = lambda t: t.permute(0, 2, 3, 1).reshape(shape)  # noqa: E731
    x, gy = rows(s["x"]), rows(s["gy"])
    one = x.new_ones(c["c"])
    gamma = (one if s["weight"] is None else s["weight"]).view(shape[2:])
    beta = (0 * one if s["bias"] is None else s["bias"]).view(shape[2:])
    var, mu = torch.var_mean(x.double(), dim=(1, 3), keepdim=True, correction=0)
    r = torch.rsqrt(var + EPS)
    pre = lambda v: (v.double() - mu) * r * gamma.double() + beta.double()  # noqa: E731
    z = pre(x)
    y = torch.where(z > 0, z, SLOPE * z).float()
    if c["bits8"]:
        as_rows = lambda v: v.reshape(n, shape[1], c["c"])  # noqa: E731
        x = _eight_bits(as_rows(x), lambda v: as_rows(pre(v.view(shape)))).view(shape)
    xh = ((x.double() - mu) * r).float()
    slope = torch.where(z > 0, 1.0, SLOPE).float()
    gz = gy * slope
    s1, s2 = gz.sum(1, dtype=torch.float64), (gz * xh).sum(1, dtype=torch.float64)  # [N, G, Cg]
    m = shape[1] * shape[3]
    big1 = (s1 * gamma).sum(-1)[:, None, :, None] / m
    big2 = (s2 * gamma).sum(-1)[:, None, :, None] / m
    gx = r.float() * (gz * gamma - big1.float() - xh * big2.float())
    return {"rows": rows, "shape": shape, "y": y, "gx": gx, "xh": xh, "slope": slope, "gz": gz, "gamma": gamma, "r": r,
            "s1": s1, "s2": s2, "big1": big1, "big2": big2, "m": m}


def _back(t, case):
    return t.reshape(case["n"], case["h"], case["w"], case["c"]).permute(0, 3, 1, 2)


def _plain_penalty(s):
    c, f = s["case"], _plain_norm(s)
    u = f["rows"](s["u"])
    xh, gz, gamma, m, r, slope = f["xh"], f["gz"], f["gamma"], f["m"], f["r"], f["slope"]
    su, sa, sq = (t.sum(1, dtype=torch.float64) for t in (u, u * xh, u * gz))
    mean = lambda t: t.sum(-1)[:, None, :, None] / m  # noqa: E731
    mu_u, mu_a, mu_q = mean(su), mean(sa), mean(sq * gamma)
    r32 = r.float()
    inner = r32 * (u - mu_u.float() - xh * mu_a.float())
    g_gy = slope * gamma * inner
    g_gamma = (r[:, 0] * (sq - f["s1"] * mu_u[:, 0] - f["s2"] * mu_a[:, 0])).sum(0).reshape(-1).float()
    big = -r32 * (gz * gamma * mu_a.float() + u * f["big2"].float())
    mean_big, mean_bigx = -r * (f["big1"] * mu_a + mu_u * f["big2"]), -2 * r * f["big2"] * mu_a
    g_r = r ** 2 * (mu_q - f["big1"] * mu_u - f["big2"] * mu_a)
    g_x = r32 * (big - mean_big.float() - xh * mean_bigx.float()) - g_r.float() * xh
    out = {"y": _back(f["y"], c), "gx": _back(f["gx"], c), "g_x": _back(g_x, c), "g_gy": _back(g_gy, c)}
    return {**out, "g_weight": g_gamma} if c["affine"] else out


def _plain_weights(s):
    c = s["case"]
    x = torch.nn.functional.pad(_eight_bits(s["x"]), (0, 0) + (c["p"],) * 4)
    taps = x.unfold(1, c["k"], c["s"]).unfold(2, c["k"], c["s"])  # [N, Ho, Wo, Ci, k, k]
    gw = s["gy"].reshape(-1, c["co"]).t() @ taps.reshape(-1, c["ci"] * c["k"] ** 2)
    return gw.view(c["co"], c["ci"], c["k"], c["k"])


def _plain(s):
    if s["case"]["op"] == "pack":
        return _eight_bits(s["x"])
    if s["case"]["op"] == "weights":
        return _plain_weights(s)
    if s["case"]["op"] == "penalty":
        return _plain_penalty(s)
    f, c = _plain_norm(s), s["case"]
    out = {"y": _back(f["y"], c), "gx": _back(f["gx"], c)}
    if c["affine"]:
        out.update(g_weight=f["s2"].sum(0).reshape(-1).float(), g_bias=f["s1"].sum(0).reshape(-1).float())
    return out


# ---- the framework's calls --------------------------------------------------------------------------------------------
def _own(s):
    package = os.path.join(os.getcwd(), "explorable-super-resolution_old_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from esr_amd import act8, dconv, gn
    c = s["case"]
    if c["op"] == "pack":
        return act8.pack(s["x"]).unpack()
    if c["op"] == "weights":
        return dconv.conv_wgrad_act8(act8.pack(s["x"]), s["gy"], c["k"], c["s"], c["p"])
    y = gn.group_norm_lrelu(s["x"], c["groups"], s["weight"], s["bias"], EPS, SLOPE, "int8" if c["bits8"] else None)
    if c["op"] == "penalty":
        gx, = torch.autograd.grad(y, s["x"], s["gy"], create_graph=True)
        wrt = [s["x"], s["gy"]] + ([s["weight"]] if c["affine"] else [])
        names = ["g_x", "g_gy", "g_weight"]
        return {"y": y.detach(), "gx": gx.detach(), **dict(zip(names, torch.autograd.grad(gx, wrt, s["u"])))}
    wrt = [s["x"]] + ([s["weight"], s["bias"]] if c["affine"] else [])
    return {"y": y.detach(), **dict(zip(["gx", "g_weight", "g_bias"], torch.autograd.grad(y, wrt, s["gy"])))}


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _exact_bits(x, side):
    """x, side: 64-bit [P, C]; side(v) tells on which side of the kink v lies."""
    p, c = x.shape
    pad = torch.zeros(p, -c % 32, dtype=x.dtype, device=x.device)
    top = torch.cat([x, pad], 1).reshape(p, -1, 32).abs().max(2).values.clamp(min=2.0 ** -119)
    two = lambda k: ((k + 1023) << 52).view(torch.float64)  # noqa: E731  (2^k by its bits: pow is not exact)
    k = torch.ceil(torch.log2(top / 127)).long()
    k = torch.where(127 * two(k - 1) >= top, k - 1, k)
    k = torch.where(127 * two(k) < top, k + 1, k)
    step = two(k).repeat_interleave(32, 1)[:, :c]
    near = torch.round(x / step) * step
    other = near + torch.sign(x - near) * step
    return torch.where(side(near) == side(x), near, other)


def exact(case, seed):
    s = prepare(case, seed)
    s = {k: v.detach() if torch.is_tensor(v) else v for k, v in s.items()}
    if case["op"] == "pack":
        x = s["x"].double().reshape(-1, case["c"])
        return _exact_bits(x, lambda v: v > 0).reshape(s["x"].shape)
    if case["op"] == "weights":
        x = _exact_bits(s["x"].double().reshape(-1, case["ci"]), lambda v: v > 0).reshape(s["x"].shape)
        ho, wo = _out_hw(case)
        k, st, p = case["k"], case["s"], case["p"]
        big = torch.zeros(case["n"], case["h"] + 2 * p, case["w"] + 2 * p, case["ci"], dtype=x.dtype, device=x.device)
        big[:, p:p + case["h"], p:p + case["w"]] = x
        gy = s["gy"].double().reshape(-1, case["co"])
        gw = torch.zeros(case["co"], case["ci"], k, k, dtype=x.dtype, device=x.device)
        for a in range(k):
            for b in range(k):
                at = big[:, a:a + (ho - 1) * st + 1:st, b:b + (wo - 1) * st + 1:st].reshape(-1, case["ci"])
                gw[:, :, a, b] = gy.t() @ at
        return gw
    # group norm as nested functions of the input, differentiated twice by autograd
    n, c, g = case["n"], case["c"], case["groups"]
    x = s["x"].double()
    w = (torch.ones(c, dtype=x.dtype, device=x.device) if s["weight"] is None else s["weight"].double()).requires_grad_()
    b = (torch.zeros(c, dtype=x.dtype, device=x.device) if s["bias"] is None else s["bias"].double()).requires_grad_()
    gy = s["gy"].double().requires_grad_()
    per = lambda t: t.reshape(n, g, -1)  # noqa: E731
    mu = per(x).mean(2)
    sd = torch.sqrt(((per(x) - mu[..., None]) ** 2).mean(2) + EPS)
    wide = lambda t: t.repeat_interleave(c // g, 1)[:, :, None, None]  # noqa: E731
    aff = lambda v: (v - wide(mu)) / wide(sd) * w[:, None, None] + b[:, None, None]  # noqa: E731
    z = aff(x).detach()
    out = {"y": torch.where(z > 0, z, SLOPE * z)}
    at = x
    if case["bits8"]:
        shape = (n, case["h"], case["w"], c)
        side = lambda v: aff(v.reshape(shape).permute(0, 3, 1, 2)).detach().permute(0, 2, 3, 1).reshape(-1, c) > 0  # noqa: E731
        at = _exact_bits(x.permute(0, 2, 3, 1).reshape(-1, c), side).reshape(shape).permute(0, 3, 1, 2)
    # the backward at `at`, with the statistics of x as functions that have the derivatives of a mean and a deviation
    at = at.detach().requires_grad_()
    count = per(x).shape[2]
    xh0 = per((at.detach() - wide(mu)) / wide(sd))
    d = per(at) - per(at.detach())
    mu_at = mu + d.mean(2)
    sd_at = sd + (d * xh0).mean(2)  # first order suffices: the backward holds x only through xh and 1/sd
    r_at = 1 / sd_at
    xh = (per(at) - mu_at[..., None]) * r_at[..., None]
    slope = torch.where(z > 0, 1.0, SLOPE).double()
    gz = gy * slope
    h = per(gz * w[:, None, None])
    gx = r_at[..., None] * (h - h.sum(2, keepdim=True) / count - xh * (h * xh).sum(2, keepdim=True) / count)
    gx = gx.reshape(x.shape)
    out["gx"] = gx.detach()
    if case["op"] == "norm":
        if case["affine"]:
            out["g_weight"] = (gz * xh.reshape(x.shape)).sum((0, 2, 3)).detach()
            out["g_bias"] = gz.sum((0, 2, 3)).detach()
        return out
    g_x, g_gy, g_w = torch.autograd.grad(gx, [at, gy, w], s["u"].double())
    out.update(g_x=g_x, g_gy=g_gy)
    return {**out, "g_weight": g_w} if case["affine"] else out
