"""float64 NumPy definitions of GroupNorm + LeakyReLU (forward, backward, double backward) and of the 8-bit activation
blocks, with the magnitudes that bound a float32 evaluation's rounding."""
from types import SimpleNamespace as NS

import numpy as np

U = 2.0 ** -24  # half a unit in the last place of float32, relative


def case(shape, G, seed=0, affine=True, slope=0.2, eps=1e-5, scale=2.0, shift=0.5, dtype=np.float64):
    """Inputs NCHW; dtype float32 rounds them (and slope, eps) to what the GPU gets."""
    r = np.random.default_rng(seed)
    B, C, H, W = shape
    q = lambda v: np.asarray(v, dtype=dtype).astype(np.float64)  # noqa: E731
    c = NS(G=G, slope=float(q(slope)), eps=float(q(eps)))
    c.x = q(r.standard_normal(shape) * scale * (0.5 + r.random((C, 1, 1))) + shift * r.standard_normal((C, 1, 1)))
    c.w = q(1 + 0.3 * r.standard_normal(C)) if affine else None
    c.b = q(0.3 * r.standard_normal(C)) if affine else None
    c.gy, c.u = q(r.standard_normal(shape)), q(r.standard_normal(shape))
    c.ga, c.gb = q(r.standard_normal(C)), q(r.standard_normal(C))
    return c


def _ch(v, C, one):
    return np.full((C, 1, 1), float(one)) if v is None else v.reshape(-1, 1, 1)


def _grp(t, G):
    """Sum over a (sample, group), broadcast back."""
    s = t.reshape(t.shape[0], G, -1).sum(2)
    return np.repeat(s, t.shape[1] // G, 1)[:, :, None, None]


def forward(c):
    B, C, H, W = c.x.shape
    M = C // c.G * H * W
    f = NS(M=M, gamma=_ch(c.w, C, 1), beta=_ch(c.b, C, 0))
    f.mu = _grp(c.x, c.G) / M
    f.r = 1 / np.sqrt(_grp((c.x - f.mu) ** 2, c.G) / M + c.eps)
    f.pre = lambda v: (v - f.mu) * f.r * f.gamma + f.beta
    f.z = f.pre(c.x)
    f.y = np.where(f.z > 0, f.z, c.slope * f.z)
    f.at = c.x  # where the backward is evaluated (an 8-bit checkpoint's values in its place)
    return f


def backward(c, f):
    d = NS(m=np.where(f.z > 0, 1.0, c.slope), xh=(f.at - f.mu) * f.r)
    d.gz = c.gy * d.m
    d.h = f.gamma * d.gz
    d.m1, d.m2 = _grp(d.h, c.G) / f.M, _grp(d.h * d.xh, c.G) / f.M
    d.gx = f.r * (d.h - d.m1 - d.xh * d.m2)
    d.gw, d.gb = (d.gz * d.xh).sum((0, 2, 3)), d.gz.sum((0, 2, 3))
    # float32 evaluation with float64 sums.  gz and h round once each, the two means once after gz's rounding in every
    # term, x̂ and its product once each, the two differences and r's conversion and product once each
    mean = lambda t: _grp(np.abs(t), c.G) / f.M  # noqa: E731
    T = f.r * (np.abs(d.h) + mean(d.h) + np.abs(d.xh) * mean(d.h * d.xh) + np.abs(d.m1) + np.abs(d.xh * d.m2))
    d.tol_gx = 8 * U * T
    d.tol_gw = 2 * U * np.abs(d.gz * d.xh).sum((0, 2, 3))
    d.tol_gb = 2 * U * np.abs(d.gz).sum((0, 2, 3))
    return d


def backward2(c, f, d, u=True, ga=True, gb=True):
    """u, ga, gb: whether gx, dγ, dβ have an upstream gradient."""
    C = c.x.shape[1]
    u = c.u if u else np.zeros_like(c.u)
    ga = c.ga.reshape(-1, 1, 1) if ga else np.zeros((C, 1, 1))
    gb = c.gb.reshape(-1, 1, 1) if gb else np.zeros((C, 1, 1))
    mean = lambda t: _grp(t, c.G) / f.M  # noqa: E731
    mU, mA, mQ = mean(u), mean(u * d.xh), mean(u * d.h)
    inner = f.r * (u - mU - d.xh * mA)
    e = NS(g_gy=d.m * (f.gamma * inner + ga * d.xh + gb))
    e.g_w = (d.gz * inner).sum((0, 2, 3))
    big = -f.r * (d.h * mA + u * d.m2) + ga * d.gz
    g_r = (mQ - d.m1 * mU - d.m2 * mA) * f.r ** 2
    e.g_x = f.r * (big - mean(big) - d.xh * mean(big * d.xh)) - g_r * d.xh
    # roundings as in backward; the means with what their terms' roundings leave
    a = np.abs
    ab = lambda t: mean(a(t))  # noqa: E731
    e.tol_gy = 10 * U * d.m * (a(f.gamma) * f.r * (a(u) + a(mU) + a(d.xh * mA)) + a(ga * d.xh) + a(gb))
    e.tol_w = 4 * U * (f.r * a(d.gz) * (a(u) + a(mU) + a(d.xh * mA))).sum((0, 2, 3))
    bigT = f.r * (a(d.h * mA) + a(u) * ab(d.h * d.xh)) + a(ga * d.gz)
    mG = f.r * (ab(d.h) * a(mA) + a(mU) * ab(d.h * d.xh)) + ab(ga * d.gz)
    mGx = 2 * f.r * ab(d.h * d.xh) * a(mA) + ab(ga * d.gz * d.xh)
    gr = (ab(u * d.h) + ab(d.h) * a(mU) + ab(d.h * d.xh) * a(mA)) * f.r ** 2
    e.tol_x = 12 * U * (f.r * (bigT + mG + a(d.xh) * mGx) + gr * a(d.xh))
    return e


def pack(x, pre=None):
    """(codes, exps, values) of float32 [P, C]; pre: values -> pre-activations whose sign a code keeps (default: x)."""
    x = np.asarray(x, dtype=np.float32).astype(np.float64)
    P, C = x.shape
    nb = -(-C // 32)
    xb = np.pad(x, ((0, 0), (0, nb * 32 - C))).reshape(P, nb, 32)
    ok = np.isfinite(xb).all(2)
    top = np.where(ok, np.abs(np.where(np.isfinite(xb), xb, 0)).max(2), 0)
    m, e = np.frexp(top)  # top = m 2^e, m in [1/2, 1)
    k = np.where(top > 0, np.where(m > 127 / 128, e - 6, e - 7), -132)
    k = np.maximum(k, -132)
    exps = np.where(ok, k + 132, 255).astype(np.uint8)
    wide = lambda t: np.repeat(t, 32, 1)[:, :C]  # noqa: E731
    step, fine = wide(np.ldexp(1.0, k)), wide(ok)
    xs = np.where(fine, x, 0)
    most = np.where(wide(k) == 122, 63, 127)  # 64 · 2^122 is past the largest float
    code = np.clip(np.rint(xs / step), -most, most)
    pre = pre or (lambda v: v)
    wrong = fine & ((pre(code * step) > 0) != (pre(xs) > 0))
    code = code + np.where(wrong, np.where(code * step > xs, -1.0, 1.0), 0.0)
    return code.astype(np.int8), exps, np.where(fine, code * step, np.nan)


def rows(t):
    """NCHW -> [N·H·W, C]."""
    return t.transpose(0, 2, 3, 1).reshape(-1, t.shape[1])


def back(t, shape):
    B, C, H, W = shape
    return t.reshape(B, H, W, C).transpose(0, 3, 1, 2)


def wgrad(x, gy, k, s, p):
    """(gw [Co, Ci, k, k], Σ|x·gy|) in float64 of NHWC x and gy."""
    B, H, W, Ci = x.shape
    _, Ho, Wo, Co = gy.shape
    big = np.pad(x.astype(np.float64), ((0, 0), (p, p + s), (p, p + s), (0, 0)))
    g = gy.astype(np.float64).reshape(-1, Co)
    gw, mag = np.zeros((Co, Ci, k, k)), np.zeros((Co, Ci, k, k))
    for a in range(k):
        for b in range(k):
            t = big[:, a:a + (Ho - 1) * s + 1:s, b:b + (Wo - 1) * s + 1:s].reshape(-1, Ci)
            gw[:, :, a, b] = g.T @ t
            mag[:, :, a, b] = np.abs(g).T @ np.abs(t)
    return gw, mag
