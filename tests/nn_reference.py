"""Plain 64-bit forms of the operators in cudacaml_b200.nn, with, beside each
result, the sum of the magnitudes of its terms, from which the tests derive
their tolerances."""
import numpy as np
import torch

U = 2.0**-24  # unit roundoff of F32
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-140, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-24}


def words(first, n, seed, offset):
    """Philox-4x32-10 words of elements first .. first + n - 1 (numpy)."""
    lo, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    q = np.arange(first >> 2, ((first + n - 1) >> 2) + 1, dtype=np.uint64)
    c = [q & lo, q >> half, np.full_like(q, offset & 0xFFFFFFFF), np.full_like(q, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & lo, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & lo]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[first & 3:][:n]


def keep(first, shape, p, seed, offset, device):
    n = int(np.prod(shape))
    if n == 0:
        return torch.zeros(shape, dtype=torch.bool, device=device)
    k = words(first, n, seed, offset) >= np.uint64(round(p * 2.0**32))
    return torch.from_numpy(k.reshape(shape)).to(device)


def close(got, want, slack, name=""):
    """|got - want| <= unit(got) * |want| + slack, element by element."""
    w = want.double()
    g = got.double()
    assert g.shape == w.shape, (name, g.shape, w.shape)
    bound = UNIT[got.dtype] * w.abs() + slack + TINY[got.dtype]
    off = (g - w).abs() - bound
    bad = ~(off <= 0)
    assert not bool(bad.any()), (name, int(bad.sum()), float(off[bad].max()), bad.nonzero()[:3].tolist())


ACT = {
    "none": (lambda g: g, lambda g: torch.ones_like(g)),
    "sigmoid": (torch.sigmoid, lambda g: torch.sigmoid(g) * (1 - torch.sigmoid(g))),
    "tanh": (torch.tanh, lambda g: 1 - torch.tanh(g) ** 2),
}


def norm(v, kind, eps):
    """(v normalised, 1/deviation, magnitude of its terms)."""
    m = v.mean(1, keepdim=True) if kind == "layer" else torch.zeros_like(v[:, :1])
    r = 1.0 / torch.sqrt(((v - m) ** 2).mean(1, keepdim=True) + eps)
    return (v - m) * r, r, (v.abs() + (v.abs().mean(1, keepdim=True) if kind == "layer" else 0.0)) * r


def norm_grad(g, hat, r, mag, gmag, kind):
    """(gradient through the norm, magnitude of its terms)."""
    d = g - hat * (g * hat).mean(1, keepdim=True)
    m = gmag + mag * (gmag * mag).mean(1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(1, keepdim=True)
        m = m + gmag.mean(1, keepdim=True)
    return d * r, m * r


def block(x, branch, *, kind="rms", eps=1e-6, post_norm=True, w1=None, c1=None, w2=None, c2=None, gate=None, act="none", scale=1.0, mask=1.0):
    """(y, |y|, h, |h|) in 64 bits; mask: keep / (1 - p), or 1."""
    x = x.double()
    y, ymag = x, x.abs()
    if branch is not None:
        b = branch.double()
        u, _, m = norm(b, kind, eps) if post_norm else (b, None, b.abs())
        if w2 is not None:
            u, m = u * w2.double(), m * w2.double().abs()
        if c2 is not None:
            u, m = u + c2.double(), m + c2.double().abs()
        if gate is not None:
            a = ACT[act][0](gate.double())
            u, m = u * a, m * a.abs()
        y, ymag = x + scale * mask * u, x.abs() + abs(scale) * mask * m
    h, r, _ = norm(y, kind, eps)
    hmag = (ymag + (ymag.mean(1, keepdim=True) if kind == "layer" else 0.0)) * r + h.abs()
    if kind == "layer" or branch is not None:  # errors of the row's statistics come in through hat as well
        hmag = hmag + h.abs() * (ymag * y.abs()).mean(1, keepdim=True) * r * r
    if w1 is not None:
        h, hmag = h * w1.double(), hmag * w1.double().abs()
    if c1 is not None:
        h, hmag = h + c1.double(), hmag + c1.double().abs()
    return y, ymag, h, hmag


def block_grad(y, branch, dy, dh, *, kind="rms", eps=1e-6, post_norm=True, w1=None, w2=None, c2=None, gate=None, act="none", scale=1.0, mask=1.0):
    """{name: (gradient, magnitude)} in 64 bits."""
    y = y.double()
    out = {}
    d = torch.zeros_like(y) if dy is None else dy.double()
    dm = d.abs()
    if dh is not None:
        g = dh.double() if w1 is None else dh.double() * w1.double()
        hat, r, mag = norm(y, kind, eps)
        b, m = norm_grad(g, hat, r, mag, g.abs(), kind)
        d, dm = d + b, dm + m
        out["dpre_weight"] = ((dh.double() * hat).sum(0), (dh.double().abs() * mag).sum(0))
        out["dpre_bias"] = (dh.double().sum(0), dh.double().abs().sum(0))
    out["dx"] = (d, dm)
    if branch is None:
        return out
    b = branch.double()
    hat, r, mag = norm(b, kind, eps) if post_norm else (b, torch.ones_like(b[:, :1]), b.abs())
    one = torch.ones_like(b)
    a, slope = (one, None) if gate is None else (ACT[act][0](gate.double()), ACT[act][1](gate.double()))
    u, um = hat, mag
    if w2 is not None:
        u, um = u * w2.double(), um * w2.double().abs()
    if c2 is not None:
        u, um = u + c2.double(), um + c2.double().abs()
    dz, dzm = scale * mask * d, abs(scale) * mask * dm
    du, dum = dz * a, dzm * a.abs()
    if gate is not None:
        # 1 - a^2 and a (1 - a) lose bits where they are small: their error is of a's size
        dg, dgm = dz * u * slope, dzm * um * (slope.abs() + a.abs() + a * a)
        out["dgate"] = (dg, dgm) if gate.dim() == 2 else (dg.sum(0), dgm.sum(0))
    out["dpost_weight"] = ((du * hat).sum(0), (dum * mag).sum(0))
    out["dpost_bias"] = (du.sum(0), dum.sum(0))
    if post_norm:
        g, gm = (du, dum) if w2 is None else (du * w2.double(), dum * w2.double().abs())
        out["dbranch"] = norm_grad(g, hat, r, mag, gm, kind)
    else:
        out["dbranch"] = (du, dum)
    return out


def grouped(x, w, offsets, transpose_w=False):
    """(product, magnitude) in 64 bits, experts' rows by a list of offsets."""
    w = w.transpose(1, 2) if transpose_w else w
    out = torch.zeros((x.shape[0], w.shape[2]), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    for e, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        out[a:b] = x[a:b].double() @ w[e].double()
        mag[a:b] = x[a:b].double().abs() @ w[e].double().abs()
    return out, mag


def grouped_dw(x, dy, offsets):
    out = torch.zeros((len(offsets) - 1, x.shape[1], dy.shape[1]), dtype=torch.float64, device=x.device)
    mag = torch.zeros_like(out)
    for e, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
        out[e] = x[a:b].double().T @ dy[a:b].double()
        mag[e] = x[a:b].double().abs().T @ dy[a:b].double().abs()
    return out, mag
