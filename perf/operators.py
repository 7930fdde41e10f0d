"""Cases of the operators of a residual block with experts: dropout from a
counter-based generator, the norms around a block fused with its gate and
residual scale, and products grouped by expert, each in its directions.

``run`` computes them in plain torch operations in 32 bits, or, where ``own``
is true, by the calls a user makes of ``cudacaml_b200.nn``. ``exact`` gives
the same outputs from the definitions in 64 bits.
"""
import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_DEV = "cuda"
_nn = None


def _own():
    global _nn
    if _nn is None:
        from cudacaml_b200 import nn

        _nn = nn
    return _nn


# ----------------------------------------------------------------- the cases
def _dropout(**k):
    # xtype has no meaning for dropout; dir "bwd" is the same mask on a gradient
    return {"op": "dropout", "dir": "fwd", "type": "bf16", "p": 0.1, "residual": False, "base": 0, **k}


def _norm(**k):
    # act: the gate's function, "off" without a gate; gate: "full" (rows x cols) or "channel" (cols);
    # xtype: the residual stream's type
    return {"op": "norm", "dir": "fwd", "kind": "rms", "type": "bf16", "xtype": "bf16", "act": "sigmoid", "gate": "full", "p": 0.1, "bias": False, **k}


def _grouped(**k):
    # active: experts that get rows; spare: rows at the end that belong to none
    return {"op": "grouped", "dir": "fwd", "type": "bf16", "spare": 0, **k}


def listed():
    return [
        # the first tokens of a short prompt: a launch and little else
        _dropout(name="dropout_few_rows", rows=16, cols=1024),
        # residual dropout over the tokens of one training step
        _dropout(name="dropout_residual", rows=16384, cols=4096, residual=True),
        # its gradient in 32 bits, ragged, on a slice of rows that starts inside the whole
        _dropout(name="dropout_grad_odd", rows=4099, cols=1021, type="f32", dir="bwd", p=0.3, base=1021 * 77),
        # one token through the join of two blocks while serving
        _norm(name="norm_one_token", rows=1, cols=4096, act="off", p=0.0),
        # a training step's tokens
        _norm(name="norm_train", rows=8192, cols=4096),
        _norm(name="norm_train_grad", rows=8192, cols=4096, dir="bwd"),
        # layer norms with biases, a gate for each channel, odd sizes, 32 bits
        _norm(name="norm_layer_grad_odd", rows=1531, cols=1001, dir="bwd", kind="layer", type="f32", xtype="f32", act="tanh", gate="channel", p=0.25, bias=True),
        # a decoding step: 16 sequences, two experts each, of 64
        _grouped(name="grouped_decode", rows=32, experts=64, active=26, k=4096, n=1024),
        # a training step's products: up, and both gradients of a smaller one with rows that were dropped
        _grouped(name="grouped_train", rows=16384, experts=16, active=16, k=4096, n=4096),
        _grouped(name="grouped_train_grad", rows=8192, experts=32, active=30, k=4096, n=1024, dir="bwd", spare=100),
        # 32 bits, and 32 bits in odd sizes
        _grouped(name="grouped_f32", rows=4096, experts=8, active=8, k=1024, n=4096, type="f32"),
        _grouped(name="grouped_grad_odd", rows=1003, experts=7, active=6, k=515, n=129, type="f32", dir="bwd", spare=3),
    ]


def _log(rng, low, high, odd):
    v = int(round(low * (high / low) ** rng.random()))
    v = max(low, min(high, v))
    return v if odd else max(8, v // 8 * 8)


def draw(rng):
    op = rng.choice(["dropout", "norm", "norm", "grouped", "grouped", "grouped"])
    odd = rng.random() < 0.35
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    way = rng.choice(["fwd", "bwd"])
    if op == "dropout":
        cols = _log(rng, 8, 8192, odd)
        rows = min(_log(rng, 1, 16384, True), (16384 * 4096) // (cols * (2 if dtype == "f32" else 1)))
        return _dropout(rows=rows, cols=cols, type=dtype, dir=way, p=rng.choice([0.05, 0.1, 0.2, 0.5]),
                        residual=way == "fwd" and rng.random() < 0.5, base=rng.randrange(1 << 34) if odd else 4 * rng.randrange(1 << 32))
    if op == "norm":
        cols = _log(rng, 32, 8192, odd)
        xtype = dtype if rng.random() < 0.6 else "f32"
        rows = min(_log(rng, 1, 8192, True), (8192 * 4096) // (cols * (2 if xtype == "f32" else 1)))
        return _norm(rows=rows, cols=cols, type=dtype, xtype=xtype, dir=way, kind=rng.choice(["rms", "rms", "layer"]),
                     act=rng.choice(["off", "none", "sigmoid", "tanh"]), gate=rng.choice(["full", "channel"]),
                     p=rng.choice([0.0, 0.1, 0.3]), bias=rng.random() < 0.3)
    experts = _log(rng, 1, 64, True)
    k, n = _log(rng, 64, 4096, odd), _log(rng, 64, 4096, odd)
    most = (2.0 * 16384 * 4096 * 4096) / (2.0 * k * n) / (2 if way == "bwd" else 1) / (6 if dtype == "f32" else 1)
    rows = max(1, min(_log(rng, 1, 16384, True), int(most)))
    return _grouped(rows=rows, experts=experts, active=max(1, min(experts - experts // 8, rows)), k=k, n=n, type=dtype, dir=way,
                    spare=rng.choice([0, 0, rows // 16]))


# ------------------------------------------------------------ what is in hand
def _rand(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=_DEV, dtype=torch.float32) * scale).to(dtype)


def _counts(case, seed):
    """Rows of each expert: `active` of them have some, unevenly."""
    r = np.random.RandomState(seed % (1 << 31))
    e, a, t = case["experts"], case["active"], case["rows"] - case["spare"]
    share = r.lognormal(0.0, 0.4, a)
    extra = r.multinomial(t - a, share / share.sum()) if t > a else np.zeros(a, np.int64)
    counts = np.zeros(e, np.int64)
    counts[r.permutation(e)[:a]] = 1 + extra
    return counts


def prepare(case, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    s = {"case": case}
    t = _TYPES[case["type"]]
    rows = case["rows"]
    if case["op"] == "dropout":
        shape = (rows, case["cols"])
        s["x"] = _rand(g, shape, t)
        s["residual"] = _rand(g, shape, t) if case["residual"] else None
        s["seed"], s["offset"] = 1 + 7919 * seed, 1000 + seed
        s["out"] = torch.empty(shape, dtype=t, device=_DEV)
        return s
    if case["op"] == "norm":
        cols, xt = case["cols"], _TYPES[case["xtype"]]
        shape = (rows, cols)
        level = 1.0 + 3.0 * (torch.rand(cols, generator=g, device=_DEV) < 0.01)  # a few channels stand out
        s["y" if case["dir"] == "bwd" else "x"] = (_rand(g, shape, torch.float32) * level).to(xt)
        s["branch"] = _rand(g, shape, t, 2.0)
        for name in ("pre_weight", "post_weight"):
            s[name] = 1.0 + _rand(g, (cols,), torch.float32, 0.2)
        for name in ("pre_bias", "post_bias"):
            s[name] = _rand(g, (cols,), torch.float32, 0.1) if case["bias"] else None
        s["gate"] = None
        if case["act"] != "off":
            s["gate"] = _rand(g, shape, t) if case["gate"] == "full" else _rand(g, (cols,), torch.float32)
        s["scale"], s["seed"], s["offset"] = 0.5, 1 + 104729 * seed, 3 + seed
        if case["dir"] == "fwd":
            s["out"] = {"y": torch.empty(shape, dtype=xt, device=_DEV), "h": torch.empty(shape, dtype=t, device=_DEV)}
        else:
            s["dy"], s["dh"] = _rand(g, shape, xt, 0.01), _rand(g, shape, t, 0.01)
            out = {"dx": torch.empty(shape, dtype=xt, device=_DEV), "dbranch": torch.empty(shape, dtype=t, device=_DEV)}
            if s["gate"] is not None:
                out["dgate"] = torch.empty_like(s["gate"])
            for name in ("pre_weight", "post_weight", "pre_bias", "post_bias"):
                if s[name] is not None:
                    out["d" + name] = torch.empty(cols, dtype=torch.float32, device=_DEV)
            s["out"] = out
        return s
    e, k, n = case["experts"], case["k"], case["n"]
    counts = _counts(case, seed)
    s["counts"] = counts.tolist()
    offsets = np.concatenate([[0], np.cumsum(counts)])
    s["offsets"] = torch.from_numpy(offsets.astype(np.int32)).to(_DEV)
    # the plain form's plan: the experts with rows, and where each row sits in their padded batch
    some = np.nonzero(counts)[0]
    s["some"] = torch.from_numpy(some).to(_DEV)
    s["most"] = int(counts.max())
    who = np.repeat(np.arange(len(some)), counts[some])
    place = np.arange(int(counts.sum())) - np.repeat(offsets[some], counts[some])
    s["place"] = torch.from_numpy(who * s["most"] + place).to(_DEV)
    s["x"] = _rand(g, (rows, k), t)
    s["w"] = _rand(g, (e, k, n), t, k**-0.5)
    if case["dir"] == "fwd":
        s["out"] = torch.empty((rows, n), dtype=t, device=_DEV)
    else:
        s["dy"] = _rand(g, (rows, n), t, 0.01)
        s["out"] = {"dx": torch.empty((rows, k), dtype=t, device=_DEV), "dw": torch.empty((e, k, n), dtype=t, device=_DEV)}
    return s


# ------------------------------------------------------------------ one pass
def _scratch(nbytes):
    return torch.empty(nbytes, dtype=torch.uint8, device=_DEV) if nbytes else None


def _run_own(s):
    nn, c = _own(), s["case"]
    stream = torch.cuda.current_stream().cuda_stream
    if c["op"] == "dropout":
        if c["dir"] == "bwd":
            nn.dropout_backward(s["x"], c["p"], s["seed"], s["out"], offset=s["offset"], base=c["base"], stream=stream)
        else:
            nn.dropout(s["x"], c["p"], s["seed"], s["out"], offset=s["offset"], base=c["base"], residual=s["residual"], stream=stream)
        return s["out"]
    if c["op"] == "norm":
        how = dict(kind=c["kind"], eps=1e-6, branch=s["branch"], post_weight=s["post_weight"], post_bias=s["post_bias"], gate=s["gate"],
                   gate_act="none" if c["act"] == "off" else c["act"], scale=s["scale"], p=c["p"], seed=s["seed"], offset=s["offset"],
                   pre_weight=s["pre_weight"], pre_bias=s["pre_bias"], stream=stream)
        if c["dir"] == "fwd":
            nn.block_norm(s["x"], **s["out"], **how)
        else:
            ws = _scratch(nn.block_norm_backward_workspace(c["rows"], c["cols"]))
            nn.block_norm_backward(s["y"], dy=s["dy"], dh=s["dh"], **s["out"], workspace=ws, **how)
        return s["out"]
    if c["dir"] == "fwd":
        ws = _scratch(nn.grouped_matmul_workspace(s["x"], s["w"], s["out"]))
        nn.grouped_matmul(s["x"], s["w"], s["offsets"], s["out"], workspace=ws, stream=stream)
    else:
        dx, dw = s["out"]["dx"], s["out"]["dw"]
        ws = _scratch(max(nn.grouped_matmul_workspace(s["dy"], s["w"], dx, transpose_w=True), nn.grouped_matmul_dw_workspace(s["x"], s["dy"], dw)))
        nn.grouped_matmul(s["dy"], s["w"], s["offsets"], dx, transpose_w=True, workspace=ws, stream=stream)
        nn.grouped_matmul_dw(s["x"], s["dy"], s["offsets"], dw, workspace=ws, stream=stream)
    return s["out"]


def _plain_keep(n, base, p, seed, offset):
    """n truth values: Philox-4x32-10, four words a counter, from element `base` on."""
    first = base // 4
    q = torch.arange(first, (base + n + 3) // 4, device=_DEV, dtype=torch.int64)
    low = 0xFFFFFFFF
    c0, c1 = q & low, q >> 32
    c2, c3 = torch.full_like(q, offset & low), torch.full_like(q, offset >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack([c0, c1, c2, c3], dim=1).reshape(-1)
    return (words >= round(p * 2.0**32))[base - 4 * first : base - 4 * first + n]


def _plain_norm(v, kind, eps):
    """(v normalised, 1 over its deviation), row by row."""
    if kind == "layer":
        v = v - v.mean(dim=1, keepdim=True)
    r = torch.rsqrt((v * v).mean(dim=1, keepdim=True) + eps)
    return v * r, r


def _plain_norm_grad(g, vhat, r, kind):
    d = g - vhat * (g * vhat).mean(dim=1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(dim=1, keepdim=True)
    return d * r


def _plain_act(gate, act):
    """The gate's value and its slope."""
    if act == "sigmoid":
        a = 1.0 / (1.0 + torch.exp(-gate))
        return a, a * (1.0 - a)
    if act == "tanh":
        a = torch.tanh(gate)
        return a, 1.0 - a * a
    return gate, torch.ones_like(gate)


def _plain_block(s):
    c = s["case"]
    t, xt = _TYPES[c["type"]], _TYPES[c["xtype"]]
    bhat, r2 = _plain_norm(s["branch"].float(), c["kind"], 1e-6)
    u = bhat * s["post_weight"]
    if s["post_bias"] is not None:
        u = u + s["post_bias"]
    act, slope = _plain_act(s["gate"].float(), c["act"]) if s["gate"] is not None else (None, None)
    n = c["rows"] * c["cols"]
    keep = None
    if c["p"] > 0:
        keep = _plain_keep(n, 0, c["p"], s["seed"], s["offset"]).reshape(c["rows"], c["cols"]) * (1.0 / (1.0 - c["p"]))
    if c["dir"] == "fwd":
        z = u if act is None else u * act
        z = z if keep is None else z * keep
        y = s["x"].float() + s["scale"] * z
        h = _plain_norm(y, c["kind"], 1e-6)[0] * s["pre_weight"]
        if s["pre_bias"] is not None:
            h = h + s["pre_bias"]
        return {"y": y.to(xt), "h": h.to(t)}
    dh = s["dh"].float()
    yhat, r1 = _plain_norm(s["y"].float(), c["kind"], 1e-6)
    dx = s["dy"].float() + _plain_norm_grad(dh * s["pre_weight"], yhat, r1, c["kind"])
    dz = s["scale"] * dx
    dz = dz if keep is None else dz * keep
    du = dz if act is None else dz * act
    out = {"dx": dx.to(xt), "dbranch": _plain_norm_grad(du * s["post_weight"], bhat, r2, c["kind"]).to(t)}
    if act is not None:
        dg = dz * u * slope
        out["dgate"] = dg.to(t) if c["gate"] == "full" else dg.sum(dim=0)
    out["dpre_weight"], out["dpost_weight"] = (dh * yhat).sum(dim=0), (du * bhat).sum(dim=0)
    if c["bias"]:
        out["dpre_bias"], out["dpost_bias"] = dh.sum(dim=0), du.sum(dim=0)
    return out


def _plain_padded(s, v):
    """The rows of v in 32 bits, as a batch with one padded block for each expert that has rows."""
    batch = torch.zeros((len(s["some"]) * s["most"], v.shape[1]), dtype=torch.float32, device=_DEV)
    batch[s["place"]] = v[: len(s["place"])].float()
    return batch.reshape(len(s["some"]), s["most"], v.shape[1])


def _plain_unpadded(s, batch, rows):
    out = torch.zeros((rows, batch.shape[2]), dtype=torch.float32, device=_DEV)
    out[: len(s["place"])] = batch.reshape(-1, batch.shape[2])[s["place"]]
    return out


def _plain_grouped(s):
    c = s["case"]
    t = _TYPES[c["type"]]
    x, w = _plain_padded(s, s["x"]), s["w"][s["some"]].float()
    if c["dir"] == "fwd":
        return _plain_unpadded(s, torch.bmm(x, w), c["rows"]).to(t)
    dy = _plain_padded(s, s["dy"])
    dw = torch.zeros((c["experts"], c["k"], c["n"]), dtype=t, device=_DEV)
    dw[s["some"]] = torch.bmm(x.transpose(1, 2), dy).to(t)
    return {"dx": _plain_unpadded(s, torch.bmm(dy, w.transpose(1, 2)), c["rows"]).to(t), "dw": dw}


def run(s):
    if own:
        return _run_own(s)
    c = s["case"]
    if c["op"] == "dropout":
        x = s["x"].float()
        keep = _plain_keep(x.numel(), c["base"], c["p"], s["seed"], s["offset"]).reshape(x.shape)
        y = torch.where(keep, x * (1.0 / (1.0 - c["p"])), torch.zeros_like(x))
        y = y if s["residual"] is None else y + s["residual"].float()
        return y.to(_TYPES[c["type"]])
    return _plain_block(s) if c["op"] == "norm" else _plain_grouped(s)


# --------------------------------------------------------- what it cannot do without
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    b, rows = size[case["type"]], case["rows"]
    if case["op"] == "dropout":
        n = rows * case["cols"]
        return {"bytes": n * b * (3 if case["residual"] else 2), "flops": n * 2}
    if case["op"] == "norm":
        n, xb, cols = rows * case["cols"], size[case["xtype"]], case["cols"]
        full = case["act"] != "off" and case["gate"] == "full"
        vectors = (4 if case["bias"] else 2) + (1 if case["act"] != "off" and not full else 0)
        if case["dir"] == "fwd":
            return {"bytes": n * (2 * xb + 2 * b + (b if full else 0)) + 4 * cols * vectors, "flops": n * 12}
        return {"bytes": n * (3 * xb + 3 * b + (2 * b if full else 0)) + 8 * cols * vectors, "flops": n * 30}
    k, n, taken = case["k"], case["n"], rows - case["spare"]
    one, weights = 2.0 * taken * k * n, case["active"] * k * n * b
    if case["dir"] == "fwd":
        return {"bytes": taken * k * b + weights + rows * n * b, "flops": one}
    return {"bytes": taken * (k + n) * b + weights + rows * k * b + case["experts"] * k * n * b, "flops": 2 * one}


# ------------------------------------------------------------- the definitions in 64 bits
def _exact_keep(n, base, p, seed, offset):
    """Element by element from the generator's definition, on the host."""
    e = np.arange(base, base + n, dtype=np.uint64)
    q, low, half = np.arange(base >> 2, ((base + n - 1) >> 2) + 1, dtype=np.uint64), np.uint64(0xFFFFFFFF), np.uint64(32)
    ctr = [q & low, q >> half, np.uint64(offset) & low, np.uint64(offset) >> half]
    key = [seed & 0xFFFFFFFF, seed >> 32]
    for i in range(10):
        p0, p1 = np.uint64(0xD2511F53) * ctr[0], np.uint64(0xCD9E8D57) * ctr[2]
        ctr = [(p1 >> half) ^ ctr[1] ^ np.uint64((key[0] + i * 0x9E3779B9) % 2**32), p1 & low,
               (p0 >> half) ^ ctr[3] ^ np.uint64((key[1] + i * 0xBB67AE85) % 2**32), p0 & low]
    words = np.empty((len(q), 4), np.uint64)
    for j in range(4):
        words[:, j] = ctr[j]
    w = words.reshape(-1)[(e - np.uint64(4) * (e[0] >> np.uint64(2))).astype(np.int64)]
    return torch.from_numpy(w.astype(np.int64)).to(_DEV) >= int(round(p * 2.0**32))


def _exact_stats(v, kind):
    mean = v.mean(1) if kind == "layer" else torch.zeros(v.shape[0], dtype=torch.float64, device=_DEV)
    var = ((v - mean[:, None]) ** 2).mean(1)
    return mean[:, None], 1.0 / torch.sqrt(var + 1e-6)[:, None]


def _exact_back(v, kind, g):
    """d(sum g * norm(v)) / dv."""
    mean, r = _exact_stats(v, kind)
    hat, d = (v - mean) * r, v.shape[1]
    along = (g * hat).sum(1)[:, None] / d
    flat = g.sum(1)[:, None] / d if kind == "layer" else 0.0
    return (g - flat - hat * along) * r, hat


def _exact_norm(s):
    c, d = s["case"], torch.float64
    shape = (c["rows"], c["cols"])
    b = s["branch"].to(d)
    mean, r = _exact_stats(b, c["kind"])
    w1, w2 = s["pre_weight"].to(d), s["post_weight"].to(d)
    c1, c2 = (s["pre_bias"].to(d), s["post_bias"].to(d)) if c["bias"] else (0.0, 0.0)
    u = (b - mean) * r * w2 + c2
    gate = s["gate"].to(d) if s["gate"] is not None else None
    a = 1.0 if gate is None else {"none": lambda v: v, "sigmoid": torch.special.expit, "tanh": torch.tanh}[c["act"]](gate)
    m = 1.0
    if c["p"] > 0:
        m = _exact_keep(shape[0] * shape[1], 0, c["p"], s["seed"], s["offset"]).reshape(shape).to(d) / (1.0 - c["p"])
    if c["dir"] == "fwd":
        y = s["x"].to(d) + s["scale"] * m * a * u
        mean, r = _exact_stats(y, c["kind"])
        return {"y": y, "h": (y - mean) * r * w1 + c1}
    dh = s["dh"].to(d)
    back, yhat = _exact_back(s["y"].to(d), c["kind"], dh * w1)
    dx = s["dy"].to(d) + back
    du = s["scale"] * m * dx * a
    db, bhat = _exact_back(b, c["kind"], du * w2)
    out = {"dx": dx, "dbranch": db, "dpre_weight": (dh * yhat).sum(0), "dpost_weight": (du * bhat).sum(0)}
    if gate is not None:
        slope = {"none": lambda v: 1.0, "sigmoid": lambda v: v * (1.0 - v), "tanh": lambda v: 1.0 - v * v}[c["act"]](a)
        dg = s["scale"] * m * dx * u * slope
        out["dgate"] = dg if c["gate"] == "full" else dg.sum(0)
    if c["bias"]:
        out["dpre_bias"], out["dpost_bias"] = dh.sum(0), du.sum(0)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    d = torch.float64
    if case["op"] == "dropout":
        keep = _exact_keep(s["x"].numel(), case["base"], case["p"], s["seed"], s["offset"]).reshape(s["x"].shape)
        y = keep * (s["x"].to(d) / (1.0 - case["p"]))
        return y if s["residual"] is None else y + s["residual"].to(d)
    if case["op"] == "norm":
        return _exact_norm(s)
    k, n, rows = case["k"], case["n"], case["rows"]
    if case["dir"] == "fwd":
        out = {"y": torch.zeros((rows, n), dtype=d, device=_DEV)}
    else:
        out = {"dx": torch.zeros((rows, k), dtype=d, device=_DEV), "dw": torch.zeros((case["experts"], k, n), dtype=d, device=_DEV)}
    at = 0
    for e, count in enumerate(s["counts"]):
        x, w = s["x"][at : at + count].to(d), s["w"][e].to(d)
        if case["dir"] == "fwd":
            out["y"][at : at + count] = x @ w
        else:
            dy = s["dy"][at : at + count].to(d)
            out["dx"][at : at + count] = dy @ w.T
            out["dw"][e] = x.T @ dy
        at += count
    return out["y"] if case["dir"] == "fwd" else out
