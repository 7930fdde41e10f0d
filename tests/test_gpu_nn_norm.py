"""nn.block_norm and its gradient on a B200 against their formulas in 64 bits.

Tolerance: with M the sum of the magnitudes of the terms that make up an
element (nn_reference returns it beside the value), each term has a few F32
roundings of its own and those of its row's sums, whose running error is at
most one rounding for each addend of a thread's part plus the tree's:
|y - e| <= unit * |e| + (cols / 32 + 64) * 2^-24 * M, and rows more roundings
for sums over rows."""
import pytest
import torch
from nn_reference import U, block, block_grad, close, keep

from cudacaml_b200 import nn
from cudacaml_b200 import runtime as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rand(shape, dtype, seed, scale=1.0, mean=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale + mean).to(dtype)


def slack(mag, cols, rows=0):
    return (cols / 32 + 64 + rows) * U * mag


class Case:
    def __init__(self, rows, cols, t, xt, kind="rms", gate="full", act="sigmoid", p=0.0, bias=False, post_norm=True, weights=True, wt=torch.float32, pad=0, mean=0.0):
        def mat(dtype, seed, scale=1.0, m=0.0):
            return rand((rows, cols + pad), dtype, seed, scale, m)[:, pad // 2 : pad // 2 + cols]

        self.rows, self.cols, self.p = rows, cols, p
        self.x, self.branch = mat(xt, 1, 1.0, mean), mat(t, 2, 2.0, mean)
        self.w1 = rand((cols,), wt, 3, 0.3, 1.0) if weights else None
        self.w2 = rand((cols,), wt, 4, 0.3, 1.0) if weights and post_norm else None
        self.c1 = rand((cols,), wt, 5, 0.2) if bias else None
        self.c2 = rand((cols,), wt, 6, 0.2) if bias and post_norm else None
        self.gate = None if gate is None else mat(t, 7) if gate == "full" else rand((cols,), torch.float32, 8)
        self.dy, self.dh = mat(xt, 9, 0.1), mat(t, 10, 0.1)
        self.seed, self.offset, self.base, self.scale, self.eps = 1234567, 5, (1 << 35) + 4, 0.7, 1e-5
        self.mask = keep(self.base, (rows, cols), p, self.seed, self.offset, DEV).double() / (1 - p) if p > 0 else 1.0
        self.plain = dict(kind=kind, eps=self.eps, post_norm=post_norm, w1=self.w1, w2=self.w2, c2=self.c2, gate=self.gate, act=act, scale=self.scale, mask=self.mask)
        self.how = dict(kind=kind, eps=self.eps, branch=self.branch, post_norm=post_norm, post_weight=self.w2, post_bias=self.c2, gate=self.gate,
                        gate_act=act, scale=self.scale, p=p, seed=self.seed, offset=self.offset, base=self.base, pre_weight=self.w1, pre_bias=self.c1)
        self.t, self.xt, self.kind = t, xt, kind

    def out(self, dtype):
        return torch.full((self.rows, self.cols), float("nan"), dtype=dtype, device=DEV)

    def forward(self, check=True):
        y, h = self.out(self.xt), self.out(self.t)
        nn.block_norm(self.x, y, h, **self.how)
        if check:
            ye, ym, he, hm = block(self.x, self.branch, c1=self.c1, **self.plain)
            close(y, ye, slack(ym, self.cols), "y")
            close(h, he, slack(hm, self.cols), "h")
        return y, h

    def backward(self, y, dy, dh):
        out = {"dx": self.out(self.xt), "dbranch": self.out(self.t)}
        vec = lambda: torch.full((self.cols,), float("nan"), device=DEV)  # noqa: E731
        if self.gate is not None:
            out["dgate"] = self.out(self.t) if self.gate.dim() == 2 else vec()
        if dh is not None:
            out["dpre_weight"], out["dpre_bias"] = vec(), vec()
        if self.plain["post_norm"]:
            out["dpost_weight"], out["dpost_bias"] = vec(), vec()
        ws = torch.full((nn.block_norm_backward_workspace(self.rows, self.cols),), 255, dtype=torch.uint8, device=DEV)
        how = dict(self.how)
        if dh is None:
            how["pre_weight"] = None
        nn.block_norm_backward(y, dy=dy, dh=dh, workspace=ws, **out, **how)
        want = block_grad(y, self.branch, dy, dh, **self.plain)
        for name, got in out.items():
            e, m = want[name]
            close(got, e, slack(m, self.cols, self.rows if got.dim() == 1 else 0), name)
        return out


T = [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")]


@pytest.mark.parametrize("t,xt", T)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 8), (3, 33), (5, 64), (37, 200), (2, 1000), (130, 512), (9, 4096), (3, 8192), (2, 9001), (2, 20480)])
def test_values_and_gradients(t, xt, kind, rows, cols):
    c = Case(rows, cols, TYPES[t], TYPES[xt], kind=kind, p=0.2, bias=True)
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)


@pytest.mark.parametrize("t,xt", T)
@pytest.mark.parametrize("kind,gate,bias", [("rms", "full", False), ("layer", "channel", True)])
@pytest.mark.parametrize("rows,cols", [(300, 4097), (5, 6147), (161, 6499), (4, 8191), (3, 12287)])
def test_long_rows_of_odd_length(t, xt, kind, gate, bias, rows, cols):
    c = Case(rows, cols, TYPES[t], TYPES[xt], kind=kind, gate=gate, act="tanh", p=0.2, bias=bias)
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)


@pytest.mark.parametrize("gate,act", [(None, "none"), ("full", "none"), ("full", "tanh"), ("channel", "sigmoid"), ("channel", "none"), ("channel", "tanh")])
@pytest.mark.parametrize("t,rows,cols", [("bf16", 65, 1024), ("f32", 17, 257), ("f16", 300, 96)])
def test_gates(gate, act, t, rows, cols):
    c = Case(rows, cols, TYPES[t], TYPES[t], gate=gate, act=act)
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)
    c.backward(y, None, c.dh)
    c.backward(y, c.dy, None)


@pytest.mark.parametrize("t,cols,pad,wt", [("bf16", 256, 16, "bf16"), ("bf16", 250, 6, "f32"), ("f32", 260, 8, "f16"), ("f16", 1024, 2, "f16"), ("bf16", 4096, 24, "bf16")])
@pytest.mark.parametrize("post_norm", [True, False])
def test_strides_weight_types_and_plain_branch(t, cols, pad, wt, post_norm):
    c = Case(21, cols, TYPES[t], torch.float32 if cols == 256 else TYPES[t], pad=pad, wt=TYPES[wt], post_norm=post_norm, bias=True, p=0.1)
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)
    c = Case(21, cols, TYPES[t], TYPES[t], pad=pad, weights=False, post_norm=post_norm, gate=None, act="none")
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)


@pytest.mark.parametrize("t,xt", T)
@pytest.mark.parametrize("cols", [48, 1001, 4096, 10000])
def test_norm_alone(t, xt, cols):
    c = Case(11, cols, TYPES[t], TYPES[xt], gate=None, act="none")
    h = c.out(c.t)
    nn.block_norm(c.x, h=h, eps=c.eps, pre_weight=c.w1)
    _, _, he, hm = block(c.x, None, eps=c.eps, w1=c.w1)
    close(h, he, slack(hm, cols), "h")
    dx, dw = c.out(c.xt), torch.empty(cols, device=DEV)
    ws = torch.empty(nn.block_norm_backward_workspace(11, cols), dtype=torch.uint8, device=DEV)
    nn.block_norm_backward(c.x, dy=c.dy, dh=c.dh, dx=dx, dpre_weight=dw, workspace=ws, eps=c.eps, pre_weight=c.w1)
    want = block_grad(c.x, None, c.dy, c.dh, eps=c.eps, w1=c.w1)
    close(dx, want["dx"][0], slack(want["dx"][1], cols), "dx")
    close(dw, want["dpre_weight"][0], slack(want["dpre_weight"][1], cols, 11), "dw")


@pytest.mark.parametrize("cols", [64, 777, 4096, 16384])
def test_large_mean_and_constant_rows(cols):
    # a mean of 100 deviations; the error of v - mean is of v's size, which the magnitude counts
    c = Case(7, cols, torch.float32, torch.float32, kind="layer", mean=200.0, gate=None, act="none")
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)
    # rows without deviation: norm 0 for the layer norm, 0 for an all-zero rms row
    x = torch.full((3, cols), 2.0, device=DEV)
    h = torch.empty_like(x)
    nn.block_norm(x, h=h, kind="layer", eps=1e-5)
    assert not bool(h.any())
    nn.block_norm(torch.zeros_like(x), h=h, eps=1e-6)
    assert not bool(h.any())
    nn.block_norm(torch.zeros_like(x), h=h, eps=0.0)  # 0 * inf
    assert bool(torch.isnan(h).all())


def test_all_dropped_and_none_dropped():
    c = Case(40, 512, torch.bfloat16, torch.float32, p=0.0)
    c.how["p"], c.plain["mask"] = 1.0, 0.0
    y, _ = c.forward()
    assert torch.equal(y, c.x)
    out = c.backward(y, c.dy, c.dh)
    assert not bool(out["dbranch"].any()) and not bool(out["dgate"].any()) and not bool(out["dpost_weight"].any())


@pytest.mark.parametrize("cols", [200, 201, 12000])
def test_one_bad_row_stays_in_its_row(cols):
    c = Case(9, cols, torch.bfloat16, torch.bfloat16)
    clean = c.forward(check=False)
    for bad in (float("nan"), float("inf")):
        c.branch[4, 7] = bad
        y, h = c.forward(check=False)
        for got, want in zip((y, h), clean):
            keepers = [r for r in range(9) if r != 4]
            assert torch.equal(got[keepers], want[keepers]) and not bool(torch.isfinite(got[4]).all())


@pytest.mark.parametrize("cols", [512, 513, 9000])
def test_in_place_and_partial_outputs(cols):
    c = Case(33, cols, torch.bfloat16, torch.bfloat16, p=0.1)
    y, h = c.forward()
    x = c.x.clone()
    nn.block_norm(x, x, None, **{**c.how, "pre_weight": None, "pre_bias": None})
    assert torch.equal(x, y)
    h2 = torch.empty_like(h)
    nn.block_norm(c.x, None, h2, **c.how)
    assert torch.equal(h2, h)
    full = c.backward(y, c.dy, c.dh)
    dy, dh = c.dy.clone(), c.dh.clone()
    nn.block_norm_backward(y, dy=dy, dh=dh, dx=dy, dbranch=dh, **c.how)
    assert torch.equal(dy, full["dx"]) and torch.equal(dh, full["dbranch"])


def test_rows_do_not_depend_on_their_neighbours_and_runs_repeat():
    c = Case(700, 1024, torch.bfloat16, torch.bfloat16, p=0.1)
    y, h = c.forward()
    one = c.backward(y, c.dy, c.dh)
    two = c.backward(y, c.dy, c.dh)
    assert all(torch.equal(one[k], two[k]) for k in one)
    y1, h1 = torch.empty_like(y[:1]), torch.empty_like(h[:1])
    how = {**c.how, "branch": c.branch[600:601], "gate": c.gate[600:601], "base": c.base + 600 * 1024}
    nn.block_norm(c.x[600:601], y1, h1, **how)
    assert torch.equal(y1[0], y[600]) and torch.equal(h1[0], h[600])


@pytest.mark.parametrize("t,xt", T)
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("gate,p", [("full", 0.2), ("full", 0.0), (None, 0.2), (None, 0.0)])
@pytest.mark.parametrize("rows,cols", [(1, 8), (70, 96), (33, 1000), (301, 1024), (9, 4096), (3, 8192)])
def test_rows_do_not_depend_on_the_results_asked_for(t, xt, kind, gate, p, rows, cols):
    c = Case(rows, cols, TYPES[t], TYPES[xt], kind=kind, gate=gate, act="sigmoid" if gate else "none", p=p)
    y, h = c.forward()
    alone = torch.empty_like(y), torch.empty_like(h)
    nn.block_norm(c.x, alone[0], **{**c.how, "pre_weight": None})
    nn.block_norm(c.x, h=alone[1], **c.how)
    assert torch.equal(alone[0], y) and torch.equal(alone[1], h)
    every = c.backward(y, c.dy, c.dh)
    names = [n for n in every if n not in ("dpre_bias", "dpost_bias")]
    some = {n: torch.empty_like(every[n]) for n in names}
    ws = torch.full((nn.block_norm_backward_workspace(rows, cols),), 255, dtype=torch.uint8, device=DEV)
    nn.block_norm_backward(y, dy=c.dy, dh=c.dh, workspace=ws, **some, **c.how)
    assert all(torch.equal(some[n], every[n]) for n in names)
    dx = torch.empty_like(some["dx"])
    nn.block_norm_backward(y, dy=c.dy, dh=c.dh, dx=dx, **c.how)
    assert torch.equal(dx, every["dx"])


@pytest.mark.parametrize("rows,cols", [(0, 64), (2000, 64), (3000, 136), (1000, 31)])
def test_many_or_no_rows(rows, cols):
    c = Case(rows, cols, torch.bfloat16, torch.bfloat16, gate="channel", act="tanh", bias=True)
    y, _ = c.forward(check=rows > 0)
    if rows:
        c.backward(y, c.dy, c.dh)
        return
    out = {k: torch.full((cols,), 7.0, device=DEV) for k in ("dpre_weight", "dpre_bias", "dpost_weight", "dpost_bias", "dgate")}
    nn.block_norm_backward(y, dy=c.dy, dh=c.dh, **out, **c.how)
    assert all(not bool(v.any()) for v in out.values())


def test_offsets_past_32_bits():
    stride, cols = (1 << 31) + 64, 1024
    buf = torch.empty(stride + cols, dtype=torch.bfloat16, device=DEV)
    c = Case(2, cols, torch.bfloat16, torch.bfloat16)
    for field in ("x", "branch"):
        v = torch.as_strided(buf, (2, cols), (stride, 1))
        v.copy_(getattr(c, field))
        setattr(c, field, v)
        c.how["branch"] = c.branch
        y, _ = c.forward()
        c.backward(y, c.dy, c.dh)
        setattr(c, field, v.clone())
        c.how["branch"] = c.branch


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("cols", [96, 515])
def test_gradient_against_differences(kind, cols):
    # L = sum(cy * y + ch * h). The central difference along v has the formula's own truncation
    # (taken from the 64-bit form) and the rounding of L's terms, each bounded as above.
    rows, eps = 6, 2.0**-6
    c = Case(rows, cols, torch.float32, torch.float32, kind=kind, bias=True)
    cy, ch = rand((rows, cols), torch.float32, 20), rand((rows, cols), torch.float32, 21)
    y, _ = c.forward()
    c.dy, c.dh = cy, ch
    grads = c.backward(y, cy, ch)
    for field, name in (("x", "dx"), ("branch", "dbranch"), ("gate", "dgate"), ("w1", "dpre_weight"), ("w2", "dpost_weight"), ("c2", "dpost_bias")):
        at = getattr(c, field)
        v = rand(at.shape, torch.float32, 22)
        found, plain, rounding = [], [], 0.0
        for s in (eps, -eps):
            moved = at + s * v
            how, formula, x = dict(c.how), dict(c.plain), c.x
            key = {"branch": "branch", "gate": "gate", "w1": "pre_weight", "w2": "post_weight", "c2": "post_bias"}.get(field)
            if field == "x":
                x = moved
            else:
                how[key] = moved
                if field != "branch":
                    formula[field] = moved
            yo, ho = c.out(torch.float32), c.out(torch.float32)
            nn.block_norm(x, yo, ho, **how)
            ye, ym, he, hm = block(x, how["branch"], c1=c.c1, **formula)
            found.append(float((cy.double() * yo.double() + ch.double() * ho.double()).sum()))
            plain.append(float((cy.double() * ye + ch.double() * he).sum()))
            rounding += float((cy.abs() * (slack(ym, cols) + U * ye.abs()) + ch.abs() * (slack(hm, cols) + U * he.abs())).sum()) / (2 * eps)
        e, m = block_grad(y, c.branch, cy, ch, **c.plain)[name]
        along = float((grads[name].double() * v.double()).sum())
        truncation = abs((plain[0] - plain[1]) / (2 * eps) - float((e * v.double()).sum()))
        # y was rounded before the gradient was taken at it, and moved points are rounded
        inputs = 8 * U * float((m * (1 + v.abs())).sum()) / eps
        grad_error = float((slack(m, cols, rows) * v.abs()).sum())
        assert abs((found[0] - found[1]) / (2 * eps) - along) <= truncation + rounding + inputs + grad_error, name


def test_another_stream_and_capture():
    c = Case(64, 2048, torch.bfloat16, torch.bfloat16, p=0.1)
    y, h = c.forward()
    g0 = c.backward(y, c.dy, c.dh)
    st = R.Stream()
    y2, h2 = torch.empty_like(y), torch.empty_like(h)
    dx, dw = torch.empty_like(y), torch.empty(2048, device=DEV)
    ws = torch.empty(nn.block_norm_backward_workspace(64, 2048), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    with R.Graph.capture(st) as g:
        nn.block_norm(c.x, y2, h2, stream=st, **c.how)
        nn.block_norm_backward(y2, dy=c.dy, dh=c.dh, dx=dx, dpost_weight=dw, workspace=ws, stream=st, **c.how)
    for _ in range(2):
        for t in (y2, h2, dx, dw, ws):
            t.zero_()
        torch.cuda.synchronize()
        g.launch(st)
        st.synchronize()
        assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(dx, g0["dx"]) and torch.equal(dw, g0["dpost_weight"])
    g.destroy()
    st.destroy()


@pytest.mark.parametrize("base", [3, (1 << 34) - 700, (1 << 34) - 702, (1 << 63) + 8])
@pytest.mark.parametrize("t,cols", [("bf16", 256), ("f32", 130)])
def test_masks_of_any_first_index(base, t, cols):
    # a first index that is no multiple of the generator's four, and one whose counters' high word changes on the way
    c = Case(9, cols, TYPES[t], TYPES[t], p=0.3)
    c.base = c.how["base"] = base
    c.plain["mask"] = keep(base, (9, cols), 0.3, c.seed, c.offset, DEV).double() / 0.7
    y, _ = c.forward()
    c.backward(y, c.dy, c.dh)


@pytest.mark.parametrize("t", ["bf16", "f32"])
def test_f32_gate_of_every_element(t):
    rows, cols = 19, 264
    c = Case(rows, cols, TYPES[t], torch.float32, act="tanh")
    c.gate = rand((rows, cols), torch.float32, 31, 0.4)
    c.how["gate"], c.plain["gate"] = c.gate, c.gate
    y, _ = c.forward()
    dgate = torch.empty_like(c.gate)
    nn.block_norm_backward(y, dy=c.dy, dh=c.dh, dgate=dgate, **c.how)
    e, m = block_grad(y, c.branch, c.dy, c.dh, **c.plain)["dgate"]
    close(dgate, e, slack(m, cols), "dgate")


def test_tanh_gate_near_zero_keeps_its_relative_error():
    g = torch.cat([torch.logspace(-30, 0.7, 2000), -torch.logspace(-30, 0.7, 2000), torch.tensor([0.0, 0.5499, 0.5501, float("inf"), -float("inf")])]).to(DEV)
    cols = g.numel()
    x, y = torch.zeros((1, cols), device=DEV), torch.empty((1, cols), device=DEV)
    nn.block_norm(x, y, branch=torch.ones_like(x), post_norm=False, gate=g.reshape(1, -1), gate_act="tanh")
    # series, exponential and reciprocal: eight units in the last place
    close(y, torch.tanh(g.double()).reshape(1, -1), 8 * U * torch.tanh(g.double()).abs().reshape(1, -1), "tanh")
