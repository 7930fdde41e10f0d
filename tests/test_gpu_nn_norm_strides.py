"""nn.block_norm and its gradient on a B200 with outputs whose rows are padded,
each by another width: the results and tolerances of test_gpu_nn_norm.py, and
padding that stays as it was."""
import pytest
import torch
from nn_reference import block, block_grad, close
from test_gpu_nn_norm import DEV, TYPES, Case, slack

from cudacaml_b200 import nn

pytestmark = pytest.mark.gpu
MARK = 7.0


class Padded:
    """A rows x cols view that begins `left` columns into rows of left + cols + right, all MARK."""

    def __init__(self, rows, cols, dtype, left, right):
        self.all = torch.full((rows, left + cols + right), MARK, dtype=dtype, device=DEV)
        self.view, self.left, self.cols = self.all[:, left : left + cols], left, cols

    def kept(self):
        return bool((self.all[:, : self.left] == MARK).all()) and bool((self.all[:, self.left + self.cols :] == MARK).all())


# multiples of 8 for 16-byte rows, odd ones for the others; rows too long for the ring of either direction
@pytest.mark.parametrize("t,xt", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("cols", [200, 203, 4096, 4097, 12296, 12297])
@pytest.mark.parametrize("gate,bias", [("full", False), ("channel", True)])
def test_padded_outputs(t, xt, kind, cols, gate, bias):
    rows = 37 if cols < 1000 else 5
    step = 8 if cols % 8 == 0 else 1
    pads = iter((step * a, step * b) for a, b in ((1, 1), (1, 2), (2, 3), (3, 3), (2, 5)))
    c = Case(rows, cols, TYPES[t], TYPES[xt], kind=kind, gate=gate, act="tanh", p=0.2, bias=bias)
    out = lambda dtype: Padded(rows, cols, dtype, *next(pads))  # noqa: E731
    y, h = out(c.xt), out(c.t)
    nn.block_norm(c.x, y.view, h.view, **c.how)
    ye, ym, he, hm = block(c.x, c.branch, c1=c.c1, **c.plain)
    close(y.view, ye, slack(ym, cols), "y")
    close(h.view, he, slack(hm, cols), "h")
    grads = {"dx": out(c.xt), "dbranch": out(c.t)}
    if gate == "full":
        grads["dgate"] = out(c.t)
    dy = y.view.clone()
    nn.block_norm_backward(dy, dy=c.dy, dh=c.dh, **{n: g.view for n, g in grads.items()}, **c.how)
    want = block_grad(dy, c.branch, c.dy, c.dh, **c.plain)
    for name, g in grads.items():
        close(g.view, want[name][0], slack(want[name][1], cols), name)
    for p in (y, h, *grads.values()):
        assert p.kept()


@pytest.mark.parametrize("cols", [264, 267, 9000])
def test_padded_gradient_of_an_f32_gate(cols):
    c = Case(19, cols, torch.bfloat16, torch.float32, act="sigmoid")
    c.gate = c.how["gate"] = c.plain["gate"] = torch.randn((19, cols), generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    dgate = Padded(19, cols, torch.float32, 8, 16) if cols % 8 == 0 else Padded(19, cols, torch.float32, 1, 3)
    y, _ = c.forward()
    nn.block_norm_backward(y, dy=c.dy, dh=c.dh, dgate=dgate.view, **c.how)
    e, m = block_grad(y, c.branch, c.dy, c.dh, **c.plain)["dgate"]
    close(dgate.view, e, slack(m, cols), "dgate")
    assert dgate.kept()
