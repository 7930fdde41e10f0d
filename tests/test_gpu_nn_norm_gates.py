"""The sigmoid gate of nn.block_norm on a B200: its relative error over all of
F32's exponentials, by every way that a gate is read.

Units of 2^-24: 4 of the hardware's exponential (2^-22), 1 of its correction, 1 of
the sum, 2 of the reciprocal, 1 of the product, 1 of the result: 10. The slope
a (1 - a) of a gate below 0 has two roundings more, dgate two products and a
channel's two sums over three rows: 16."""
import pytest
import torch
from nn_reference import U

from cudacaml_b200 import nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
LEAST = 2.0**-126


def gates(cols):
    g = torch.linspace(-80, 80, cols, device=DEV)
    g[:8] = torch.tensor([-80.0, -1e-30, 0.0, 1e-30, -17.3, 79.9, -40.0, -79.99], device=DEV)
    return g


def sigmoid(g, cols, t, rank):
    x = torch.zeros((3, cols), device=DEV)
    branch, y = torch.ones((3, cols), dtype=t, device=DEV), torch.full((3, cols), float("nan"), device=DEV)
    gate = g if rank == 1 else g.expand(3, cols).contiguous()
    nn.block_norm(x, y, branch=branch, post_norm=False, gate=gate, gate_act="sigmoid")
    return y, x, branch, gate


# the ring by 16 bytes, by elements, and rows too long for it; f32 and 16-bit branches
@pytest.mark.parametrize("cols", [200, 201, 2048, 20000])
@pytest.mark.parametrize("t", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rank", [1, 2])
def test_relative_error(cols, t, rank):
    g = gates(cols)
    y, x, branch, gate = sigmoid(g, cols, t, rank)
    want = torch.sigmoid(g.double()).expand(3, cols)
    assert float(((y.double() - want).abs() / want).max()) <= 10 * U
    dy, dgate = torch.ones_like(x), torch.empty_like(gate)
    ws = torch.empty(nn.block_norm_backward_workspace(3, cols), dtype=torch.uint8, device=DEV)
    nn.block_norm_backward(y, dy=dy, dgate=dgate, branch=branch, post_norm=False, gate=gate, gate_act="sigmoid", workspace=ws)
    slope = (want * torch.sigmoid(-g.double())).sum(0) if rank == 1 else want * torch.sigmoid(-g.double())
    low = (g < 0).expand_as(slope)
    assert float(((dgate.double() - slope).abs() / slope)[low].max()) <= 16 * U


@pytest.mark.parametrize("cols", [200, 201, 20000])
@pytest.mark.parametrize("rank", [1, 2])
def test_ends(cols, rank):
    g = gates(cols)
    g[:7] = torch.tensor([float("inf"), -float("inf"), float("nan"), 100.0, -100.0, 3e38, -3e38], device=DEV)
    y = sigmoid(g, cols, torch.float32, rank)[0]
    assert bool((y[:, [0, 3, 5]] == 1).all()) and bool((y[:, [1, 4, 6]].abs() < LEAST).all()) and bool(y[:, 2].isnan().all())
    assert not bool(y[:, 3:].isnan().any())
