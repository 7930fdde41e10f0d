"""F32 grouped products of infinite operands on a B200: infinities and NaN where
the definition has them, whatever the number of rows, and every other result
within the bound of test_gpu_nn_grouped.py."""
import pytest
import torch
from nn_reference import grouped, grouped_dw
from test_gpu_nn_grouped import DEV, rand, slack, space

from cudacaml_b200 import nn

pytestmark = pytest.mark.gpu
INF = float("inf")


def spread(a, seed, share):
    """Infinities of both signs in a few places of a, and zeros and round numbers (whose lower planes are 0) in others."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    u = torch.rand(a.shape, generator=g, device=DEV)
    a = torch.where(u < 0.3, a.round(), a)
    a = torch.where(u < share, torch.full_like(a, INF), a)
    return torch.where(u > 1 - share, torch.full_like(a, -INF), a)


def same(got, want, mag, k):
    w = want.double()
    assert torch.equal(got.isnan(), w.isnan())
    inf = w.isinf()
    assert bool(inf.any()) and torch.equal(got.double()[inf], w[inf])
    fine = w.isfinite()
    off = (got.double() - w).abs() - (2.0**-24 * w.abs() + slack(mag, k))
    assert bool(fine.any()) and float(off[fine].max()) <= 0


@pytest.mark.parametrize("rows,experts,k,n", [(6, 3, 96, 40), (64, 2, 64, 72), (200, 3, 515, 129), (700, 4, 1024, 264), (2050, 2, 300, 520), (300, 1, 4000, 64)])
def test_infinities(rows, experts, k, n):
    offsets = [rows * e // experts for e in range(experts)] + [rows - 1]
    x, w, dy = rand((rows, k), torch.float32, 1), rand((experts, k, n), torch.float32, 2), rand((rows, n), torch.float32, 3)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    some = 1.0 / (8 * max(k, rows))  # leaves most rows and columns without one
    for xs, ws in ((spread(x, 4, 4 * some), w), (x, spread(w, 5, some)), (spread(x, 6, some), spread(w, 7, some / 4))):
        xs[0, 0] = INF
        for wt in (False, True):
            v = ws.transpose(1, 2).contiguous() if wt else ws
            out = torch.empty((rows, n), device=DEV)
            nn.grouped_matmul(xs, v, off, out, transpose_w=wt, workspace=space(nn.grouped_matmul_workspace(xs, v, out, transpose_w=wt)))
            same(out, *grouped(xs, v, offsets, wt), k)
            assert not bool(out[-1].any())
    for xs, ys in ((spread(x, 8, 4 * some), dy), (x, spread(dy, 9, 4 * some))):
        xs[0, 0] = ys[0, 0] = INF
        out = torch.empty((experts, k, n), device=DEV)
        nn.grouped_matmul_dw(xs, ys, off, out, workspace=space(nn.grouped_matmul_dw_workspace(xs, ys, out)))
        same(out, *grouped_dw(xs, ys, offsets), rows)


def test_nothing_but_infinities_or_nan():
    x, w = torch.full((300, 2000), INF, device=DEV), rand((1, 2000, 300), torch.float32, 10).abs() + 0.5
    off = torch.tensor([0, 300], dtype=torch.int32, device=DEV)
    out = torch.empty((300, 300), device=DEV)
    ws = space(nn.grouped_matmul_workspace(x, w, out))
    nn.grouped_matmul(x, w, off, out, workspace=ws)
    assert bool((out == INF).all())
    w[0, 1::2] *= -1
    nn.grouped_matmul(x, w, off, out, workspace=ws)
    assert bool(out.isnan().all())
    x.fill_(float("nan"))
    nn.grouped_matmul(x, w, off, out, workspace=ws)
    assert bool(out.isnan().all())
