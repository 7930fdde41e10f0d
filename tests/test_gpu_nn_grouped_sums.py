"""How exact the grouped products' sums are on a B200, norm-wise against 64 bits,
where the bound for each element would hide a mistake.

F32 results of 16-bit operands of one sign: an MMA may cut its accumulator and
its sixteen products below 2^-23 of the running sum, together at most 3 * 2^-23
of it. A chunk is 32 MMAs from 0, whose sums grow evenly: 32 / 2 * 3 * 2^-23 =
5.7e-6 at most, whatever the number of rows; adding up to 128 chunks (or parts)
rounds to nearest, at most 2^-24 of the sum each time and of either sign, some
sqrt(128) * 2^-25: 3e-7. Together 6e-6.

F32 operands of random signs: the planes leave 2^-24 of each number's size or
less, a chunk's sums and those of the chunks as above but of either sign:
1e-6 in all, where any one of the six plane products left out is 4e-6 or more
(test_nn_planes_host.py).

Operands of which one pair of planes carries the result: products of 4 at most
cancel, in one MMA, which may cut four of them and the sum below 2^-23 of the
largest; the pairs of lower planes add a hundredth of that: 5 * 4 * 2^-23 * 1.1 =
2.7e-6, of results of 1.5e-5 or more.

Operands down to the least normal number: the lowest plane that there is ends at
2^-133, so that either operand may be off by that: 2^-133 * (|a| + |b|) for each
product beside the bound of test_gpu_nn_grouped.py, and a product below 2^-126
may be lost whole in each of its six terms."""
import numpy as np
import pytest
import torch
from nn_planes import TERMS, carried_by
from nn_reference import grouped, grouped_dw

from cudacaml_b200 import nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def space(n):
    return torch.full((n,), 255, dtype=torch.uint8, device=DEV) if n else None


def gradient(x, dy, offsets, dtype):
    out = torch.full((len(offsets) - 1, x.shape[1], dy.shape[1]), float("nan"), dtype=dtype, device=DEV)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    nn.grouped_matmul_dw(x, dy, off, out, workspace=space(nn.grouped_matmul_dw_workspace(x, dy, out)))
    return out


def forward(x, w, offsets, wt):
    out = torch.full((x.shape[0], w.shape[1] if wt else w.shape[2]), float("nan"), dtype=x.dtype, device=DEV)
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    nn.grouped_matmul(x, w, off, out, transpose_w=wt, workspace=space(nn.grouped_matmul_workspace(x, w, out, transpose_w=wt)))
    return out


def error(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,k,n", [(300, 264, 520), (5000, 256, 512), (16384, 2048, 2048), (65536, 256, 512)])
def test_f32_gradient_of_w_has_no_bias_that_grows_with_the_rows(dtype, rows, k, n):
    x, dy = rand((rows, k), TYPES[dtype], 1).abs(), rand((rows, n), TYPES[dtype], 2).abs()
    offsets = [0, rows // 100, rows]
    out = gradient(x, dy, offsets, torch.float32)
    want, _ = grouped_dw(x, dy, offsets)
    for e in range(2):
        assert error(out[e], want[e]) <= 6e-6


# the product on the tensor cores takes 16 rows an expert or more; K below a chunk of 256, just past one, over many, and cut into parts
@pytest.mark.parametrize("rows,experts,k,n", [(96, 2, 64, 64), (64, 2, 72, 200), (300, 3, 256, 264), (129, 2, 264, 520), (515, 4, 1000, 136), (64, 1, 5000, 64),
                                              (4000, 8, 640, 1024)])
def test_f32_products_norm_wise(rows, experts, k, n):
    offsets = [rows * e // experts for e in range(experts + 1)]
    x, w, dy = rand((rows, k), torch.float32, 3), rand((experts, k, n), torch.float32, 4), rand((rows, n), torch.float32, 5)
    for got, want in ((forward(x, w, offsets, False), grouped(x, w, offsets)[0]), (forward(dy, w, offsets, True), grouped(dy, w, offsets, True)[0])):
        for a, b in zip(offsets[:-1], offsets[1:]):
            assert error(got[a:b], want[a:b]) <= 1e-6
    got, want = gradient(x, dy, offsets, torch.float32), grouped_dw(x, dy, offsets)[0]
    for e in range(experts):
        assert error(got[e], want[e]) <= 1e-6


@pytest.mark.parametrize("term", TERMS)
@pytest.mark.parametrize("rows,k,n", [(64, 64, 72), (200, 600, 264), (48, 2000, 64)])
def test_f32_products_by_every_pair_of_planes(term, rows, k, n):
    pairs = [carried_by(term, rows, k, n, e) for e in range(3)]
    xs, ws = (torch.from_numpy(np.stack(v)).to(DEV) for v in zip(*pairs))
    want = torch.bmm(xs.double(), ws.double())
    offsets, x = [0, rows, 2 * rows, 3 * rows], xs.reshape(3 * rows, k)
    steps = [0, k, 2 * k, 3 * k]
    for got in (forward(x, ws, offsets, False).reshape(want.shape), forward(x, ws.transpose(1, 2).contiguous(), offsets, True).reshape(want.shape),
                gradient(xs.transpose(1, 2).reshape(3 * k, rows).contiguous(), ws.reshape(3 * k, n), steps, torch.float32)):
        assert float((got.double() - want).abs().max()) <= 2.7e-6


@pytest.mark.parametrize("small", [-100, -110, -112, -118, -123])
@pytest.mark.parametrize("large", [0, 60, 120])
def test_f32_products_of_very_small_operands(small, large):
    rows, k, n = 96, 200, 72
    offsets = [0, rows // 3, rows]
    x, w = rand((rows, k), torch.float32, 6) * 2.0**small, rand((2, k, n), torch.float32, 7) * 2.0**large
    dy = rand((rows, n), torch.float32, 8) * 2.0**large

    def check(got, want, mag, others, terms):
        bound = 2.0**-24 * want.abs() + (terms + 16) * 2.0**-23 * mag + 2.0**-133 * others + 6 * terms * 2.0**-126
        assert float((got.double() - want).abs().sub(bound).max()) <= 0

    ones, onesw, onesd = torch.ones_like(x), torch.ones_like(w), torch.ones_like(dy)
    check(forward(x, w, offsets, False), *grouped(x, w, offsets), grouped(x, onesw, offsets)[1] + grouped(ones, w, offsets)[1], k)
    check(forward(x, w.transpose(1, 2).contiguous(), offsets, True), *grouped(x, w, offsets), grouped(x, onesw, offsets)[1] + grouped(ones, w, offsets)[1], k)
    check(gradient(x, dy, offsets, torch.float32), *grouped_dw(x, dy, offsets), grouped_dw(x, onesd, offsets)[1] + grouped_dw(ones, dy, offsets)[1], rows)
