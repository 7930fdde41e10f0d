"""How exact the grouped products' sums are on a B200, norm-wise against 64 bits,
where the bound for each element would hide a mistake.

F32 results of 16-bit operands of one sign: an MMA may cut its accumulator and
its sixteen products below 2^-23 of the running sum, together at most 3 * 2^-23
of it. A chunk is 32 MMAs from 0, whose sums grow evenly: 32 / 2 * 3 * 2^-23 =
5.7e-6 at most, whatever the number of rows; adding up to 128 chunks (or parts)
rounds to nearest, at most 2^-24 of the sum each time and of either sign, some
sqrt(128) * 2^-25: 3e-7. Together 6e-6."""
import pytest
import torch
from nn_reference import grouped_dw

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
