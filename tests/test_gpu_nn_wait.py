"""Grouped products whose waits run out on a B200: the call ends, says so in its
error word, and leaves the device, the stream and the next call as they were.

The bound of a wait is set to a few polls, of 4 us each; a draining warp waits for
a tile's contraction, at the two larger sizes 100 us and more, or a chunk of it,
from 7 us on for F32."""
import pytest
import torch

from cudacaml_b200 import nn

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def space(n):
    return torch.full((n,), 255, dtype=torch.uint8, device=DEV) if n else None


def calls(t, rows, k, n):
    """The three products of two experts (one of a ragged end), as functions of an error word."""
    x, dy, w = rand((rows, k), t, 1), rand((rows, n), t, 2), rand((2, k, n), t, 3, k**-0.5)
    off = torch.tensor([0, rows // 2 - 5, rows], dtype=torch.int32, device=DEV)
    outs = torch.empty((rows, n), dtype=t, device=DEV), torch.empty((rows, k), dtype=t, device=DEV), torch.empty((2, k, n), dtype=t, device=DEV)
    ws = space(max(nn.grouped_matmul_workspace(x, w, outs[0]), nn.grouped_matmul_workspace(dy, w, outs[1], transpose_w=True),
                   nn.grouped_matmul_dw_workspace(x, dy, outs[2])))

    def forward(err):
        nn.grouped_matmul(x, w, off, outs[0], workspace=ws, err=err)
        return outs[0]

    def transposed(err):
        nn.grouped_matmul(dy, w, off, outs[1], transpose_w=True, workspace=ws, err=err)
        return outs[1]

    def gradient(err):
        nn.grouped_matmul_dw(x, dy, off, outs[2], workspace=ws, err=err)
        return outs[2]

    return forward, transposed, gradient


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,k,n", [(512, 65536, 2048), (131072, 512, 2048), (700, 264, 520)])
def test_a_wait_that_runs_out_ends_the_call_and_is_reported(dtype, rows, k, n):
    every = calls(TYPES[dtype], rows, k, n)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    clean = [f(err).clone() for f in every]
    assert int(err) == 0
    seen = 0
    try:
        for polls in (1, 2, 3):
            nn.wait_polls(polls)
            for f, want in zip(every, clean):
                for _ in range(5):
                    err.zero_()
                    out = f(err)
                    got = int(err)
                    assert got in (0, 16)
                    assert got or torch.equal(out, want)
                    seen |= got
    finally:
        nn.wait_polls()
    assert seen == 16 or rows == 700
    err.zero_()
    for f, want in zip(every, clean):
        assert torch.equal(f(err), want)
    assert int(err) == 0


def test_polls_out_of_range_are_refused():
    for polls in (-1, 1 << 32):
        with pytest.raises(ValueError):
            nn.wait_polls(polls)
