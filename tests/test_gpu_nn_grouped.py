"""nn.grouped_matmul and grouped_matmul_dw on a B200 against each expert's
product in 64 bits.

Tolerance: sums over K are F32 in any order, K roundings of at most 2^-23 of
the running sum (tensor-core accumulation may truncate), and a few for 32-bit
operands taken in parts: |y - e| <= unit * |e| + (K + 16) * 2^-23 * sum |a||b|."""
import numpy as np
import pytest
import torch
from nn_reference import close, grouped, grouped_dw

from cudacaml_b200 import nn
from cudacaml_b200 import runtime as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def rand(shape, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def space(n):
    return torch.full((n,), 255, dtype=torch.uint8, device=DEV) if n else None


def slack(mag, k):
    return (k + 16) * 2.0**-23 * mag


def forward(x, w, offsets, wt, out=None, check=True):
    n = w.shape[1] if wt else w.shape[2]
    out = torch.full((x.shape[0], n), float("nan"), dtype=x.dtype, device=DEV) if out is None else out
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    nn.grouped_matmul(x, w, off, out, transpose_w=wt, workspace=space(nn.grouped_matmul_workspace(x, w, out, transpose_w=wt)), err=err)
    assert int(err) == 0
    if check:
        e, m = grouped(x, w, offsets, wt)
        close(out, e, slack(m, x.shape[1]), "out")
    return out


def backward_w(x, dy, offsets, out_dtype=None, out=None):
    out = torch.full((len(offsets) - 1, x.shape[1], dy.shape[1]), float("nan"), dtype=out_dtype or x.dtype, device=DEV) if out is None else out
    off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    nn.grouped_matmul_dw(x, dy, off, out, workspace=space(nn.grouped_matmul_dw_workspace(x, dy, out)), err=err)
    assert int(err) == 0
    e, m = grouped_dw(x, dy, offsets)
    rows = max(b - a for a, b in zip(offsets[:-1], offsets[1:]))
    close(out, e, slack(m, rows), "dw")
    return out


def cut(rows, experts, seed, spare=0):
    """Uneven offsets with empty experts, `spare` rows left over at the end."""
    r = np.random.RandomState(seed)
    share = r.rand(experts) ** 3 * (r.rand(experts) > 0.25) + 1e-9
    counts = r.multinomial(rows - spare, share / share.sum())
    return [0] + np.cumsum(counts).tolist()


SHAPES = [(1, 1, 1, 1), (1, 4, 8, 16), (5, 3, 7, 9), (64, 2, 64, 64), (33, 8, 128, 264), (200, 5, 72, 136), (300, 9, 256, 512), (257, 1, 640, 384),
          (1000, 17, 192, 200), (129, 4, 1031, 77), (700, 3, 520, 1032), (40, 64, 512, 256), (2, 33, 4096, 128), (17, 40, 1000, 1000)]


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,experts,k,n", SHAPES)
def test_every_direction(dtype, rows, experts, k, n):
    t = TYPES[dtype]
    offsets = cut(rows, experts, rows + k, spare=rows // 10)
    x, w, dy = rand((rows, k), t, 1), rand((experts, k, n), t, 2, k**-0.5), rand((rows, n), t, 3)
    y = forward(x, w, offsets, False)
    assert not bool(y[offsets[-1] :].any())
    forward(dy, w, offsets, True)
    backward_w(x, dy, offsets)
    if t != torch.float32:
        backward_w(x, dy, offsets, out_dtype=torch.float32)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_row_ranges(dtype):
    t, k, n = TYPES[dtype], 136, 72
    x, dy = rand((400, k), t, 4), rand((400, n), t, 5)
    for offsets in ([0, 400], [0, 0, 400], [0, 400, 400], [0, 0, 0, 0], [0, 127, 128, 256, 257, 400], [0, 128, 256, 384], [0, 1, 2, 3, 400],
                    [0, 129, 129, 129, 130], [7, 100, 399], [400, 400, 400]):
        w = rand((len(offsets) - 1, k, n), t, 6, 0.1)
        y = forward(x, w, offsets, False)
        assert not bool(y[: offsets[0]].any()) and not bool(y[offsets[-1] :].any())
        forward(dy, w, offsets, True)
        dw = backward_w(x, dy, offsets)
        for e, (a, b) in enumerate(zip(offsets[:-1], offsets[1:])):
            assert a < b or not bool(dw[e].any())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_what_other_rows_hold_does_not_reach_an_expert(dtype):
    # the last rows of a range and the first of the next share tiles: NaN there must stay there
    t, k, n = TYPES[dtype], 192, 256
    for offsets in ([0, 100, 230, 360], [0, 3, 20, 37], [5, 70, 135, 300]):
        x, dy = rand((offsets[-1] + 9, k), t, 7), rand((offsets[-1] + 9, n), t, 8)
        w = rand((3, k, n), t, 9, 0.1)
        clean, cleanw = forward(x, w, offsets, False), backward_w(x, dy, offsets)
        a, b = offsets[1], offsets[2]
        for bad in (float("nan"), float("inf")):
            xb, dyb = x.clone(), dy.clone()
            xb[a:b] = bad
            dyb[a:b] = bad
            xb[offsets[-1] :] = bad
            dyb[offsets[-1] :] = bad
            xb[: offsets[0]] = bad
            got = forward(xb, w, offsets, False, check=False)
            assert torch.equal(got[:a], clean[:a]) and torch.equal(got[b:], clean[b:])
            assert not bool(torch.isfinite(got[a:b]).any())
            dw = torch.empty_like(cleanw)
            off = torch.tensor(offsets, dtype=torch.int32, device=DEV)
            nn.grouped_matmul_dw(xb, dyb, off, dw, workspace=space(nn.grouped_matmul_dw_workspace(xb, dyb, dw)))
            assert torch.equal(dw[0], cleanw[0]) and torch.equal(dw[2], cleanw[2]) and not bool(torch.isfinite(dw[1]).any())


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("pad", [8, 3])
def test_strides(dtype, pad):
    t, rows, k, n, e = TYPES[dtype], 150, 128, 200, 3
    offsets = [0, 60, 60, 150]
    x = rand((rows, k + pad), t, 10)[:, :k]
    w = rand((e, k + 2, n + pad), t, 11, 0.1)[:, :k, :n]
    dy = rand((rows, n + 2 * pad), t, 12)[:, pad : pad + n]
    big = torch.zeros((rows, n + pad), dtype=t, device=DEV)
    forward(x, w, offsets, False, out=big[:, :n])
    assert not bool(big[:, n:].any())
    forward(dy, w, offsets, True)
    bigw = torch.zeros((e, k + 1, n + pad), dtype=t, device=DEV)
    backward_w(x, dy, offsets, out=bigw[:, :k, :n])
    assert not bool(bigw[:, k:].any()) and not bool(bigw[:, :, n:].any())


def test_offsets_out_of_order_are_clamped_and_reported():
    x, w = rand((50, 64), torch.bfloat16, 13), rand((4, 64, 64), torch.bfloat16, 14, 0.1)
    for raw, used in (([0, 30, 20, 40, 50], [0, 30, 30, 40, 50]), ([0, 10, 20, 30, 99], [0, 10, 20, 30, 50]), ([-5, 10, 20, 30, 40], [0, 10, 20, 30, 40]),
                      ([0, 2**31 - 1, 5, 6, 7], [0, 50, 50, 50, 50])):
        off = torch.tensor(raw, dtype=torch.int32, device=DEV)
        for t in (torch.bfloat16, torch.float32):
            err = torch.zeros(1, dtype=torch.int32, device=DEV)
            xt, wt = x.to(t), w.to(t)
            out = torch.empty((50, 64), dtype=t, device=DEV)
            nn.grouped_matmul(xt, wt, off, out, err=err, workspace=space(nn.grouped_matmul_workspace(xt, wt, out)))
            assert int(err) == 64
            e, m = grouped(xt, wt, used)
            close(out, e, slack(m, 64), "clamped")
            err.zero_()
            dw = torch.empty((4, 64, 64), dtype=t, device=DEV)
            nn.grouped_matmul_dw(xt, xt, off, dw, err=err, workspace=space(nn.grouped_matmul_dw_workspace(xt, xt, dw)))
            assert int(err) == 64
            e, m = grouped_dw(xt, xt, used)
            close(dw, e, slack(m, 50), "clamped")


@pytest.mark.parametrize("dtype", list(TYPES))
def test_many_experts(dtype):
    t = TYPES[dtype]
    r = np.random.RandomState(3)
    offsets = [0] + np.cumsum(r.randint(0, 4, 1024)).tolist()
    rows = offsets[-1] + 2
    x, w, dy = rand((rows, 32), t, 15), rand((1024, 32, 24), t, 16), rand((rows, 24), t, 17)
    forward(x, w, offsets, False)
    forward(dy, w, offsets, True)
    backward_w(x, dy, offsets)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,experts,k,n", [(3000, 6, 1024, 1536), (64, 16, 2048, 512)])
def test_runs_repeat(dtype, rows, experts, k, n):
    t = TYPES[dtype]
    offsets = cut(rows, experts, 9)
    x, w, dy = rand((rows, k), t, 18), rand((experts, k, n), t, 19, k**-0.5), rand((rows, n), t, 20)
    a, b, c = forward(x, w, offsets, False), forward(dy, w, offsets, True), backward_w(x, dy, offsets)
    assert torch.equal(a, forward(x, w, offsets, False, check=False))
    assert torch.equal(b, forward(dy, w, offsets, True, check=False))
    assert torch.equal(c, backward_w(x, dy, offsets))


def test_matrices_past_32_bits():
    # the second expert's matrix starts past 2^31 elements; x's second row too
    k, n, t = 128, 256, torch.bfloat16
    stride = (1 << 31) + 64
    buf = torch.empty(stride + k * n, dtype=t, device=DEV)
    w = torch.as_strided(buf, (2, k, n), (stride, n, 1))
    w.copy_(rand((2, k, n), t, 21, 0.1))
    x = rand((10, k), t, 22)
    forward(x, w, [0, 4, 10], False)
    backward_w(x, rand((10, n), t, 23), [0, 4, 10], out=w)
    xs = torch.as_strided(buf, (2, k), (stride, 1))
    xs.copy_(x[:2])
    forward(xs, rand((2, k, n), t, 24, 0.1), [0, 1, 2], False)


def test_empty_contraction_gives_zero():
    out = torch.ones((5, 8), device=DEV)
    nn.grouped_matmul(torch.empty((5, 0), device=DEV), torch.empty((2, 0, 8), device=DEV), torch.tensor([0, 2, 5], dtype=torch.int32, device=DEV), out)
    assert not bool(out.any())
    dw = torch.ones((2, 3, 8), device=DEV)
    nn.grouped_matmul_dw(torch.empty((0, 3), device=DEV), torch.empty((0, 8), device=DEV), torch.tensor([0, 0, 0], dtype=torch.int32, device=DEV), dw)
    assert not bool(dw.any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_gradients_against_differences(dtype):
    # bilinear: f(x + v) - f(x) along g is <v, dx> exactly, up to the rounding of both sides
    t, offsets, k, n = TYPES[dtype], [0, 70, 70, 150], 96, 160
    x, w, g = rand((160, k), t, 25), rand((3, k, n), t, 26, 0.1), rand((160, n), t, 27)
    dx, dw = forward(g, w, offsets, True), backward_w(x, g, offsets, out_dtype=torch.float32)
    unit = {"bf16": 2.0**-8, "f32": 2.0**-24}[dtype]
    v = (2 * x).to(t) - x  # x + v is exact in the type
    y0, y1 = forward(x, w, offsets, False), forward((x + v).to(t), w, offsets, False)
    quotient = ((y1.double() - y0.double()) * g.double()).sum()
    _, m = grouped(x + v, w, offsets)
    _, mx = grouped(g, w, offsets, True)
    tol = ((unit + (k + 16) * 2.0**-23) * 2 * m * g.double().abs()).sum() + ((unit + (n + 16) * 2.0**-23) * mx * v.double().abs()).sum()
    assert abs(float(quotient - (dx.double() * v.double()).sum())) <= float(tol)
    y2 = forward(x, (2 * w.double()).to(t), offsets, False)  # w + w
    _, m = grouped(x, 2 * w, offsets)
    _, mw = grouped_dw(x, g, offsets)
    quotient = ((y2.double() - y0.double()) * g.double()).sum()
    tol = ((unit + (k + 16) * 2.0**-23) * 2 * m * g.double().abs()).sum() + ((96 + 16) * 2.0**-23 * mw * w.double().abs()).sum()
    assert abs(float(quotient - (dw.double() * w.double()).sum())) <= float(tol)


def test_capture_with_offsets_that_change():
    t, k, n = torch.bfloat16, 256, 256
    x, w = rand((300, k), t, 28), rand((3, k, n), t, 29, 0.1)
    off = torch.zeros(4, dtype=torch.int32, device=DEV)
    out = torch.empty((300, n), dtype=t, device=DEV)
    dw = torch.empty((3, k, n), dtype=t, device=DEV)
    ws = space(max(nn.grouped_matmul_workspace(x, w, out), nn.grouped_matmul_dw_workspace(x, out, dw)))
    st = R.Stream()
    torch.cuda.synchronize()
    with R.Graph.capture(st) as g:
        nn.grouped_matmul(x, w, off, out, workspace=ws, stream=st)
        nn.grouped_matmul_dw(x, x, off, dw, workspace=ws, stream=st)
    for offsets in ([0, 100, 200, 300], [0, 0, 299, 300], [0, 0, 0, 0]):
        off.copy_(torch.tensor(offsets, dtype=torch.int32))
        torch.cuda.synchronize()
        g.launch(st)
        st.synchronize()
        e, m = grouped(x, w, offsets)
        close(out, e, slack(m, k), "captured")
        e, m = grouped_dw(x, x, offsets)
        close(dw, e, slack(m, 300), "captured dw")
    g.destroy()
    st.destroy()


@pytest.mark.parametrize("rows,k,n", [(96, 200, 72), (6, 200, 72)])
@pytest.mark.parametrize("wt", [False, True])
def test_f32_holds_over_the_whole_range(rows, k, n, wt):
    # numbers of very different size, down to where the lowest of three planes vanishes, each row and matrix of one size
    offsets = [0, rows // 3, rows // 3, rows]
    scale = torch.tensor([2.0**e for e in (-60, -20, 0, 30, 90)], device=DEV)
    x = rand((rows, k), torch.float32, 30) * scale[torch.arange(rows, device=DEV) % 5][:, None]
    w = rand((3, n, k) if wt else (3, k, n), torch.float32, 31)
    forward(x, w, offsets, wt)


def test_f32_nan_reaches_its_row_alone():
    x, w = rand((64, 96), torch.float32, 32), rand((2, 96, 40), torch.float32, 33)
    x[5, 7] = float("nan")
    for offsets in ([0, 32, 64], [0, 5, 6]):
        y = forward(x, w, offsets, False, check=False)
        bad = torch.isnan(y).any(1)
        assert bool(bad[5]) and int(bad.sum()) == 1 and bool(torch.isnan(y[5]).all())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_a_long_contraction_over_one_expert(dtype):
    t = TYPES[dtype]
    x, dy = rand((5000, 24), t, 34), rand((5000, 40), t, 35)
    backward_w(x, dy, [0, 4990])
    backward_w(x, dy, [0, 10, 4000, 5000])
    forward(rand((3, 9000), t, 36), rand((2, 9000, 40), t, 37, 0.01), [0, 1, 3], False)
    forward(rand((3, 9000), t, 36), rand((2, 40, 9000), t, 37, 0.01), [0, 1, 3], True)
