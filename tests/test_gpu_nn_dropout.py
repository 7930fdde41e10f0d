"""nn.dropout on a B200 against the generator's definition, element by element.

Tolerance: the kept value x * factor has two roundings of F32 (the factor and
the product), the sum with the residual one more, storage one of its type:
|y - e| <= unit * |e| + 4 * 2^-24 * (|x / (1-p)| + |residual|)."""
import pytest
import torch
from nn_reference import U, close, keep

from cudacaml_b200 import backend_cuda as cuda
from cudacaml_b200 import nn
from cudacaml_b200 import runtime as R
from cudacaml_b200.ir import F32, Value

pytestmark = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
DEV = "cuda"


def rand(shape, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def check(x, out, p, seed, offset, base, residual=None):
    k = keep(base, tuple(x.shape), p, seed, offset, x.device)
    v = torch.where(k, x.double() / (1 - p) if p < 1 else torch.zeros_like(x, dtype=torch.float64), torch.zeros((), dtype=torch.float64, device=DEV))
    want = v if residual is None else v + residual.double()
    slack = 4 * U * (v.abs() + (0 if residual is None else residual.double().abs()))
    close(out, want, slack, "dropout")


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("shape", [(1, 1), (1, 7), (3, 5), (16, 1024), (129, 33), (257, 4096), (1, 100003), (5000, 8)])
@pytest.mark.parametrize("p,base,offset", [(0.1, 0, 0), (0.5, 3, 1 << 40), (0.37, (1 << 33) + 2, 17)])
def test_values(dtype, shape, p, base, offset):
    t = TYPES[dtype]
    x, res = rand(shape, t, 1), rand(shape, t, 2)
    seed = 0x123456789ABCDEF
    for r in (None, res):
        out = torch.full_like(x, float("nan"))
        nn.dropout(x, p, seed, out, offset=offset, base=base, residual=r)
        check(x, out, p, seed, offset, base, r)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_p_zero_and_one_and_tiny(dtype):
    x = rand((33, 70), TYPES[dtype], 3)
    out = torch.empty_like(x)
    nn.dropout(x, 0.0, 5, out)
    assert torch.equal(out, x)
    nn.dropout(x, 1.0, 5, out)
    assert not bool(out.any())
    nn.dropout(x, 1.0, 5, out, residual=x)
    assert torch.equal(out, x)
    nn.dropout(x, 2.0**-40, 5, out)  # rounds to no element
    assert torch.equal(out, x)


def test_dropped_places_give_zero_whatever_they_hold():
    shape, p, seed = (64, 515), 0.4, 9
    k = keep(0, shape, p, seed, 0, DEV)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t in TYPES.values():
            x = torch.where(k, torch.ones((), device=DEV), torch.full((), bad, device=DEV)).to(t)
            out = torch.empty_like(x)
            nn.dropout(x, p, seed, out)
            assert bool((out[~k] == 0).all()) and bool(torch.isfinite(out).all())
            x = torch.full(shape, bad, dtype=t, device=DEV)
            nn.dropout(x, p, seed, out)
            assert bool((out[~k] == 0).all()) and not bool(torch.isfinite(out[k]).any())


@pytest.mark.parametrize("dtype", list(TYPES))
def test_strided_rows_in_place_and_slices(dtype):
    t, p, seed = TYPES[dtype], 0.25, 77
    for cols, stride in ((24, 32), (33, 57), (8, 9)):
        big = rand((50, stride), t, 4)
        x = big[:, :cols]
        res = rand((50, stride + 8), t, 5)[:, 8 : 8 + cols]
        outbig = torch.zeros((50, stride + 1), dtype=t, device=DEV)
        out = outbig[:, 1 : 1 + cols]
        nn.dropout(x, p, seed, out, residual=res)
        check(x, out, p, seed, 0, 0, res)
        assert not bool(outbig[:, 0].any()) and not bool(outbig[:, 1 + cols :].any())
        # a slice of rows with its first element's index as base draws the whole's mask
        part = torch.empty((20, cols), dtype=t, device=DEV)
        nn.dropout(x[10:30], p, seed, part, base=10 * cols)
        whole = torch.empty((50, cols), dtype=t, device=DEV)
        nn.dropout(x, p, seed, whole)
        assert torch.equal(part, whole[10:30])
        # in place
        y = x.clone()
        nn.dropout(y, p, seed, y)
        assert torch.equal(y, whole)


def test_unaligned_start():
    big = rand((100001,), torch.bfloat16, 6)
    for shift in (1, 3, 8):
        x = big[shift:]
        out = torch.empty(100001 + 5, dtype=torch.bfloat16, device=DEV)[5 : 5 + x.numel()]
        nn.dropout(x, 0.3, 8, out)
        check(x, out, 0.3, 8, 0, 0)


def test_offsets_past_32_bits():
    stride = (1 << 31) + 24
    buf = torch.empty(stride + 4096, dtype=torch.bfloat16, device=DEV)
    for cols in (4096, 1001):
        x = torch.as_strided(buf, (2, cols), (stride, 1))
        x.copy_(rand((2, cols), torch.bfloat16, 7))
        out = torch.empty((2, cols), dtype=torch.bfloat16, device=DEV)
        nn.dropout(x, 0.2, 3, out)
        check(x, out, 0.2, 3, 0, 0)


def test_more_than_2_to_31_elements():
    n = (1 << 31) + 4100
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    nn.dropout(x, 0.5, 11, x)  # in place: 2 where kept, 0 where dropped
    for first in (0, (1 << 31) - 64, n - 4000):
        part = x[first : first + 4000]
        check(torch.ones_like(part), part, 0.5, 11, 0, first)


def test_gradient_is_the_forwards_mask():
    # the operator is linear in x: <dropout(v), g> = <v, dropout_backward(g)> up to F32 rounding
    v, g = rand((77, 130), torch.float32, 8), rand((77, 130), torch.float32, 9)
    a, b = torch.empty_like(v), torch.empty_like(v)
    nn.dropout(v, 0.3, 21, a, offset=4)
    nn.dropout_backward(g, 0.3, 21, b, offset=4)
    lhs, rhs = (a.double() * g.double()), (v.double() * b.double())
    assert bool(((lhs - rhs).abs() <= 4 * U * lhs.abs()).all())
    # and a difference quotient of it, exact but for rounding: x and x + v
    x, y0, y1 = rand((77, 130), torch.float32, 10), torch.empty_like(v), torch.empty_like(v)
    nn.dropout(x, 0.3, 21, y0, offset=4)
    nn.dropout(x + v, 0.3, 21, y1, offset=4)
    quotient = ((y1.double() - y0.double()) * g.double()).sum()
    slack = (4 * U * (y1.double().abs() + y0.double().abs()) * g.double().abs()).sum()
    assert abs(float(quotient - rhs.sum())) <= float(slack)


def test_another_stream_and_capture():
    x = torch.empty((512, 1024), dtype=torch.bfloat16, device=DEV)
    out = torch.empty_like(x)
    src = rand((512, 1024), torch.bfloat16, 12)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        x.copy_(src)
        nn.dropout(x, 0.1, 2, out, stream=s.cuda_stream)
    s.synchronize()
    check(src, out, 0.1, 2, 0, 0)
    st = R.Stream()
    out.zero_()
    torch.cuda.synchronize()
    with R.Graph.capture(st) as g:
        nn.dropout(x, 0.1, 2, out, stream=st)
    for _ in range(2):
        out.zero_()
        torch.cuda.synchronize()
        g.launch(st)
        st.synchronize()
        check(src, out, 0.1, 2, 0, 0)
    g.destroy()
    st.destroy()


def test_residents_and_arrays():
    import numpy as np

    host = np.random.default_rng(0).standard_normal((6, 40)).astype(np.float32)
    x, out = cuda.upload(Value.of_array(F32, (6, 40), host)), cuda.upload(Value.of_array(F32, (6, 40), np.zeros((6, 40), np.float32)))
    nn.dropout(x, 0.5, 31, out)
    view = nn.Array(x.buf.ptr, "f32", (6, 40))
    R.synchronize()
    got = torch.from_numpy(cuda.download(out).data.reshape(6, 40).copy()).to(DEV)
    check(torch.from_numpy(host).to(DEV), got, 0.5, 31, 0, 0)
    nn.dropout(view, 0.5, 31, view)
    R.synchronize()
    assert np.array_equal(cuda.download(x).data.reshape(-1), got.cpu().numpy().reshape(-1))
    cuda.free_resident(x)
    cuda.free_resident(out)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("base", [(1 << 34) - 21, (1 << 34) - 4000])
def test_counters_whose_high_word_changes_on_the_way(dtype, base):
    x = rand((40, 200), TYPES[dtype], 13)
    out = torch.empty_like(x)
    nn.dropout(x, 0.3, 5, out, base=base, offset=(1 << 33) + 7)
    check(x, out, 0.3, 5, (1 << 33) + 7, base)
