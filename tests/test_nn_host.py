"""cudacaml_b200.nn without a GPU: the argument blocks against the header, the
refusals (each raised before anything is issued), and the plain generator of
the GPU tests against the framework's own on the oracle."""
import os
import re
import struct
import subprocess

import numpy as np
import pytest

from cudacaml_b200 import dsl as D
from cudacaml_b200 import nn
from cudacaml_b200 import rng as Rng
from cudacaml_b200 import runtime as R
from cudacaml_b200.ir import I32, Graph, Value
from oracle import interp

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def A(*shape, dtype="f32", ptr=1 << 20, strides=None):
    return nn.Array(ptr, dtype, shape, strides)


BLOCKS = {"ccb_nn_dropout_t": nn._DROPOUT, "ccb_nn_block_norm_t": nn._NORM, "ccb_nn_block_norm_backward_t": nn._NORM_BACK,
          "ccb_nn_grouped_matmul_t": nn._GROUPED, "ccb_nn_grouped_matmul_dw_t": nn._GROUPED_DW}


def test_argument_blocks_have_the_headers_layout(tmp_path):
    src = tmp_path / "sizes.c"
    src.write_text('#include "ccb.h"\n#include <stdio.h>\nint main(void){%s return 0;}\n' %
                   "".join('printf("%%zu\\n", sizeof(%s));' % n for n in BLOCKS))
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    sizes = [int(v) for v in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [b.size for b in BLOCKS.values()]
    header = open(os.path.join(ROOT, "include", "ccb.h")).read()
    kinds = {"*": "P", "long long": "q", "unsigned long long": "Q", "double": "d", "int": "i"}
    for name, block in BLOCKS.items():
        body = re.search(r"typedef struct \{([^}]*)\} " + name, header).group(1)
        letters = ""
        for field in filter(None, (f.strip() for f in body.split(";"))):
            n = field.count(",") + 1
            if "*" in field:
                letters += "P" * n
            else:
                letters += next(v for k, v in sorted(kinds.items(), key=lambda kv: -len(kv[0])) if field.startswith(k)) * n
        want = "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([PqQdi])", block.format.replace("0P", "")))
        assert letters == want, name


def test_plain_generator_is_the_frameworks_philox():
    from nn_reference import words

    seed = 20240607
    g = Graph("w", [("w", Rng.u32(D.scalar("seed", I32), (64,)))])
    got = interp.run(interp.compile(g), [("seed", Value.of_array(I32, (), np.array([seed], np.int32)))])[0][1].data
    # word 0 of the block with counter (q, 0, 0, 0) is Rng's element q
    assert np.array_equal(words(0, 256, seed, 0)[::4].astype(np.uint32), got.view(np.uint32))


def refused(match, f, *a, **k):
    with pytest.raises(ValueError, match=match):
        f(*a, **k)


def test_dropout_refusals():
    x = A(4, 8)
    refused("outside \\[0, 1\\]", nn.dropout, x, 1.5, 1, x)
    refused("outside \\[0, 1\\]", nn.dropout, x, float("nan"), 1, x)
    refused("shape", nn.dropout, x, 0.1, 1, A(8, 4))
    refused("element type", nn.dropout, x, 0.1, 1, A(4, 8, dtype="bf16"))
    refused("element type", nn.dropout, A(4, 8, dtype="f64"), 0.1, 1, x)
    refused("i32", nn.dropout, A(4, 8, dtype="i32"), 0.1, 1, A(4, 8, dtype="i32"))
    refused("residual", nn.dropout, x, 0.1, 1, x, residual=A(4, 9))
    refused("seed", nn.dropout, x, 0.1, -1, x)
    refused("2\\^64", nn.dropout, x, 0.1, 1, x, offset=1 << 64)
    refused("passes 2\\^64", nn.dropout, x, 0.1, 1, x, base=(1 << 64) - 4)
    refused("along its rows", nn.dropout, A(4, 8, strides=(1, 4)), 0.1, 1, x)
    refused("shorter than a row", nn.dropout, A(4, 8, strides=(7, 1)), 0.1, 1, x)
    refused("not dense", nn.dropout, A(2, 2, 8, strides=(64, 8, 1)), 0.1, 1, x)
    refused("null pointer", nn.dropout, A(4, 8, ptr=0), 0.1, 1, x)
    refused("aligned", nn.dropout, A(4, 8, ptr=(1 << 20) + 2), 0.1, 1, x)
    refused("device memory", nn.dropout, np.zeros((4, 8), np.float32), 0.1, 1, x)


def test_block_norm_refusals():
    x, h = A(4, 8), A(4, 8)
    refused("kind", nn.block_norm, x, h=h, kind="batch")
    refused("gate_act", nn.block_norm, x, x, h, branch=x, gate=x, gate_act="relu")
    refused("eps", nn.block_norm, x, h=h, eps=-1.0)
    refused("scale", nn.block_norm, x, x, h, branch=x, scale=float("inf"))
    refused("p = ", nn.block_norm, x, x, h, branch=x, p=-0.1)
    refused("without a branch", nn.block_norm, x, x, h)
    refused("without a branch", nn.block_norm, x, h=h, post_weight=A(8))
    refused("need post_norm", nn.block_norm, x, x, h, branch=x, post_norm=False, post_weight=A(8))
    refused("need h", nn.block_norm, x, x, branch=x, pre_weight=A(8))
    refused("neither y nor h", nn.block_norm, x, branch=x)
    refused("elements, expected 8", nn.block_norm, x, h=h, pre_weight=A(7))
    refused("different element types", nn.block_norm, x, h=h, pre_weight=A(8), pre_bias=A(8, dtype="bf16"))
    refused("x has neither", nn.block_norm, A(4, 8, dtype="bf16"), h=A(4, 8, dtype="f16"))
    refused("gate has neither", nn.block_norm, x, x, h, branch=x, gate=A(4, 8, dtype="bf16"))
    refused("shape", nn.block_norm, x, x, h, branch=x, gate=A(3, 8))
    refused("overlap", nn.block_norm, x, x, h, branch=x, gate=A(4, 8, strides=(0, 1)))
    refused("null pointer", nn.block_norm, A(4, 8, ptr=0), h=h)


def test_block_norm_backward_refusals():
    y, v = A(4, 8), A(8)
    need = nn.block_norm_backward_workspace(4, 8)
    assert need > 0
    back = nn.block_norm_backward
    refused("workspace", back, y, dh=y, dx=y, dpre_weight=v)
    refused("workspace", back, y, dh=y, dx=y, dpre_weight=v, workspace=A(need // 4 - 1))
    refused("workspace", back, y, dh=y, dx=y, dpre_weight=v, workspace=A(need // 4, ptr=(1 << 20) + 4))
    refused("neither dy nor dh", back, y, dx=y)
    refused("need dh", back, y, dy=y, dpre_weight=v, workspace=A(need))
    refused("dgate without a gate", back, y, dy=y, branch=y, dgate=y)
    refused("element type", back, y, dy=y, branch=y, gate=v, dgate=A(8, dtype="bf16"))
    refused("without a branch", back, y, dy=y, dbranch=y)
    refused("need post_norm", back, y, dy=y, branch=y, post_norm=False, dpost_weight=v, workspace=A(need))
    refused("element type", back, y, dh=y, dpre_weight=A(8, dtype="bf16"), workspace=A(need))
    refused("dy has shape", back, y, dy=A(4, 9))
    refused("rows", nn.block_norm_backward_workspace, -1, 8)


def test_grouped_refusals():
    x, w, off, out = A(6, 8), A(3, 8, 5), A(4, dtype="i32"), A(6, 5)
    gm = nn.grouped_matmul
    refused("columns and each matrix", gm, x, A(3, 7, 5), off, out)
    refused("transposed", gm, x, w, off, out, transpose_w=True)
    refused("offsets has shape", gm, x, w, A(3, dtype="i32"), out)
    refused("offsets has element type", gm, x, w, A(4), out)
    refused("shape", gm, x, w, off, A(6, 6))
    refused("element type", gm, x, A(3, 8, 5, dtype="bf16"), off, out)
    refused("rank 2", gm, x, A(8, 5), off, out)
    refused("experts must be", gm, x, A(1025, 8, 5), A(1026, dtype="i32"), out)
    refused("experts must be", gm, x, A(0, 8, 5), A(1, dtype="i32"), out)
    refused("w's stride", gm, x, A(3, 8, 5, strides=(39, 5, 1)), off, out)
    refused("null pointer", gm, x, w, A(4, dtype="i32", ptr=0), out)
    refused("err", gm, x, w, off, out, err=A(1))
    refused("aligned to 4", gm, x, w, off, out, err=(1 << 20) + 2)
    dw = nn.grouped_matmul_dw
    dy, o = A(6, 5), A(3, 8, 5)
    refused("rows and dy", dw, x, A(7, 5), off, o)
    refused("matrix of out", dw, x, dy, off, A(3, 5, 8))
    refused("neither x's", dw, x, dy, off, A(3, 8, 5, dtype="bf16"))
    refused("offsets has shape", dw, x, dy, A(5, dtype="i32"), o)
    assert nn.grouped_matmul_workspace(x, w, out) >= 0 and nn.grouped_matmul_dw_workspace(x, dy, o) >= 0


@pytest.mark.skipif(R.available(), reason="needs a machine without a GPU")
def test_without_a_device_a_valid_call_says_so():
    with pytest.raises(R.CcbError) as e:
        nn.dropout(A(4, 8), 0.1, 1, A(4, 8))
    assert e.value.code == 2


def test_empty_tensors_need_no_device():
    nn.dropout(A(0, 8, ptr=0), 0.1, 1, A(0, 8, ptr=0))
    nn.block_norm(A(0, 8), h=A(0, 8))
    nn.grouped_matmul(A(0, 8), A(3, 8, 5), A(4, dtype="i32"), A(0, 5))
    nn.grouped_matmul_dw(A(6, 0), A(6, 5), A(4, dtype="i32"), A(3, 0, 5))
    assert struct.calcsize("P") == 8


def test_expert_block_graphs_lower_to_one_launch_each():
    from cudacaml_b200 import backend_cuda as B
    from cudacaml_b200 import expert_block as E

    for g in (E.activation((24, 40)), E.activation_grad((24, 40)), E.squared_error((24, 16)), E.descent((3, 16, 40), 0.1)):
        assert B.lower_info(g)["launches"] == 1
