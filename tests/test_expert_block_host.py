"""The graphs of the expert block's update, on the oracle."""
import numpy as np

from cudacaml_b200 import backend_cuda as B
from cudacaml_b200 import expert_block as E
from cudacaml_b200.ir import F32, I32, Value
from oracle import interp


def values(shape, seed):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def test_one_graph_takes_every_rate():
    shape = (3, 5, 7)
    g = E.descent(shape)
    assert B.lower_info(g)["launches"] == 1
    c = interp.compile(g)
    p, d = values(shape, 1), values(shape, 2)
    for rate in (0.5, 1e-3, 0.0):
        ok = ("err", Value.of_array(I32, (), np.array([0], np.int32)))
        ins = [("p", Value.of_array(F32, shape, p)), ("g", Value.of_array(F32, shape, d)), ("rate", Value.of_array(F32, (), np.array([rate], np.float32))), ok]
        q = dict(interp.run(c, ins))["q"].data.reshape(shape)
        assert np.array_equal(q, p - np.float32(rate) * d)
        built_in = dict(interp.run(interp.compile(E.descent(shape, rate)), ins[:2] + [ok]))["q"].data.reshape(shape)
        assert np.array_equal(q, built_in)


def test_a_raised_error_word_keeps_the_parameters():
    shape = (6, 11)
    c = interp.compile(E.descent(shape))
    p, d = values(shape, 3), values(shape, 4)
    d[2, 3], d[5, 0] = np.nan, np.inf
    for err in (16, 64, 80, -1):
        ins = [("p", Value.of_array(F32, shape, p)), ("g", Value.of_array(F32, shape, d)), ("rate", Value.of_array(F32, (), np.array([0.5], np.float32))),
               ("err", Value.of_array(I32, (), np.array([err], np.int32)))]
        assert np.array_equal(dict(interp.run(c, ins))["q"].data.reshape(shape), p)
