"""The expert block's update on a B200: rates that change from step to step, and
steps whose device checks failed."""
import numpy as np
import pytest

from cudacaml_b200 import backend_cuda as cuda
from cudacaml_b200 import runtime as R
from cudacaml_b200.expert_block import ExpertBlock

pytestmark = pytest.mark.gpu


def filled(tokens, dim, hidden, offsets, seed=3):
    block = ExpertBlock(tokens, dim, hidden, len(offsets) - 1, p=0.1, seed=5)
    r = np.random.default_rng(seed)
    for k in ("x", "target") + ExpertBlock.WEIGHTS:
        block.put(k, 0.3 * r.standard_normal(block.shapes[k]))
    block.put("offsets", offsets)
    return block


def step(block, rate):
    block.forward()
    block.backward()
    block.update(rate)


def test_a_schedule_of_rates_compiles_nothing(monkeypatch):
    block = filled(48, 32, 40, [0, 20, 48])
    try:
        def refuse(*a, **k):
            raise AssertionError("compiled in a training step")

        monkeypatch.setattr(cuda, "compile_on", refuse)
        held = len(block.graphs)
        for rate in (0.5, 0.25, 0.125, 0.5):
            before = {k: block.get(k).astype(np.float64) for k in ExpertBlock.WEIGHTS}
            step(block, rate)
            for k, was in before.items():
                moved = was - rate * block.get("d" + k).astype(np.float64)
                assert np.all(np.abs(block.get(k) - moved) <= 2.0**-22 * (np.abs(moved) + np.abs(was)) + 1e-30), k
        assert len(block.graphs) == held
    finally:
        block.release()


def test_a_failed_step_is_reported_once_and_moves_nothing():
    block = filled(48, 32, 40, [0, 20, 48])
    try:
        step(block, 0.5)
        block.loss()
        before = {k: block.get(k) for k in ExpertBlock.WEIGHTS}
        block.put("offsets", [0, 20, 99])
        step(block, 0.5)
        block.put("offsets", [0, 20, 48])
        step(block, 0.5)  # not reported yet
        for k, was in before.items():
            assert np.array_equal(block.get(k), was), k
        with pytest.raises(R.CcbError, match="error word 64"):
            block.loss()
        block.forward()
        first = block.loss()
        block.backward()
        block.update(0.25)
        for k, was in before.items():
            assert not np.array_equal(block.get(k), was), k
        for _ in range(20):
            step(block, 0.25)
        block.forward()
        assert block.loss() < first
    finally:
        block.release()
