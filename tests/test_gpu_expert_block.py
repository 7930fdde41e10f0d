"""The expert block's training step on a B200: its loss and every gradient
against automatic differentiation in 64 bits with the same masks, and a loss
that descends."""
import numpy as np
import pytest
import torch
from nn_reference import keep

from cudacaml_b200 import runtime as R
from cudacaml_b200.expert_block import ExpertBlock

pytestmark = pytest.mark.gpu


def norm(v, eps=1e-6):
    return v / torch.sqrt((v * v).mean(1, keepdim=True) + eps)


def reference(v, offsets, scale, p, seed, step):
    """(loss, gradients) by torch's autograd in 64 bits."""
    t = {k: torch.from_numpy(a).double().cuda().requires_grad_(k != "target") for k, a in v.items()}
    shape, wide = v["x"].shape, (v["x"].shape[0], v["up"].shape[2])
    m1 = keep(0, wide, p, seed, 2 * step, "cuda").double() / (1 - p)
    m2 = keep(0, shape, p, seed, 2 * step + 1, "cuda").double() / (1 - p)
    h = norm(t["x"]) * t["w_in"]
    cut = list(zip(offsets[:-1], offsets[1:]))
    z = torch.cat([h[a:b] @ t["up"][e] for e, (a, b) in enumerate(cut)])
    a = torch.tanh(z) * m1
    b = torch.cat([a[i:j] @ t["down"][e] for e, (i, j) in enumerate(cut)])
    y = t["x"] + scale * m2 * torch.sigmoid(t["gate"]) * norm(b) * t["w_post"]
    loss = ((norm(y) * t["w_out"] - t["target"]) ** 2).mean()
    loss.backward()
    return float(loss.detach()), {k: x.grad for k, x in t.items() if x.grad is not None}


@pytest.mark.parametrize("tokens,dim,hidden,offsets", [(96, 64, 128, [0, 30, 30, 96]), (131, 72, 40, [0, 1, 64, 100, 131]), (520, 256, 512, [0, 100, 260, 520])])
def test_step_against_autograd(tokens, dim, hidden, offsets):
    e = len(offsets) - 1
    r = np.random.default_rng(5)
    g = lambda *s, k=1.0, m=0.0: (m + k * r.standard_normal(s)).astype(np.float32)  # noqa: E731
    v = {"x": g(tokens, dim), "target": g(tokens, dim), "w_in": g(dim, k=0.2, m=1.0), "w_post": g(dim, k=0.2, m=1.0), "w_out": g(dim, k=0.2, m=1.0),
         "gate": g(dim), "up": g(e, dim, hidden, k=dim**-0.5), "down": g(e, hidden, dim, k=hidden**-0.5)}
    block = ExpertBlock(tokens, dim, hidden, e, p=0.2, seed=77)
    try:
        for k, a in v.items():
            block.put(k, a)
        block.put("offsets", offsets)
        losses = []
        for step in range(3):
            block.forward()
            block.backward()
            losses.append(block.loss())
            want, grads = reference(v, offsets, block.scale, block.p, block.seed, step)
            # a chain of five norms and products in f32: some hundred roundings of each value's size
            assert abs(losses[-1] - want) <= 1e-5 * abs(want)
            for k in ("x",) + ExpertBlock.WEIGHTS:
                got, e64 = torch.from_numpy(block.get("d" + k)).double().cuda(), grads[k]
                assert float((got - e64).norm()) <= 2e-5 * float(e64.norm()), k
            block.update(0.5)
            for k in ExpertBlock.WEIGHTS:
                moved = v[k].astype(np.float64) - 0.5 * block.get("d" + k).astype(np.float64)
                v[k] = block.get(k)
                assert np.all(np.abs(v[k] - moved) <= 2.0**-22 * (np.abs(moved) + np.abs(v[k])) + 1e-30), k
        for _ in range(10):
            block.forward()
            block.backward()
            block.update(0.5)
        block.forward()
        assert block.loss() < losses[0]
    finally:
        block.release()


def test_offsets_out_of_range_are_reported():
    block = ExpertBlock(16, 32, 32, 2)
    try:
        for k in ("x", "target", "w_in", "w_post", "w_out", "gate", "up", "down"):
            block.put(k, np.ones(block.shapes[k], np.float32))
        block.put("offsets", [0, 8, 99])
        block.forward()
        with pytest.raises(R.CcbError, match="error word 64"):
            block.loss()
    finally:
        block.release()
