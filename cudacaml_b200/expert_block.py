"""A residual block with experts, trained on one device: the operators of ``nn``
beside compiled graphs, on one stream.

``ExpertBlock`` holds f32 parameters, activations and gradients of::

    h   = norm(x) * w_in
    z_e = h_e @ up[e];  a = dropout(tanh_like(z));  b_e = a_e @ down[e]
    y   = x + scale * dropout(sigmoid(gate) * norm(b) * w_post)
    out = norm(y) * w_out;  loss = mean((out - target)^2)

for tokens that arrive grouped by expert (rows ``offsets[e] .. offsets[e+1]``
of x are expert e's; the offsets stay on the device). Norms, products and masks
are ``nn`` calls; the activation, its derivative, the loss and the update are
graphs, built with ``dsl`` and ``grad`` like any other. Nothing synchronises
but ``loss`` and the accessors.
"""
from __future__ import annotations

import numpy as np

from . import backend_cuda as cuda
from . import dsl as D
from . import examples as X
from . import grad as Grad
from . import nn
from . import runtime as R
from .ir import F32, I32, Graph, numel


def activation(shape) -> Graph:
    z = D.param("z", F32, shape)
    return Graph("act", [("a", D.map(X.tanh_like, z))])


def activation_grad(shape) -> Graph:
    """z, da -> da * tanh_like'(z), as the gradient of sum(tanh_like(z) * da)."""
    z, da = D.param("z", F32, shape), D.param("da", F32, shape)
    g = Graph("actg", [("s", D.reduce(D.add, D.const(F32, 0.0), D.map2(D.mul, D.map(X.tanh_like, z), da)))])
    return Graph("actg", [o for o in Grad.grad(g, "s", ["z"]).outputs if o[0] == Grad.grad_name("s", "z")])


def squared_error(shape) -> Graph:
    """loss = mean((out - target)^2) and its gradient by ``out``."""
    out, target = D.param("out", F32, shape), D.param("target", F32, shape)
    d = D.map2(D.sub, out, target)
    scale = 1.0 / numel(shape)
    loss = D.reduce(D.add, D.const(F32, 0.0), D.map(lambda e: D.mul(D.mul(e, e), D.const(F32, scale)), d))
    return Grad.grad(Graph("mse", [("loss", loss)]), "loss", ["out"])


def descent(shape, rate=None) -> Graph:
    """q = p - rate * g, or p where the scalar parameter ``err`` is not 0 (whatever g
    holds); the rate is the scalar parameter ``rate``, or a number built into the graph."""
    p, g = D.param("p", F32, shape), D.param("g", F32, shape)
    r = D.broadcast(shape, D.scalar("rate", F32)) if rate is None else D.full(F32, shape, rate)
    step = D.map2(lambda e, s: D.select(D.eq(e, D.const(I32, 0)), s, D.const(F32, 0.0)), D.broadcast(shape, D.scalar("err", I32)), D.map2(D.mul, r, g))
    return Graph("sgd", [("q", D.map2(D.sub, p, step))])


class ExpertBlock:
    WEIGHTS = ("w_in", "up", "down", "w_post", "gate", "w_out")

    def __init__(self, tokens: int, dim: int, hidden: int, experts: int, *, device: int = 0, scale: float = 0.5, p: float = 0.1, seed: int = 1):
        self.tokens, self.scale, self.p, self.seed, self.device, self.step_no = tokens, scale, p, seed, device, 0
        act, wide = (tokens, dim), (tokens, hidden)
        self.shapes = {"x": act, "target": act, "h": act, "z": wide, "a": wide, "b": act, "y": act, "out": act, "loss": (1,),
                       "w_in": (dim,), "w_post": (dim,), "w_out": (dim,), "gate": (dim,), "up": (experts, dim, hidden), "down": (experts, hidden, dim)}
        self.shapes.update({"d" + n: self.shapes[n] for n in ("out", "b", "a", "z", "h", "x", "y") + self.WEIGHTS})
        with R.with_device(device):
            self.stream = R.Stream()
            self.buf = {n: R.Buffer(4 * numel(s)) for n, s in self.shapes.items()}
            self.buf.update({n + "'": R.Buffer(4 * numel(self.shapes[n])) for n in self.WEIGHTS})  # the update writes beside
            self.buf["offsets"], self.buf["err"], self.buf["rate"] = R.Buffer(4 * (experts + 1)), R.Buffer(4), R.Buffer(4)
            self.offsets = nn.Array(self.buf["offsets"].ptr, "i32", (experts + 1,))
            R.check(R.lib().ccb_memset_d8(self.buf["err"].ptr, 0, 4, self.stream.h))
            need = [nn.block_norm_backward_workspace(tokens, dim)]
            for x, w, o, t in (("h", "up", "z", False), ("a", "down", "b", False), ("db", "down", "da", True), ("dz", "up", "dh", True)):
                need.append(nn.grouped_matmul_workspace(self[x], self[w], self[o], transpose_w=t))
            need.append(nn.grouped_matmul_dw_workspace(self["a"], self["db"], self["ddown"]))
            need.append(nn.grouped_matmul_dw_workspace(self["h"], self["dz"], self["dup"]))
            self.space = R.Buffer(max(need))
        self.graphs = {"act": cuda.compile_on(device, activation(wide)), "act_grad": cuda.compile_on(device, activation_grad(wide)),
                       "loss": cuda.compile_on(device, squared_error(act))}
        self.graphs.update({s: cuda.compile_on(device, descent(s)) for s in {self.shapes[n] for n in self.WEIGHTS}})
        self.rate = None  # the one on the device

    def __getitem__(self, name) -> nn.Array:
        return nn.Array(self.buf[name].ptr, "f32", self.shapes[name])

    def put(self, name, value) -> None:
        """Upload an input, a parameter, or "offsets" (ascending, experts + 1)."""
        with R.with_device(self.device):
            self.stream.synchronize()
            self.buf[name].upload(np.asarray(value, np.int32 if name == "offsets" else np.float32))

    def get(self, name):
        out = np.empty(self.shapes[name], np.float32)
        with R.with_device(self.device):
            self.stream.synchronize()
            self.buf[name].download(out)
        return out

    def _graph(self, which, ins, outs):
        c = self.graphs[which]
        cuda.run_device_ptrs(c, [self.buf[ins[n]].ptr for n, _, _ in c.params], [self.buf[outs[n]].ptr for n, _, _ in c.outputs], self.stream.h)

    def _join(self):
        return dict(branch=self["b"], post_weight=self["w_post"], gate=self["gate"], gate_act="sigmoid", scale=self.scale, p=self.p, seed=self.seed,
                    offset=2 * self.step_no + 1, pre_weight=self["w_out"], stream=self.stream)

    def forward(self) -> None:
        s, kw = self.stream, dict(workspace=self.space, err=self.buf["err"], stream=self.stream)
        with R.with_device(self.device):
            nn.block_norm(self["x"], h=self["h"], pre_weight=self["w_in"], stream=s)
            nn.grouped_matmul(self["h"], self["up"], self.offsets, self["z"], **kw)
            self._graph("act", {"z": "z"}, {"a": "a"})
            nn.dropout(self["a"], self.p, self.seed, self["a"], offset=2 * self.step_no, stream=s)
            nn.grouped_matmul(self["a"], self["down"], self.offsets, self["b"], **kw)
            nn.block_norm(self["x"], self["y"], self["out"], **self._join())
            self._graph("loss", {"out": "out", "target": "target"}, {"loss": "loss", Grad.grad_name("loss", "out"): "dout"})

    def backward(self) -> None:
        s, kw = self.stream, dict(workspace=self.space, err=self.buf["err"], stream=self.stream)
        with R.with_device(self.device):
            nn.block_norm_backward(self["y"], dh=self["dout"], dx=self["dy"], dbranch=self["db"], dgate=self["dgate"], dpre_weight=self["dw_out"],
                                   dpost_weight=self["dw_post"], workspace=self.space, **self._join())
            nn.grouped_matmul_dw(self["a"], self["db"], self.offsets, self["ddown"], **kw)
            nn.grouped_matmul(self["db"], self["down"], self.offsets, self["da"], transpose_w=True, **kw)
            nn.dropout_backward(self["da"], self.p, self.seed, self["da"], offset=2 * self.step_no, stream=s)
            self._graph("act_grad", {"z": "z", "da": "da"}, {Grad.grad_name("s", "z"): "dz"})
            nn.grouped_matmul_dw(self["h"], self["dz"], self.offsets, self["dup"], **kw)
            nn.grouped_matmul(self["dz"], self["up"], self.offsets, self["dh"], transpose_w=True, **kw)
            nn.block_norm_backward(self["x"], dy=self["dy"], dh=self["dh"], dx=self["dx"], dpre_weight=self["dw_in"], pre_weight=self["w_in"],
                                   workspace=self.space, stream=s)

    def update(self, rate: float) -> None:
        """One step of gradient descent on every parameter, and the next step's masks. While a device check of the
        products has failed and ``loss`` has not reported it, the parameters stay as they are."""
        with R.with_device(self.device):
            if rate != self.rate:
                self.buf["rate"].upload(np.array([rate], np.float32), self.stream.h)
                self.rate = rate
            for n in self.WEIGHTS:
                self._graph(self.shapes[n], {"p": n, "g": "d" + n, "rate": "rate", "err": "err"}, {"q": n + "'"})
                self.buf[n], self.buf[n + "'"] = self.buf[n + "'"], self.buf[n]
        self.step_no += 1

    def loss(self) -> float:
        """The last forward pass's loss; raises if a device check of the products has failed since the last call, once."""
        err = np.empty(1, np.int32)
        with R.with_device(self.device):
            self.stream.synchronize()
            self.buf["err"].download(err)
            if err[0]:
                R.check(R.lib().ccb_memset_d8(self.buf["err"].ptr, 0, 4, self.stream.h))
        if err[0]:
            raise R.CcbError(6, f"ExpertBlock: error word {int(err[0])} (64: offsets out of order or range, 16: a wait ran out)")
        return float(self.get("loss")[0])

    def release(self) -> None:
        with R.with_device(self.device):
            self.stream.synchronize()
            for c in self.graphs.values():
                cuda.release(c)
            for b in self.buf.values():
                b.free()
            self.space.free()
            self.stream.destroy()
