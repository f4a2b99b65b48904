"""One layer of a graph model, trained in 16 bits and served in 8.

Nodes have a type, types have a learnt row of features, and a node's class is to be told from its own features and
its neighbours':

    x      = table[types] * scale                 trspmm.embed
    h      = A x                                  Plan.spmm (float32)
    y, r   = norm(h + x) * weight                 trspmm.rms_norm
    logits = y W^T

The training step goes back through it: rms_norm_grad, the SpMM again (A is symmetric) and embed_grad.  Serving takes
the norm's output as 8-bit codes and multiplies them by 8-bit weights: rms_norm_i8 and matmul_i8.

    python examples/graph_layer.py [--nodes 4096] [--width 64] [--steps 40]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tr-spmm_zzx_amd"))

import trspmm  # noqa: E402
from trspmm import graphs  # noqa: E402

CLASSES, SCALE, EPS = 16, 8.0, 1e-5


class GraphLayer:
    def __init__(self, nodes: int, width: int, types: int, seed: int = 0):
        g = graphs.erdos_renyi_gcn(nodes=nodes, edges=4 * nodes)
        self.plan = trspmm.Plan.from_format(trspmm.build_format(g.rowptr, g.col, g.val), g.m, g.n)
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.types = torch.randint(types, (g.n,), generator=gen, device="cuda")
        self.table = torch.randn((types, width), generator=gen, device="cuda") * 0.1    # float32 masters
        self.weight = torch.ones(width, device="cuda")
        self.w = torch.randn((CLASSES, width), generator=gen, device="cuda") * 0.05
        self.labels = self.types % CLASSES

    def features(self):
        """Features of the nodes (fp16, the SpMM's operand) and of their neighbourhoods (float32)."""
        x = trspmm.embed(self.table, self.types, SCALE, dtype=torch.float16)
        return x, self.plan.spmm(x)

    def train_step(self, rate: float) -> float:
        x, h = self.features()
        y, r = trspmm.rms_norm(h, self.weight, x, eps=EPS, dtype=torch.float16)
        w16 = self.w.half()
        logits = (y @ w16.t()).float()
        loss = torch.nn.functional.cross_entropy(logits, self.labels)
        # back: the classes, the norm, the graph, the table
        d = torch.softmax(logits, 1)
        d[torch.arange(d.shape[0], device="cuda"), self.labels] -= 1
        d = d.half()                                                  # the rate brings in 1 / nodes
        dw = (d.t() @ y).float()
        dr, dweight = trspmm.rms_norm_grad(d @ w16, r, self.weight, eps=EPS)
        dx = self.plan.spmm(dr).add_(dr)                              # A^T dh + the residual's own
        dtable = trspmm.embed_grad(dx, self.types, self.table.shape[0], SCALE)
        rate /= d.shape[0]
        self.w.sub_(dw, alpha=rate)
        self.weight.sub_(dweight, alpha=rate)
        self.table.sub_(dtable, alpha=rate)
        return loss

    def logits16(self) -> torch.Tensor:
        x, h = self.features()
        y, _ = trspmm.rms_norm(h, self.weight, x, eps=EPS, dtype=torch.float16)
        return (y @ self.w.half().t()).float()

    def serving_weights(self):
        """W in 8 bits with a scale for each class, laid out once."""
        scale = self.w.abs().amax(1) / 127
        return torch.round(self.w / scale[:, None]).to(torch.int8), scale

    def logits8(self, codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        x, h = self.features()
        q, s, _ = trspmm.rms_norm_i8(h, self.weight, x, eps=EPS, r_out=x)
        return trspmm.matmul_i8(q, s, codes, scale, dtype=torch.float32)


def run(nodes: int = 4096, width: int = 64, types: int = 512, steps: int = 40, rate: float = 4.0) -> dict:
    layer = GraphLayer(nodes, width, types)
    losses = torch.stack([layer.train_step(rate) for _ in range(steps)])
    full, served = layer.logits16(), layer.logits8(*layer.serving_weights())
    same = (full.argmax(1) == served.argmax(1)).float().mean()
    right = (served.argmax(1) == layer.labels).float().mean()
    return {"first": float(losses[0]), "last": float(losses[-1]), "same": float(same), "right": float(right),
            "off": float((served - full).norm() / full.norm())}


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("nodes", 4096), ("width", 64), ("types", 512), ("steps", 40)):
        ap.add_argument("--" + name, type=int, default=value)
    got = run(**vars(ap.parse_args()))
    print("loss %(first).3f -> %(last).3f; served in 8 bits: %(right).1f%% right, %(same).1f%% as in 16 bits, logits off by "
          "%(off).2g" % {**got, "right": 100 * got["right"], "same": 100 * got["same"]})
