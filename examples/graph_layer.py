"""One layer of a graph model, trained in 16 bits and served in 8 or 4.

Nodes have a type, types have a learnt row of features, and a node's class is to be told from its own features and
its neighbours':

    x      = table[types] * scale                 trspmm.embed
    h      = A x                                  Plan.spmm (float32)
    y, r   = norm(h + x) * weight                 trspmm.rms_norm
    logits = y W^T

The training step goes back through it: rms_norm_grad, the SpMM again (A is symmetric) and embed_grad.  Parameters are updated by plain descent, or by AdamW with its states in 8 bits,
which writes the 16-bit copies of the next step's forward pass as it goes (trspmm.adamw).  Serving takes the norm's output as
8-bit codes and multiplies them by 8-bit weights (rms_norm_i8 and matmul_i8), or both as 4-bit codes with block scales
(rms_norm_mx4 and matmul_mx4, the weights by quant_mx4).

    python examples/graph_layer.py [--nodes 4096] [--width 64] [--steps 40] [--optimiser adamw]
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

    def features(self, table=None):
        """Features of the nodes (fp16, the SpMM's operand) and of their neighbourhoods (float32)."""
        x = trspmm.embed(self.table if table is None else table, self.types, SCALE, dtype=torch.float16)
        return x, self.plan.spmm(x)

    def gradients(self, table=None, w16=None):
        """The loss and the gradients of table, weight and w, summed over the nodes; table and w16: copies to use."""
        x, h = self.features(table)
        y, r = trspmm.rms_norm(h, self.weight, x, eps=EPS, dtype=torch.float16)
        w16 = self.w.half() if w16 is None else w16
        logits = (y @ w16.t()).float()
        loss = torch.nn.functional.cross_entropy(logits, self.labels)
        # back: the classes, the norm, the graph, the table
        d = torch.softmax(logits, 1)
        d[torch.arange(d.shape[0], device="cuda"), self.labels] -= 1
        d = d.half()                                                  # the rate brings in 1 / nodes
        dw = (d.t() @ y).float()
        dr, dweight = trspmm.rms_norm_grad(d @ w16, r, self.weight, eps=EPS)
        dx = self.plan.spmm(dr).add_(dr)                              # A^T dh + the residual's own
        return loss, (trspmm.embed_grad(dx, self.types, self.table.shape[0], SCALE), dweight, dw)

    def train_step(self, rate: float) -> float:
        loss, (dtable, dweight, dw) = self.gradients()
        rate /= self.labels.shape[0]
        self.w.sub_(dw, alpha=rate)
        self.weight.sub_(dweight, alpha=rate)
        self.table.sub_(dtable, alpha=rate)
        return loss

    def start_adamw(self, bits: int = 8):
        self.params = [self.table, self.weight, self.w]
        self.states = [trspmm.adamw_state(p, bits) for p in self.params]
        self.copies = [self.table.half(), None, self.w.half()]
        self.steps = 0

    def adamw_step(self, rate: float) -> float:
        loss, grads = self.gradients(self.copies[0], self.copies[2])
        self.steps += 1
        trspmm.adamw(self.params, grads, self.states, self.steps, lr=rate, weight_decay=[0.0, 0.0, 0.01], copies=self.copies,
                     grad_scale=1 / self.labels.shape[0])
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


    def serving_weights4(self):
        """W as 4-bit codes with a scale for each 32 of a class's weights."""
        return trspmm.quant_mx4(self.w)

    def logits4(self, codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
        x, h = self.features()
        q, s, _ = trspmm.rms_norm_mx4(h, self.weight, x, eps=EPS, r_out=x)
        return trspmm.matmul_mx4(q, s, codes, scale, dtype=torch.float32)


def run(nodes: int = 4096, width: int = 64, types: int = 512, steps: int = 40, rate: float = None,
        optimiser: str = "descent") -> dict:
    layer = GraphLayer(nodes, width, types)
    if optimiser == "adamw":
        layer.start_adamw()
        rate = 0.01 if rate is None else rate
        losses = torch.stack([layer.adamw_step(rate) for _ in range(steps)])
    else:
        rate = 4.0 if rate is None else rate
        losses = torch.stack([layer.train_step(rate) for _ in range(steps)])
    full = layer.logits16()
    got = {"first": float(losses[0]), "last": float(losses[-1])}
    for name, served in (("", layer.logits8(*layer.serving_weights())), ("4", layer.logits4(*layer.serving_weights4()))):
        got["same" + name] = float((full.argmax(1) == served.argmax(1)).float().mean())
        got["right" + name] = float((served.argmax(1) == layer.labels).float().mean())
        got["off" + name] = float((served - full).norm() / full.norm())
    return got


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, value in (("nodes", 4096), ("width", 64), ("types", 512), ("steps", 40)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--optimiser", choices=("descent", "adamw"), default="descent")
    got = run(**vars(ap.parse_args()))
    print("loss %(first).3f -> %(last).3f" % got)
    for bits, name in ((8, ""), (4, "4")):
        print("served in %d bits: %.1f%% right, %.1f%% as in 16 bits, logits off by %.2g"
              % (bits, 100 * got["right" + name], 100 * got["same" + name], got["off" + name]))
