"""The 4-bit operators and AdamW as a layer uses them: examples/graph_layer.py's gradients and steps, and training and serving
captured into one graph.

The example's gradients are held against the formula's in 64 bits with bounds that are carried along: a number stands with a bound of its
error, a product or sum adds what its operands' bounds give and its own rounding.  Half precision rounds by 2^-11 of a value (2^-25 where
it is subnormal), sums of k terms in 32 bits by k 2^-23 of the terms' sizes (to nearest or towards zero)."""
import os
import sys

import pytest
import torch

import trspmm
from conftest import ROOT

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(ROOT, "examples"))
try:
    import graph_layer
finally:
    sys.path.pop(0)

F32, HALF = 2.0 ** -23, 2.0 ** -11


def say(*a):
    print(*a, flush=True)


class Near:
    """A tensor in 64 bits and a bound of the distance to it."""

    def __init__(self, value, off=0.0):
        self.v = value.double()
        self.e = torch.zeros_like(self.v) + off

    def half(self):
        return Near(self.v, self.e + HALF * (self.v.abs() + self.e) + 2.0 ** -25)

    def mm(self, other, terms=None):
        most = (self.v.abs() + self.e) @ (other.v.abs() + other.e)
        off = self.v.abs() @ other.e + self.e @ other.v.abs() + self.e @ other.e
        return Near(self.v @ other.v, off + (terms or self.v.shape[1]) * F32 * most)

    def t(self):
        return Near(self.v.t(), self.e.t())

    def __add__(self, other):
        v = self.v + other.v
        return Near(v, (self.e + other.e) + F32 * (v.abs() + self.e + other.e))

    def __mul__(self, other):
        v = self.v * other.v
        off = self.v.abs() * other.e + self.e * other.v.abs() + self.e * other.e
        return Near(v, off + F32 * (v.abs() + off))

    def mean(self):
        return Near(self.v.mean(1, True), self.e.mean(1, True) + self.v.shape[1] * F32 * (self.v.abs() + self.e).mean(1, True))

    def root(self):
        """1 / sqrt(self + eps): at most 1 / 2 (self + eps - e)^-3/2 e off, and 4 roundings."""
        s = self.v + graph_layer.EPS
        low = (s - self.e).clamp_min(graph_layer.EPS)
        return Near(s.rsqrt(), 0.5 * low ** -1.5 * self.e + 4 * F32 * low.rsqrt())


def expected(layer, table, w16):
    """Gradients of the summed loss in 64 bits, and their bounds."""
    n = layer.labels.shape[0]
    dense = torch.zeros((n, n), dtype=torch.float64)
    graph = graph_layer.graphs.erdos_renyi_gcn(nodes=n, edges=4 * n)
    rows = torch.repeat_interleave(torch.arange(len(graph.rowptr) - 1), torch.as_tensor(graph.rowptr).long().diff())
    dense[rows, torch.as_tensor(graph.col).long()] = torch.as_tensor(graph.val).half().double()
    dense = Near(dense.cuda())
    pick = torch.nn.functional.one_hot(layer.types, table.shape[0]).double()
    weight, w = Near(layer.weight), Near(w16)
    x = Near(table.double()[layer.types] * graph_layer.SCALE).half()      # times 8: exact before it
    r32 = dense.mm(x) + x
    s = (r32 * r32).mean().root()
    y = (r32 * s * weight).half()
    r = r32.half()
    logits = y.mm(w.t()).half()
    p = torch.softmax(logits.v, 1)
    # logits off by at most b move a softmax's p by at most p (exp(2 b) - 1)
    d = Near(p - torch.nn.functional.one_hot(layer.labels, p.shape[1]),
             p * torch.expm1(2 * logits.e.amax(1, True)) + 16 * F32).half()
    dw = d.t().mm(y).half()
    g = d.mm(w).half()
    s = (r * r).mean().root()
    dweight = Near(torch.ones((1, n), device="cuda")).mm(g * r * s)
    gw = g * weight
    inner = (gw * r).mean()
    back = r * s * s * s * inner
    dr = (gw * s + Near(-back.v, back.e)).half()
    dx = dense.t().mm(dr) + dr
    dtable = Near(pick.t()).mm(dx, n)
    return Near(dtable.v * graph_layer.SCALE, dtable.e * graph_layer.SCALE * (1 + F32)), Near(dweight.v[0], dweight.e[0]), dw


def layer_of(nodes=272, width=40, types=20):
    layer = graph_layer.GraphLayer(nodes, width, types)
    layer.weight.add_(0.3 * torch.randn(width, generator=torch.Generator(device="cuda").manual_seed(5), device="cuda"))
    return layer


def test_the_layers_gradients():
    say("layer gradients")
    layer = layer_of()
    _, grads = layer.gradients()
    for name, got, want in zip(("table", "weight", "w"), grads, expected(layer, layer.table, layer.w.half())):
        off = (got.double() - want.v).abs()
        say(name, "off", float(off.norm() / want.v.norm()), "bound", float(want.e.norm() / want.v.norm()))
        assert want.e.norm() < 0.5 * want.v.norm()      # a bound that says something
        assert bool((off <= want.e).all()), name


@pytest.mark.parametrize("bits", [32, 8])
def test_the_layers_steps(bits):
    """Two steps by AdamW are the formula's with the layer's own gradients; the copies are the parameters rounded."""
    say("layer steps", bits)
    layer = layer_of()
    layer.start_adamw(bits)
    scale = 1 / layer.labels.shape[0]
    for step in (1, 2):
        _, grads = layer.gradients(layer.copies[0], layer.copies[2])
        before = [(p.double(), *(t.double() for t in s.values())) for p, s in zip(layer.params, layer.states)]
        layer.adamw_step(0.01)
        for (p, m, v), g, got, decay in zip(before, grads, layer.params, (0.0, 0.0, 0.01)):
            g = g.double() * scale
            m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
            root = (v / (1 - 0.999 ** step)).sqrt() + 1e-8
            want = p * (1 - 0.01 * decay) - 0.01 / (1 - 0.9 ** step) * m / root
            # a dozen roundings of the step (of its terms' sizes: m is a sum), three of the parameter, each at most 2^-23
            size = 0.01 / (1 - 0.9 ** step) * ((m - 0.1 * g).abs() + 0.1 * g.abs()) / root
            assert bool(((got.double() - want).abs() <= 16 * F32 * size + 3 * F32 * want.abs()).all())
        assert torch.equal(layer.copies[0], layer.table.half()) and torch.equal(layer.copies[2], layer.w.half())
        assert layer.copies[1] is None


def test_the_layer_served_in_4_bits():
    say("layer in 4 bits")
    layer = layer_of()
    codes, scale = layer.serving_weights4()
    got = layer.logits4(codes, scale)
    x, h = layer.features()
    q, s, _ = trspmm.rms_norm_mx4(h, layer.weight, x, eps=graph_layer.EPS)
    y, w = (trspmm.dequant_mx4(c, e, 40, torch.float32).double() for c, e in ((q, s), (codes, scale)))
    assert bool(((got.double() - y @ w.t()).abs() <= 64 * F32 * (y.abs() @ w.abs().t())).all())
    # codes are at most a quarter of their value off, or a quarter of the block's scale (half the least step): an eighth of its largest value
    full = layer.w.double()
    top = torch.nn.functional.pad(full.abs(), (0, 24)).view(16, 2, 32).amax(2).repeat_interleave(32, 1)[:, :40]
    assert bool(((w - full).abs() <= torch.maximum(full.abs() / 4, top / 8)).all())


@pytest.mark.parametrize("optimiser", ["descent", "adamw"])
def test_the_example_runs(optimiser):
    say("example", optimiser)
    got = graph_layer.run(nodes=500, width=33, types=40, steps=3, optimiser=optimiser)
    say(got)
    assert all(value == value and abs(value) < 1e3 for value in got.values())


def chain(bits):
    """A layer of 300 numbers to 96: its norm, their gradients, a step of both, the weights laid out again, and served."""
    gen = torch.Generator(device="cuda").manual_seed(bits)
    x, dy, res = (torch.randn((130, 300), generator=gen, device="cuda").half() for _ in range(3))
    weight = 1 + 0.1 * torch.randn(300, generator=gen, device="cuda")
    w = torch.randn((96, 300), generator=gen, device="cuda") / 8
    w_grad = torch.randn((96, 300), generator=gen, device="cuda").half()
    bias = torch.randn(96, generator=gen, device="cuda")
    step = torch.ones((), dtype=torch.int64, device="cuda")
    states = [trspmm.adamw_state(weight, 32), trspmm.adamw_state(w, bits)]
    w16 = w.half()
    codes, scale = trspmm.quant_mx4(w16)
    out = torch.empty((130, 96), dtype=torch.bfloat16, device="cuda")

    def run():
        y, r = trspmm.rms_norm(x, weight, res, eps=1e-5)
        dr, dweight = trspmm.rms_norm_grad(dy, r, weight, eps=1e-5)
        trspmm.adamw([weight, w], [dweight, w_grad], states, step, lr=0.01, weight_decay=[0.0, 0.1], copies=[None, w16],
                     grad_scale=0.5, seed=9)
        trspmm.quant_mx4(w16, out=codes, scale=scale)
        q, s, _ = trspmm.rms_norm_mx4(x, weight, res, 1e-5)
        trspmm.matmul_mx4(q, s, codes, scale, bias, out=out)
        step.add_(1)
        return y, dr
    kept = [weight, w, w16, codes, scale.view(torch.uint8), out, step]
    kept += [t if t.dtype == torch.float32 else t.view(torch.uint8) for state in states for t in state if t is not None]
    return run, kept, (x, dy)


@pytest.mark.parametrize("bits", [32, 8])
def test_training_and_serving_in_one_graph(bits):
    """Replays of a captured step change parameters, states, copies and codes as eager steps of the same numbers do."""
    say("one graph", bits)
    run, kept, inputs = chain(bits)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    eager, wanted, others = chain(bits)
    for turn in range(5):
        graph.replay()
        want = eager()
        torch.cuda.synchronize()
        assert int(kept[6]) == turn + 2
        for a, b in zip([*kept, *held], [*wanted, *want]):
            assert torch.equal(a, b), turn
        for a, b in zip(inputs, others):
            a.mul_(-0.5)
            b.mul_(-0.5)


def test_two_streams_at_once():
    """Two chains of their own on two streams give what they give alone."""
    say("two streams")
    alone = []
    for bits in (32, 8):
        run, kept, _ = chain(bits)
        for _ in range(4):
            run()
        alone.append(kept)
    both = [chain(bits) for bits in (32, 8)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in both]
    for _ in range(4):
        for stream, (run, _, _) in zip(streams, both):
            with torch.cuda.stream(stream):
                run()
    torch.cuda.synchronize()
    for want, (_, kept, _) in zip(alone, both):
        assert all(torch.equal(a, b) for a, b in zip(want, kept))
