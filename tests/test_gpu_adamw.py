"""trspmm.adamw against its formula.

m and v are single products and sums, each rounded to 32 bits: numpy's float32 gives the same bits, and with them the
8-bit codes, whose rounding bits are a function of seed, step and index.  The parameter is compared with the formula in 64 bits
from those m and v: its change is a chain of at most 12 roundings (the step's factors among them) of 2^-23 or better."""
import math

import numpy as np
import pytest
import torch

import trspmm
from trspmm import _native as nat

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
ROUND = {t: torch.finfo(t).eps / 2 for t in TYPES}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)
MASK = 0xFFFFFFFF


def say(*a):
    print(*a, flush=True)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rand(shape, dtype, seed, std=1.0):
    return (torch.randn(shape, generator=gen(seed), device="cuda") * std).to(dtype)


def words(n, seed, step):
    """The rounding bits of n elements, in Python's integers' arithmetic."""
    key = (seed * 0x6A09E667 + step * 0xB7E15163) & MASK
    key = ((key ^ key >> 16) * 0xBB67AE85) & MASK
    x = (np.uint64(key) + np.arange(n, dtype=np.uint64) * np.uint64(0x9E3779B9)) & np.uint64(MASK)
    x = ((x ^ x >> np.uint64(15)) * np.uint64(0xBB67AE85)) & np.uint64(MASK)
    return x ^ x >> np.uint64(16)


E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()


def decoded(codes, scale):
    """float32: an 8-bit value times a power of two is one."""
    unit = np.ldexp(1.0, scale.astype(np.int64) - 127).repeat(32)[:codes.size]
    return (E4M3[codes] * unit).astype(np.float32)


def encoded(x, chance, floor):
    """(codes, scales) of float32 x; chance: of 2^16, for each element."""
    n = x.size
    full = np.zeros((n + 31) // 32 * 32, np.float64)
    full[:n] = x
    fine = np.isfinite(full)
    peak = np.where(fine, np.abs(full), 0.0).reshape(-1, 32).max(1)
    e = np.where(peak > 0, np.frexp(peak)[1] - 1, -1000)
    byte = np.maximum(e + 127 - 7, 1)
    t = np.where(fine, np.abs(full), 0.0).reshape(-1, 32) / np.ldexp(1.0, byte - 127)[:, None]
    t = t.reshape(-1)[:n]
    gap = np.ldexp(1.0, np.maximum(np.frexp(t)[1] - 1, -6) - 3)
    up = np.floor(t / gap + (16.0 * chance + 8) / 2 ** 20) * gap
    if floor:
        up = np.where(x > 0, np.maximum(up, 2.0 ** -9), up)
    size = np.searchsorted(E4M3[:127], up)
    assert np.array_equal(E4M3[size], up)
    code = np.where(fine[:n], size, 127) | (np.signbit(x).astype(np.int64) << 7 if not floor else 0)
    return code.astype(np.uint8), byte.astype(np.uint8)


class Case:
    """One tensor's operands on the GPU, and what the step has to make of them."""

    def __init__(self, n, p_type, g_type, bits, copy_type, seed, decay=0.1, offset=0, state_std=0.1):
        self.bits, self.decay, self.n = bits, decay, n

        def on(values, dtype):
            buf = torch.full((n + offset + 16,), 7, dtype=torch.uint8, device="cuda") if dtype is torch.float8_e4m3fn else \
                torch.full((n + offset + 16,), 7, dtype=dtype, device="cuda")
            view = buf[offset:offset + n]
            view.copy_(values)
            self.buffers.append((buf, offset, n))
            return view.view(dtype)

        self.buffers = []
        self.p, self.g = on(rand((n,), p_type, seed), p_type), on(rand((n,), g_type, seed + 1, 0.3), g_type)
        m, v = rand((n,), torch.float32, seed + 2, state_std), rand((n,), torch.float32, seed + 3, state_std).square()
        if bits == 8:
            parts = []
            for x, floor in ((m, False), (v, True)):
                codes, scale = encoded(x.cpu().numpy(), np.full(n, 32768.0), floor)
                parts.append((on(torch.from_numpy(codes), torch.float8_e4m3fn), torch.from_numpy(scale).cuda().view(torch.float8_e8m0fnu)))
            self.state = trspmm.AdamWState(parts[0][0], parts[1][0], parts[0][1], parts[1][1])
        else:
            self.state = trspmm.AdamWState(on(m, torch.float32), on(v, torch.float32))
        self.copy = None if copy_type is None else on(torch.zeros(n, device="cuda"), copy_type)
        self.before = self.host()

    def host(self):
        as8 = (lambda x: x.view(torch.uint8).cpu().numpy().copy())
        s = self.state
        if self.bits == 8:
            m, v, ms, vs = map(as8, s)
            state = (m, v, ms, vs)
        else:
            state = (s.m.cpu().numpy().copy(), s.v.cpu().numpy().copy())
        return self.p.double().cpu().numpy().copy(), self.g.float().cpu().numpy().copy(), state

    def check(self, step, seed=0, scale=1.0, lr=HYPER["lr"], betas=HYPER["betas"], eps=HYPER["eps"]):
        p, g, state = self.before
        f = np.float32
        m, v = (decoded(state[0], state[2]), decoded(state[1], state[3])) if self.bits == 8 else state
        with np.errstate(all="ignore"):
            x = g * f(scale)
            m = f(betas[0]) * m + f(1 - betas[0]) * x
            v = f(betas[1]) * v + f(1 - betas[1]) * (x * x)
            now = self.host()
            if self.bits == 8:
                w = words(self.n, seed, step)
                for k, (y, chance, floor) in enumerate(((m, w >> np.uint64(16), False), (v, w & np.uint64(0xFFFF), True))):
                    codes, byte = encoded(y, chance.astype(np.float64), floor)
                    assert np.array_equal(now[2][2 + k], byte), "scales of state %d" % k
                    assert np.array_equal(now[2][k], codes), "codes of state %d" % k
            else:
                assert np.array_equal(now[2][0], m, equal_nan=True) and np.array_equal(now[2][1], v, equal_nan=True)
            way = m.astype(np.float64) / (1 - betas[0] ** step) / (np.sqrt(v.astype(np.float64) / (1 - betas[1] ** step)) + eps)
            want = p * (1 - lr * self.decay) - lr * way
            room = 2.0 ** -23 * (2 * np.abs(p) + 12 * np.abs(lr * way))
            for got in [self.p] + ([] if self.copy is None else [self.copy]):
                off = np.abs(got.double().cpu().numpy() - want)
                bound = room + (ROUND[got.dtype] * 1.01) * (np.abs(want) + room) + TINY[got.dtype]
                assert np.all((off <= bound) | (np.isnan(want) & np.isnan(got.double().cpu().numpy()))), float(np.nanmax(off - bound))
        for buf, a, n in self.buffers:       # nothing beside the tensors
            rest = torch.cat((buf[:a], buf[a + n:]))
            assert bool((rest.view(torch.uint8) == 7).all() if buf.dtype is torch.uint8 else (rest == 7).all())


def step_all(cases, step, **more):
    args = {**HYPER, "weight_decay": [c.decay for c in cases], **more}
    trspmm.adamw([c.p for c in cases], [c.g for c in cases], [c.state for c in cases], step,
                 copies=[c.copy for c in cases], **args)


@pytest.mark.parametrize("p_type", TYPES)
@pytest.mark.parametrize("g_type", TYPES)
@pytest.mark.parametrize("bits", [32, 8])
def test_types(p_type, g_type, bits):
    say("types", p_type, g_type, bits)
    cases = [Case(777, p_type, g_type, bits, c, 10 * i) for i, c in enumerate([None, *TYPES])]
    step_all(cases, 3)
    for c in cases:
        c.check(3)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 31, 32, 33, 63, 255, 256, 257, 1023, 1024, 1025, 2047, 2048, 2049, 4097, 70_001])
def test_sizes(n, bits):
    say("size", n, bits)
    for offset in (0, 1):      # a start off every vector's boundary
        c = Case(n, torch.float32, torch.bfloat16, bits, torch.bfloat16, n, offset=offset)
        step_all([c], 1)
        c.check(1)


def test_many_tensors_of_all_kinds():
    say("many")
    cases = []
    for i in range(150):
        cases.append(Case([1, 40, 3000, 0, 515, 9001][i % 6], TYPES[i % 3], TYPES[i // 3 % 3], (32, 8)[i // 9 % 2],
                          [None, *TYPES][i // 18 % 4], 5 * i, decay=(0.0, 0.1)[i % 2], offset=i % 2))
    step_all(cases, 12, seed=5)
    for c in cases:
        if c.n:
            c.check(12, seed=5)


@pytest.mark.parametrize("bits", [32, 8])
def test_steps_follow_one_another(bits):
    """20 steps, each from what the one before left."""
    say("steps", bits)
    c = Case(3000, torch.float32, torch.float32, bits, torch.float16, 1)
    c.state = trspmm.adamw_state(c.p, bits)
    c.buffers = c.buffers[:2]
    for step in range(1, 21):
        c.g.copy_(rand((3000,), torch.float32, 100 + step, 0.1 * (step % 3)))
        c.before = c.host()
        step_all([c], step, seed=9)
        c.check(step, seed=9)


def test_a_late_step_and_other_numbers():
    say("late")
    for step, betas, eps in [(1, (0.0, 0.0), 1e-8), (100_000, (0.95, 0.99), 1e-3), (2 ** 31 + 5, (0.9, 0.9999), 1e-12)]:
        for bits in (32, 8):
            c = Case(500, torch.float32, torch.float32, bits, None, 3)
            step_all([c], step, betas=betas, eps=eps, seed=MASK)
            c.check(step % 2 ** 32 if step > MASK else step, seed=MASK, betas=betas, eps=eps)


@pytest.mark.parametrize("bits", [32, 8])
def test_numbers_from_the_gpu(bits):
    say("from the gpu", bits)
    c = Case(900, torch.float32, torch.bfloat16, bits, None, 3)
    d = Case(900, torch.float32, torch.bfloat16, bits, None, 3)
    one = (lambda x, t: torch.tensor([x], dtype=t, device="cuda"))
    zero = one(0.0, torch.float32)
    step_all([c], one(7, torch.int64), lr=one(2e-3, torch.float32), grad_scale=one(0.37, torch.float32), skip=zero, seed=2)
    c.check(7, seed=2, scale=np.float32(0.37), lr=float(np.float32(2e-3)))
    step_all([d], 7, lr=2e-3, grad_scale=0.37, seed=2)
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(c.state, d.state) if a is not None)
    # the factor's powers differ in their last bits
    assert float((c.p - d.p).abs().max()) <= 12 * 2.0 ** -23 * float(d.p.abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_skipped_step_writes_nothing(bits):
    say("skip", bits)
    for flag in (1.0, float("inf"), float("nan")):
        c = Case(900, torch.float32, torch.bfloat16, bits, torch.float16, 3)
        step_all([c], 7, skip=torch.tensor(flag, device="cuda"))
        now = c.host()
        assert np.array_equal(now[0], c.before[0]) and all(np.array_equal(a, b) for a, b in zip(now[2], c.before[2]))
        assert bool((c.copy == 0).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite_reach_their_element_alone(bits):
    say("not finite", bits)
    c = Case(400, torch.float32, torch.float32, bits, None, 3)
    for at, x in ((5, float("nan")), (70, float("inf")), (399, -float("inf")), (200, 1e30)):
        c.g[at] = x
    c.before = c.host()
    step_all([c], 2)
    c.check(2)
    assert torch.nonzero(torch.isnan(c.p)).flatten().tolist() == [5, 70, 399]


def test_8_bit_states_keep_their_means():
    """A state that decays towards nothing and one that grows: nearest codes would stay where they are (v changes by
    0.1% a step).  Of 2^16 elements a step's mean is known to 2^-8 of a gap's half; the bound is 6 of that."""
    say("means")
    n = 1 << 16
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.5, device="cuda")
    state = trspmm.adamw_state(p, 8)
    state.m.copy_(torch.ones(n, device="cuda"))
    state.v.copy_(torch.ones(n, device="cuda"))
    for s in (state.m_scale, state.v_scale):
        s.view(torch.uint8).fill_(127)
    m = v = 1.0
    for step in range(1, 201):
        trspmm.adamw([p], [g], [state], step, lr=0.0, weight_decay=0.0, seed=3)
        m, v = 0.9 * m + 0.1 * 0.5, 0.999 * v + 0.001 * 0.25
    got = [float(x.double().mean()) for x in state.values()]
    # a rounding is off by a gap (1/8 of the value) at most with a variance of at most gap^2 / 4, and its share in the mean
    # fades by beta a step: sum of beta^(2k) <= 1 / (1 - beta^2)
    for x, want, beta in zip(got, (m, v), (0.9, 0.999)):
        sigma = 1.0 / 8 / 2 * math.sqrt(min(200, 1 / (1 - beta ** 2))) / math.sqrt(n)
        assert abs(x - want) <= 6 * sigma + 2.0 ** -16, (x, want, sigma)


def test_a_small_second_moment_does_not_vanish():
    say("floor")
    n = 64
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 1e-6, device="cuda")
    g[0] = g[32] = 1e3
    state = trspmm.adamw_state(p, 8)
    for step in range(1, 30):
        if step > 3:
            g.zero_()          # m lives on: a v of 0 would make its step m / eps
        trspmm.adamw([p], [g], [state], step, lr=1e-3, weight_decay=0.0)
    assert bool((state.v.view(torch.uint8) > 0).all()) and float(p.abs().max()) < 29 * 1e-3 * 10


def test_a_captured_step():
    """Replayed with the program's own work between: step's number, rate and gradients change, an eager twin follows."""
    say("graph")
    a = [Case(5000, torch.float32, torch.bfloat16, b, torch.bfloat16, 3) for b in (32, 8)]
    b = [Case(5000, torch.float32, torch.bfloat16, b, torch.bfloat16, 3) for b in (32, 8)]
    step, lr = torch.tensor([0], device="cuda"), torch.tensor([0.0], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step.add_(1)
        step_all(a, step, lr=lr, seed=4)
    for turn in range(1, 5):
        for x, y in zip(a, b):
            x.g.copy_(rand((5000,), torch.bfloat16, 50 + turn))
            y.g.copy_(x.g)
        lr.fill_(1e-3 * turn)
        graph.replay()
        step_all(b, torch.tensor([turn], device="cuda"), lr=lr, seed=4)
        torch.cuda.synchronize()
        for x, y in zip(a, b):
            assert int(step) == turn and torch.equal(x.p, y.p) and torch.equal(x.copy, y.copy)
            assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(x.state, y.state) if s is not None)


def test_shapes_and_other_streams():
    say("shapes")
    p = rand((30, 50), torch.float32, 1)
    want, g = p.clone(), rand((50, 30), torch.float16, 2).t()       # a gradient whose rows are columns
    trspmm.adamw([want.view(-1)], [g.contiguous().view(-1)], [trspmm.adamw_state(want.view(-1))], 1)
    state = trspmm.adamw_state(p, 32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    trspmm.adamw([p], [g], [state], 1, stream=side)
    side.synchronize()
    assert torch.equal(p, want) and state.m.shape == p.shape
    scalar = torch.ones((), device="cuda")
    trspmm.adamw([scalar], [scalar * 2], [trspmm.adamw_state(scalar, 8)], 1, lr=0.1, weight_decay=0.0)
    assert abs(float(scalar) - 0.9) < 1e-6
    trspmm.adamw([], [], [], 1)


def test_against_differences():
    """With beta1 = beta2 = 0 and no decay a step is lr g / (|g| + eps): its sign is the gradient's.  The gradient of a
    quadratic, taken by differences in 64 bits, gives the same step."""
    say("differences")
    target, p = rand((300,), torch.float32, 1), rand((300,), torch.float32, 2)
    loss = (lambda x: ((x - target.double()) ** 2).sum())
    h = 1e-4
    eye = torch.eye(300, dtype=torch.float64, device="cuda") * h
    diff = torch.stack([(loss(p.double() + e) - loss(p.double() - e)) / (2 * h) for e in eye])
    want = p.double() - 0.01 * diff / (diff.abs() + 1e-8)
    trspmm.adamw([p], [2 * (p - target)], [trspmm.adamw_state(p)], 1, lr=0.01, betas=(0.0, 0.0), weight_decay=0.0)
    assert float((p.double() - want).abs().max()) < 1e-6


def test_refusals():
    say("refusals")
    p, g = torch.ones(100, device="cuda"), torch.ones(100, device="cuda")
    s, s8 = trspmm.adamw_state(p), trspmm.adamw_state(p, 8)
    half = torch.ones(100, dtype=torch.float16, device="cuda")
    for args, more in [(([p], [g], []), {}), (([p], [], [s]), {}), (([p.cpu()], [g], [s]), {}), (([p], [g.cpu()], [s]), {}),
                       (([p], [g[:99]], [s]), {}), (([p.int()], [g], [s]), {}), (([p], [g.double()], [s]), {}),
                       (([p[::2]], [g[:50]], [trspmm.adamw_state(p[:50])]), {}), (([p], [g], [(s.m,)]), {}),
                       (([p], [g], [(s.m, s.v, s8.m_scale, None)]), {}), (([p], [g], [(half, half)]), {}),
                       (([p], [g], [(s8.m, s8.v)]), {}), (([p], [g], [(s8.m, s8.v, s8.m_scale[:3], s8.v_scale[:3])]), {}),
                       (([p], [g], [(s.m, s.v, s8.m_scale, s8.v_scale)]), {}), (([p], [g], [(s.m[:99], s.v[:99])]), {}),
                       (([p], [g], [s]), {"weight_decay": [0.1, 0.1]}), (([p], [g], [s]), {"copies": [half[:99]]}),
                       (([p], [g], [s]), {"copies": []}), (([p], [g], [s]), {"copies": [half.int()]}),
                       (([p], [g], [s]), {"lr": torch.ones(2, device="cuda")}), (([p], [g], [s]), {"lr": half[:1]}),
                       (([p], [g], [s]), {"skip": torch.ones(1, dtype=torch.int32, device="cuda")}),
                       (([p], [g], [s]), {"grad_scale": torch.ones(1)}), (([p], [None], [s]), {}), (([p], [g], [s]), {"seed": -1}),
                       (([p], [g], [s]), {"seed": 2 ** 32}), (([p], [g], [s]), {"lr": "1"}), (([p], [g], [s]), {"weight_decay": "1"}),
                       (([p], [g], [s]), {"weight_decay": [None]})]:
        with pytest.raises(ValueError):
            trspmm.adamw(*args, 1, **more)
    other = trspmm.adamw_state(p)
    for args, more in [(([p, p], [g, g], [s, other]), {}), (([p, half], [g, g], [s, s]), {}), (([p], [g], [(s.m, s.m)]), {}),
                       (([p[:60], p[40:]], [g[:60], g[40:]], [trspmm.adamw_state(p[:60]), trspmm.adamw_state(p[40:])]), {}),
                       (([p], [g], [s]), {"copies": [p]}), (([p], [g], [s]), {"copies": [g]}), (([p], [p], [s]), {}), (([p], [s.v], [s]), {}),
                       (([p], [g], [s]), {"betas": (1.0, 0.9)}), (([p], [g], [s]), {"betas": (0.9, -0.1)}),
                       (([p], [g], [s]), {"eps": 0.0}), (([p], [g], [s]), {"lr": float("nan")}), (([p], [g], [s]), {"weight_decay": float("inf")}),
                       (([p], [g], [s]), {"grad_scale": float("inf")})]:
        with pytest.raises(nat.TrsError):
            trspmm.adamw(*args, 1, **more)
    with pytest.raises(nat.TrsError):
        trspmm.adamw([p], [g], [s], 0)
    with pytest.raises(ValueError):
        trspmm.adamw([p], [g], [s], torch.ones(1, device="cuda"))
    with pytest.raises(ValueError):
        trspmm.adamw([p], [g], [s], 1.5)
    with pytest.raises(ValueError):
        trspmm.adamw_state(p, 16)
    assert bool((p == 1).all()) and bool((s.m == 0).all())


def test_numbers_of_other_kinds_and_a_shared_gradient():
    say("numpy numbers, shared gradient")
    g = rand((1000,), torch.float32, 1)
    first, second, third = (rand((1000,), torch.float32, 2) for _ in range(3))
    states = [trspmm.adamw_state(first) for _ in range(3)]
    trspmm.adamw([first, second], [g, g], states[:2], np.int64(1), np.float32(0.125), weight_decay=np.float32(0.25), grad_scale=np.float64(0.5))
    trspmm.adamw((third,), (g,), states[2:], 1, 0.125, weight_decay=(0.25,), grad_scale=0.5)
    assert torch.equal(first, third) and torch.equal(second, third)


def test_autograd_sees_the_change():
    """A backward pass through what was saved of a parameter before the step is refused, as after torch's own in-place operations."""
    say("versions")
    p = rand((64,), torch.float32, 1).requires_grad_()
    copy = p.detach().clone().requires_grad_()
    loss, other = (p * p).sum(), (copy * copy).sum()
    g = torch.ones(64, device="cuda")
    trspmm.adamw([p], [g], [trspmm.adamw_state(p)], 1, copies=[copy])
    for x in (loss, other):
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            x.backward()
    with torch.inference_mode():
        q = torch.ones(64, device="cuda")
        trspmm.adamw([q], [g], [trspmm.adamw_state(q)], 1)
    assert bool((q != 1).all())


def test_an_index_past_32_bits():
    """2^32 + 5000 elements: those with a gradient, at the start, around 2^31 and at the end, are stepped as in a tensor of their own."""
    say("long tensor")
    n = 2 ** 32 + 5000
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("not enough memory")
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    state = trspmm.adamw_state(p, 8)
    parts = [slice(0, 640), slice(2 ** 31 - 320, 2 ** 31 + 320), slice(2 ** 32 - 320, 2 ** 32 + 320), slice(n - 584, n)]
    alone = []
    for i, at in enumerate(parts):
        count = at.stop - at.start
        mine, grad = (rand((count,), torch.bfloat16, 10 * i + k) for k in range(2))
        p[at], g[at] = mine, grad
        alone.append((mine, trspmm.adamw_state(mine, 8)))
        trspmm.adamw([mine], [grad], [alone[-1][1]], 1, lr=0.5)
    trspmm.adamw([p], [g], [state], 1, lr=0.5)
    for at, (mine, its) in zip(parts, alone):
        assert torch.equal(p[at], mine), at
        blocks = slice(at.start // 32, (at.stop + 31) // 32)
        for long, short in ((state.m_scale, its.m_scale), (state.v_scale, its.v_scale)):
            assert torch.equal(long[blocks].view(torch.uint8), short.view(torch.uint8)), at
        # codes: one of the same two neighbours, by other bits
        for long, short in ((state.m, its.m), (state.v, its.v)):
            off = long[at].view(torch.uint8).int() - short.view(torch.uint8).int()
            assert int(off.abs().max()) <= 1
        p[at] = 0
    assert not bool(p.any())


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_from_the_gpu_below_1_writes_nothing(bits):
    """Steps count from 1; a counter that is raised behind the call starts at 0, where the bias corrections divide by 0."""
    say("step below 1", bits)
    for step in (0, -1, -2 ** 40):
        c = Case(900, torch.float32, torch.bfloat16, bits, torch.float16, 3)
        step_all([c], torch.tensor(step, device="cuda"))
        now = c.host()
        assert np.array_equal(now[0], c.before[0]) and all(np.array_equal(a, b) for a, b in zip(now[2], c.before[2]))
        assert bool((c.copy == 0).all())


def test_a_captured_step_that_counts_behind_the_call():
    say("graph, counted behind")
    c, twin = (Case(3000, torch.float32, torch.float32, 8, torch.bfloat16, 3) for _ in range(2))
    step = torch.tensor([0], device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        step_all([c], step, seed=4)
        step.add_(1)
    for turn in range(4):
        graph.replay()
        if turn > 0:
            step_all([twin], torch.tensor([turn], device="cuda"), seed=4)
        torch.cuda.synchronize()
        assert torch.equal(c.p, twin.p) and torch.equal(c.copy, twin.copy), turn
        assert all(torch.equal(s.view(torch.uint8), t.view(torch.uint8)) for s, t in zip(c.state, twin.state))


@pytest.mark.parametrize("byte", [0, 1, 200, 254])
def test_states_with_every_scale(byte):
    """Scale byte b stands for 2^(b - 127), also where that is no ordinary float: a state that was written elsewhere may hold it."""
    say("scale", byte)
    c = Case(640, torch.float32, torch.float32, 8, None, 3)
    for codes, scale in ((c.state.m, c.state.m_scale), (c.state.v, c.state.v_scale)):
        scale.view(torch.uint8).fill_(byte)
        codes.view(torch.uint8).clamp_(max=0x3F if byte == 254 else 0x78)      # 2^127 times 1.875 is finite
    c.g.zero_()
    c.before = c.host()
    assert all(np.array_equal(decoded(c.before[2][k], c.before[2][2 + k]), x.cpu().numpy()) for k, x in enumerate(c.state.values()))
    step_all([c], 2)
    c.check(2)
    if byte == 0:       # 0.9 and 0.999 of values up to 2^-119: they live on at the smallest scale that is written
        assert bool((c.state.m.view(torch.uint8) & 127 > 0).any()) and bool((c.state.v.view(torch.uint8) > 0).any())


def test_a_nan_scale_is_a_block_of_nan():
    say("nan scale")
    c = Case(640, torch.float32, torch.float32, 8, None, 3)
    for scale in (c.state.m_scale, c.state.v_scale):
        scale.view(torch.uint8)[3] = 255
    c.state.m.view(torch.uint8)[96:128] = torch.arange(32, dtype=torch.uint8, device="cuda")
    step_all([c], 2)
    assert torch.nonzero(torch.isnan(c.p)).flatten().tolist() == list(range(96, 128))
    for codes in (c.state.m, c.state.v):
        assert torch.nonzero(torch.isnan(codes.float())).flatten().tolist() == list(range(96, 128))


def test_numbers_on_the_gpu_that_the_step_would_write():
    """A factor, a rate, a step or a flag inside of what is written would be read by some workgroups before the write and by others
    after it."""
    say("overlapping numbers")
    p, g = torch.ones(5000, device="cuda"), torch.ones(5000, device="cuda")
    s, s8 = trspmm.adamw_state(p), trspmm.adamw_state(p, 8)
    copy = torch.zeros(5000, device="cuda")
    for state, more in [(s, {"lr": p[7:8]}), (s, {"grad_scale": s.m[4999:]}), (s, {"skip": s.v[:1]}), (s, {"skip": copy[3:4], "copies": [copy]}),
                        (s8, {"lr": s8.v.view(torch.uint8)[8:12].view(torch.float32)}),
                        (s8, {"skip": s8.m_scale.view(torch.uint8)[8:12].view(torch.float32)})]:
        with pytest.raises(nat.TrsError, match="overlaps"):
            trspmm.adamw([p], [g], [state], 1, **more)
    with pytest.raises(nat.TrsError, match="overlaps"):
        trspmm.adamw([p], [g], [s], s.m[:2].view(torch.int64))
    assert bool((p == 1).all()) and bool((s.m == 0).all())
    trspmm.adamw([p], [g], [s], 1, lr=g[:1])      # one that is only read
    assert bool((p < 1).all())


def words_from(first, n, seed, step):
    """The rounding bits of n elements from index `first` on."""
    key = (seed * 0x6A09E667 + step * 0xB7E15163) & MASK
    key = ((key ^ key >> 16) * 0xBB67AE85) & MASK
    out = np.empty(n, np.uint64)
    for i in range(n):
        at = first + i
        x = (key + at * 0x9E3779B9 + (at >> 32) * 0x243F6A89) & MASK
        x = ((x ^ x >> 15) * 0xBB67AE85) & MASK
        out[i] = x ^ x >> 16
    return out


def test_rounding_bits_past_32_bits():
    """Codes around element 2^32 and at the end are those of the formula, whose bits depend on the index's upper half."""
    say("long tensor's codes")
    n = 2 ** 32 + 5000
    if torch.cuda.mem_get_info()[0] < 80e9:
        pytest.skip("not enough memory")
    assert np.array_equal(words_from(0, 100, 5, 9), words(100, 5, 9))
    p, g = (torch.zeros(n, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    state = trspmm.adamw_state(p, 8)
    parts = [slice(0, 640), slice(2 ** 31 - 320, 2 ** 31 + 320), slice(2 ** 32 - 320, 2 ** 32 + 320), slice(n - 584, n)]
    for i, at in enumerate(parts):
        g[at] = rand((at.stop - at.start,), torch.bfloat16, 10 + i)
    step = 2 ** 32 + 3
    trspmm.adamw([p], [g], [state], step, seed=6)
    f = np.float32
    for at in parts:
        x = g[at].float().cpu().numpy()
        w = words_from(at.start, x.size, 6, step)
        blocks = slice(at.start // 32, (at.stop + 31) // 32)
        for codes, scale, y, chance, floor in ((state.m, state.m_scale, f(1 - 0.9) * x, w >> np.uint64(16), False),
                                               (state.v, state.v_scale, f(1 - 0.999) * (x * x), w & np.uint64(0xFFFF), True)):
            want, byte = encoded(y, chance.astype(np.float64), floor)
            assert np.array_equal(scale[blocks].view(torch.uint8).cpu().numpy(), byte), at
            assert np.array_equal(codes[at].view(torch.uint8).cpu().numpy(), want), at


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("step", [2 ** 32, 2 ** 32 + 3, 2 ** 40 + 7])
def test_steps_past_32_bits(step, bits):
    """The hash takes the step modulo 2^32, the bias corrections the step itself."""
    say("step", step, bits)
    for number in (step, torch.tensor([step], device="cuda")):
        c = Case(700, torch.float32, torch.float32, bits, None, 3)
        step_all([c], number, betas=(0.9, 1 - 2.0 ** -30), seed=8)
        c.check(step, betas=(0.9, 1 - 2.0 ** -30), seed=8)


def test_a_second_moment_far_below_its_blocks_largest():
    """v below 2^-17 of its block's largest is held at the smallest code, 2^-9 of the scale, 2^-17 to 2^-16 of the largest: never
    0, no longer its mean, and the parameter's change is smaller by the root of that."""
    say("v's floor")
    n = 32
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 2.0 ** -20, device="cuda")
    g[0] = 1.0
    state = trspmm.adamw_state(p, 8)
    for step in range(1, 6):
        trspmm.adamw([p], [g], [state], step, weight_decay=0.0, seed=1)
        v = state.values()[1]
        unit = 2.0 ** (int(state.v_scale.view(torch.uint8)[0]) - 127)
        assert bool((v[1:] == unit * 2.0 ** -9).all())
        share = float(v[1] / v[0])
        assert 2.0 ** -17.2 <= share <= 2.0 ** -16
