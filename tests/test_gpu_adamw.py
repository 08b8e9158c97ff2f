"""AdamW over many tensors against the float64 oracle and, for the 8-bit states, against the float32
definition of their codes bit for bit.

Tolerances, u = 2^-24: a moment is two rounded products (and rounded constants) and a rounded sum,
so within 6u of the sum of the magnitudes of its parts; the weight is p*keep (2u with the constant)
minus a quotient: 8u for the denominator's square root, product, sum and quotient, 3u for the step's
constant and product, plus what the moment's error passes on (v enters under a square root), and u
of the result."""
import numpy as np
import pytest
import torch

from _util import np64
from colabfold_legacy_kernels import ops
from oracle import adamw as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HP = dict(lr=1e-2, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.02, grad_scale=0.5)


def buffer(n, dtype, dev, off=0):
    """A tensor of n elements, `off` elements into a larger one whose rest must not change."""
    whole = torch.full((n + off + 37,), 77, dtype=dtype, device=dev)
    return whole[off:off + n], whole


class Set:
    """Tensors of given sizes with states, and guards around all of them."""

    def __init__(self, sizes, bits, grad, copy, dev, seed=0, off=0, off8=0):
        g = torch.Generator().manual_seed(seed)
        self.sizes, self.bits, self.guards = sizes, bits, []

        def one(values, dtype, at):
            t, whole = buffer(values.numel(), dtype, dev, at)
            t.copy_(values)
            self.guards.append((whole, at, values.numel()))
            return t
        self.p, self.g, self.m, self.v, self.s, self.c = [], [], [], [], [], []
        for n in sizes:
            size = torch.exp(2 * torch.randn(n, generator=g)) * 1e-2
            self.p.append(one(torch.randn(n, generator=g), torch.float32, off))
            self.g.append(one(torch.randn(n, generator=g) * size, grad, off))
            m = (torch.randn(n, generator=g) * size).float()
            v = (torch.randn(n, generator=g).square() * size.square()).float()
            if bits == 8:
                qm, qv, s = ref.encode(m.numpy(), v.numpy())
                m, v = torch.from_numpy(qm), torch.from_numpy(qv)
                s = torch.from_numpy(s)
                flat = one(s.reshape(-1), torch.float32, off)
                self.s.append(flat.view(-1, 2))
            self.m.append(one(m, torch.int8 if bits == 8 else torch.float32, off8 or off))
            self.v.append(one(v, torch.uint8 if bits == 8 else torch.float32, off8 or off))
            self.c.append(None if copy is None else one(torch.zeros(n), copy, off))

    def plan(self):
        return ops.AdamWPlan(self.p, self.g, self.m, self.v, self.s if self.bits == 8 else None,
                             self.c)

    def states(self):
        """float32 states per tensor."""
        if self.bits == 32:
            return [(m.cpu().numpy(), v.cpu().numpy()) for m, v in zip(self.m, self.v)]
        return [ref.decode(m.cpu().numpy(), v.cpu().numpy(), s.cpu().numpy())
                for m, v, s in zip(self.m, self.v, self.s)]

    def check_guards(self):
        for whole, at, n in self.guards:
            assert (whole[:at] == 77).all() and (whole[at + n:] == 77).all()


def check_step(s, before, step, hp):
    """The set's values after a step from `before` = ([p], [g], [(m, v)])."""
    for i, n in enumerate(s.sizes):
        p0, g0, (m0, v0) = before[0][i], before[1][i], before[2][i]
        p, m, v = ref.step(p0, g0, m0, v0, step, **hp)
        g = np.abs(g0 * hp["grad_scale"])
        em = 6 * U * (np.abs(hp["beta1"] * m0) + (1 - hp["beta1"]) * g)
        ev = 6 * U * v
        if s.bits == 32:
            assert (np.abs(np64(s.m[i]) - m) <= em + 1e-44).all()
            assert (np.abs(np64(s.v[i]) - v) <= ev + 1e-44).all()
        else:
            m32, v32 = ref.moments32(g0.astype(np.float32), m0, v0, hp["beta1"], hp["beta2"],
                                     hp["grad_scale"])
            qm, qv, scales = ref.encode(m32, v32)
            assert (s.m[i].cpu().numpy() == qm).all() and (s.v[i].cpu().numpy() == qv).all()
            assert (s.s[i].cpu().numpy() == scales).all()
        rate = hp["lr"] / (1 - hp["beta1"] ** step)
        denom = np.sqrt(v) / np.sqrt(1 - hp["beta2"] ** step) + hp["eps"]
        tol = rate * (em / denom + 14 * U * np.abs(m) / denom) + 3 * U * np.abs(p0) + U * np.abs(p)
        assert (np.abs(np64(s.p[i]) - p) <= tol + 1e-44).all(), float(
            (np.abs(np64(s.p[i]) - p) / tol).max())
        if s.c[i] is not None:
            assert torch.equal(s.c[i], s.p[i].to(s.c[i].dtype))


def snapshot(s):
    return ([np64(p) for p in s.p], [np64(g) for g in s.g], s.states())


SETS = [[1], [2, 255, 256, 257, 3], [1024, 1023, 1025, 5000], [0, 7, 0, 300], [100000, 13],
        [37] * 500]


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("grad", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("copy", [None, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("sizes", SETS)
def test_steps(cuda, bits, grad, copy, sizes):
    s = Set(sizes, bits, grad, copy, cuda, seed=len(sizes))
    plan = s.plan()
    for step in (1, 2, 1000):
        before = snapshot(s)
        ops.adamw_step(plan, step, **HP)
        check_step(s, before, step, HP)
    s.check_guards()


@pytest.mark.parametrize("bits,off8", [(32, 0), (8, 4)])
@pytest.mark.parametrize("off", [1, 2, 3, 5])
def test_tensors_at_any_element(cuda, bits, off8, off):
    """Views that begin at any element of a larger buffer (codes at multiples of four)."""
    for grad, copy in ((torch.float32, torch.bfloat16), (torch.bfloat16, torch.float16)):
        s = Set([5, 256, 1030, 4099], bits, grad, copy, cuda, seed=off, off=off, off8=off8)
        before = snapshot(s)
        ops.adamw_step(s.plan(), 3, **HP)
        check_step(s, before, 3, HP)
        s.check_guards()


@pytest.mark.parametrize("bits", [8, 32])
def test_large_and_mixed(cuda, bits):
    """Sizes that take the long chunks, gradients of all types and single copies in one plan."""
    sizes = [9_000_001, 3, 70_000]
    s = Set(sizes, bits, torch.float32, torch.bfloat16, cuda, seed=3)
    s.g[1], s.g[2] = s.g[1].bfloat16(), s.g[2].half()
    s.c[0] = None
    before = snapshot(s)
    ops.adamw_step(s.plan(), 7, **HP)
    check_step(s, before, 7, HP)
    s.check_guards()


@pytest.mark.parametrize("bits", [8, 32])
def test_states_as_float32(cuda, bits):
    s = Set([3, 700, 0, 256, 5000], bits, torch.float32, None, cuda)
    plan = s.plan()
    ops.adamw_step(plan, 1, **HP)
    m, v = ops.adamw_states(plan)
    assert m.shape == v.shape == (plan.size,) and plan.starts == [0, 256, 1024, 1024, 1280]
    rest = torch.ones(plan.size, dtype=torch.bool)
    for (dm, dv), at, n in zip(s.states(), plan.starts, plan.numel):
        assert (m[at:at + n].cpu().numpy() == dm).all() and (v[at:at + n].cpu().numpy() == dv).all()
        rest[at:at + n] = False
    assert not m[rest.to(cuda)].any() and not v[rest.to(cuda)].any()


def test_zero_states_and_zero_gradients(cuda):
    for bits in (8, 32):
        p = [torch.randn(300, device=cuda), torch.randn(4, 5, device=cuda)]
        g = [torch.zeros_like(t) for t in p]
        m, v, scales = ops.adamw_zero_states(p, bits)
        plan = ops.AdamWPlan(p, g, m, v, scales)
        want = [t.clone() for t in p]
        ops.adamw_step(plan, 1, 0.1)
        assert all(torch.equal(a, b) for a, b in zip(p, want))  # 0 / (0 + eps), no decay
        ops.adamw_step(plan, 2, 0.1, weight_decay=0.5)
        for a, b in zip(p, want):
            torch.testing.assert_close(a, 0.95 * b, rtol=4 * U, atol=0)
        g[0][::2] = 2.0
        ops.adamw_step(plan, 3, 0.1)
        assert torch.isfinite(p[0]).all() and (p[0][::2] != 0.95 * want[0][::2]).all()
        assert all(not t.any() for t in (m[1], v[1]))


def test_small_and_large_scales(cuda):
    """Gradients from the subnormal range to 1e18: the codes follow the float32 definition."""
    for size in (1e-42, 1e-38, 1e-30, 1e-19, 1e-10, 1e10, 1e18):
        s = Set([700], 8, torch.float32, None, cuda)
        s.m[0].zero_(), s.v[0].zero_(), s.s[0].zero_()
        s.g[0].copy_(torch.randn(700, generator=torch.Generator().manual_seed(1)) * size)
        m32, v32 = ref.moments32(s.g[0].cpu().numpy(), np.zeros(700, np.float32),
                                 np.zeros(700, np.float32), 0.9, 0.99)
        qm, qv, scales = ref.encode(m32, v32)
        ops.adamw_step(s.plan(), 1, 1e-3, 0.9, 0.99, 1e-8)
        assert (s.s[0].cpu().numpy() == scales).all(), size
        assert (s.m[0].cpu().numpy() == qm).all() and (s.v[0].cpu().numpy() == qv).all(), size
        assert torch.isfinite(s.p[0]).all()


def test_special_gradients(cuda):
    """32-bit states: an infinite or NaN gradient stays with its element. 8-bit states: within its
    block of 256, from the next step on."""
    s = Set([600], 32, torch.float32, None, cuda)
    s.g[0][5], s.g[0][300] = float("inf"), float("nan")
    plan = s.plan()
    for t in (1, 2):
        ops.adamw_step(plan, t, **HP)
    bad = torch.zeros(600, dtype=torch.bool, device=cuda)
    bad[5], bad[300] = True, True
    assert torch.equal(~torch.isfinite(s.p[0]), bad)
    s = Set([900], 8, torch.float32, None, cuda)
    s.g[0][300] = float("nan")
    plan = s.plan()
    ops.adamw_step(plan, 1, **HP)
    assert torch.isfinite(s.p[0]).sum() == 899 and s.s[0][1].isnan().all()
    assert torch.isfinite(s.s[0][[0, 2, 3]]).all()
    ops.adamw_step(plan, 2, **HP)
    assert torch.isfinite(s.p[0][:256]).all() and torch.isfinite(s.p[0][512:]).all()
    m, _ = ops.adamw_states(plan)
    assert m[256:512].isnan().all() and not m[900:].any()


def test_hyper_replays_with_other_values(cuda):
    """A captured step reads lr, the bias corrections and the gradient scale at replay."""
    for bits in (8, 32):
        a = Set([1000, 77], bits, torch.float32, torch.bfloat16, cuda, seed=5)
        plan = a.plan()
        hyper = ops.adamw_hyper(1, 0.0).to(cuda)
        kw = dict(beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.02, hyper=hyper)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.adamw_step(plan, None, None, **kw)
        for t, lr, scale in ((1, 1e-2, 1.0), (2, 3e-3, 0.25), (9, 1e-2, 0.5)):
            before = snapshot(a)
            hyper.copy_(ops.adamw_hyper(t, lr, 0.9, 0.99, scale))
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            hp = dict(HP, lr=lr, grad_scale=scale)
            # lr and 1 - beta^t are rounded to float32 and used in float32: 8u more of each part.
            for i in range(2):
                p, m, v = ref.step(before[0][i], before[1][i], *before[2][i], t, **hp)
                step = np.abs(before[0][i] * (1 - lr * 0.02) - p)
                em = 6 * U * (0.9 * np.abs(before[2][i][0]) + 0.1 * np.abs(before[1][i] * scale))
                rate = lr / (1 - 0.9 ** t) / (np.sqrt(v) / np.sqrt(1 - 0.99 ** t) + 1e-8)
                tol = rate * em + 24 * U * step + 5 * U * np.abs(before[0][i])
                assert (np.abs(np64(a.p[i]) - p) <= tol).all()
                assert torch.equal(a.c[i], a.p[i].bfloat16())


def test_autograd_notices_the_change(cuda):
    w = torch.randn(8, 8, device=cuda, requires_grad=True)
    g = torch.ones_like(w)
    m, v, _ = ops.adamw_zero_states([w])
    plan = ops.AdamWPlan([w], [g], m, v)
    y = (w * w).sum()
    ops.adamw_step(plan, 1, 1e-3)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_refusals(cuda):
    z = lambda *s, **k: torch.zeros(*s, device=cuda, **k)  # noqa: E731
    p, g = z(300), z(300)
    q8 = (z(300, dtype=torch.int8), z(300, dtype=torch.uint8))
    sc = z(2, 2)
    P = ops.AdamWPlan
    bad = [lambda: P([p], [g, g], [z(300)], [z(300)]), lambda: P([p], [z(299)], [z(300)], [z(300)]),
           lambda: P([p.half()], [g], [z(300)], [z(300)]),
           lambda: P([p], [g.double()], [z(300)], [z(300)]),
           lambda: P([p], [g.int()], [z(300)], [z(300)]),
           lambda: P([p], [g], [z(300).half()], [z(300)]), lambda: P([p], [g], [q8[0]], [z(300)]),
           lambda: P([p], [g], [q8[0]], [q8[1]]), lambda: P([p], [g], [q8[0]], [q8[1]], [z(3, 2)]),
           lambda: P([p], [g], [z(300)], [z(300)], [sc]),
           lambda: P([p], [g], [z(300)], [z(300)], copies=[z(300)]),
           lambda: P([p], [g], [z(300)], [None]), lambda: P([p, p], [g, g], [z(300)] * 2, [z(300)] * 2),
           lambda: P([p], [g], [p], [z(300)]), lambda: P([p], [p], [z(300)], [z(300)]),
           lambda: P([z(20, 30).t()], [z(30, 20)], [z(30, 20)], [z(30, 20)]),
           lambda: P([p], [g.cpu()], [z(300)], [z(300)])]
    for call in bad:
        with pytest.raises(ops.InvalidArgument):
            call()
    plan = P([p], [g], [q8[0]], [q8[1]], [sc])
    for kw in (dict(step=0, lr=0.1), dict(step=1, lr=float("nan")), dict(step=1, lr=0.1, beta1=1.0),
               dict(step=1, lr=0.1, eps=0.0), dict(step=1, lr=0.1, hyper=z(3)),
               dict(step=1, lr=0.1, hyper=torch.zeros(4))):
        with pytest.raises(ops.InvalidArgument):
            ops.adamw_step(plan, **kw)
