"""The embedding, the residual join and AdamW together with the blocks between them: one training
step of a pair representation, against float64 autograd; the same step captured and replayed; and
calls at once from several threads and streams.

The step rounds what it hands on to bf16 eight times between the table and its gradient (z, its norm,
the projection, the stream, and on the way back the projection's gradient, the norm's input's, the
two parts of dz), each within half a step, 2^-9 of the value; norms and gates pass such errors on
about as large as they are (their Jacobians on normed rows have norms near 1). 2-norms of gradients
are therefore held to 8 * 2^-8, twice the sum of the roundings."""
import threading

import numpy as np
import pytest
import torch

from _util import np64
from colabfold_legacy_kernels import ops
from oracle import adamw as ref_adamw

pytestmark = pytest.mark.gpu

C, N = 64, 24
HP = dict(lr=3e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.01, grad_scale=0.5)
# Weights that the kernels read in bf16 (working copies), and float32 vectors.
SHAPES = {"table": (65, C), "wp": (C, C), "bp": (C,), "wg": (C, C), "bg": (C,)}
VECTORS = ["ln_w", "ln_b", "post_w", "post_b", "res", "pre_w", "pre_b"]


class Step:
    def __init__(self, dev, bits, seed=0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s, std=1.0, mean=0.0: (torch.randn(s, generator=g) * std + mean).to(dev)  # noqa
        self.p = {k: rand(*s, std=0.5 if k == "table" else 0.12) for k, s in SHAPES.items()}
        for k in VECTORS:
            self.p[k] = rand(C, std=0.2, mean=0.0 if k.endswith("_b") else 0.8)
        self.names = list(self.p)
        self.copy = {k: self.p[k].bfloat16() for k in SHAPES}
        self.grad = {k: torch.zeros_like(t) for k, t in self.p.items()}
        params = [self.p[k] for k in self.names]
        self.states = ops.adamw_zero_states(params, bits)
        self.plan = ops.AdamWPlan(params, [self.grad[k] for k in self.names], *self.states,
                                  copies=[self.copy.get(k) for k in self.names])
        self.hyper = torch.zeros(4, device=dev)
        at = torch.arange(N, device=dev)
        self.ids = (at[:, None] - at[None, :]).clamp(-32, 32).add(32).reshape(-1)
        self.ids[::17] = -1  # padded pairs
        self.mask = (self.ids >= 0).bfloat16()
        self.dr, self.dh = rand(N * N, C).bfloat16(), rand(N * N, C).bfloat16()

    def gradients(self):
        p, c = self.p, self.copy
        z = ops.embedding(c["table"], self.ids, 8.0)
        y = ops.layer_norm(z, p["ln_w"], p["ln_b"])
        gdp = (c["wp"], c["bp"], c["wg"], c["bg"], self.mask)
        o = ops.gated_dual_proj(y, *gdp)
        post, pre = (p["post_w"], p["post_b"]), (p["pre_w"], p["pre_b"])
        r, h = ops.residual_norm(z, o, y, post, p["res"], pre)
        dz, do, dgate, *joined = ops.residual_norm_bwd(r, o, y, post, p["res"], pre, self.dr,
                                                       self.dh)
        dy, *projected = ops.gated_dual_proj_bwd(y, *gdp, do, dx=dgate)  # y is the gate as well
        dz2, dln_w, dln_b = ops.layer_norm_bwd(z, p["ln_w"], dy)
        dtable = ops.embedding_bwd(dz + dz2, self.ids, 65, 8.0)
        names = ["table", "wp", "bp", "wg", "bg", "ln_w", "ln_b", "post_w", "post_b", "res",
                 "pre_w", "pre_b"]
        for k, t in zip(names, [dtable] + projected + [dln_w, dln_b] + joined):
            self.grad[k].copy_(t)
        return r, h

    def run(self):
        out = self.gradients()
        ops.adamw_step(self.plan, None, None, HP["beta1"], HP["beta2"], HP["eps"],
                       HP["weight_decay"], hyper=self.hyper)
        return out

    def tensors(self):
        return ([self.p[k] for k in self.names] + list(self.copy.values()) +
                [t for ts in self.states if ts is not None for t in ts])


def float64_gradients(s):
    leaf = {k: (s.copy[k] if k in s.copy else s.p[k]).double().cpu().requires_grad_()
            for k in s.names}
    ids, mask = s.ids.cpu(), s.mask.double().cpu()[:, None]
    norm = lambda x, w, b: torch.nn.functional.layer_norm(x, (C,), leaf[w], leaf[b], 1e-5)  # noqa
    z = torch.where(ids[:, None] >= 0, leaf["table"][ids.clamp(min=0)] * 8.0, 0.0)
    y = norm(z, "ln_w", "ln_b")
    o = mask * (y @ leaf["wp"] + leaf["bp"]) * torch.sigmoid(y @ leaf["wg"] + leaf["bg"])
    r = z + leaf["res"] * torch.sigmoid(y) * norm(o, "post_w", "post_b")
    h = norm(r, "pre_w", "pre_b")
    grads = torch.autograd.grad([r, h], list(leaf.values()),
                                [s.dr.double().cpu(), s.dh.double().cpu()])
    return r.detach(), h.detach(), dict(zip(s.names, grads))


@pytest.mark.parametrize("bits", [8, 32])
def test_training_steps(cuda, bits):
    s = Step(cuda, bits)
    for t in (1, 2, 3):
        r, h, grads = float64_gradients(s)
        got_r, got_h = s.gradients()
        rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())  # noqa: E731
        assert rel(got_r, r) < 8 * 2.0 ** -8 and rel(got_h, h) < 8 * 2.0 ** -8
        for k in s.names:
            assert rel(s.grad[k], grads[k]) < 8 * 2.0 ** -8, (t, k, rel(s.grad[k], grads[k]))
        m0, v0 = (a.clone() for a in ops.adamw_states(s.plan))
        before = {k: np64(s.p[k]) for k in s.names}
        ops.adamw_step(s.plan, t, **HP)
        for i, k in enumerate(s.names):
            at = slice(s.plan.starts[i], s.plan.starts[i] + s.plan.numel[i])
            shape = before[k].shape
            want, m, v = ref_adamw.step(before[k], np64(s.grad[k]), np64(m0[at]).reshape(shape),
                                        np64(v0[at]).reshape(shape), t, **HP)
            u = 2.0 ** -24
            big = np.abs(HP["beta1"] * np64(m0[at]).reshape(shape)) + 0.1 * np.abs(
                np64(s.grad[k]) * HP["grad_scale"])
            rate = HP["lr"] / (1 - 0.9 ** t) / (np.sqrt(v / (1 - 0.99 ** t)) + 1e-8)
            tol = rate * (6 * u * big + 14 * u * np.abs(m)) + 4 * u * np.abs(before[k])
            assert (np.abs(np64(s.p[k]) - want) <= tol).all(), (t, k)
            if k in s.copy:
                assert torch.equal(s.copy[k], s.p[k].bfloat16())


@pytest.mark.parametrize("bits", [8, 32])
def test_captured_training_step(cuda, bits):
    """One captured step, replayed with new hyperparameters and eager work in between, leaves the
    bits that eager steps leave."""
    eager, s = Step(cuda, bits), Step(cuda, bits)
    warm = Step(cuda, bits, seed=1)  # allocations and code objects, outside the capture
    warm.hyper.copy_(ops.adamw_hyper(1, 1e-3))
    warm.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = s.run()
    for t in (1, 2, 3, 4):
        hyper = ops.adamw_hyper(t, 3e-3 / t, HP["beta1"], HP["beta2"], 0.5)
        for x in out:
            x.fill_(float("nan"))
        for x in s.grad.values():
            x.fill_(float("nan"))
        s.hyper.copy_(hyper)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager.hyper.copy_(hyper)
        want = eager.run()
        for a, b in zip(list(out) + s.tensors(), list(want) + eager.tensors()):
            assert torch.equal(a, b), t


@pytest.mark.parametrize("m,v", [(300, 500), (6000, 3000), (40000, 500), (5000, 60)])
def test_captured_embedding_gradient(cuda, m, v):
    """Each way of the gradient in a graph, replayed on new ids and gradients."""
    c = 72
    dout, ids = torch.zeros(m, c, device=cuda).bfloat16(), torch.zeros(m, device=cuda).long()
    ops.embedding_bwd(dout, ids, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.embedding_bwd(dout, ids, v, 2.0)
    for seed in range(3):
        g = torch.Generator().manual_seed(seed)
        dout.copy_(torch.randn(m, c, generator=g).bfloat16())
        ids.copy_(torch.randint(-2, v, (m,), generator=g))
        got.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, ops.embedding_bwd(dout, ids, v, 2.0)), seed


def test_calls_at_once(cuda):
    """Calls from four threads on streams of their own: each has its own workspace and result."""
    torch.cuda.synchronize()
    errors = []

    def work(k):
        try:
            stream = torch.cuda.Stream()
            g = torch.Generator().manual_seed(k)
            with torch.cuda.stream(stream):
                ids = torch.randint(-1, 700, (9000,), generator=g).to(cuda)
                d = torch.randn(9000, 96, generator=g).bfloat16().to(cuda)
                want = ops.embedding_bwd(d, ids, 700).clone()
                joined = [t.clone() for t in ops.residual_norm_bwd(
                    d, d, d, None, None, (want[0, :96].contiguous(), None), d, d) if t is not None]
                for _ in range(20):
                    again = ops.embedding_bwd(d, ids, 700)
                    more = [t for t in ops.residual_norm_bwd(
                        d, d, d, None, None, (want[0, :96].contiguous(), None), d, d)
                        if t is not None]
                    stream.synchronize()
                    assert torch.equal(again, want)
                    assert all(torch.equal(a, b) for a, b in zip(more, joined))
        except Exception as e:  # noqa: BLE001
            errors.append((k, e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
