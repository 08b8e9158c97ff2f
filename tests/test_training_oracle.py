"""The float64 oracle of the embedding, the residual join and AdamW, on the CPU: against torch's own
routines and autograd in float64, and against central differences."""
import numpy as np
import pytest
import torch

from oracle import adamw, embedding, residual_norm


def test_embedding_against_torch():
    rng = np.random.default_rng(0)
    table = rng.normal(size=(7, 5))
    ids = rng.integers(0, 7, size=(4, 6))
    dout = rng.normal(size=(4, 6, 5))
    t = torch.tensor(table, requires_grad=True)
    y = 1.5 * torch.nn.functional.embedding(torch.tensor(ids), t)
    y.backward(torch.tensor(dout))
    np.testing.assert_allclose(embedding.embedding(table, ids, 1.5), y.detach().numpy())
    np.testing.assert_allclose(embedding.embedding_bwd(dout, ids, 7, 1.5), t.grad.numpy())


def test_embedding_absent_tokens():
    table, ids = np.arange(6.0).reshape(3, 2), np.array([-1, 2, 3, 0])
    np.testing.assert_array_equal(embedding.embedding(table, ids, 2.0),
                                  [[0, 0], [8, 10], [0, 0], [0, 2]])
    np.testing.assert_array_equal(embedding.embedding_bwd(np.ones((4, 2)), ids, 3),
                                  [[1, 1], [0, 0], [1, 1]])


def _torch_norm(x, scale, offset, kind):
    c = (x.shape[-1],)
    if kind == "layer":
        return torch.nn.functional.layer_norm(x, c, scale, offset, 1e-5)
    y = torch.nn.functional.rms_norm(x, c, scale, 1e-5)
    return y if offset is None else y + offset


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("gate,post,scale", [(True, True, True), (False, True, True),
                                             (True, False, False)])
def test_residual_norm_against_autograd(kind, gate, post, scale):
    g = torch.Generator().manual_seed(3)
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64).requires_grad_()  # noqa
    m, c = 5, 12
    x, o, lg = rand(m, c), rand(m, c), rand(m, c) if gate else None
    pw, pb = (rand(c), rand(c)) if post else (None, None)
    a, nw, nb = rand(c) if scale else None, rand(c), rand(c)
    dr, dh = rand(m, c).detach(), rand(m, c).detach()
    t = _torch_norm(o, pw, pb, kind) if post else o
    t = torch.sigmoid(lg) * t if gate else t
    r = x + (a * t if scale else t)
    h = _torch_norm(r, nw, nb, kind)
    leaves = [t_ for t_ in (x, o, lg, pw, pb, a, nw, nb) if t_ is not None]
    grads = torch.autograd.grad([r, h], leaves, [dr, dh])
    np_ = lambda t_: None if t_ is None else t_.detach().numpy()  # noqa: E731
    args = (np_(o), np_(lg), (np_(pw), np_(pb)) if post else None, np_(a), (np_(nw), np_(nb)))
    r_ref, h_ref = residual_norm.residual_norm(np_(x), *args, kind)
    np.testing.assert_allclose(r_ref, np_(r), rtol=1e-12)
    np.testing.assert_allclose(h_ref, np_(h), rtol=1e-10, atol=1e-12)
    got = residual_norm.residual_norm_bwd(r_ref, *args, np_(dr), np_(dh), kind)
    got = [t_ for t_ in got if t_ is not None]
    assert len(got) == len(grads)
    for t_, ref in zip(got, grads):
        np.testing.assert_allclose(t_, ref.numpy(), rtol=1e-9, atol=1e-11)


def test_residual_norm_against_differences():
    rng = np.random.default_rng(5)
    m, c, step = 3, 6, 1e-6
    x, o, gate, dr, dh = (rng.normal(size=(m, c)) for _ in range(5))
    post, pre = (rng.normal(size=c), rng.normal(size=c)), (rng.normal(size=c), rng.normal(size=c))
    a = rng.normal(size=c)

    def loss(x, o, gate, a):
        r, h = residual_norm.residual_norm(x, o, gate, post, a, pre)
        return (r * dr).sum() + (h * dh).sum()

    r, _ = residual_norm.residual_norm(x, o, gate, post, a, pre)
    grads = residual_norm.residual_norm_bwd(r, o, gate, post, a, pre, dr, dh)
    for k, (v, grad) in enumerate(zip((x, o, gate, a), (grads[0], grads[1], grads[2], grads[5]))):
        for i in np.ndindex(v.shape):
            args = [x, o, gate, a]
            hi, lo = v.copy(), v.copy()
            hi[i] += step
            lo[i] -= step
            d = (loss(*args[:k], hi, *args[k + 1:]) - loss(*args[:k], lo, *args[k + 1:])) / (2 * step)
            assert abs(d - grad[i]) < 1e-6 * max(1.0, abs(d)), (k, i)


def test_adamw_against_torch():
    g = torch.Generator().manual_seed(1)
    p = torch.randn(40, generator=g, dtype=torch.float64)
    q = p.clone().requires_grad_()
    opt = torch.optim.AdamW([q], lr=1e-2, betas=(0.8, 0.99), eps=1e-6, weight_decay=0.1)
    pn, m, v = p.numpy(), np.zeros(40), np.zeros(40)
    for t in range(1, 6):
        q.grad = torch.randn(40, generator=g, dtype=torch.float64)
        opt.step()
        pn, m, v = adamw.step(pn, q.grad.numpy() * 4, m, v, t, 1e-2, 0.8, 0.99, 1e-6, 0.1, 0.25)
        np.testing.assert_allclose(pn, q.detach().numpy(), rtol=1e-12)


def test_adamw_codes():
    """Codes stand for values within half a step in the coded variable; zero blocks are zeros;
    a v above zero stays above zero; a second rounding changes nothing."""
    rng = np.random.default_rng(2)
    m = (rng.normal(size=700) * np.exp(3 * rng.normal(size=700))).astype(np.float32)
    v = np.exp(6 * rng.normal(size=700)).astype(np.float32)
    m[256:512], v[256:512] = 0, 0
    v[0] = 1e-30
    qm, qv, s = adamw.encode(m, v)
    dm, dv = adamw.decode(qm, qv, s)
    assert not dm[256:512].any() and not dv[256:512].any() and s[1].tolist() == [0, 0]
    assert (dv[v > 0] > 0).all() and qv[0] == 1
    sm, sv = (np.repeat(s[:, i], 256)[:700].astype(np.float64) for i in (0, 1))
    rm = np.sqrt(np.abs(m) / np.where(sm > 0, sm, 1))
    # Half a step of the coded variable, and float32's rounding of five operations.
    low, high = (np.maximum(rm + e * 0.5 / 127, 0) ** 2 * sm for e in (-1, 1))
    assert (np.abs(dm) <= high * (1 + 1e-6)).all() and (np.abs(dm) >= low * (1 - 1e-6)).all()
    assert (np.sign(dm) * np.sign(m) >= 0).all()
    rv = np.where(sv > 0, v / np.where(sv > 0, sv, 1), 0) ** 0.25
    high = np.maximum(rv + 0.5 / 255, 1 / 255) ** 4 * sv
    low = np.maximum(rv - 0.5 / 255, 0) ** 4 * sv
    assert (dv <= high * (1 + 1e-6)).all() and (dv >= low * (1 - 1e-6)).all()
    again = adamw.encode(dm, dv)
    assert (again[0] == qm).all() and (again[1] == qv).all()
