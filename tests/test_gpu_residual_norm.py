"""The residual join with its norms, forward and backward, against the float64 oracle.

Tolerances: u = 2^-24. A sum over a row is made of at most C/256 + 32 float32 additions one after
the other (a lane's own, then the lanes', then the waves'), so statistics are off by at most
d*u, d = C/256 + 32, times the mean magnitude of what is summed. Every later operation adds a few u;
the bounds below follow the formula with magnitudes in place of values (sums of absolute terms, no
cancellation), times K = 3*d + 40 + 4*max|gate| roundings, which counts every operation between
input and output (three sums deep in the backward; the sigmoid's argument scales its error by
|gate|). Results in 16 bits add half a step, eps/2 of the value."""
import numpy as np
import pytest
import torch

from _util import np64
from colabfold_legacy_kernels import _native, ops
from oracle import residual_norm as ref

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]
# (gate, post, res_scale, pre), post and pre: 0 none, 1 scale, 2 scale and offset
FULL = (True, 2, True, 2)
FORMS = [FULL, (False, 2, True, 2), (True, 0, True, 2), (True, 2, False, 2), (True, 2, True, 0),
         (False, 0, False, 2), (False, 0, False, 0), (True, 1, True, 1), (False, 1, False, 1)]


def make(shape, dtype, form, seed, dev):
    g = torch.Generator().manual_seed(seed)
    rows = lambda std=1.0, mean=0.0: (torch.randn(shape, generator=g) * std + mean).to(dtype).to(dev)  # noqa
    c = shape[-1]
    vec = lambda std, mean: (torch.randn(c, generator=g) * std + mean).to(dev)  # noqa: E731
    pair = lambda k: None if k == 0 else (vec(0.3, 1.0), vec(0.3, 0.0) if k == 2 else None)  # noqa
    gate, post, scale, pre = form
    return {"x": rows(2.0, 0.3), "o": rows(0.7, 0.2), "gate": rows() if gate else None,
            "post": pair(post), "res_scale": vec(0.2, 0.5) if scale else None, "pre": pair(pre),
            "r": rows(2.0, 0.3), "dr": rows(), "dh": rows() if pre else None}


def h64(t):
    if t is None:
        return None
    return tuple(map(h64, t)) if isinstance(t, tuple) else np64(t)


def _abs_norm(v, pair, kind, eps):
    """(magnitudes of N(v) and of vhat, rstd) with the mean's error counted as if it were not
    cancelled."""
    mean = v.mean(-1, keepdims=True) if kind == "layer" else 0.0
    rstd = 1 / np.sqrt(((v - mean) ** 2).mean(-1, keepdims=True) + eps)
    hat = np.abs((v - mean) * rstd) + rstd * np.abs(v).mean(-1, keepdims=True)
    y = hat * np.abs(pair[0])
    return (y if pair[1] is None else y + np.abs(pair[1])), hat, rstd


def depth(c, gate):
    return 3 * (c / 256 + 32) + 40 + (4 * np.abs(gate).max() if gate is not None and gate.size else 0)


def within(name, got, want, size, k, dtype):
    """|got - want| <= k*u*size, and half a step of the type (with its smallest subnormal)."""
    if want is None:
        assert got is None, name
        return
    info = torch.finfo(dtype)
    half = 0.0 if dtype == torch.float32 else info.eps / 2
    tiny = info.smallest_normal * info.eps
    err = np.abs(np64(got) - want)
    assert np.isfinite(np64(got)).all(), name
    tol = k * U * size * (1 + half) + half * np.abs(want) + tiny
    assert (err <= tol).all(), (name, float((err / tol).max()))


def check_forward(s, r, h, kind, eps):
    a = {k: h64(s[k]) for k in ("x", "o", "gate", "post", "res_scale", "pre")}
    want, _ = ref.residual_norm(**a, kind=kind, eps=eps)
    size = np.abs(a["o"]) if a["post"] is None else _abs_norm(a["o"], a["post"], kind, eps)[0]
    if a["gate"] is not None:
        size = size / (1 + np.exp(-a["gate"]))
    size = size * (1.0 if a["res_scale"] is None else np.abs(a["res_scale"])) + np.abs(a["x"])
    k = depth(r.shape[-1], a["gate"])
    within("r", r, want, size, k, r.dtype)
    if a["pre"] is None:
        assert h is None
        return
    # h is the norm of the stream as it was kept.
    kept = np64(r)
    within("h", h, ref.norm(kept, a["pre"], kind, eps), _abs_norm(kept, a["pre"], kind, eps)[0], k,
           r.dtype)


NAMES = ("dx", "do", "dgate", "dpost_scale", "dpost_offset", "dres_scale", "dpre_scale",
         "dpre_offset")


def check_backward(s, got, kind, eps):
    a = {k: h64(s[k]) for k in ("r", "o", "gate", "post", "res_scale", "pre", "dr", "dh")}
    want = ref.residual_norm_bwd(**a, kind=kind, eps=eps)
    mean = lambda v: v.mean(-1, keepdims=True)  # noqa: E731
    ax = tuple(range(a["o"].ndim - 1))
    sums = {}
    d = np.zeros_like(a["o"]) if a["dr"] is None else np.abs(a["dr"])
    if a["pre"] is not None:
        _, hat, rstd = _abs_norm(a["r"], a["pre"], kind, eps)
        g = np.abs(a["dh"]) * np.abs(a["pre"][0])
        d = d + rstd * (g + mean(g) + hat * mean(g * hat))
        sums["dpre_scale"], sums["dpre_offset"] = np.abs(a["dh"]) * hat, np.abs(a["dh"])
    u = np.abs(a["o"])
    if a["post"] is not None:
        u, ohat, rstd = _abs_norm(a["o"], a["post"], kind, eps)
    sig = 1.0 if a["gate"] is None else 1 / (1 + np.exp(-a["gate"]))
    dt = d * (1.0 if a["res_scale"] is None else np.abs(a["res_scale"]))
    sums["dres_scale"] = d * sig * u
    sizes = {"dx": d, "dgate": dt * u * sig}
    du = dt * sig
    if a["post"] is not None:
        sums["dpost_scale"], sums["dpost_offset"] = du * ohat, du
        g = du * np.abs(a["post"][0])
        du = rstd * (g + mean(g) + ohat * mean(g * ohat))
    sizes["do"] = du
    rows = a["o"].size // a["o"].shape[-1]
    k = depth(a["o"].shape[-1], a["gate"])
    for name, t, w in zip(NAMES, got, want):
        if name in sums:  # a lane's rows one after the other, then slots, waves and blocks
            size = sums[name].sum(ax)
            within(name, t, w, size, k + rows / 256 + 128, torch.float32)
            assert t is None or t.dtype == torch.float32
        else:
            within(name, t, w, sizes.get(name), k, s["r"].dtype)


def backward(s, kind, eps):
    return ops.residual_norm_bwd(s["r"], s["o"], s["gate"], s["post"], s["res_scale"], s["pre"],
                                 s["dr"], s["dh"], kind, eps)


def forward(s, kind, eps):
    return ops.residual_norm(s["x"], s["o"], s["gate"], s["post"], s["res_scale"], s["pre"], kind,
                             eps)


SIZES = [(1, 1), (1, 128), (2, 8), (3, 7), (5, 33), (17, 64), (130, 128), (203, 384), (65, 256),
         (9, 449), (31, 512), (4, 1000), (3, 1344), (2, 2048), (3, 2049), (5, 4096), (2, 4104),
         (2, 5003), (1, 20000), (2053, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("m,c", SIZES)
def test_sizes(cuda, dtype, kind, m, c):
    s = make((m, c), dtype, FULL, m + c, cuda)
    check_forward(s, *forward(s, kind, 1e-5), kind, 1e-5)
    got = backward(s, kind, 1e-5)
    check_backward(s, got, kind, 1e-5)
    for a, b in zip(got, backward(s, kind, 1e-5)):  # the same bits again
        assert torch.equal(a, b)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("m,c", [(70, 128), (9, 61), (3, 3000), (2, 9000)])
def test_forms(cuda, form, kind, m, c):
    for dtype in (torch.bfloat16, torch.float32):
        s = make((m, c), dtype, form, 3, cuda)
        check_forward(s, *forward(s, kind, 1e-3), kind, 1e-3)
        check_backward(s, backward(s, kind, 1e-3), kind, 1e-3)
        if s["dh"] is not None:  # no gradient from the stream's other readers
            s["dr"] = None
            check_backward(s, backward(s, kind, 1e-3), kind, 1e-3)


@pytest.mark.parametrize("m", [40000, 262144 + 3])
def test_many_rows(cuda, m):
    s = make((m, 64), torch.bfloat16, FULL, 7, cuda)
    check_forward(s, *forward(s, "layer", 1e-5), "layer", 1e-5)
    check_backward(s, backward(s, "layer", 1e-5), "layer", 1e-5)


def test_shapes_and_empty(cuda):
    s = make((3, 5, 2, 32), torch.float16, FULL, 1, cuda)
    r, h = forward(s, "layer", 1e-5)
    assert r.shape == h.shape == (3, 5, 2, 32)
    check_forward(s, r, h, "layer", 1e-5)
    check_backward(s, backward(s, "layer", 1e-5), "layer", 1e-5)
    s = make((0, 24), torch.float16, FULL, 1, cuda)
    r, h = forward(s, "layer", 1e-5)
    assert r.shape == h.shape == (0, 24)
    got = backward(s, "layer", 1e-5)
    assert got[0].shape == (0, 24) and all(not t.any() and t.shape == (24,) for t in got[3:])


@pytest.mark.parametrize("c", [128, 129, 5000])
def test_rows_without_variance_and_special_values(cuda, c):
    """Constant rows have a finite norm (eps) and zero eps does not reach other rows; gates of both
    infinities are 0 and 1; a NaN stays in its row."""
    s = make((6, c), torch.float32, FULL, 2, cuda)
    for k in ("x", "o", "r"):
        s[k][1] = 0.0 if k != "o" else 3.0
    s["gate"][2, ::2], s["gate"][2, 1::2] = float("inf"), float("-inf")
    r, h = forward(s, "layer", 1e-5)
    assert torch.isfinite(r).all() and torch.isfinite(h).all()
    assert torch.equal(r[2, 1::2], s["x"][2, 1::2])
    got = backward(s, "layer", 1e-5)
    assert all(torch.isfinite(t).all() for t in got) and not got[2][2].any()
    clean = forward(s, "layer", 1e-5)
    s["o"][4, c // 2] = float("nan")
    r, h = forward(s, "layer", 1e-5)
    assert r[4].isnan().all() and h[4].isnan().all()
    keep = [0, 1, 2, 3, 5]
    assert torch.equal(r[keep], clean[0][keep]) and torch.equal(h[keep], clean[1][keep])
    s = make((5, c), torch.float32, FULL, 2, cuda)  # eps 0: rows of the launch that do not exist
    check_forward(s, *forward(s, "rms", 0.0), "rms", 0.0)
    check_backward(s, backward(s, "rms", 0.0), "rms", 0.0)


def test_extreme_gates(cuda):
    """Gates of the type's lowest and highest values."""
    for dtype in TYPES:
        s = make((4, 64), dtype, FULL, 5, cuda)
        s["gate"][0], s["gate"][1] = torch.finfo(dtype).min, torch.finfo(dtype).max
        r, h = forward(s, "layer", 1e-5)
        assert torch.equal(r[0], s["x"][0])
        got = backward(s, "layer", 1e-5)
        assert all(torch.isfinite(t).all() for t in got)
        assert not got[1][0].any() and not got[2][:2].any()


def test_refusals(cuda):
    s = make((4, 32), torch.bfloat16, FULL, 1, cuda)
    x, o, w = s["x"], s["o"], s["post"]
    bad = [lambda: ops.residual_norm(x, o[:3]), lambda: ops.residual_norm(x, o.half()),
           lambda: ops.residual_norm(x.double(), o.double()),
           lambda: ops.residual_norm(x.t(), o.t()), lambda: ops.residual_norm(x, o, o[:, :16]),
           lambda: ops.residual_norm(x, o, kind="batch"),
           lambda: ops.residual_norm(x, o, post=(w[0].bfloat16(), None)),
           lambda: ops.residual_norm(x, o, post=(w[0][:16], None)),
           lambda: ops.residual_norm(x, o, post=(None, w[1])),
           lambda: ops.residual_norm(x, o, pre=(w[0], w[1][:5])),
           lambda: ops.residual_norm(x, o, res_scale=w[0].half()),
           lambda: ops.residual_norm(x, o, res_scale=w[0].cpu()),
           lambda: ops.residual_norm(x.reshape(-1)[4:100].reshape(3, 32), o[:3]),  # misaligned
           lambda: ops.residual_norm_bwd(x, o, None, None, None, None, None, None),
           lambda: ops.residual_norm_bwd(x, o, None, None, None, None, x, x),
           lambda: ops.residual_norm_bwd(x, o, None, None, None, s["pre"], x, None),
           lambda: ops.residual_norm_bwd(x, o, None, None, None, None, x.float(), None)]
    for call in bad:
        with pytest.raises(ops.InvalidArgument):
            call()


@pytest.mark.parametrize("m,c", [(5, 128), (3, 77), (2, 4999), (300, 64)])
def test_writes_stay_in_their_buffers(cuda, m, c):
    lib, st = _native.lib(), torch.cuda.current_stream(cuda).cuda_stream
    s = make((m, c), torch.float32, FULL, 9, cuda)
    need = lib.clk_residual_norm_bwd_workspace_size(m, c)
    ws = torch.full((need + 512,), 0xA5, dtype=torch.uint8, device=cuda)
    rows = [torch.full((m * c + 64,), 7.5, device=cuda) for _ in range(3)]
    sums = [torch.full((c + 64,), 7.5, device=cuda) for _ in range(5)]
    p = lambda t: t.data_ptr()  # noqa: E731
    assert lib.clk_residual_norm_bwd(
        st, _native.F32, 0, p(s["r"]), p(s["o"]), p(s["gate"]), p(s["post"][0]), p(s["post"][1]),
        p(s["res_scale"]), p(s["pre"][0]), p(s["dr"]), p(s["dh"]), *map(p, rows), *map(p, sums),
        p(ws), need, m, c, 1e-5) == _native.OK
    assert (ws[need:] == 0xA5).all()
    assert all((t[m * c:] == 7.5).all() for t in rows) and all((t[c:] == 7.5).all() for t in sums)
    got = [t[:m * c].reshape(m, c) for t in rows] + [t[:c] for t in sums]
    check_backward(s, got, "layer", 1e-5)
    out = [torch.full((m * c + 64,), 7.5, device=cuda) for _ in range(2)]
    assert lib.clk_residual_norm_fwd(
        st, _native.F32, 0, p(s["x"]), p(s["o"]), p(s["gate"]), p(s["post"][0]), p(s["post"][1]),
        p(s["res_scale"]), p(s["pre"][0]), p(s["pre"][1]), *map(p, out), m, c, 1e-5) == _native.OK
    assert all((t[m * c:] == 7.5).all() for t in out)


def test_offsets_past_32_bits(cuda):
    """More than 2^31 elements: the last rows and the sums over all of them."""
    m, c = 2_200_000, 1024
    o = torch.zeros(m, c, dtype=torch.bfloat16, device=cuda)
    tail = make((6, c), torch.bfloat16, (False, 0, True, 0), 3, cuda)
    o[-6:] = tail["o"]
    x = torch.zeros_like(o)
    x[-6:] = tail["x"]
    r, _ = ops.residual_norm(x, o, None, None, tail["res_scale"])
    assert torch.equal(r[-6:], ops.residual_norm(tail["x"], tail["o"], None, None,
                                                 tail["res_scale"])[0]) and not r[:100].any()
    del r
    x[-6:] = tail["dr"]
    got = ops.residual_norm_bwd(x, o, None, None, tail["res_scale"], None, x, None)
    want = ops.residual_norm_bwd(tail["dr"], tail["o"], None, None, tail["res_scale"], None,
                                 tail["dr"], None)
    assert torch.equal(got[0][-6:], want[0]) and torch.equal(got[1][-6:], want[1])
    torch.testing.assert_close(got[5], want[5], rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("form", [FULL, (False, 0, False, 2), (True, 1, True, 0)])
def test_autograd(cuda, form):
    s = make((6, 5, 64), torch.bfloat16, form, 11, cuda)
    leaf = lambda t: None if t is None else t.clone().requires_grad_()  # noqa: E731
    post, pre = s["post"] or (None, None), s["pre"] or (None, None)
    leaves = [leaf(t) for t in (s["x"], s["o"], s["gate"], post[0], post[1], s["res_scale"],
                                pre[0], pre[1])]
    r, h = ops.ResidualNormFunction.apply(*leaves, "layer", 1e-5)
    there = [t for t in leaves if t is not None]
    outs, douts = ([r], [s["dr"]]) if h is None else ([r, h], [s["dr"], s["dh"]])
    grads = torch.autograd.grad(outs, there, douts, retain_graph=True)
    want = ops.residual_norm_bwd(r.detach(), s["o"], s["gate"], s["post"], s["res_scale"],
                                 s["pre"], s["dr"], s["dh"])
    want = [t for t in want if t is not None]
    assert len(grads) == len(want)
    for a, b in zip(grads, want):
        assert torch.equal(a, b)
    # One output alone.
    gx, = torch.autograd.grad(r, leaves[0], s["dr"], retain_graph=True)
    assert torch.equal(gx, s["dr"])
    if h is not None:
        gx, = torch.autograd.grad(h.sum(), leaves[0])
        zero = torch.zeros_like(s["dr"])
        assert torch.equal(gx, ops.residual_norm_bwd(
            r.detach(), s["o"], s["gate"], s["post"], s["res_scale"], s["pre"], zero,
            torch.ones_like(zero))[0])
