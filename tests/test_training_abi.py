"""Refusals of the embedding, residual-join and AdamW entries, and AdamW's table, on the CPU: every
call below fails in the host's checks or works on host memory only; nothing is launched."""
import ctypes

import numpy as np
import pytest
import torch

import colabfold_legacy_kernels as clk
from colabfold_legacy_kernels import _native, ops

pytestmark = pytest.mark.skipif(not clk.available("gfx950"), reason="library not built")

OK, INVALID = _native.OK, _native.INVALID_ARGUMENT
BF16, F16, F32, U8, S32, S64 = (_native.BF16, _native.F16, _native.F32, _native.U8, _native.S32,
                                _native.S64)
FAKE = 0x100000  # a non-null, 16-byte aligned address that is never dereferenced


def embedding(**kw):
    a = dict(stream=None, dtype=BF16, table=FAKE, ids_dtype=S32, ids=FAKE, out=FAKE, M=4, V=8,
             C=16, scale=1.0)
    a.update(kw)
    return _native.lib().clk_embedding_fwd(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=U8), "dtype"), (dict(ids_dtype=F32), "ids"), (dict(M=-1), "expected"),
    (dict(C=0), "expected"), (dict(V=-1), "expected"), (dict(M=(1 << 30) + 1), "too large"),
    (dict(V=1 << 30), "too large"), (dict(M=1 << 20, C=1 << 19), "too large"),
    (dict(table=None), "null"), (dict(ids=None), "null"), (dict(out=None), "null"),
    (dict(table=FAKE + 2), "aligned"), (dict(out=FAKE + 8), "aligned"),
])
def test_embedding_refuses(kw, msg):
    assert embedding(**kw) == INVALID
    assert msg in _native.last_error()


def test_embedding_without_tokens():
    assert embedding(M=0, ids=None, out=None) == OK


def embedding_bwd(**kw):
    a = dict(stream=None, dtype=BF16, dout=FAKE, ids_dtype=S64, ids=FAKE, dtable=FAKE,
             workspace=FAKE, workspace_bytes=1 << 40, M=4, V=8, C=16, scale=1.0)
    a.update(kw)
    return _native.lib().clk_embedding_bwd(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=U8), "dtype"), (dict(ids_dtype=U8), "ids"), (dict(M=-1), "expected"),
    (dict(dout=None), "null"), (dict(dtable=None), "null"), (dict(workspace=None), "null"),
    (dict(dout=FAKE + 2), "aligned"), (dict(dtable=FAKE + 4), "aligned"),
    (dict(workspace=FAKE + 8), "aligned"), (dict(M=1 << 20, C=1 << 19), "too large"),
])
def test_embedding_bwd_refuses(kw, msg):
    assert embedding_bwd(**kw) == INVALID
    assert msg in _native.last_error()


@pytest.mark.parametrize("m,v,c", [(1, 1, 1), (4, 8, 16), (8192, 65, 128), (8193, 65, 128),
                                   (100000, 70000, 33), (1 << 20, 1 << 25, 8)])
def test_embedding_bwd_workspace(m, v, c):
    lib = _native.lib()
    need = lib.clk_embedding_bwd_workspace_size(m, v, c)
    assert 0 < need < 64 * (m + v) + 2 * (m * c * 4) + (1 << 26)
    assert embedding_bwd(M=m, V=v, C=c, workspace_bytes=need - 1) == INVALID
    assert "workspace" in _native.last_error()


def test_embedding_bwd_empty():
    lib = _native.lib()
    assert lib.clk_embedding_bwd_workspace_size(0, 8, 16) == 0
    assert lib.clk_embedding_bwd_workspace_size(-1, 8, 16) == 0
    assert embedding_bwd(V=0, dtable=None) == OK  # no table, no gradient


def residual(**kw):
    a = dict(stream=None, dtype=BF16, norm=0, x=FAKE, o=FAKE, gate=FAKE, post_scale=FAKE,
             post_offset=FAKE, res_scale=FAKE, pre_scale=FAKE, pre_offset=FAKE, r=FAKE, h=FAKE,
             M=4, C=16, eps=1e-5)
    a.update(kw)
    return _native.lib().clk_residual_norm_fwd(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=U8), "dtype"), (dict(norm=2), "norm"), (dict(norm=-1), "norm"),
    (dict(M=-1), "[M,C]"), (dict(C=0), "[M,C]"), (dict(C=(1 << 20) + 1), "too large"),
    (dict(post_scale=None), "offset without"), (dict(pre_scale=None, h=None), "offset without"),
    (dict(h=None), "only with it"), (dict(pre_scale=None, pre_offset=None), "only with it"),
    (dict(x=None), "null"), (dict(o=None), "null"), (dict(r=None), "null"),
    (dict(x=FAKE + 2), "aligned"), (dict(gate=FAKE + 8), "aligned"), (dict(h=FAKE + 4), "aligned"),
])
def test_residual_norm_refuses(kw, msg):
    assert residual(**kw) == INVALID
    assert msg in _native.last_error()


def test_residual_norm_without_rows():
    assert residual(M=0) == OK


def residual_bwd(**kw):
    a = dict(stream=None, dtype=BF16, norm=0, r=FAKE, o=FAKE, gate=FAKE, post_scale=FAKE,
             post_offset=FAKE, res_scale=FAKE, pre_scale=FAKE, dr=FAKE, dh=FAKE, dx=FAKE, d_o=FAKE,
             dgate=FAKE, dpost_scale=FAKE, dpost_offset=FAKE, dres=FAKE, dpre_scale=FAKE,
             dpre_offset=FAKE, ws=FAKE, ws_bytes=1 << 40, M=4, C=16, eps=1e-5)
    a.update(kw)
    return _native.lib().clk_residual_norm_bwd(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(dtype=U8), "dtype"), (dict(norm=7), "norm"), (dict(C=0), "[M,C]"),
    (dict(o=None), "null"), (dict(dx=None), "null"), (dict(d_o=None), "null"),
    (dict(ws=None), "null"), (dict(dr=None, dh=None), "null"), (dict(dh=None), "needed"),
    (dict(r=None), "needed"), (dict(gate=None), "dgate"), (dict(dgate=None), "dgate"),
    (dict(post_scale=None, post_offset=None), "not there"), (dict(res_scale=None), "not there"),
    (dict(pre_scale=None, dh=None), "not there"), (dict(dr=FAKE + 2), "aligned"),
    (dict(ws=FAKE + 4), "aligned"), (dict(ws_bytes=0), "workspace"),
])
def test_residual_norm_bwd_refuses(kw, msg):
    assert residual_bwd(**kw) == INVALID
    assert msg in _native.last_error()


def spread(names, step=1 << 20):
    """Addresses far apart for the named arrays."""
    return {n: FAKE + (i + 1) * step for i, n in enumerate(names)}


@pytest.mark.parametrize("first,second,off", [("out", "table", 0), ("out", "table", 240),
                                              ("table", "out", 112), ("out", "ids", 0),
                                              ("ids", "out", 124)])
def test_embedding_refuses_overlaps(first, second, off):
    at = spread(("table", "ids", "out"))  # out has 4 rows of 32 bytes, the table 8
    at[first] = at[second] + off
    assert embedding(**at) == INVALID
    assert "overlap" in _native.last_error()


@pytest.mark.parametrize("first,second,off", [("dtable", "dout", 0), ("dtable", "dout", 112),
                                              ("dout", "dtable", 496), ("ids", "dtable", 504),
                                              ("workspace", "dout", 112), ("workspace", "ids", 16),
                                              ("workspace", "dtable", 496)])
def test_embedding_bwd_refuses_overlaps(first, second, off):
    at = spread(("dout", "ids", "dtable", "workspace"))
    at[first] = at[second] + off
    assert embedding_bwd(**at) == INVALID
    assert "overlap" in _native.last_error()


@pytest.mark.parametrize("first,second,off", [("r", "x", 0), ("r", "o", 112), ("o", "r", 112),
                                              ("h", "gate", 16), ("h", "r", 0), ("r", "h", 112)])
def test_residual_norm_refuses_overlaps(first, second, off):
    at = spread(("x", "o", "gate", "r", "h"))
    at[first] = at[second] + off
    assert residual(**at) == INVALID
    assert "overlap" in _native.last_error()


@pytest.mark.parametrize("first,second,off", [("dx", "dr", 0), ("dx", "r", 112), ("d_o", "o", 0),
                                              ("dgate", "gate", 0), ("dh", "dx", 16),
                                              ("dx", "d_o", 0), ("dgate", "dx", 112)])
def test_residual_norm_bwd_refuses_overlaps(first, second, off):
    at = spread(("r", "o", "gate", "dr", "dh", "dx", "d_o", "dgate"))
    at[first] = at[second] + off
    assert residual_bwd(**at) == INVALID
    assert "overlap" in _native.last_error()


def test_ops_refuse_host_tensors():
    t = torch.zeros(4, 8)
    for call in (lambda: ops.embedding(t, torch.zeros(3, dtype=torch.long)),
                 lambda: ops.embedding_bwd(t, torch.zeros(4, dtype=torch.long), 3),
                 lambda: ops.residual_norm(t, t),
                 lambda: ops.residual_norm_bwd(t, t, None, None, None, None, t, None),
                 lambda: ops.AdamWPlan([t], [t], [t], [t])):
        with pytest.raises(ops.InvalidArgument):
            call()
    with pytest.raises(ops.InvalidArgument):
        ops.AdamWPlan([], [], [], [])
    with pytest.raises(ops.InvalidArgument):
        ops.adamw_zero_states([t], 4)


# ---- AdamW's table: host memory only ---------------------------------------------------------

def tensors(sizes, bits=32, grad=F32, copy=0, base=1 << 32, gap=4096):
    """clk_adamw_tensor entries of made-up, disjoint addresses."""
    arr = (_native.AdamwTensor * max(1, len(sizes)))()
    at = base
    for i, n in enumerate(sizes):
        t = arr[i]
        for name, size in (("param", 4 * n), ("grad", (4 if grad == F32 else 2) * n),
                           ("exp_avg", n * bits // 8), ("exp_avg_sq", n * bits // 8),
                           ("scales", 8 * -(-n // 256) if bits == 8 else 0),
                           ("copy", 2 * n if copy else 0)):
            if size:
                setattr(t, name, at)
                at += -(-size // gap) * gap
        t.numel, t.grad_dtype, t.copy_dtype = n, grad, copy
    return arr


ENTRY = np.dtype([("p", "<u8"), ("g", "<u8"), ("m", "<u8"), ("v", "<u8"), ("scales", "<u8"),
                  ("copy", "<u8"), ("at", "<i8"), ("n", "<u4"), ("grad", "<u2"), ("cp", "<u2")])


def table(arr, n, bits):
    lib, chunks = _native.lib(), ctypes.c_int64(-1)
    st = lib.clk_adamw_table(arr, n, bits, None, 0, ctypes.byref(chunks))
    if st != OK:
        return st, None
    out = np.zeros(chunks.value, ENTRY)
    count = ctypes.c_int64(-1)
    assert lib.clk_adamw_table(arr, n, bits, out.ctypes.data, out.nbytes, ctypes.byref(count)) == OK
    assert count.value == chunks.value
    if out.nbytes:
        assert lib.clk_adamw_table(arr, n, bits, out.ctypes.data, out.nbytes - 1,
                                   ctypes.byref(count)) == INVALID
    return OK, out


@pytest.mark.parametrize("bits", [8, 32])
@pytest.mark.parametrize("sizes", [[1], [255, 256, 257], [0, 5, 0, 1025, 4096, 3], [10 ** 7 + 3],
                                   [1000] * 3000, [5 * 10 ** 9]])
def test_adamw_table_covers_every_element_once(sizes, bits):
    arr = tensors(sizes, bits, BF16, F16)
    st, rows = table(arr, len(sizes), bits)
    assert st == OK, _native.last_error()
    k, base = 0, 0
    for t, n in zip(arr, sizes):
        done, skipped = 0, False
        while done < n:
            row = rows[k]
            assert row["p"] == t.param + 4 * done and row["g"] == t.grad + 2 * done
            assert row["m"] == t.exp_avg + done * bits // 8
            assert row["v"] == t.exp_avg_sq + done * bits // 8
            assert row["scales"] == (t.scales + 8 * (done // 256) if bits == 8 else 0)
            assert row["copy"] == t.copy + 2 * done and row["at"] == base + done
            assert (row["grad"], row["cp"]) == (BF16, F16)
            assert 0 < row["n"] <= n - done and (row["n"] == n - done or row["n"] % 256 == 0)
            done += int(row["n"])
            k += 1
            if n > 10 ** 6 and not skipped and done > 10 ** 5:  # its first and last chunks
                skipped, k = True, len(rows) - 1
                done = int(rows[k]["p"] - t.param) // 4
        base += -(-n // 256) * 256
    assert k == len(rows)


@pytest.mark.parametrize("change,msg", [
    (dict(param=0), "null"), (dict(grad=0), "null"), (dict(exp_avg=0), "null"),
    (dict(exp_avg_sq=0), "null"), (dict(scales=0), "null"), (dict(numel=-1), "elements"),
    (dict(grad_dtype=U8), "gradient"), (dict(copy=1 << 40, copy_dtype=F32), "copy"),
    (dict(param=(1 << 40) + 2), "misaligned"), (dict(exp_avg=(1 << 40) + 1), "misaligned"),
    (dict(grad=(1 << 40) + 2), "misaligned"),
])
def test_adamw_table_refuses(change, msg):
    arr = tensors([300, 700], 8)
    for k, v in change.items():
        setattr(arr[1], k, v)
    assert table(arr, 2, 8)[0] == INVALID
    assert msg in _native.last_error()


def test_adamw_table_refuses_overlaps():
    def overlap(name, other, off, sizes=(300, 700), which=1):
        arr = tensors(list(sizes), 8, F32, BF16)
        setattr(arr[which], name, getattr(arr[0], other) + off)
        return table(arr, len(sizes), 8)[0]

    assert overlap("param", "param", 0) == INVALID and "overlap" in _native.last_error()
    assert overlap("param", "param", 4 * 299) == INVALID
    assert overlap("param", "param", -4 * 699) == INVALID
    assert overlap("grad", "param", 0) == INVALID        # read while it is written
    assert overlap("copy", "grad", 0) == INVALID
    assert overlap("scales", "exp_avg", 0) == INVALID
    assert overlap("exp_avg_sq", "exp_avg", 0, which=0) == INVALID
    assert overlap("grad", "grad", 0) == OK              # a shared gradient is only read
    arr = tensors([300, 700, 5], 8, gap=4)               # neighbours that touch do not overlap
    assert table(arr, 3, 8)[0] == OK


def test_adamw_table_empty_and_bad_calls():
    lib, chunks = _native.lib(), ctypes.c_int64(-1)
    assert lib.clk_adamw_table(None, 0, 32, None, 0, ctypes.byref(chunks)) == OK
    assert chunks.value == 0
    assert lib.clk_adamw_table(None, 1, 32, None, 0, ctypes.byref(chunks)) == INVALID
    assert lib.clk_adamw_table(None, 0, 16, None, 0, ctypes.byref(chunks)) == INVALID
    assert lib.clk_adamw_table(tensors([1 << 37]), 1, 32, None, 0, ctypes.byref(chunks)) == INVALID


def adamw(**kw):
    a = dict(stream=None, table=FAKE, chunks=1, bits=32, step=1, lr=1e-3, beta1=0.9, beta2=0.999,
             eps=1e-8, decay=0.0, grad_scale=1.0, hyper=None)
    a.update(kw)
    return _native.lib().clk_adamw_step(*a.values())


@pytest.mark.parametrize("kw,msg", [
    (dict(table=None), "table"), (dict(table=FAKE + 8), "table"), (dict(chunks=-1), "chunks"),
    (dict(bits=4), "bits"), (dict(step=0), "step"), (dict(beta1=1.0), "betas"),
    (dict(beta2=-0.1), "betas"), (dict(beta1=float("nan")), "betas"), (dict(eps=0.0), "eps"),
    (dict(eps=1e-60), "eps"), (dict(eps=float("inf")), "eps"), (dict(lr=float("nan")), "lr"),
    (dict(grad_scale=float("inf")), "grad_scale"), (dict(decay=float("nan")), "weight_decay"),
    (dict(hyper=FAKE + 2), "hyper"),
])
def test_adamw_refuses(kw, msg):
    assert adamw(**kw) == INVALID
    assert msg in _native.last_error()


def test_adamw_states_refuses():
    lib = _native.lib()
    assert lib.clk_adamw_states(None, FAKE, 1, 8, None, FAKE) == INVALID
    assert lib.clk_adamw_states(None, FAKE, 1, 8, FAKE, FAKE + 4) == INVALID
    assert lib.clk_adamw_states(None, None, 1, 8, FAKE, FAKE) == INVALID
    assert lib.clk_adamw_states(None, None, 0, 8, None, None) == OK
    assert adamw(chunks=0, table=None) == OK
