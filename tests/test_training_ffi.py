"""The XLA FFI targets of the embedding and the residual join through a fake XLA runtime: every decode
error on the CPU (nothing is launched), and on the GPU the same bits as the ops calls."""
import ctypes

import pytest
import torch

import colabfold_legacy_kernels as clk
from colabfold_legacy_kernels import ops
from _xla_ffi import BF16, F16, F32, F64, S32, S64, U8, FakeXla, ApiVersion, ExtensionBase, \
    Metadata, MetadataExtension

pytestmark = pytest.mark.skipif(not clk.available("gfx950"), reason="library not built")

TARGETS = ["ClkEmbedding", "ClkEmbeddingBwd", "ClkResidualNorm", "ClkResidualNormBwd"]
FAKE = 0x100000
DT = {torch.bfloat16: BF16, torch.float16: F16, torch.float32: F32, torch.uint8: U8,
      torch.int32: S32, torch.int64: S64}


def library():
    return ctypes.CDLL(clk.library_path("attention", "gfx950"))


def test_locator_names_the_targets():
    assert [clk.symbol(k, "gfx950") for k in ("embedding", "embedding_bwd", "residual_norm",
                                              "residual_norm_bwd")] == TARGETS


@pytest.mark.parametrize("name", TARGETS)
def test_metadata_and_other_stages(name):
    x, lib = FakeXla(), library()
    md = Metadata(ctypes.sizeof(Metadata), ApiVersion(), 0)
    ext = MetadataExtension(ExtensionBase(ctypes.sizeof(MetadataExtension), 1, None),
                            ctypes.pointer(md))
    assert x.call(lib, name, x.frame([], [], extension=ext)) is None
    assert md.traits == 1
    for stage in (0, 1, 2):
        assert x.call(lib, name, x.frame([], [], stage=stage)) is None
    assert x.errors == []


def refused(name, args, rets, attrs, msg):
    x = FakeXla()
    frame = x.frame([x.buffer(d, s, FAKE) for d, s in args], [x.buffer(d, s, FAKE) for d, s in rets],
                    attrs)
    assert x.call(library(), name, frame) is not None
    code, text = x.errors[-1]
    assert code == 3 and msg in text, text


SCALE = [("scale", F32, 1.0)]


@pytest.mark.parametrize("args,rets,attrs,msg", [
    ([(BF16, (8, 16))], [(BF16, (4, 16))], SCALE, "expects"),
    ([(U8, (8, 16)), (S32, (4,))], [(BF16, (4, 16))], SCALE, "table"),
    ([(BF16, (8, 16)), (F32, (4,))], [(BF16, (4, 16))], SCALE, "ids"),
    ([(BF16, (8, 16)), (S64, (4, 2))], [(BF16, (4, 16))], SCALE, "out"),
    ([(BF16, (8, 16)), (S64, (4,))], [(F16, (4, 16))], SCALE, "out"),
    ([(BF16, (8, 16)), (S64, (4,))], [(BF16, (4, 16))], [], "scale"),
])
def test_embedding_refuses(args, rets, attrs, msg):
    refused("ClkEmbedding", args, rets, attrs, msg)


@pytest.mark.parametrize("args,rets,attrs,msg", [
    ([(BF16, (4, 16)), (S32, (4,))], [(F32, (8, 16))], SCALE, "expects"),
    ([(BF16, (4, 16)), (S32, (4,))], [(BF16, (8, 16)), (U8, (64,))], SCALE, "dtable"),
    ([(BF16, (4, 16)), (U8, (4,))], [(F32, (8, 16)), (U8, (64,))], SCALE, "ids"),
    ([(BF16, (5, 16)), (S32, (4,))], [(F32, (8, 16)), (U8, (64,))], SCALE, "dout"),
    ([(BF16, (4, 16)), (S32, (4,))], [(F32, (8, 16)), (F32, (64,))], SCALE, "workspace"),
    ([(BF16, (4, 16)), (S32, (4,))], [(F32, (200, 16)), (U8, (1,))], SCALE, "workspace 1 bytes"),
    ([(BF16, (4, 16)), (S32, (4,))], [(F32, (8, 16)), (U8, (64,))], [], "scale"),
])
def test_embedding_bwd_refuses(args, rets, attrs, msg):
    refused("ClkEmbeddingBwd", args, rets, attrs, msg)


def join_attrs(gate=1, post=2, res_scale=1, pre=2, rms=0, drop=None):
    a = [("gate", S64, gate), ("post", S64, post), ("res_scale", S64, res_scale),
         ("pre", S64, pre), ("rms", S64, rms), ("eps", F32, 1e-5)]
    return [t for t in a if t[0] != drop]


ROW, VEC = (BF16, (4, 16)), (F32, (16,))
FULL = [ROW] * 3 + [VEC] * 5


@pytest.mark.parametrize("args,rets,attrs,msg", [
    ([ROW], [ROW], join_attrs(), "first two"),
    ([ROW, (BF16, (5, 16))], [ROW], join_attrs(), "first two"),
    ([(U8, (4, 16))] * 2, [ROW], join_attrs(), "first two"),
    (FULL, [ROW, ROW], join_attrs(drop="rms"), "missing"),
    (FULL, [ROW, ROW], join_attrs(drop="eps"), "missing"),
    (FULL, [ROW, ROW], join_attrs(post=3), "post and pre"),
    (FULL, [ROW, ROW], join_attrs(rms=2), "norm"),
    ([ROW, ROW, (BF16, (4, 8))] + [VEC] * 5, [ROW, ROW], join_attrs(), "gate"),
    ([ROW] * 3 + [VEC] * 4 + [(F16, (16,))], [ROW, ROW], join_attrs(), "f32 [C]"),
    (FULL, [ROW], join_attrs(), "do not match"),
    (FULL + [VEC], [ROW, ROW], join_attrs(), "do not match"),
    (FULL, [ROW, (F16, (4, 16))], join_attrs(), "results"),
])
def test_residual_norm_refuses(args, rets, attrs, msg):
    refused("ClkResidualNorm", args, rets, attrs, msg)


@pytest.mark.parametrize("args,rets,attrs,msg", [
    (FULL + [ROW], [ROW] * 3 + [VEC] * 5 + [(U8, (64,))], join_attrs(), "do not match"),
    (FULL + [ROW, ROW], [ROW] * 3 + [VEC] * 4 + [(U8, (64,))], join_attrs(), "do not match"),
    (FULL + [ROW, VEC], [ROW] * 3 + [VEC] * 5 + [(U8, (64,))], join_attrs(), "dr and dh"),
    (FULL + [ROW, ROW], [ROW, ROW, VEC] + [VEC] * 5 + [(U8, (64,))], join_attrs(), "dx, do"),
    (FULL + [ROW, ROW], [ROW] * 3 + [VEC] * 4 + [ROW, (U8, (64,))], join_attrs(), "gradients"),
    (FULL + [ROW, ROW], [ROW] * 3 + [VEC] * 5 + [(F32, (64,))], join_attrs(), "workspace"),
    (FULL + [ROW, ROW], [ROW] * 3 + [VEC] * 5 + [(U8, (1,))], join_attrs(), "workspace 1 bytes"),
])
def test_residual_norm_bwd_refuses(args, rets, attrs, msg):
    refused("ClkResidualNormBwd", args, rets, attrs, msg)


def buf(x, t):
    return x.buffer(DT[t.dtype], tuple(t.shape), t.data_ptr())


@pytest.mark.gpu
@pytest.mark.parametrize("idt", [torch.int32, torch.int64])
def test_embedding_targets_on_the_gpu(cuda, idt):
    lib, x = library(), FakeXla(stream=torch.cuda.current_stream(cuda).cuda_stream)
    table = torch.randn(300, 40, device=cuda).bfloat16()
    ids = torch.randint(-1, 300, (6, 50), device=cuda).to(idt)
    out = torch.empty(6, 50, 40, dtype=torch.bfloat16, device=cuda)
    fr = x.frame([buf(x, table), buf(x, ids)], [buf(x, out)], [("scale", F64, 2.5)])
    assert x.call(lib, "ClkEmbedding", fr) is None, x.errors
    assert torch.equal(out, ops.embedding(table, ids, 2.5))
    size = lib.clk_embedding_bwd_workspace_size
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_int64] * 3
    ws = torch.empty(size(300, 300, 40), dtype=torch.uint8, device=cuda)
    dtable = torch.empty(300, 40, device=cuda)
    fr = x.frame([buf(x, out), buf(x, ids)], [buf(x, dtable), buf(x, ws)], [("scale", F32, 2.5)])
    assert x.call(lib, "ClkEmbeddingBwd", fr) is None, x.errors
    assert torch.equal(dtable, ops.embedding_bwd(out, ids, 300, 2.5))


@pytest.mark.gpu
@pytest.mark.parametrize("gate,post,res_scale,pre,rms", [(1, 2, 1, 2, 0), (0, 1, 1, 1, 1),
                                                         (1, 0, 0, 2, 0), (0, 0, 1, 0, 0)])
def test_residual_norm_targets_on_the_gpu(cuda, gate, post, res_scale, pre, rms):
    lib, xla = library(), FakeXla(stream=torch.cuda.current_stream(cuda).cuda_stream)
    g = torch.Generator().manual_seed(3)
    row = lambda: torch.randn((3, 7, 96), generator=g).bfloat16().to(cuda)  # noqa: E731
    vec = lambda: torch.randn(96, generator=g).to(cuda)  # noqa: E731
    x, o, dr, dh = row(), row(), row(), row()
    gt = row() if gate else None
    pair = lambda n: (vec(), vec() if n == 2 else None) if n else None  # noqa: E731
    pst, a, pr = pair(post), vec() if res_scale else None, pair(pre)
    extra = [t for t in (gt, *(pst or ()), a, *(pr or ())) if t is not None]
    attrs = join_attrs(gate, post, res_scale, pre, rms)
    kind = "rms" if rms else "layer"
    r, h = torch.empty_like(x), torch.empty_like(x)
    fr = xla.frame([buf(xla, t) for t in [x, o] + extra],
                   [buf(xla, t) for t in ([r, h] if pre else [r])], attrs)
    assert xla.call(lib, "ClkResidualNorm", fr) is None, xla.errors
    want = ops.residual_norm(x, o, gt, pst, a, pr, kind)
    assert torch.equal(r, want[0]) and (not pre or torch.equal(h, want[1]))
    want = [t for t in ops.residual_norm_bwd(r, o, gt, pst, a, pr, dr, dh if pre else None, kind)
            if t is not None]
    got = [torch.empty_like(t) for t in want]
    size = lib.clk_residual_norm_bwd_workspace_size
    size.restype, size.argtypes = ctypes.c_size_t, [ctypes.c_int64] * 2
    ws = torch.empty(size(21, 96), dtype=torch.uint8, device=cuda)
    fr = xla.frame([buf(xla, t) for t in [r, o] + extra + ([dr, dh] if pre else [dr])],
                   [buf(xla, t) for t in got + [ws]], attrs)
    assert xla.call(lib, "ClkResidualNormBwd", fr) is None, xla.errors
    for t, w in zip(got, want):
        assert torch.equal(t, w)
