"""Token embedding and its gradient against the float64 oracle.

Tolerances. Forward: a float32 product and one rounding to the type t, so at most half a step of
each, relative to the value: eps(t)/2 + 2^-24, and half a smallest subnormal below the normal range.
Gradient: a float32 sum of n terms in any order is off by at most (n - 1) 2^-24 times the sum of
their magnitudes; the scale's rounding and its product add two more."""
import numpy as np
import pytest
import torch

from _util import np64
from colabfold_legacy_kernels import _native, ops
from oracle import embedding as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]
U32 = 2.0 ** -24


def make_ids(m, v, law, g, dtype, absent=0.0):
    if law == "uniform":
        ids = (torch.rand(m, generator=g) * v).long().clamp(max=v - 1)
    elif law == "long_tail":
        ids = torch.exp(torch.rand(m, generator=g) * np.log(v)).long().sub(1).clamp(0, v - 1)
    elif law == "one":
        ids = torch.full((m,), v // 2)
    else:  # sorted runs
        ids = torch.arange(m) * v // max(m, 1)
    if absent:
        bad = torch.tensor([-1, v, -2 ** 31, 2 ** 31 - 1])[torch.randint(0, 4, (m,), generator=g)]
        ids = torch.where(torch.rand(m, generator=g) < absent, bad, ids)
    return ids.to(dtype)


def check_forward(out, table, ids, scale):
    want = ref.embedding(np64(table), ids.cpu().numpy(), scale)
    half = torch.finfo(table.dtype).eps / 2 + U32 + 2.0 ** -23 * (scale != 1.0)
    tiny = torch.finfo(table.dtype).smallest_normal * torch.finfo(table.dtype).eps / 2
    err = np.abs(np64(out) - want)
    assert (err <= half * np.abs(want) + tiny).all(), float((err - half * np.abs(want)).max())


def check_gradient(got, dout, ids, rows, scale):
    d, i = np64(dout), ids.cpu().numpy()
    want = ref.embedding_bwd(d, i, rows, scale)
    size = ref.embedding_bwd(np.abs(d), i, rows, abs(scale))
    count = np.bincount(i[(i >= 0) & (i < rows)].reshape(-1), minlength=rows)[:, None]
    err = np.abs(np64(got) - want)
    assert (err <= (count + 3) * U32 * size + 1e-37).all(), float((err / (size + 1e-30)).max())
    assert not np64(got)[count[:, 0] == 0].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,v,c", [(1, 1, 1), (3, 2, 7), (64, 22, 256), (129, 65, 128), (7, 5, 8),
                                   (1000, 300, 449), (33, 9, 24), (5, 4, 20000), (300, 11, 3)])
def test_forward(cuda, dtype, m, v, c):
    g = torch.Generator().manual_seed(m + c)
    table = torch.randn(v, c, generator=g).to(dtype).to(cuda)
    for idt in (torch.int32, torch.int64):
        ids = make_ids(m, v, "uniform", g, idt, 0.2).to(cuda)
        for scale in (1.0, 11.25, 0.3):
            check_forward(ops.embedding(table, ids, scale), table, ids, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("law", ["uniform", "long_tail", "one", "runs"])
@pytest.mark.parametrize("m,v,c", [
    (1, 1, 1), (1, 9, 16), (31, 3, 8), (32, 3, 8), (33, 3, 8), (64, 22, 256), (257, 300, 129),
    (1500, 65, 128), (8192, 40, 24), (8193, 65, 64), (9000, 255, 40), (9000, 256, 40),
    (20000, 70000, 12), (70000, 23, 36), (5000, 2, 1100)])
def test_gradient(cuda, dtype, law, m, v, c):
    g = torch.Generator().manual_seed(m + v + c)
    dout = torch.randn(m, c, generator=g).to(dtype).to(cuda)
    ids = make_ids(m, v, law, g, torch.int64 if m % 2 else torch.int32, 0.1).to(cuda)
    got = ops.embedding_bwd(dout, ids, v, 1.5)
    check_gradient(got, dout, ids, v, 1.5)
    assert torch.equal(got, ops.embedding_bwd(dout, ids, v, 1.5))  # the same bits again


@pytest.mark.parametrize("m", [40, 30000])
def test_gradient_of_absent_tokens_only(cuda, m):
    dout = torch.full((m, 16), float("nan"), device=cuda, dtype=torch.bfloat16)
    ids = torch.full((m,), -1, device=cuda)
    assert torch.equal(ops.embedding_bwd(dout, ids, 7), torch.zeros(7, 16, device=cuda))
    # Absent among others: what their rows of dout hold reaches nothing.
    dout[::2] = 1
    ids[::2] = 3
    got = ops.embedding_bwd(dout, ids, 7)
    assert (got[3] == (m + 1) // 2).all() and got.sum() == 16 * ((m + 1) // 2)


def test_special_values(cuda):
    table = torch.tensor([[float("inf"), -0.0, float("nan"), 65504.0]], device=cuda).half()
    ids = torch.tensor([0, 5, -1], device=cuda)
    out = ops.embedding(table, ids, 2.0)
    assert out[0, 0] == float("inf") and out[0, 2].isnan() and out[0, 3] == float("inf")
    assert not out[1:].any()
    assert not ops.embedding(table, ids, float("inf"))[1:].any()
    # A NaN gradient stays in its row.
    dout = torch.ones(4, 8, device=cuda)
    dout[1] = float("nan")
    got = ops.embedding_bwd(dout, torch.tensor([0, 1, 2, 2], device=cuda), 4, 3.0)
    assert got[1].isnan().all()
    assert torch.equal(got[[0, 2, 3]], torch.tensor([3.0, 6.0, 0.0], device=cuda)[:, None].expand(3, 8))


def test_shapes_and_empty(cuda):
    table = torch.randn(6, 16, device=cuda)
    ids = torch.randint(0, 6, (2, 3, 5), device=cuda)
    out = ops.embedding(table, ids)
    assert out.shape == (2, 3, 5, 16) and torch.equal(out, table[ids])
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    assert ops.embedding(table, none).shape == (0, 16)
    got = ops.embedding_bwd(torch.empty(0, 16, device=cuda), none, 6)
    assert torch.equal(got, torch.zeros(6, 16, device=cuda))
    assert ops.embedding_bwd(out, ids, 0).shape == (0, 16)
    assert not ops.embedding(table[:0], ids).any()
    one = torch.tensor(4, device=cuda)
    assert torch.equal(ops.embedding(table, one), table[4])


def test_refusals(cuda):
    table, ids = torch.randn(6, 16, device=cuda), torch.zeros(4, dtype=torch.int64, device=cuda)
    dout = torch.randn(4, 16, device=cuda)
    bad = [lambda: ops.embedding(table.double(), ids), lambda: ops.embedding(table, ids.short()),
           lambda: ops.embedding(table.t(), ids), lambda: ops.embedding(table[0], ids),
           lambda: ops.embedding(table.reshape(-1)[4:84].reshape(5, 16)[:, 1:], ids),
           lambda: ops.embedding(table.reshape(-1)[1:81].reshape(5, 16), ids),  # misaligned
           lambda: ops.embedding(table, ids.cpu()), lambda: ops.embedding_bwd(dout, ids[:3], 6),
           lambda: ops.embedding_bwd(dout, ids.float(), 6),
           lambda: ops.embedding_bwd(dout.double(), ids, 6),
           lambda: ops.embedding_bwd(dout, ids, -1),
           lambda: ops.embedding_bwd(dout.t().contiguous().t(), ids, 6)]
    for call in bad:
        with pytest.raises(ops.InvalidArgument):
            call()


@pytest.mark.parametrize("m,v,c", [(50, 30, 33), (9001, 300, 64), (70, 3, 128)])
def test_writes_stay_in_their_buffers(cuda, m, v, c):
    """Guard bytes behind the table's gradient and the workspace, and around out, stay."""
    g = torch.Generator().manual_seed(4)
    lib, st = _native.lib(), torch.cuda.current_stream(cuda).cuda_stream
    ids = make_ids(m, v, "long_tail", g, torch.int32, 0.1).to(cuda)
    dout = torch.randn(m, c, generator=g).to(cuda)
    need = lib.clk_embedding_bwd_workspace_size(m, v, c)
    ws = torch.full((need + 512,), 0xA5, dtype=torch.uint8, device=cuda)
    dt = torch.full((v * c + 64,), 7.5, device=cuda)
    assert lib.clk_embedding_bwd(st, _native.F32, dout.data_ptr(), _native.S32, ids.data_ptr(),
                                 dt.data_ptr(), ws.data_ptr(), need, m, v, c, 1.0) == _native.OK
    assert (ws[need:] == 0xA5).all() and (dt[v * c:] == 7.5).all()
    check_gradient(dt[:v * c].reshape(v, c), dout, ids, v, 1.0)
    out = torch.full((m * c + 64,), 7.5, device=cuda)
    table = torch.randn(v, c, generator=g).to(cuda)
    assert lib.clk_embedding_fwd(st, _native.F32, table.data_ptr(), _native.S32, ids.data_ptr(),
                                 out.data_ptr(), m, v, c, 1.0) == _native.OK
    assert (out[m * c:] == 7.5).all()


def test_offsets_past_32_bits(cuda):
    """A table, an output and a gradient of more than 2^31 elements; rows of both ends."""
    v, c = 2_200_000, 1024
    table = torch.empty(v, c, dtype=torch.bfloat16, device=cuda)
    far = torch.tensor([0, 1, v // 2, v - 2, v - 1], device=cuda)
    rows = torch.randn(5, c, device=cuda).bfloat16()
    table[far] = rows
    assert torch.equal(ops.embedding(table, far), rows)
    ids = torch.zeros(v, dtype=torch.int32, device=cuda)
    ids[far] = far.int()
    out = ops.embedding(table, ids)
    assert torch.equal(out[far], rows) and torch.equal(out[v - 5:v - 2], rows[:1].expand(3, c))
    del table
    out.zero_()
    out[far] = rows
    got = ops.embedding_bwd(out, ids, v)
    assert torch.equal(got[far], rows.float()) and not got[2:v // 2].any()


def test_autograd_and_streams(cuda):
    table = torch.randn(40, 64, device=cuda, dtype=torch.bfloat16, requires_grad=True)
    ids = torch.randint(-1, 40, (50, 3), device=cuda)
    dout = torch.randn(50, 3, 64, device=cuda).bfloat16()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = ops.EmbeddingFunction.apply(table, ids, 8.0)
        grad, = torch.autograd.grad(y, table, dout)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(y, ops.embedding(table.detach(), ids, 8.0))
    assert grad.dtype == torch.bfloat16
    assert torch.equal(grad, ops.embedding_bwd(dout, ids, 40, 8.0).bfloat16())
    # A gradient that is not contiguous (an expanded one).
    y = ops.EmbeddingFunction.apply(table, ids, 8.0)
    grad, = torch.autograd.grad(y.sum(), table)
    assert torch.equal(grad, ops.embedding_bwd(torch.ones_like(dout), ids, 40, 8.0).bfloat16())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,v,c", [
    (2048, 145, 8), (2049, 500, 16), (8192, 1000, 40), (16384, 3000, 24), (20481, 145, 72),
    (65536, 100000, 8), (65537, 200, 8), (70001, 255, 17), (70001, 256, 8), (140000, 70000, 12),
    (70000, 20_000_000, 1)])
@pytest.mark.parametrize("law", ["uniform", "long_tail", "one"])
def test_gradient_by_sorted_tokens(cuda, dtype, m, v, c, law):
    """Every way of sorting, at its first and last number of tokens, and of 1 to 4 digits of ids."""
    g = torch.Generator().manual_seed(m + v)
    dout = torch.randn(m, c, generator=g).to(dtype).to(cuda)
    ids = make_ids(m, v, law, g, torch.int64 if m % 2 else torch.int32, 0.1).to(cuda)
    got = ops.embedding_bwd(dout, ids, v, 0.5)
    if v > 10 ** 6:  # compare the rows that are named; the others are zero
        there = ids[(ids >= 0) & (ids < v)].unique().long()
        named = torch.zeros(v, dtype=torch.bool, device=cuda)
        named[there] = True
        assert not got[~named].any()
        index = torch.full((v + 1,), -1, device=cuda)
        index[there] = torch.arange(len(there), device=cuda)
        ids = torch.where((ids >= 0) & (ids < v), index[ids.clamp(0, v - 1)], -1)
        got, v = got[there], len(there)
    check_gradient(got, dout, ids, v, 0.5)


@pytest.mark.parametrize("seed", range(4))
@pytest.mark.parametrize("c", [4, 300])
def test_gradient_of_runs_of_all_lengths(cuda, seed, c):
    """Runs of equal tokens that end on, before and behind the multiples of any chunk of the sorted
    order, up to thousands of tokens, after a shift of 0 to 40 tokens."""
    rng = np.random.default_rng(seed)
    lengths = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 511, 512, 513,
               1007, 1008, 1009, 1023, 1024, 1025, 1040, 1041, 2047, 2048, 2049, 2064, 3100, 5000]
    rng.shuffle(lengths)
    lengths = [int(rng.integers(0, 41))] + lengths
    ids = np.repeat(np.arange(len(lengths)) * 7 + 3, lengths)
    v = 7 * len(lengths) + 150
    order = rng.permutation(len(ids))
    ids = torch.from_numpy(ids[order]).to(cuda)
    dout = torch.randn(len(ids), c, generator=torch.Generator().manual_seed(seed)).to(cuda)
    check_gradient(ops.embedding_bwd(dout, ids, v), dout, ids, v, 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,v,c", [
    (1, 5000, 16), (31, 5000, 9), (2048, 1153, 40), (4096, 5000, 8), (4097, 5000, 24),
    (8192, 70000, 136), (32768, 5000, 20), (32769, 1153, 8), (40000, 70000, 72)])
@pytest.mark.parametrize("law", ["long_tail", "one", "runs"])
def test_gradient_of_larger_tables(cuda, dtype, m, v, c, law):
    """Tables that are always sorted: by counting (up to 4096 tokens), by digits with few tiles of
    tokens and with more."""
    g = torch.Generator().manual_seed(m + v)
    dout = torch.randn(m, c, generator=g).to(dtype).to(cuda)
    ids = make_ids(m, v, law, g, torch.int64 if m % 2 else torch.int32, 0.1).to(cuda)
    got = ops.embedding_bwd(dout, ids, v, 0.5)
    check_gradient(got, dout, ids, v, 0.5)
    assert torch.equal(got, ops.embedding_bwd(dout, ids, v, 0.5))


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("c", [2, 8, 20, 300])
def test_gradient_of_sorted_runs_of_all_lengths(cuda, seed, c):
    rng = np.random.default_rng(100 + seed)
    lengths = [1, 2, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 239, 240, 241, 255,
               256, 257, 272, 500, 511, 512, 513, 1007, 1008, 1009, 1023, 1024, 1025, 1040, 1041,
               2047, 2048, 2049, 2064, 4095, 4096, 4097, 5000]
    rng.shuffle(lengths)
    lengths = [int(rng.integers(0, 41))] + lengths[:6 if seed == 0 else 12 if seed == 1 else None]
    ids = np.repeat(np.arange(len(lengths)) * 70 + 3, lengths)
    v = 70 * len(lengths) + 1200
    ids = torch.from_numpy(ids[rng.permutation(len(ids))]).to(cuda)
    dout = torch.randn(len(ids), c, generator=torch.Generator().manual_seed(seed)).to(cuda)
    got = ops.embedding_bwd(dout, ids, v)
    check_gradient(got, dout, ids, v, 1.0)
    # Where tokens are sorted, a row's sum has the order of its tokens: another mix of the rows
    # gives the same bits.
    back = torch.argsort(ids, stable=True)
    assert torch.equal(got, ops.embedding_bwd(dout[back].contiguous(), ids[back].contiguous(), v))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("v", [143, 144, 145, 287, 288, 289, 1152])
def test_gradient_at_the_borders_of_row_blocks(cuda, dtype, v):
    """Small calls on tables of up to eight blocks of 144 rows; NaN and infinite gradients stay in
    their rows, those of absent tokens reach nothing."""
    g = torch.Generator().manual_seed(v)
    m, c = 1500, 68
    dout = torch.randn(m, c, generator=g).to(dtype).to(cuda)
    ids = make_ids(m, v, "uniform", g, torch.int64, 0.2).to(cuda)
    ids[:v] = torch.arange(min(v, m), device=cuda)
    clean = ops.embedding_bwd(dout, ids, v, 0.5)
    check_gradient(clean, dout, ids, v, 0.5)
    dout[0], dout[142, 5] = float("nan"), float("inf")
    dout[(ids < 0) | (ids >= v)] = float("nan")
    got = ops.embedding_bwd(dout, ids, v, 0.5)
    hit = torch.zeros(v, dtype=torch.bool, device=cuda)
    hit[0] = hit[142] = True
    size = ref.embedding_bwd(np.abs(np64(dout)), ids.cpu().numpy(), v, 0.5)
    count = np.bincount(ids.cpu().numpy()[((ids >= 0) & (ids < v)).cpu().numpy()], minlength=v)
    ok = (~hit).cpu().numpy()
    err = np.abs(np64(got) - np64(clean))[ok]  # both in some order of the same float32 sums
    assert (err <= 2 * (count[ok][:, None] + 3) * U32 * size[ok] + 1e-37).all()
    assert got[0].isnan().all() and got[142, 5] == float("inf")
    assert torch.isfinite(got[142, torch.arange(c, device=cuda) != 5]).all()


@pytest.mark.parametrize("dtype,unit", [(torch.float16, 2.0 ** -24), (torch.bfloat16, 2.0 ** -133),
                                        (torch.float32, 2.0 ** -133)])
@pytest.mark.parametrize("v", [20, 65, 129, 3000])
def test_gradient_of_subnormal_numbers(cuda, dtype, unit, v):
    """Small multiples of a unit below the normal range: every sum of them is exact."""
    g = torch.Generator().manual_seed(7)
    dout = (torch.randint(-3, 4, (640, 43), generator=g).double() * unit).to(dtype).to(cuda)
    ids = torch.randint(0, v, (640,), generator=g).to(cuda)
    got = ops.embedding_bwd(dout, ids, v)
    want = ref.embedding_bwd(np64(dout), ids.cpu().numpy(), v, 1.0)
    assert np.array_equal(np64(got), want)


@pytest.mark.parametrize("m,v,c", [(1, 1, 5), (700, 30, 100), (5000, 65, 131), (5000, 65, 128),
                                   (900, 129, 256), (4000, 144, 77), (2500, 300, 64)])
def test_float32_gradient_of_single_tokens_is_exact(cuda, m, v, c):
    """A row that one token names is that token's row, to the last bit, at every size from the
    smallest normal number that holds 24 bits above 2^-133 to the largest finite one."""
    g = torch.Generator().manual_seed(11)
    ids = torch.randint(0, max(v // 2, 1), (m,), generator=g)
    alone = torch.arange(max(v // 2, 1), v)[:m]  # rows of one token each
    at = torch.randperm(m, generator=g)[:alone.numel()]
    ids[at] = alone
    x = torch.randn(m, c, generator=g)
    x[at] = torch.randn(alone.numel(), c, generator=g) * 2.0 ** torch.randint(
        -100, 120, (alone.numel(), 1), generator=g).float()
    if m > 1:
        x[at[0], 0] = torch.finfo(torch.float32).max
    got = ops.embedding_bwd(x.to(cuda), ids.to(cuda), v).cpu()
    assert torch.equal(got[ids[at]], x[at])
