"""Compressed SH coefficients on the GPU against plain implementations in 64 bits. u = 2^-24 below
(fp32 unit roundoff); half precisions add half a step of their type."""
import numpy as np
import pytest
import torch

import gs3d
from gs3d import MX4Rows, RenderBuffers, RenderOnlyGaussiansVector, RenderOptions, RenderOutputs, Tiling
from gs3d import compressed as gc
from gs3d.render import render_given_colour
from gs3d.scene import SceneSpec, look_at_camera, synthetic_gaussians
from gs3d.structs import GaussiansVector

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rng(seed):
    return torch.Generator().manual_seed(seed)


def make_indices(n, rows, gen, skew=0.0, invalid=True):
    i = (torch.rand(n, generator=gen) ** (1 + skew) * rows).to(torch.int32).clamp(0, max(rows - 1, 0)) + 1
    if invalid and n >= 8:
        i[:: max(1, n // 7)] = torch.tensor([0, -1, rows + 1, 2**31 - 1, -2**31, 0, rows + 7, 0, -5],
                                            dtype=torch.int32)[: len(i[:: max(1, n // 7)])]
    return i


# -- lookup -----------------------------------------------------------------------------------
LOOKUP_SHAPES = [(1, 1, 1), (1, 5, 48), (7, 1, 3), (33, 4, 27), (1000, 64, 48), (1001, 300, 12), (257, 9, 130),
                 (64, 3, 1021), (5, 2, 65536), (20_003, 5000, 48), (700, 50, 2), (700, 50, 4), (700, 50, 6), (701, 9, 54),
             (300, 9, 514)]


def lookup_exact(table, idx, scale, dtype):
    """The product of two fp32 values is exact in 64 bits, so rounding it to fp32 and then to the
    type is what the kernel is specified to give, bit for bit."""
    padded = torch.cat([torch.zeros(1, table.shape[1], dtype=torch.float64), table.double()])
    i = idx.long()
    i = torch.where((i >= 1) & (i <= table.shape[0]), i, 0)
    return (padded[i] * float(np.float32(scale))).float().to(dtype)


@pytest.mark.parametrize("n,rows,dim", LOOKUP_SHAPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("out_kind", TYPES)
def test_lookup(cuda, n, rows, dim, kind, out_kind):
    gen = rng(n + dim)
    table = torch.randn(rows, dim, generator=gen).to(kind)
    idx = make_indices(n, rows, gen)
    out = gc.table_lookup(table.to(cuda), idx.to(cuda), scale=1.7, dtype=out_kind)
    assert out.dtype == out_kind and out.shape == (n, dim)
    assert torch.equal(out.cpu(), lookup_exact(table, idx, 1.7, out_kind))


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,table_stride,out_stride,offset", [(48, 48, 60, 0), (48, 64, 48, 0), (27, 31, 29, 1),
                                                               (48, 52, 50, 3), (3, 4, 4, 1), (16, 17, 19, 0),
                                                               (20, 20, 20, 4), (20, 22, 24, 2), (54, 56, 54, 2)])
def test_lookup_strides(cuda, kind, dim, table_stride, out_stride, offset):
    """Row strides and starts of every alignment; what lies between the rows stays as it was."""
    gen = rng(5)
    n, rows = 301, 40
    tbuf = torch.randn(rows * table_stride + offset, generator=gen).to(kind).to(cuda)
    table = torch.as_strided(tbuf, (rows, dim), (table_stride, 1), offset)
    obuf = torch.full((n * out_stride + offset,), -3.0, dtype=kind, device=cuda)
    out = torch.as_strided(obuf, (n, dim), (out_stride, 1), offset)
    idx = make_indices(n, rows, gen)
    gc.table_lookup(table, idx.to(cuda), scale=0.5, out=out)
    want = torch.full((n * out_stride + offset,), -3.0, dtype=kind)
    torch.as_strided(want, (n, dim), (out_stride, 1), offset).copy_(lookup_exact(table.cpu(), idx, 0.5, kind))
    assert torch.equal(obuf.cpu(), want)


def test_lookup_edges(cuda):
    table = torch.tensor([[float("inf"), float("nan"), -0.0, 1e38]], device=cuda)
    one = torch.ones(2, dtype=torch.int32, device=cuda)
    out = gc.table_lookup(table, one, scale=100.0).cpu()
    assert torch.isinf(out[:, 0]).all() and torch.isnan(out[:, 1]).all() and torch.isinf(out[:, 3]).all()
    assert gc.table_lookup(table, one[:0]).shape == (0, 4)
    # an empty table has no valid index
    assert torch.equal(gc.table_lookup(table[:0], one), torch.zeros(2, 4, device=cuda))
    with pytest.raises(ValueError):
        gc.table_lookup(table, one, out=torch.empty(3, 4, device=cuda))
    with pytest.raises(ValueError):
        gc.table_lookup(table, one, dtype=torch.float16, out=torch.empty(2, 4, device=cuda))


# -- gradient -----------------------------------------------------------------------------------
def gradient_exact(grads, idx, rows, scale, f2g=None, live=None):
    """(gradient, bound) in 64 bits. A sum of m fp32 terms in any order is within (m - 1) u sum|g| of
    the exact one to first order; one more rounding by the scale's product, one by the scale itself
    and one by an accumulation: (m + 2) u |scale| sum|g| covers them with second-order terms for
    m < 2^20."""
    n = grads.shape[0] if live is None else live
    i = torch.zeros(n, dtype=torch.int64)
    if f2g is None:
        i[:] = idx[:n].long()
    else:
        g = f2g[:n].long()
        ok = (g >= 1) & (g <= idx.shape[0])
        i[ok] = idx.long()[g[ok] - 1]
    i = torch.where((i >= 1) & (i <= rows), i, 0)
    d = grads[:n].double().flatten(1)
    s = float(np.float32(scale))
    out = torch.zeros(rows + 1, d.shape[1], dtype=torch.float64).index_add_(0, i, d)[1:] * s
    mag = torch.zeros(rows + 1, d.shape[1], dtype=torch.float64).index_add_(0, i, d.abs())[1:] * abs(s)
    m = torch.bincount(i, minlength=rows + 1)[1:, None].double()
    return out, (m + 2) * U * mag + 1e-45


GRAD_SHAPES = [(1, 1, 1, 0.0), (1, 5, 48, 0.0), (7, 3, 3, 0.0), (31, 64, 27, 0.0), (1000, 64, 48, 0.0),
               (4097, 1, 48, 0.0), (5000, 300, 12, 1.0), (20_003, 70_000, 48, 0.0), (50_001, 1000, 27, 2.0),
               (3000, 7, 130, 0.0), (300, 4, 1021, 0.0), (9, 2, 65536, 0.0), (100_000, 4096, 48, 3.0),
               (70_000, 2, 16, 0.0), (66_000, 65_536, 4, 0.0), (40_000, 3_000_000, 5, 0.0)]


@pytest.mark.parametrize("n,rows,dim,skew", GRAD_SHAPES)
@pytest.mark.parametrize("kind", TYPES)
def test_gradient(cuda, n, rows, dim, skew, kind):
    gen = rng(n + rows)
    grads = torch.randn(n, dim, generator=gen).to(kind)
    idx = make_indices(n, rows, gen, skew)
    got = gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, scale=1.3)
    want, bound = gradient_exact(grads, idx, rows, 1.3)
    assert got.dtype == torch.float32 and got.shape == want.shape
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [900, 3000, 20_001])
@pytest.mark.parametrize("dim,stride,offset", [(2, 2, 0), (4, 4, 0), (6, 6, 0), (8, 8, 2), (12, 12, 0), (12, 16, 4), (20, 22, 0),
                                               (42, 42, 0), (42, 43, 1), (106, 106, 0), (254, 254, 0), (516, 516, 0)])
@pytest.mark.parametrize("kind", TYPES)
def test_gradient_units(cuda, n, dim, stride, offset, kind):
    """Rows that are read 2, 4, 8 and 16 bytes at a time, by every path of the sizes."""
    gen = rng(n + dim)
    rows = 33
    buf = torch.randn(n * stride + offset, generator=gen).to(kind).to(cuda)
    grads = torch.as_strided(buf, (n, dim), (stride, 1), offset)
    idx = make_indices(n, rows, gen, 1.0)
    got = gc.table_gradient(grads, idx.to(cuda), rows, scale=-0.7)
    want, bound = gradient_exact(grads.cpu(), idx, rows, -0.7)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [1025, 8191, 8192, 8193, 16_383, 16_384, 16_385])
@pytest.mark.parametrize("rows", [1, 256, 257, 65_536, 65_537, (1 << 24) + 1])
def test_gradient_sizes_of_the_cluster_sort(cuda, n, rows):
    """One or two rows a thread of a cluster, one to four passes of 8 bits; filtered rows; equal bits again."""
    gen = rng(n + rows)
    grads = torch.randn(n, 2, generator=gen)
    idx = make_indices(n, rows, gen, 0.5)
    out = torch.full((rows, 2), 7.0, device=cuda)
    gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, out=out)
    want, bound = gradient_exact(grads, idx, rows, 1.0)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    live = n - n // 5
    f2g = (torch.randperm(n, generator=gen) + 1).to(torch.int32)
    counts = torch.tensor([live, 0, 0, 0], dtype=torch.int32)
    a = gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, fgidx_to_gidx=f2g.to(cuda), device_counts=counts.to(cuda))
    want, bound = gradient_exact(grads, idx, rows, 1.0, f2g, live)
    assert ((a.cpu().double() - want).abs() <= bound).all()
    b = gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, fgidx_to_gidx=f2g.to(cuda), device_counts=counts.to(cuda))
    assert torch.equal(a.view(torch.int32), b.view(torch.int32))


@pytest.mark.parametrize("n", [1, 30, 1000])
@pytest.mark.parametrize("rows,dim,out_stride", [(3, 1, 1), (60_000, 48, 48), (60_000, 48, 52), (5_000, 27, 29),
                                                 (17_000_000, 2, 2), (900, 130, 132), (40_000, 3, 4)])
def test_gradient_of_few_rows_zeroes_the_rest(cuda, n, rows, dim, out_stride):
    gen = rng(n + rows)
    grads = torch.randn(n, dim, generator=gen)
    idx = make_indices(n, rows, gen)
    idx[-1] = rows
    buf = torch.full((rows * out_stride,), 5.0, device=cuda)
    out = torch.as_strided(buf, (rows, dim), (out_stride, 1))
    gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, out=out)
    named = idx[(idx >= 1) & (idx <= rows)].long().unique() - 1
    assert int((out != 0).any(dim=1).sum()) <= len(named)
    keep = torch.ones(rows, dtype=torch.bool, device=cuda)
    keep[named.to(cuda)] = False
    assert (out[keep] == 0).all()
    order = torch.full((rows + 1,), 0, dtype=torch.int64)
    order[named + 1] = torch.arange(1, len(named) + 1)
    safe = torch.where((idx >= 1) & (idx <= rows), idx.long(), 0)
    want, bound = gradient_exact(grads, order[safe].to(torch.int32), len(named), 1.0)
    assert ((out[named.to(cuda)].cpu().double() - want).abs() <= bound).all()
    if out_stride > dim:
        assert (torch.as_strided(buf, (rows, out_stride - dim), (out_stride, 1), dim) == 5.0).all()


@pytest.mark.parametrize("n", [303_104, 303_105, 606_208, 606_209])
@pytest.mark.parametrize("rows", [700, 90_000])
def test_gradient_sizes_where_the_tiles_change(cuda, n, rows):
    """Tiles of 1024, 2048 and 4096 rows; few of them leave blocks that zero the table."""
    gen = rng(n + rows)
    grads = torch.randn(n, 3, generator=gen)
    idx = make_indices(n, rows, gen, 1.0)
    got = gc.table_gradient(grads.to(cuda), idx.to(cuda), rows)
    want, bound = gradient_exact(grads, idx, rows, 1.0)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("n,dim", [(700_000, 119), (500_000, 260), (300_000, 1)])
def test_gradient_of_long_runs(cuda, n, dim):
    """Few rows used by very many: runs over hundreds and thousands of chunks, beside short ones."""
    gen = rng(n)
    grads = torch.randn(n, dim, generator=gen).to(torch.bfloat16)
    idx = torch.full((n,), 4, dtype=torch.int32)
    idx[::1000] = (torch.arange(n)[::1000] % 3).to(torch.int32) + 1
    idx[n // 3 : n // 2] = 5
    idx[:70] = 6
    got = gc.table_gradient(grads.to(cuda), idx.to(cuda), 7)
    want, bound = gradient_exact(grads, idx, 7, 1.0)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    assert torch.equal(gc.table_gradient(grads.to(cuda), idx.to(cuda), 7), got)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4095, 4096, 4097, 8193])
@pytest.mark.parametrize("rows", [1, 2, 256, 257, 1024, 1025, 70_000, (1 << 20) + 1])
def test_gradient_sizes_where_the_sort_changes(cuda, n, rows):
    """One launch up to 1024 rows, then one cluster that sorts; one to three passes of 8 bits."""
    gen = rng(n + rows)
    grads = torch.randn(n, 4, generator=gen)
    idx = make_indices(n, rows, gen)
    got = gc.table_gradient(grads.to(cuda), idx.to(cuda), rows)
    want, bound = gradient_exact(grads, idx, rows, 1.0)
    assert ((got.cpu().double() - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [5, 1000, 3000, 60_000])
@pytest.mark.parametrize("dim", [3, 48])
def test_gradient_of_one_row_used_by_all(cuda, n, dim):
    """Every row of the gradients has the same index: one run over all slots, chunks and blocks."""
    grads = torch.randn(n, dim, generator=rng(n))
    idx = torch.full((n,), 7, dtype=torch.int32)
    out = torch.full((9, dim), 2.0, device=cuda)
    got = gc.table_gradient(grads.to(cuda), idx.to(cuda), 9)
    gc.table_gradient(grads.to(cuda), idx.to(cuda), 9, out=out, accumulate=True)
    want, bound = gradient_exact(grads, idx, 9, 1.0)
    assert ((got.cpu().double() - want).abs() <= bound).all()
    # the accumulation rounds once more
    assert ((out.cpu().double() - 2.0 - want).abs() <= bound + 2 * U * (2.0 + want.abs())).all()
    assert (out[torch.arange(9) != 6] == 2.0).all()


@pytest.mark.parametrize("n,rows,dim,skew", [(1000, 64, 48, 0.0), (20_003, 70_000, 48, 0.0), (50_001, 1000, 27, 2.0)])
def test_gradient_repeats_bit_for_bit(cuda, n, rows, dim, skew):
    gen = rng(2)
    grads = torch.randn(n, dim, generator=gen).to(cuda)
    idx = make_indices(n, rows, gen, skew).to(cuda)
    first = gc.table_gradient(grads, idx, rows)
    for _ in range(5):
        assert torch.equal(gc.table_gradient(grads, idx, rows).view(torch.int32), first.view(torch.int32))


@pytest.mark.parametrize("n,kept", [(1000, 0), (1000, 1), (1000, 999), (5003, 2500), (5003, 5003)])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
def test_gradient_of_filtered_rows(cuda, n, kept, kind):
    """The rows behind the count hold NaN and wild indices: they take no part and are not followed."""
    gen = rng(n + kept)
    rows = 37
    grads = torch.randn(n, 3, 9, generator=gen).to(kind)
    grads[kept:] = float("nan")
    idx = make_indices(n, rows, gen)
    f2g = torch.full((n,), 2**31 - 1, dtype=torch.int32)
    f2g[:kept] = (torch.randperm(n, generator=gen)[:kept].sort().values + 1).to(torch.int32)
    if kept > 10:
        f2g[3:6] = torch.tensor([0, -7, n + 1], dtype=torch.int32)
    counts = torch.tensor([kept, 123456, -1, 7], dtype=torch.int32)
    got = gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, scale=-2.0, fgidx_to_gidx=f2g.to(cuda),
                            device_counts=counts.to(cuda))
    want, bound = gradient_exact(grads, idx, rows, -2.0, f2g, kept)
    assert got.shape == (rows, 3, 9)
    assert ((got.cpu().double().reshape(rows, -1) - want).abs() <= bound).all()
    # a count beyond the rows, or negative, is clamped
    for c, live in ((n + 5, n), (-3, 0)):
        counts[0] = c
        f = torch.arange(1, n + 1, dtype=torch.int32)
        clean = torch.nan_to_num(grads)
        got = gc.table_gradient(clean.to(cuda), idx.to(cuda), rows, fgidx_to_gidx=f.to(cuda),
                                device_counts=counts.to(cuda))
        want, bound = gradient_exact(clean, idx, rows, 1.0, f, live)
        assert ((got.cpu().double().reshape(rows, -1) - want).abs() <= bound).all()


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,stride,out_stride,offset", [(48, 64, 52, 0), (27, 29, 28, 1), (48, 50, 49, 3), (4, 7, 6, 1)])
def test_gradient_strides_and_accumulation(cuda, kind, dim, stride, out_stride, offset):
    gen = rng(11)
    n, rows = 3001, 50
    gbuf = torch.randn(n * stride + offset, generator=gen).to(kind).to(cuda)
    grads = torch.as_strided(gbuf, (n, dim), (stride, 1), offset)
    idx = make_indices(n, rows, gen)
    idx[idx == 13] = 14  # a row without gradients keeps what it holds when accumulating
    obuf = torch.full((rows * out_stride + offset,), 3.0, device=cuda)
    out = torch.as_strided(obuf, (rows, dim), (out_stride, 1), offset)
    gc.table_gradient(grads, idx.to(cuda), rows, scale=0.25, out=out, accumulate=True)
    want, bound = gradient_exact(grads.cpu(), idx, rows, 0.25)
    got = obuf.cpu()
    # the accumulation rounds once more, at the size of the result
    assert ((torch.as_strided(got, (rows, dim), (out_stride, 1), offset).double() - 3.0 - want).abs()
            <= bound + U * (3.0 + want.abs()) * 2).all()
    assert (torch.as_strided(got, (rows, dim), (out_stride, 1), offset)[12] == 3.0).all()
    if out_stride > dim:
        between = torch.as_strided(got, (rows - 1, out_stride - dim), (out_stride, 1), offset + dim)
        assert (between == 3.0).all()
    gc.table_gradient(grads, idx.to(cuda), rows, scale=0.25, out=out)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert (out[12] == 0).all()


@pytest.mark.parametrize("n", [3000, 100_000])
def test_gradient_into_a_large_table_with_rows_apart(cuda, n):
    """The table's rows are zeroed element by element, over several turns of the blocks that do it."""
    gen = rng(n)
    rows, dim, stride, offset = 120_000, 27, 29, 1
    grads = torch.randn(n, dim, generator=gen)
    idx = make_indices(n, rows, gen, 2.0)
    buf = torch.full((rows * stride + offset,), 5.0, device=cuda)
    out = torch.as_strided(buf, (rows, dim), (stride, 1), offset)
    gc.table_gradient(grads.to(cuda), idx.to(cuda), rows, out=out)
    want, bound = gradient_exact(grads, idx, rows, 1.0)
    assert ((out.cpu().double() - want).abs() <= bound).all()
    assert (torch.as_strided(buf, (rows - 1, stride - dim), (stride, 1), offset + dim) == 5.0).all() and float(buf[0]) == 5.0


def test_gradient_edges(cuda):
    idx = torch.ones(4, dtype=torch.int32, device=cuda)
    g = torch.ones(4, 3, device=cuda)
    assert torch.equal(gc.table_gradient(g[:0], idx[:0], 5), torch.zeros(5, 3, device=cuda))
    assert gc.table_gradient(g, idx, 0).shape == (0, 3)
    assert torch.equal(gc.table_gradient(g, idx * 0, 2), torch.zeros(2, 3, device=cuda))
    assert torch.equal(gc.table_gradient(g, idx, 1), torch.full((1, 3), 4.0, device=cuda))
    keep = torch.full((2, 3), 7.0, device=cuda)
    gc.table_gradient(g[:0], idx[:0], 2, out=keep, accumulate=True)
    assert (keep == 7.0).all()
    # non-finite gradients stay in their row
    g[1, 1] = float("inf")
    out = gc.table_gradient(g, torch.tensor([1, 2, 1, 3], dtype=torch.int32, device=cuda), 3).cpu()
    assert torch.isinf(out[1, 1]) and torch.isfinite(out).sum() == 8
    with pytest.raises(ValueError):
        gc.table_gradient(g, idx, 3, accumulate=True)
    with pytest.raises(ValueError):
        gc.table_gradient(g, idx, 3, out=torch.empty(2, 3, device=cuda))
    with pytest.raises(ValueError):
        gc.table_gradient(g, idx, 3, fgidx_to_gidx=idx[:3])
    with pytest.raises(gs3d.Gs3dError):
        gc.table_gradient(g, idx[:3], 3)


def test_results_over_inputs(cuda):
    """Refused; beside one another's rows in one buffer they are what they are elsewhere."""
    gen = rng(31)
    buf = torch.randn(400, 96, generator=gen).to(cuda)
    table, idx = buf[:, :48], make_indices(400, 400, gen).to(cuda)
    want = gc.table_lookup(table, idx, scale=2.0)
    want_grad = gc.table_gradient(table, idx, 400)
    for out in (table, buf[:, 20:68], buf[:200].view(400, 48)):
        with pytest.raises(ValueError, match="overlap"):
            gc.table_lookup(table, idx, out=out)
        with pytest.raises(ValueError, match="overlap"):
            gc.table_gradient(table, idx, 400, out=out)
    assert torch.equal(gc.table_lookup(table, idx, scale=2.0, out=buf[:, 48:]), want) and torch.equal(buf[:, 48:], want)
    gc.table_gradient(table, idx, 400, out=buf[:, 48:])
    assert torch.equal(buf[:, 48:], want_grad)
    q = gc.mx4_quantise(table, "mxfp4")
    inside = q.codes.view(-1)[: 24 * 4 * 20].view(torch.float32).view(10, 48)
    with pytest.raises(ValueError, match="overlap"):
        gc.mx4_dequantise(MX4Rows(q.codes[:10], q.scales[:10], None, 48, "mxfp4"), out=inside)


def test_gradient_is_the_lookups(cuda):
    """<d_out, lookup(table + h v)> differences: the lookup is linear in the table, so with values that
    fp32 holds exactly the difference quotient equals <gradient, v> exactly."""
    gen = rng(3)
    n, rows, dim = 500, 20, 12
    idx = make_indices(n, rows, gen).to(cuda)
    table = torch.randint(-64, 64, (rows, dim), generator=gen).float().to(cuda)
    v = torch.randint(-8, 8, (rows, dim), generator=gen).float().to(cuda)
    d_out = torch.randint(-8, 8, (n, dim), generator=gen).float().to(cuda)
    grad = gc.table_gradient(d_out, idx, rows, scale=0.5)
    f = lambda t: (gc.table_lookup(t, idx, scale=0.5).double() * d_out.double()).sum()  # noqa: E731
    assert float(f(table + v) - f(table)) == float((grad.double() * v.double()).sum())


# -- 4-bit rows -----------------------------------------------------------------------------------
GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1])


def nearest(grid, y):
    """Index of the nearest grid value, ties to the even index, beyond the last: the last."""
    hi = np.minimum(np.searchsorted(grid, y), len(grid) - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - y, y - grid[lo]
    return np.where(y >= grid[-1], len(grid) - 1, np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi))


def quantise_exact(x, fmt, g):
    """(codes, scales, values) in 64 bits, where a quotient of two 24-bit values never meets a border
    that the exact one does not."""
    x = x.double().numpy()
    n, dim = x.shape
    block = 16 if fmt == "nvfp4" else 32
    nb = -(-dim // block)
    pad = np.zeros((n, nb * block))
    pad[:, :dim] = x
    b = pad.reshape(n, nb, block)
    nan = np.isnan(b).any(axis=2)
    a = np.abs(np.nan_to_num(b, nan=0.0, posinf=np.inf, neginf=-np.inf)).max(axis=2)
    if fmt == "nvfp4":
        byte = nearest(E4M3, a / (6.0 * g))
        s = E4M3[byte] * g
        byte = np.where(nan, 0x7F, byte)
    else:
        e = np.floor(np.log2(np.where((a > 0) & np.isfinite(a), a, 1.0)))
        byte = np.clip(e - 2 + 127, 0, 254)
        byte = np.where(np.isinf(a), 253, np.where(a == 0, 0, byte)).astype(int)
        s = np.exp2(byte - 127.0)
        byte = np.where(nan, 0xFF, byte)
    with np.errstate(divide="ignore", invalid="ignore"):
        y = np.where(s[..., None] > 0, np.abs(b) / s[..., None], 0.0)
    code = nearest(GRID, np.nan_to_num(y, nan=0.0, posinf=np.inf))
    with np.errstate(over="ignore", invalid="ignore"):  # an infinity of an mxfp4 block overflows again
        val = (np.where(np.signbit(b), -1.0, 1.0) * GRID[code] * s[..., None]).astype(np.float32)
    val = np.where(nan[..., None], np.float32(np.nan), val).reshape(n, -1)[:, :dim]
    code = (code | np.where(np.signbit(b), 8, 0)).reshape(n, -1)
    codes = code[:, 0::2] | (code[:, 1::2] << 4)
    return codes[:, : (dim + 1) // 2], byte, val, nan


MX_SHAPES = [(1, 1), (1, 48), (5, 3), (33, 27), (1000, 48), (257, 12), (64, 130), (7, 1021), (2, 65535), (10_001, 48),
             (1031, 4), (515, 8), (777, 20), (130, 92), (301, 44), (99, 16), (65, 17), (1025, 2), (37, 72), (3, 4100)]


def mx_input(n, dim, kind, gen, spread):
    x = torch.randn(n, dim, generator=gen) * 0.1
    if spread:  # magnitudes over many binades, exact borders, zeros, empty rows
        x = x * torch.exp2(torch.randint(-20, 20, (n, dim), generator=gen).float())
        x.view(-1)[::7] = torch.randint(-14, 15, (x.view(-1)[::7].shape[0],), generator=gen).float() * 0.25
        x.view(-1)[::11] = 0.0
        x[::5] = 0.0
        x[1::6] = torch.randint(-28, 29, x[1::6].shape, generator=gen).float() * 0.25
    return x.to(kind)


@pytest.mark.parametrize("n,dim", MX_SHAPES)
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("spread", [False, True])
def test_quantise(cuda, n, dim, kind, fmt, spread):
    gen = rng(n + dim)
    x = mx_input(n, dim, kind, gen, spread)
    scales = [None]
    if fmt == "nvfp4":
        ts = gc.mx4_tensor_scale(x.to(cuda))
        a = x.float().abs()  # the widest spread overflows fp16: infinities do not count
        want = max(np.float32(a[a.isfinite()].max().numpy()) * (np.float32(1) / np.float32(2688)), np.float32(2.0 ** -100))
        assert ts.cpu().numpy()[0] == want
        # its own scale; one that makes blocks saturate; a power of two, where borders are met exactly
        scales = [None, torch.tensor([float(want) * 0.013]), torch.tensor([2.0 ** -6])]
    for s in scales:
        q = gc.mx4_quantise(x.to(cuda), fmt, tensor_scale=None if s is None else s.to(cuda))
        g = float(q.tensor_scale.cpu()) if fmt == "nvfp4" else 1.0
        codes, byte, val, _ = quantise_exact(x, fmt, g)
        assert np.array_equal(q.scales.cpu().numpy(), byte)
        got = q.codes.cpu().numpy()
        assert np.array_equal(got, codes)
        for out_kind in TYPES:
            back = gc.mx4_dequantise(q, out_kind)
            assert torch.equal(back.cpu(), torch.from_numpy(val).to(out_kind))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantise_borders(cuda, fmt):
    """Every border of the grid times scale, its two fp32 neighbours, and block maxima at the borders
    of the scales: where a rounded quotient would decide wrongly."""
    rows, g = [], 0.0123
    for u in range(1, 127):
        s = np.float32(E4M3[u]) * np.float64(np.float32(g)) if fmt == "nvfp4" else 2.0 ** ((u % 60) - 30)
        row = [np.float32(6.0 * s)]
        for b in (0.25, 0.75, 1.25, 1.75, 2.5):
            t = np.float32(b * s)
            row += [np.nextafter(t, np.float32(0)), t, np.nextafter(t, np.float32(np.inf))]
        rows.append(row)
        for mid in ([(E4M3[u] + E4M3[u + 1]) / 2] if fmt == "nvfp4" and u < 126 else [1.0]):
            t = np.float32(6.0 * mid * np.float64(np.float32(g)))
            for a in (np.nextafter(t, np.float32(0)), t, np.nextafter(t, np.float32(np.inf))):
                rows.append([a] + [np.float32(a * k / 16) for k in range(1, 16)])
    x = torch.from_numpy(np.array(rows, dtype=np.float32))
    ts = torch.tensor([g], device=cuda) if fmt == "nvfp4" else None
    q = gc.mx4_quantise(x.to(cuda), fmt, tensor_scale=ts)
    codes, byte, val, _ = quantise_exact(x, fmt, float(np.float32(g)))
    assert np.array_equal(q.scales.cpu().numpy(), byte)
    assert np.array_equal(q.codes.cpu().numpy(), codes)
    assert np.array_equal(gc.mx4_dequantise(q).cpu().numpy(), val)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantise_non_finite(cuda, fmt):
    x = torch.randn(12, 48, generator=rng(1))
    x[0, 3] = float("nan")
    x[1, 20] = float("inf")
    x[2, 40] = -float("inf")
    x[3] = 0.0
    x[4, :16] = 1e-42   # subnormal
    x[5] = 3e38
    x[6, 5], x[6, 6] = float("inf"), float("nan")
    x[7] = -0.0
    q = gc.mx4_quantise(x.to(cuda), fmt, tensor_scale=torch.tensor([0.01], device=cuda) if fmt == "nvfp4" else None)
    codes, byte, val, nan = quantise_exact(x, fmt, float(np.float32(0.01)))
    assert np.array_equal(q.scales.cpu().numpy(), byte)
    assert np.array_equal(gc.mx4_dequantise(q).cpu().numpy(), val, equal_nan=True)
    block = 16 if fmt == "nvfp4" else 32
    clean = ~np.repeat(nan, block, axis=1)[:, :48]
    got = q.codes.cpu().numpy()
    got = np.stack([got & 15, got >> 4], axis=2).reshape(12, 48)
    want = np.stack([codes & 15, codes >> 4], axis=2).reshape(12, 48)
    assert np.array_equal(got[clean], want[clean])
    # the tensor scale looks at finite values only
    ts = gc.mx4_tensor_scale(torch.tensor([[float("inf"), 2688.0, float("nan"), -1.0]], device=cuda))
    assert float(ts) == 1.0
    assert float(gc.mx4_tensor_scale(torch.zeros(3, 4, device=cuda))) == 2.0 ** -100
    assert float(gc.mx4_tensor_scale(torch.zeros(0, 4, device=cuda))) == 2.0 ** -100


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("n", [3, 50_001, 1_200_007])
def test_tensor_scale(cuda, kind, n):
    """The largest finite magnitude wherever it lies, among infinities and NaN."""
    x = torch.zeros(n, 48, dtype=kind, device=cuda)
    flat = x.view(-1)
    for at in (0, flat.shape[0] // 2 + 1, flat.shape[0] - 1):
        flat[at] = -3.0
        assert float(gc.mx4_tensor_scale(x)) == float(np.float32(3.0) * (np.float32(1) / np.float32(2688)))
        for other in (float("inf"), -float("inf"), float("nan")):
            flat[(at + 77) % flat.shape[0]] = other
            assert float(gc.mx4_tensor_scale(x)) == float(np.float32(3.0) * (np.float32(1) / np.float32(2688)))
        flat[at] = 0.0
        flat[(at + 77) % flat.shape[0]] = 0.0


@pytest.mark.parametrize("kind", TYPES)
def test_tensor_scale_is_the_quotient_up_to_its_two_roundings(cuda, kind):
    """The definition is largest / 2688; the reciprocal of 2688 and the product with it round by at most
    2^-24 each: within (1 + 2^-24)^2 - 1 of the quotient."""
    gen = rng(9)
    for k in range(-12, 13):
        x = (torch.randn(9, 48, generator=gen) * 2.0 ** k).to(kind)
        top = x.double().abs().max()
        got = gc.mx4_tensor_scale(x.to(cuda)).cpu().double()
        assert float((got * 2688 - top).abs()) <= ((1 + 2.0 ** -24) ** 2 - 1) * float(top)


@pytest.mark.parametrize("kind", [torch.float16, torch.bfloat16])
def test_quantise_ratios_of_small_numbers(cuda, kind):
    """16-bit elements and a power-of-two maximum: quotients that meet the borders exactly."""
    gen = rng(3)
    x = torch.randint(-64, 65, (4001, 48), generator=gen).float() / 8
    x[:, 0] = torch.tensor([7.0, 10.5, 21.0, 8.0]).repeat(1001)[:4001]
    x = x.to(kind)
    for s in (None, torch.tensor([21.0 / 2688]), torch.tensor([2.0 ** -9]), torch.tensor([3.0 / 448])):
        q = gc.mx4_quantise(x.to(cuda), "nvfp4", tensor_scale=None if s is None else s.to(cuda))
        codes, byte, val, _ = quantise_exact(x, "nvfp4", float(q.tensor_scale.cpu()))
        assert np.array_equal(q.scales.cpu().numpy(), byte)
        assert np.array_equal(q.codes.cpu().numpy(), codes)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dim", [48, 27])
def test_quantise_largest_and_smallest(cuda, fmt, dim):
    """Up to the largest fp32 values, whose tensor scale is the largest, and down to subnormal ones."""
    gen = rng(12)
    for top in (float(np.finfo(np.float32).max), 2.0 ** 113, 2.0 ** -110, 2.0 ** -140):
        x = torch.from_numpy((torch.rand(50, dim, generator=gen).double() * 2 - 1).numpy() * top).float()
        x[0, 1] = top
        x[3] = 0.0
        q = gc.mx4_quantise(x.to(cuda), fmt)
        g = float(q.tensor_scale.cpu()) if fmt == "nvfp4" else 1.0
        codes, byte, val, _ = quantise_exact(x, fmt, g)
        assert np.array_equal(q.scales.cpu().numpy(), byte)
        assert np.array_equal(q.codes.cpu().numpy(), codes)
        assert np.isfinite(val).all() or fmt == "mxfp4"
        assert np.array_equal(gc.mx4_dequantise(q).cpu().numpy(), val)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("dim,stride,offset", [(48, 64, 0), (48, 49, 1), (27, 31, 3), (16, 24, 8), (12, 16, 4), (92, 92, 4),
                                               (40, 48, 0), (4, 4, 4), (48, 48, 2), (64, 72, 0)])
def test_quantise_strides(cuda, kind, dim, stride, offset):
    gen = rng(4)
    n = 333
    buf = (torch.randn(n * stride + offset, generator=gen) * 0.1).to(kind).to(cuda)
    x = torch.as_strided(buf, (n, dim), (stride, 1), offset)
    for fmt in ("nvfp4", "mxfp4"):
        a, b = gc.mx4_quantise(x, fmt), gc.mx4_quantise(x.contiguous(), fmt)
        assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
        out = torch.full((n * stride + offset,), 9.0, dtype=kind, device=cuda)
        gc.mx4_dequantise(a, out=torch.as_strided(out, (n, dim), (stride, 1), offset))
        want = torch.full_like(out, 9.0)
        torch.as_strided(want, (n, dim), (stride, 1), offset).copy_(gc.mx4_dequantise(b, kind))
        assert torch.equal(out, want)


@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_quantise_strides_of_many_rows(cuda, kind, fmt):
    """Rows apart and misaligned, more of them than the element-by-element kernels' grids hold at once:
    600K (or 400K) blocks and 9.6M elements for 303K threads, and a tensor scale of many blocks."""
    n, dim, stride, offset = 200_000, 48, 49, 1
    buf = (torch.randn(n * stride + offset, generator=rng(14)) * 0.1).to(kind).to(cuda)
    x = torch.as_strided(buf, (n, dim), (stride, 1), offset)
    x[n - 2, 5] = -7.0  # the largest magnitude, in the last turn
    buf[stride * 5 : stride * 5 + 1] = 100.0  # between the rows: not part of them
    plain = x.contiguous()
    if fmt == "nvfp4":
        assert torch.equal(gc.mx4_tensor_scale(x), gc.mx4_tensor_scale(plain))
        assert float(gc.mx4_tensor_scale(x)) == float(np.float32(7.0) * (np.float32(1) / np.float32(2688)))
    a, b = gc.mx4_quantise(x, fmt), gc.mx4_quantise(plain, fmt)
    assert torch.equal(a.codes, b.codes) and torch.equal(a.scales, b.scales)
    out = torch.full((n * stride + offset,), 9.0, dtype=kind, device=cuda)
    gc.mx4_dequantise(a, out=torch.as_strided(out, (n, dim), (stride, 1), offset))
    want = torch.full_like(out, 9.0)
    torch.as_strided(want, (n, dim), (stride, 1), offset).copy_(gc.mx4_dequantise(b, kind))
    assert torch.equal(out, want)


def test_quantise_empty(cuda):
    x = torch.zeros(0, 48, device=cuda)
    q = gc.mx4_quantise(x)
    assert q.rows == 0 and gc.mx4_dequantise(q).shape == (0, 48)
    with pytest.raises(ValueError):
        gc.mx4_quantise(x, "fp8")


def test_every_code_and_scale(cuda):
    """All 16 codes under all 256 scale bytes, in both positions of a byte."""
    vals = np.concatenate([GRID, -GRID])
    for fmt, block in (("nvfp4", 16), ("mxfp4", 32)):
        codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1).view(256, -1)
        scales = torch.arange(256, dtype=torch.uint8).view(-1, 1).expand(256, 512 // block).contiguous()
        ts = torch.tensor([0.37]) if fmt == "nvfp4" else None
        q = MX4Rows(codes, scales, ts, 512, fmt).to(cuda)
        got = gc.mx4_dequantise(q).cpu().numpy()
        b = np.arange(256)
        if fmt == "nvfp4":
            s = np.append(E4M3, np.nan)[b & 127] * float(np.float32(0.37))
        else:
            s = np.where(b == 255, np.nan, np.exp2(b - 127.0))
        nib = np.stack([b & 15, b >> 4], axis=1).reshape(-1)
        with np.errstate(over="ignore"):
            want = (vals[nib][None, :] * s[:, None]).astype(np.float32)
        assert np.array_equal(got, want, equal_nan=True)


# -- colours ------------------------------------------------------------------------------------
COLOUR_U = 147  # see test_colours


def make_mx4(rows, dim, fmt, gen):
    block = 16 if fmt == "nvfp4" else 32
    codes = torch.randint(0, 256, (rows, (dim + 1) // 2), generator=gen, dtype=torch.uint8)
    lo, hi = (8, 0x48) if fmt == "nvfp4" else (118, 126)
    scales = torch.randint(lo, hi, (rows, -(-dim // block)), generator=gen, dtype=torch.uint8)
    return MX4Rows(codes, scales, torch.tensor([0.117]) if fmt == "nvfp4" else None, dim, fmt)


@pytest.mark.parametrize("n", [1, 2, 31, 129, 1000, 4099])
@pytest.mark.parametrize("degree,storage", [(0, 0), (1, 1), (2, 2), (3, 3), (0, 3), (1, 2), (2, 3)])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("table", [False, True])
def test_colours(cuda, n, degree, storage, fmt, table):
    """Near the 64-bit value. Per unit of u = 2^-24: a component of mean - position carries 1, the sum of
    squares 3, the reciprocal root half of that and 4 of its own (2 ulp), the product with it 1: at most 8
    for a component of the direction. A basis function of degree d <= 3, whose coefficients add to at
    most 3, then carries 3 (8 d + 6) <= 90, a sum of 16 products 16 of their magnitudes (at most 3 |h|)
    and the scale of a block 3 roundings of the same: (90 + 48 + 9) u sum|h|, and 2 u for the 1/2."""
    gen = rng(n + degree)
    order = (storage + 1) ** 2
    rows = max(1, n // 3) if table else n + 2
    q = make_mx4(rows, 3 * order, fmt, gen)
    idx = make_indices(n, rows, gen) if table else None
    means = torch.randn(n, 4, generator=gen) * 2
    for views in (1, 2, 5, 64):
        pos = np.random.default_rng(views).normal(size=(views, 3)).astype(np.float32) * 4
        qd = q.to(cuda)
        got = gc.mx4_colours(qd, means.to(cuda), pos, degree, indices=None if idx is None else idx.to(cuda))
        w = gc.mx4_dequantise(qd)
        w = w[:n] if idx is None else gc.table_lookup(w, idx.to(cuda))
        h = w.cpu().double().view(n, 3, order)[:, :, : (degree + 1) ** 2]
        bound = COLOUR_U * U * h.abs().sum(dim=2) + 2 * U
        for v in {0, views // 2, views - 1}:
            want = colours_exact(h, means.double(), pos[v].astype(np.float64), degree)
            assert ((got[v, :, :3].cpu().double() - want).abs() <= bound).all()
            assert (got[v, :, 3] == 0).all()


def colours_exact(h, means, p, degree):
    d = means[:, :3] - torch.from_numpy(p)
    x, y, z = (d / d.norm(dim=1, keepdim=True)).unbind(dim=1)
    b = [0.28209479177387814 + 0 * x]
    if degree > 0:
        b += [-0.4886025119029199 * y, 0.4886025119029199 * z, -0.4886025119029199 * x]
    if degree > 1:
        b += [1.0925484305920792 * x * y, -1.0925484305920792 * y * z, 0.31539156525252005 * (2 * z * z - x * x - y * y),
              -1.0925484305920792 * x * z, 0.5462742152960396 * (x * x - y * y)]
    if degree > 2:
        b += [-0.5900435899266435 * y * (3 * x * x - y * y), 2.890611442640554 * x * y * z,
              -0.4570457994644658 * y * (4 * z * z - x * x - y * y), 0.3731763325901154 * z * (2 * z * z - 3 * (x * x + y * y)),
              -0.4570457994644658 * x * (4 * z * z - x * x - y * y), 1.445305721320277 * z * (x * x - y * y),
              -0.5900435899266435 * x * (x * x - 3 * y * y)]
    return (torch.einsum("kn,nck->nc", torch.stack(b), h) + 0.5).clamp(min=0)


def test_colours_edges(cuda):
    q = make_mx4(4, 48, "nvfp4", rng(0)).to(cuda)
    pos = np.zeros((1, 3), np.float32)
    assert gc.mx4_colours(q, torch.zeros(0, 4, device=cuda), pos, 3).shape == (1, 0, 4)
    # a NaN scale makes its channel NaN, the others stay
    q.scales[2, 1] = 0x7F
    c = gc.mx4_colours(q, torch.randn(4, 4, device=cuda), pos, 3).cpu()
    assert torch.isnan(c[0, 2, 1]) and torch.isnan(c).sum() == 1
    # no valid row: the colour of zero coefficients
    c = gc.mx4_colours(q, torch.randn(3, 4, device=cuda), pos, 3, indices=torch.tensor([0, 5, -1], dtype=torch.int32, device=cuda))
    assert torch.equal(c[0, :, :3], torch.full((3, 3), 0.5, device=cuda))
    with pytest.raises(gs3d.Gs3dError):
        gc.mx4_colours(q, torch.zeros(5, 4, device=cuda), pos, 3)
    with pytest.raises(ValueError):
        gc.mx4_colours(q, torch.zeros(4, 4, device=cuda), pos, 3, indices=torch.ones(3, dtype=torch.int32, device=cuda))
    with pytest.raises(ValueError):
        gc.mx4_colours(q, torch.zeros(4, 4, device=cuda), pos, 3, out=torch.empty(1, 4, 3, device=cuda))


# -- the render ---------------------------------------------------------------------------------
def pixel_bound(sh, buf):
    """See test_render_compressed; a colour is at most 1/2 + 3 sum|h| (a basis function is at most 3)."""
    size = float(sh.abs().sum(dim=2).max())
    ends = buf.tiles_end_sdfgidx.cpu().long()
    entries = int((ends - torch.cat([ends.new_zeros(1), ends[:-1]])).max())
    return U * (2 * COLOUR_U * size + 4 + 4 * entries * (0.5 + 3 * size))


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("table", [False, True])
@pytest.mark.parametrize("sh_degree", [0, 2, 3])
@pytest.mark.parametrize("reference_order", [False, True])
def test_render_compressed(cuda, fmt, table, sh_degree, reference_order):
    """The render of a compressed model against the render-only render of its dequantised coefficients:
    the same geometry, sorting and weights bit for bit, colours that differ by at most two colour bounds
    (the plain render's is below: test_colours' chain with exact roots), so pixels (weights add to at most
    1) by as much plus the rounding of the blend, 2 u of the largest colour per entry and side."""
    g = synthetic_gaussians(SceneSpec(5_000, "uniform:1", -4.0, 0.5), 3).to(cuda)
    ro = RenderOnlyGaussiansVector.from_trainable(g)
    tab = gc.fit_table(g.sh_coeffs, 40, iterations=2) if table else None
    comp = gc.compress(ro, fmt, table=tab)
    w = gc.mx4_dequantise(comp.sh)
    if table:
        w = gc.table_lookup(w, comp.indices)
    plain = RenderOnlyGaussiansVector(ro.means_opacities, ro.covariances, w.view(-1, 3, 16).contiguous())
    cam = look_at_camera(160, 96, 60.0, (0.3, 0.4, 3))
    til, opt = Tiling.for_camera(cam), RenderOptions.for_camera(cam, sh_degree)
    images = []
    for model in (comp, plain):
        out = RenderOutputs.create(cam.width, cam.height, cuda)
        buf = RenderBuffers.create(g.n, til.nb_tiles, cuda)
        gs3d.render(out, model, cam, til, opt, buf, reference_order=reference_order)
        images.append(out)
    assert torch.equal(images[0].last_contributing_sdfgids, images[1].last_contributing_sdfgids)
    assert torch.equal(images[0].transmittance, images[1].transmittance)
    assert float((images[0].rgb - images[1].rgb).abs().max()) <= pixel_bound(plain.sh_coeffs, buf)
    assert float(images[0].rgb.std()) > 0.01


def test_render_no_gaussians(cuda):
    comp = gs3d.CompressedGaussiansVector(torch.zeros(0, 4, device=cuda), torch.zeros(0, 6, device=cuda),
                                          gc.mx4_quantise(torch.zeros(0, 48, device=cuda)))
    cam = look_at_camera(32, 32, 60.0, (0, 0, 3))
    til = Tiling.for_camera(cam)
    out = RenderOutputs.create(32, 32, cuda)
    gs3d.render(out, comp, cam, til, RenderOptions.for_camera(cam, 3), RenderBuffers.create(0, til.nb_tiles, cuda))
    assert torch.isfinite(out.rgb).all()
    with pytest.raises(gs3d.Gs3dError):
        gs3d.render(out, comp, cam, til, RenderOptions.for_camera(cam, 3), RenderBuffers.create(0, til.nb_tiles, cuda),
                    defer_colour=True)


def test_given_colours_render(cuda):
    g = synthetic_gaussians(SceneSpec(3_000, "uniform:1", -4.0, 0.5), 4).to(cuda)
    q = gc.mx4_quantise(g.sh_coeffs)
    cam = look_at_camera(96, 64, 60.0, (0, 0.5, 3))
    til, opt = Tiling.for_camera(cam), RenderOptions.for_camera(cam, 3)
    colours = gc.mx4_colours(q, g.means_opacity_features, cam.position[None], 3)
    a = RenderOutputs.create(96, 64, cuda)
    buf = RenderBuffers.create(g.n, til.nb_tiles, cuda)
    gs3d.render(a, g, cam, til, opt, buf, defer_colour=True)
    render_given_colour(a, g, cam, til, opt, buf, colours, g.n)
    b = RenderOutputs.create(96, 64, cuda)
    plain = GaussiansVector(*g.tensors()[:3], gc.mx4_dequantise(q).view(-1, 3, 16).contiguous())
    buf = RenderBuffers.create(g.n, til.nb_tiles, cuda)
    gs3d.render(b, plain, cam, til, opt, buf)
    assert float((a.rgb - b.rgb).abs().max()) <= pixel_bound(plain.sh_coeffs, buf)


# -- offsets past 32 bits ---------------------------------------------------------------------------
def test_more_than_2_31_elements(cuda):
    """46M rows of 48 (2.2e9 elements, 4.4 GB in bf16): the rows at the end, whose element offsets do not
    fit 31 bits, and 90M rows of 24 bytes of codes (2.1 GB). Products and sums of small whole numbers, exact."""
    n, rows = 46_000_000, 100
    table = (torch.arange(rows, device=cuda) % 64)[:, None].float().expand(rows, 48).contiguous().bfloat16()
    idx = (torch.arange(n, device=cuda, dtype=torch.int32) % rows) + 1
    out = gc.table_lookup(table, idx)
    tail = (torch.arange(n - 3000, n, device=cuda) % rows) % 64
    assert torch.equal(out[n - 3000:], tail[:, None].bfloat16().expand(-1, 48))
    # only the last rows have an index: sums of values below 64 over 460 rows are exact
    keep = torch.zeros_like(idx)
    keep[n - rows * 460:] = idx[n - rows * 460:]
    grad = gc.table_gradient(out, keep, rows)
    assert torch.equal(grad, table.float() * 460)
    q = gc.mx4_quantise(out, "mxfp4")
    back = gc.mx4_dequantise(q, torch.bfloat16)
    few = gc.mx4_dequantise(gc.mx4_quantise(out[n - 3000:].contiguous(), "mxfp4"), torch.bfloat16)
    assert torch.equal(back[n - 3000:], few)
    del out, back, q
    m = 90_000_000
    sh = MX4Rows(torch.zeros(m, 24, dtype=torch.uint8, device=cuda), torch.zeros(m, 2, dtype=torch.uint8, device=cuda),
                 None, 48, "mxfp4")
    sh.codes[m - 1000:] = 0x22
    sh.scales[m - 1000:] = 127
    means = torch.randn(1000, 4, generator=rng(1)).to(cuda)
    pos = np.ones((1, 3), np.float32)
    last = torch.arange(m - 999, m + 1, dtype=torch.int32, device=cuda)
    small = MX4Rows(sh.codes[m - 1000:].clone(), sh.scales[m - 1000:].clone(), None, 48, "mxfp4")
    assert torch.equal(gc.mx4_colours(sh, means, pos, 3, indices=last), gc.mx4_colours(small, means, pos, 3))


# -- a run of them, streams and graphs -------------------------------------------------------------
def pipeline(x, idx, rows, d_out, means, pos):
    """Expand a table, take its gradient, step it, quantise it and look at its colours."""
    out = gc.table_lookup(x, idx, dtype=torch.float32)
    grad = gc.table_gradient(d_out, idx, rows)
    stepped = x - 0.1 * grad
    q = gc.mx4_quantise(stepped)
    return out, grad, gc.mx4_dequantise(q), gc.mx4_colours(q, means, pos, 3, indices=idx)


def pipeline_inputs(cuda, n=3000, rows=200):
    gen = rng(8)
    return (torch.randn(rows, 48, generator=gen).to(cuda), make_indices(n, rows, gen).to(cuda), rows,
            torch.randn(n, 48, generator=gen).to(cuda), torch.randn(n, 4, generator=gen).to(cuda),
            np.array([[0.0, 0.0, 5.0], [1.0, 4.0, 0.0]], np.float32))


def test_on_another_stream(cuda):
    args = pipeline_inputs(cuda)
    want = pipeline(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream(cuda)
    with torch.cuda.stream(s):
        got = pipeline(*args)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # the stream argument: what the call allocates belongs to that stream
    s.wait_stream(torch.cuda.current_stream())
    grads = [gc.table_gradient(args[3], args[1], args[2], stream=s) for _ in range(4)]
    outs = [gc.table_lookup(args[0], args[1], stream=s) for _ in range(4)]
    s.synchronize()
    assert all(torch.equal(g, want[1]) for g in grads) and all(torch.equal(o, want[0]) for o in outs)


def test_two_calls_at_once(cuda):
    args = pipeline_inputs(cuda, 20_000, 500)
    want = pipeline(*args)
    streams = [torch.cuda.Stream(cuda) for _ in range(3)]
    got = []
    for _ in range(5):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(pipeline(*args))
    torch.cuda.synchronize()
    for g in got:
        for a, b in zip(g, want):
            assert torch.equal(a, b)


def test_captured_and_replayed(cuda):
    """Two graphs of the same calls, replayed in turn with new inputs: neither uses the other's
    workspace, and every replay reads the inputs afresh."""
    args = pipeline_inputs(cuda)
    s = torch.cuda.Stream(cuda)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pipeline(*args)
    torch.cuda.current_stream().wait_stream(s)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = pipeline(*args)
        graphs.append((g, outs))
    for step in range(3):
        args[0].mul_(1.01 + step)
        args[1].copy_(make_indices(args[1].shape[0], args[2], rng(100 + step)).to(cuda))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = pipeline(*args)
        for _, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b)


def test_fit_table(cuda):
    """Two separated clusters are found; every Gaussian's row is the mean of its cluster within the
    sum's rounding."""
    gen = rng(6)
    centre = torch.tensor([[1.0] * 12, [-1.0] * 12])
    which = torch.randint(0, 2, (500,), generator=gen)
    sh = (centre[which] + 0.01 * torch.randn(500, 12, generator=gen)).view(500, 3, 4).to(cuda)
    table = gc.fit_table(sh, 2, iterations=5, seed=3)
    rows = table.expand()
    assert table.coeffs.shape == (2, 3, 4) and float((rows - sh).abs().max()) < 0.2
    assert gc.fit_table(sh[:3], 10).rows == 3


def test_fit_table_rows_are_their_members_means(cuda):
    """Of separated clusters, where one more iteration changes nothing: a row is the mean of its m members
    within (m + 2) u mean|x| (m - 1 roundings of the sum, one of the quotient)."""
    gen = rng(7)
    which = torch.randint(0, 5, (4001,), generator=gen)
    centre = torch.eye(5).repeat_interleave(3, dim=1)[:, :12] * 4 - 2
    sh = (centre[which] + 0.05 * torch.randn(4001, 12, generator=gen)).view(-1, 3, 4)
    table = gc.fit_table(sh.to(cuda), 60, iterations=100, seed=2)
    again = gc.fit_table(sh.to(cuda), 60, iterations=101, seed=2)
    assert torch.equal(table.indices, again.indices) and torch.equal(table.coeffs, again.coeffs)
    x, c, i = sh.double().view(-1, 12), table.coeffs.cpu().double().view(60, 12), table.indices.cpu().long() - 1
    for k in i.unique().tolist():
        mine = x[i == k]
        bound = (len(mine) + 2) * U * mine.abs().mean(dim=0)
        assert ((c[k] - mine.mean(dim=0)).abs() <= bound).all()


@pytest.mark.parametrize("iterations", [1, 3])
def test_fit_table_takes_the_nearest_row(cuda, iterations):
    """The comparison is of |c|^2 / 2 - <x, c> in fp32: d products and sums a side, so that a row may be taken
    whose value is above the least by 2 (d + 2) u (|c|^2 / 2 + |x| |c|) at most."""
    x = torch.randn(3000, 27, generator=rng(5))
    table = gc.fit_table(x.view(-1, 3, 9).to(cuda), 50, iterations=iterations, seed=1)
    c, x = table.coeffs.cpu().double().view(50, 27), x.double()
    value = 0.5 * (c * c).sum(dim=1) - x @ c.t()
    size = float(0.5 * (c * c).sum(dim=1).max() + x.norm(dim=1).max() * c.norm(dim=1).max())
    mine = value.gather(1, table.indices.cpu().long()[:, None] - 1)[:, 0]
    assert ((mine - value.min(dim=1).values) <= 2 * (27 + 2) * U * size).all()


def test_fit_table_rows_without_members(cuda):
    """Two values among 40 Gaussians and ten rows: eight rows end without members and keep what they had."""
    sh = torch.tensor([[1.0] * 12, [-0.5] * 12])[torch.arange(40) % 2].view(40, 3, 4).to(cuda)
    table = gc.fit_table(sh, 10, iterations=4, seed=3)
    assert table.rows == 10 and len(table.indices.unique()) == 2
    assert torch.equal(table.expand(), sh)
    assert ((table.coeffs == 1.0) | (table.coeffs == -0.5)).all()


# -- training and scripts ---------------------------------------------------------------------------
def table_scene(cuda, n=1500, rows=60):
    g = synthetic_gaussians(SceneSpec(n, "uniform:1", -3.5, 0.4), 2).to(cuda)
    cams = [look_at_camera(96, 64, 60.0, (2.5 * np.cos(a), 0.4, 2.5 * np.sin(a))) for a in (0.0, 2.0, 4.0)]
    targets = [torch.rand(96, 64, 3, generator=rng(i)).to(cuda) for i in range(3)]
    til = Tiling.for_camera(cams[0])
    return g, gc.fit_table(g.sh_coeffs, rows, iterations=2), cams, targets, RenderOptions.for_camera(cams[0], 3), til


def test_table_trainer_step_is_its_parts(cuda):
    """One step against the chain of public calls it is made of, and against the plain trainer: the
    geometry takes the same step as Trainer's on the expanded coefficients (Adam is per scalar), and the
    table takes Adam's first step, -lr sign(gradient), on the gradient that the sums of the Gaussians'
    SH gradients give."""
    from gs3d.backward import FilteredGaussiansGradients, backward
    from gs3d.loss import LossComputer
    from gs3d.training import TableTrainer, TrainingOptions
    g, table, cams, targets, ro, til = table_scene(cuda)
    before, geometry = table.coeffs.clone(), [t.clone() for t in g.tensors()[:3]]
    opts = TrainingOptions(scene_radius=2.5)
    tr = TableTrainer(g, table, cams, targets, ro, til, opts, seed=4)
    tr.training_step()
    idx = tr.current_camera_index()
    torch.cuda.synchronize()
    # the same gradients from the parts
    expanded = gc.table_lookup(before, table.indices)
    model = GaussiansVector(*geometry, expanded.contiguous())
    out, buf = RenderOutputs.create(96, 64, cuda), RenderBuffers.create(g.n, til.nb_tiles, cuda)
    gs3d.render(out, model, cams[idx], til, ro, buf)
    grad = torch.empty(96, 64, 3, device=cuda)
    LossComputer(96, 64, cuda, opts.loss_dssim_vs_L1_weight)(out.rgb, targets[idx], grad)
    fg = FilteredGaussiansGradients.create(g.n, 3, cuda)
    backward(fg, grad, out, model, cams[idx], til, ro, buf)
    F, _ = gs3d.counts(buf)
    want, bound = gradient_exact(fg.sh_coeffs_grads[:F].cpu(), table.indices.cpu(), table.rows, 1.0,
                                 buf.fgidx_to_gidx[:F].cpu())
    # the backward's float atomics: 1e-3 of the gradient's size between two runs, as elsewhere
    got = tr._table_gradients.sh_coeffs_grads[:table.rows].cpu().double().view(table.rows, -1)
    assert float((got - want).norm()) <= 1e-3 * float(want.norm())
    used = want.abs() > 1e-3 * want.abs().max()
    step = (table.coeffs - before).cpu().double().view(table.rows, -1)
    lr = torch.full((3, 16), opts.sh_coeffs_rest_lr, dtype=torch.float64)
    lr[:, 0] = opts.sh_coeffs_dc_lr
    # m / (1 - b1) = g and v / (1 - b2) = g^2 up to a few roundings each; coefficients move by lr within
    # 16 u of that and the rounding of a coefficient below 2
    assert ((step + lr.view(-1) * want.sign())[used].abs() <= 16 * U * lr.max() + 2 * U).all()
    assert all(not torch.equal(a, b) for a, b in zip(g.tensors()[:3], geometry))
    assert torch.equal(g.sh_coeffs, expanded)  # what this step rendered


def test_table_gradient_of_larger_gradient_buffers(cuda):
    """backward() takes gradient buffers with room for more Gaussians than the render's."""
    from types import SimpleNamespace
    gen = rng(21)
    n, rows = 2000, 30
    table = gc.SHTable(torch.randn(rows, 3, 16, generator=gen).to(cuda), make_indices(n, rows, gen).to(cuda), 0.5)
    grads = torch.randn(n + 700, 3, 16, generator=gen).to(cuda)
    f2g = (torch.randperm(n, generator=gen) + 1).to(torch.int32)
    buffers = SimpleNamespace(fgidx_to_gidx=f2g.to(cuda), device_counts=torch.tensor([1500, 0, 0, 0], dtype=torch.int32, device=cuda))
    got = table.gradient(SimpleNamespace(sh_coeffs_grads=grads), buffers)
    want, bound = gradient_exact(grads.cpu(), table.indices.cpu(), rows, 0.5, f2g, 1500)
    assert ((got.cpu().double().view(rows, -1) - want).abs() <= bound).all()


def test_table_trainer_runs(cuda):
    from gs3d.training import TableTrainer, TrainingOptions
    g, table, cams, targets, ro, til = table_scene(cuda)
    n = g.n
    tr = TableTrainer(g, table, cams, targets, ro, til,
                      TrainingOptions(scene_radius=2.5, sh_degree_increase_interval=2, opacity_reset_interval=2,
                                      adc_interval=1, adc_start_iteration_nb=1))
    for _ in range(6):
        loss = tr.training_step()
    torch.cuda.synchronize()
    assert g.n == n and bool(torch.isfinite(loss[:3]).all()) and bool(torch.isfinite(table.coeffs).all())
    model = gc.compress(g, "nvfp4", table=table)  # and on to 4 bits
    out = RenderOutputs.create(96, 64, cuda)
    gs3d.render(out, model, cams[0], til, ro, RenderBuffers.create(n, til.nb_tiles, cuda))
    assert bool(torch.isfinite(out.rgb).all())
    from gs3d import io
    with pytest.raises(ValueError):
        io.save_checkpoint("/dev/null", tr)
    with pytest.raises(ValueError):
        TableTrainer(g, gc.SHTable(table.coeffs.half(), table.indices), cams, targets, ro, til,
                     TrainingOptions(scene_radius=2.5))
    with pytest.raises(ValueError):
        TableTrainer(g, gc.SHTable(table.coeffs, table.indices[:-1]), cams, targets, ro, til,
                     TrainingOptions(scene_radius=2.5))


@pytest.mark.parametrize("table_rows", [None, 30])
def test_compress_and_render_scripts(cuda, tmp_path, table_rows):
    from gs3d import io, scripts
    g = synthetic_gaussians(SceneSpec(2_000, "uniform:1", -3.5, 0.5), 7)
    io.save_ply(tmp_path / "m.ply", g)
    cams = [look_at_camera(64, 48, 60.0, (0, 0.3, 3))]
    log = []
    model = scripts.compress(tmp_path / "m.ply", tmp_path / "m.npz", table_rows=table_rows, log=log.append)
    assert len(log) == 1 and (model.indices is None) == (table_rows is None)
    a = scripts.render(tmp_path / "m.npz", cameras=cams)[0]
    out, til = RenderOutputs.create(64, 48, cuda), Tiling.for_camera(cams[0])
    gs3d.render(out, model, cams[0], til, RenderOptions.for_camera(cams[0], 3),
                RenderBuffers.create(g.n, til.nb_tiles, cuda))
    assert torch.equal(a, out.rgb)
