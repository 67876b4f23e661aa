"""Compressed SH coefficients without a GPU: the C entry points' refusals (every call below is turned
down before it touches the device) and the Python layer's checks."""
import ctypes as C

import pytest
import torch

from gs3d import CompressedGaussiansVector, MX4Rows, _abi, io, scripts
from gs3d import compressed as gc

LIB = _abi.lib()
DATA = 0x10000  # never read: the calls are refused, or have nothing to do
BIG = 1 << 40


def rows(n=4, dim=48, stride=None, kind=_abi.GS3D_F32, data=DATA):
    return _abi.RowsC(n, dim if stride is None else stride, dim, kind, data)


def mx4(n=4, dim=48, fmt=_abi.GS3D_NVFP4, codes=DATA, scales=DATA, ts=DATA):
    return _abi.MX4RowsC(n, dim, fmt, codes, scales, ts)


def refused(status, *words):
    assert status == _abi.GS3D_ERR_INVALID_ARGUMENT, status
    msg = LIB.gs3d_last_error_string().decode()
    for w in words:
        assert w in msg, msg


BAD_ROWS = [(dict(n=-1), "rows"), (dict(n=BIG), "rows"), (dict(dim=0), "dim"), (dict(dim=1 << 17), "dim"),
            (dict(stride=47), "stride"), (dict(kind=3), "type"), (dict(data=None), "NULL"),
            (dict(data=DATA + 2), "aligned"), (dict(kind=_abi.GS3D_BF16, data=DATA + 1), "aligned")]


@pytest.mark.parametrize("bad,word", BAD_ROWS)
def test_bad_rows_are_refused_everywhere(bad, word):
    r, ok, q = rows(**bad), rows(), mx4()
    refused(LIB.gs3d_table_lookup(C.byref(r), DATA, 1.0, C.byref(ok), None), word)
    refused(LIB.gs3d_table_lookup(C.byref(ok), DATA, 1.0, C.byref(r), None), word)
    refused(LIB.gs3d_table_gradient(C.byref(r), DATA, 4, None, None, 1.0, C.byref(ok), 0, DATA, BIG, None), word)
    refused(LIB.gs3d_table_gradient(C.byref(ok), DATA, 4, None, None, 1.0, C.byref(r), 0, DATA, BIG, None), word)
    refused(LIB.gs3d_mx4_tensor_scale(C.byref(r), DATA, None), word)
    refused(LIB.gs3d_mx4_quantise(C.byref(r), C.byref(q), None), word)
    refused(LIB.gs3d_mx4_dequantise(C.byref(q), C.byref(r), None), word)


def test_lookup_refusals():
    t = rows()
    refused(LIB.gs3d_table_lookup(None, DATA, 1.0, C.byref(t), None), "NULL")
    refused(LIB.gs3d_table_lookup(C.byref(t), DATA, 1.0, None, None), "NULL")
    refused(LIB.gs3d_table_lookup(C.byref(t), None, 1.0, C.byref(rows()), None), "NULL")
    refused(LIB.gs3d_table_lookup(C.byref(t), DATA, 1.0, C.byref(rows(dim=47)), None), "dim")
    # nothing to do: no launch, no error
    assert LIB.gs3d_table_lookup(C.byref(t), None, 1.0, C.byref(rows(n=0, data=None)), None) == _abi.GS3D_OK


def test_gradient_refusals():
    g, t = rows(), rows(n=7)

    def call(g=g, idx=DATA, n_idx=4, f2g=None, t=t, flags=0, ws=DATA, nbytes=BIG):
        return LIB.gs3d_table_gradient(C.byref(g), idx, n_idx, f2g, None, 1.0, C.byref(t), flags, ws, nbytes, None)

    refused(call(t=rows(n=7, dim=12)), "dim")
    refused(call(t=rows(n=7, kind=_abi.GS3D_BF16)), "GS3D_F32")
    refused(call(flags=2), "flags")
    refused(call(n_idx=3), "3 indices for 4 rows")
    refused(call(n_idx=-1, f2g=DATA), "indices")
    refused(call(idx=None), "NULL indices")
    many = dict(g=rows(n=1025), n_idx=1025)
    refused(call(ws=DATA + 128, **many), "aligned")
    size = C.c_size_t(0)
    _abi.check(LIB.gs3d_table_gradient_workspace_size(1025, 7, 48, C.byref(size)))
    assert call(nbytes=size.value - 1, **many) == _abi.GS3D_ERR_WORKSPACE
    assert call(ws=None, **many) == _abi.GS3D_ERR_WORKSPACE
    assert call(t=rows(n=0, data=None)) == _abi.GS3D_OK
    refused(LIB.gs3d_table_gradient_workspace_size(4, 7, 48, None), "NULL")
    for bad in ((-1, 7, 48), (BIG, 7, 48), (4, -1, 48), (4, BIG, 48), (4, 7, 0)):
        refused(LIB.gs3d_table_gradient_workspace_size(*bad, C.byref(size)))


def test_gradient_workspace_grows_with_the_rows():
    size, last = C.c_size_t(0), 0
    for n in (0, 1, 1024, 1025, 100_000, 3_000_000, 1 << 30):
        _abi.check(LIB.gs3d_table_gradient_workspace_size(n, 65_536, 48, C.byref(size)))
        assert size.value >= max(last, 4 * n) if n > 1024 else size.value == 0
        last = size.value


@pytest.mark.parametrize("dim", [1, 3, 27, 48, 119, 130, 1021, 65536])
@pytest.mark.parametrize("table_rows", [1, 1000, 65_536, 3_000_000])
def test_gradient_workspace_serves_fewer_rows(dim, table_rows):
    """A workspace for n rows is large enough for any smaller number: tiles and chunks change with n."""
    sizes, size = [], C.c_size_t(0)
    steps = sorted({max(0, a + d) for a in [*range(0, 30_000, 501), *(1024 * k for k in range(1, 1300, 7)), 303_104, 606_208,
                                            *(592 * 4 * s for s in (1, 2, 21, 32)), *(2368 * 48 * s for s in (1, 2, 5, 18, 21)),
                                            *(2368 * 49 * s for s in (1, 2, 5, 18, 21)), 3_000_000, 1 << 24, 1 << 30]
                    for d in (-1, 0, 1) if a + d <= 1 << 30})
    for n in steps:
        _abi.check(LIB.gs3d_table_gradient_workspace_size(n, table_rows, dim, C.byref(size)))
        sizes.append(size.value)
    assert sizes == sorted(sizes)


@pytest.mark.parametrize("bad,word", [(dict(n=-1), "rows"), (dict(n=BIG), "rows"), (dict(dim=0), "dim"),
                                      (dict(fmt=2), "format"), (dict(codes=None), "NULL"),
                                      (dict(scales=None), "NULL"), (dict(ts=None), "NULL tensor scale")])
def test_bad_mx4_rows_are_refused_everywhere(bad, word):
    q, x = mx4(**bad), rows()
    refused(LIB.gs3d_mx4_quantise(C.byref(x), C.byref(q), None), word)
    refused(LIB.gs3d_mx4_dequantise(C.byref(q), C.byref(x), None), word)
    pos = (C.c_float * 3)()
    refused(LIB.gs3d_mx4_colours(C.byref(q), 0, None, DATA, 4, pos, 1, DATA, 4, None), word)


def test_quantise_refusals():
    refused(LIB.gs3d_mx4_quantise(C.byref(rows(n=5)), C.byref(mx4()), None), "5 rows")
    refused(LIB.gs3d_mx4_dequantise(C.byref(mx4(dim=47)), C.byref(rows()), None), "47")
    refused(LIB.gs3d_mx4_tensor_scale(C.byref(rows()), None, None), "NULL")
    empty = mx4(n=0, codes=None, scales=None, fmt=_abi.GS3D_MXFP4, ts=None)
    assert LIB.gs3d_mx4_quantise(C.byref(rows(n=0, data=None)), C.byref(empty), None) == _abi.GS3D_OK
    assert LIB.gs3d_mx4_dequantise(C.byref(empty), C.byref(rows(n=0, data=None)), None) == _abi.GS3D_OK


def test_colour_refusals():
    pos = (C.c_float * 3)()

    def call(q=mx4(), deg=3, idx=None, means=DATA, n=4, p=pos, views=1, out=DATA, stride=4):
        return LIB.gs3d_mx4_colours(C.byref(q), deg, idx, means, n, p, views, out, stride, None)

    refused(call(q=mx4(dim=47)), "47")
    refused(call(deg=-1), "degree")
    refused(call(deg=3, q=mx4(dim=27)), "degree")
    refused(call(n=5, stride=5), "4 4-bit SH rows for 5 Gaussians")
    refused(call(n=-1), "-1")
    refused(call(means=None), "NULL")
    refused(call(out=None), "NULL")
    refused(call(p=None), "NULL")
    refused(call(views=0), "views")
    refused(call(views=_abi.GS3D_MAX_FACTORED_VIEWS + 1), "views")
    refused(call(stride=3), "stride")
    refused(call(means=DATA + 4), "aligned")
    refused(call(out=DATA + 8), "aligned")
    assert call(n=0, means=None, out=None, stride=0) == _abi.GS3D_OK


def covers(n, dim, stride, elem, at):
    return {at + elem * (r * stride) + b for r in range(n) for b in range(elem * dim)}


def test_results_over_inputs_are_refused():
    """A lookup into its own table and a gradient into its own gradients would read what other threads have
    written. Rows that lie between one another's are fine; where both have gaps and their strides differ,
    ranges that meet are left to the caller."""
    bf, f32 = _abi.GS3D_BF16, _abi.GS3D_F32
    elem = {bf: 2, f32: 4}
    shapes = [(6, 5, 5, f32), (6, 5, 13, f32), (3, 4, 16, f32), (1, 7, 7, bf), (9, 3, 26, bf), (4, 10, 10, bf), (0, 5, 5, f32)]
    kept = 0
    for x in shapes:
        for y in shapes:
            for at in range(-330, 331, 6):
                meet = bool(covers(*x[:3], elem[x[3]], 0) & covers(*y[:3], elem[y[3]], at))
                gap_free = any(r[0] == 1 or r[1] == r[2] for r in (x, y))
                known = gap_free or x[2] * elem[x[3]] == y[2] * elem[y[3]]
                got = gc._rows_meet(gc._row_bytes(rows(*x, DATA)), gc._row_bytes(rows(*y, DATA + at)))
                assert got == (meet and known), (x, y, at)
                kept += meet and known
    assert kept > 500


def test_misaligned_words_are_refused():
    pos = (C.c_float * 3)()
    r, out, q = rows(), rows(), mx4()
    odd = DATA + 2
    refused(LIB.gs3d_table_lookup(C.byref(r), odd, 1.0, C.byref(out), None), "indices", "aligned")
    for k, what in enumerate(("indices", "fgidx_to_gidx", "device_counts")):
        a = [DATA, DATA, DATA]
        a[k] = odd
        refused(LIB.gs3d_table_gradient(C.byref(r), a[0], 4, a[1], a[2], 1.0, C.byref(out), 0, DATA, BIG, None),
                what, "aligned")
    refused(LIB.gs3d_mx4_tensor_scale(C.byref(r), odd, None), "tensor scale", "aligned")
    bad = mx4(ts=odd)
    refused(LIB.gs3d_mx4_quantise(C.byref(r), C.byref(bad), None), "tensor scale", "aligned")
    refused(LIB.gs3d_mx4_dequantise(C.byref(bad), C.byref(out), None), "tensor scale", "aligned")
    refused(LIB.gs3d_mx4_colours(C.byref(bad), 3, None, DATA, 4, pos, 1, DATA, 4, None), "tensor scale", "aligned")
    refused(LIB.gs3d_mx4_colours(C.byref(q), 3, odd, DATA, 4, pos, 1, DATA, 4, None), "indices", "aligned")


def test_a_table_trainer_has_no_checkpoints(tmp_path):
    trainer = type("Trainer", (), {"sh_table": None})()
    torch.save({"format": "gs3d-checkpoint-1"}, tmp_path / "c.pt")
    with pytest.raises(ValueError, match="shared table"):
        io.load_checkpoint(tmp_path / "c.pt", trainer)
    with pytest.raises(ValueError, match="shared table"):
        io.save_checkpoint(tmp_path / "d.pt", trainer)


def test_render_refusals():
    cam, til, opt = _abi.Camera(), _abi.TilingC(), _abi.RenderOptionsC()
    out, buf = _abi.RenderOutputsC(), _abi.RenderBuffersC()
    cam.width = cam.height = 16
    cam.near_z, cam.far_z = 0.2, 100.0
    til.tile_width = til.tile_height = 16
    til.nb_tiles_x = til.nb_tiles_y = 1
    opt.sh_degree = 3
    ro = _abi.RenderOnlyGaussiansC(4, 3, DATA, DATA, None)

    def call(ro=ro, q=mx4(), idx=None, flags=0):
        return LIB.gs3d_render_forward_mx4(C.byref(out), C.byref(ro) if ro else None, C.byref(q) if q else None,
                                           idx, C.byref(cam), C.byref(til), C.byref(opt), C.byref(buf), None,
                                           flags, None)

    refused(call(q=None), "NULL 4-bit")
    refused(call(ro=None), "NULL Gaussians")
    refused(call(q=mx4(dim=27)), "27")
    refused(call(q=mx4(n=3)), "3 4-bit SH rows for 4 Gaussians")
    refused(call(flags=_abi.GS3D_RENDER_DEFER_COLOUR), "DEFER_COLOUR")
    opt.sh_degree = 2
    refused(call(ro=_abi.RenderOnlyGaussiansC(4, 1, DATA, DATA, None), q=mx4(dim=12)), "degree")


# -- the Python layer ---------------------------------------------------------------------------
def test_mx4_rows_checks():
    u8 = lambda *s: torch.zeros(s, dtype=torch.uint8)  # noqa: E731
    one = torch.ones(1)
    q = MX4Rows(u8(5, 14), u8(5, 2), one, 27, "nvfp4")
    assert (q.rows, q.nbytes) == (5, 5 * 16 + 4)
    assert MX4Rows(u8(5, 14), u8(5, 1), None, 27, "mxfp4").rows == 5
    for bad in ((u8(5, 13), u8(5, 2), one, 27, "nvfp4"), (u8(5, 14), u8(5, 1), one, 27, "nvfp4"),
                (u8(5, 14), u8(4, 2), one, 27, "nvfp4"), (u8(5, 14), u8(5, 2), None, 27, "nvfp4"),
                (u8(5, 14), u8(5, 2), one.double(), 27, "nvfp4"), (u8(5, 14), u8(5, 1), one, 27, "mxfp4"),
                (u8(5, 14).char(), u8(5, 2), one, 27, "nvfp4"), (u8(5, 28)[:, ::2], u8(5, 2), one, 27, "nvfp4"),
                (u8(5, 14), u8(5, 2), one, 27, "fp4")):
        with pytest.raises(ValueError):
            MX4Rows(*bad)
    with pytest.raises(ValueError):
        MX4Rows.empty(3, 48, "int4", "cpu")


def test_a_tensor_scale_of_another_device_or_type_never_reaches_a_kernel():
    """A kernel follows the pointer: a scale in host memory beside codes on the GPU would fault it."""
    for fmt, device, ts in (("nvfp4", "meta", torch.ones(1)), ("nvfp4", "cpu", torch.ones(1).double()),
                            ("nvfp4", "cpu", torch.ones(2)), ("mxfp4", "cpu", torch.ones(1))):
        with pytest.raises(ValueError, match="scale"):
            MX4Rows.empty(3, 48, fmt, device, ts)
        q = MX4Rows.empty(3, 48, fmt, device)  # without one for now
        if fmt == "nvfp4":
            q.tensor_scale = ts
            with pytest.raises(ValueError, match="scale"):
                q.to_c()
    assert MX4Rows.empty(3, 48, "nvfp4", "cpu", torch.ones(1)).to_c().tensor_scale
    q = MX4Rows.empty(3, 48, "mxfp4", "cpu")
    q.scales = q.scales.to("meta")
    with pytest.raises(ValueError, match="one device"):
        q.to_c()


def test_compressed_gaussians_checks():
    q = MX4Rows.empty(6, 48, "mxfp4", "cpu")
    mo, cov, idx = torch.zeros(6, 4), torch.zeros(6, 6), torch.ones(6, dtype=torch.int32)
    g = CompressedGaussiansVector(mo, cov, q)
    assert g.n == 6 and g.sh_degree == 3 and g.to_c().sh_coeffs is None
    assert CompressedGaussiansVector(mo, cov, MX4Rows.empty(2, 27, "mxfp4", "cpu"), idx).sh_degree == 2
    for bad in ((mo[:5], cov, q), (mo, cov[:, :5], q), (mo.double(), cov, q), (mo[:5], cov[:5], q),
                (mo, cov, MX4Rows.empty(6, 47, "mxfp4", "cpu")), (mo, cov, q, idx.long()), (mo, cov, q, idx[:5])):
        with pytest.raises(ValueError):
            CompressedGaussiansVector(*bad)


def test_compressed_gaussians_are_checked_again_before_a_render():
    """The fields can be assigned: what a kernel would follow or misread does not get there."""
    make = lambda: CompressedGaussiansVector(torch.zeros(6, 4), torch.zeros(6, 6),  # noqa: E731
                                             MX4Rows.empty(6, 48, "mxfp4", "cpu"), torch.ones(6, dtype=torch.int32))
    assert make().to_c().n == 6
    for name, value in (("indices", torch.ones(6, dtype=torch.int64)), ("indices", torch.ones(5, dtype=torch.int32)),
                        ("indices", torch.ones(6, dtype=torch.int32, device="meta")), ("means_opacities", torch.zeros(7, 4)),
                        ("covariances", torch.zeros(6, 6, device="meta")), ("sh", MX4Rows.empty(6, 47, "mxfp4", "cpu"))):
        g = make()
        setattr(g, name, value)
        with pytest.raises(ValueError):
            g.to_c()


def test_rows_of_a_tensor():
    t = torch.zeros(5, 3, 16)
    assert (lambda c: (c.rows, c.row_stride, c.dim, c.type))(gc._rows_c(t, "t")) == (5, 48, 48, _abi.GS3D_F32)
    c = gc._rows_c(torch.zeros(5, 64, dtype=torch.bfloat16)[:, 3:30], "t")
    assert (c.rows, c.row_stride, c.dim, c.type) == (5, 64, 27, _abi.GS3D_BF16)
    assert gc._rows_c(torch.zeros(9, 4)[::3], "t").row_stride == 12
    assert gc._rows_c(torch.zeros(0, 4), "t").rows == 0
    for bad in (torch.zeros(5), torch.zeros(5, 4).double(), torch.zeros(4, 5).t(), torch.zeros(1, 4).expand(5, 4),
                torch.zeros(5, 16, 3).transpose(1, 2)):
        with pytest.raises(ValueError):
            gc._rows_c(bad, "t")


def test_sizes_that_do_not_fit_the_calls_fields_are_refused():
    """The library takes a row's length and the number of Gaussians as 32 bits: what does not fit must not
    come out as the small number that its low bits are."""
    big = 1 << 32
    meta = lambda *s, **k: torch.empty(s, device="meta", **k)  # noqa: E731
    for t in (meta(1, big + 48), meta(2, 3, big // 2 + 16), meta(1, (1 << 16) + 1)):
        with pytest.raises(ValueError, match="elements a row"):
            gc._rows_c(t, "t")
    assert gc._rows_c(meta(1, 1 << 16), "t").dim == 1 << 16
    u8 = dict(dtype=torch.uint8)
    q = MX4Rows(meta(1, big // 2 + 24, **u8), meta(1, big // 32 + 2, **u8), None, big + 48, "mxfp4")
    with pytest.raises(ValueError, match="elements a row"):
        q.to_c()
    with pytest.raises(ValueError, match="Gaussians"):
        gc.mx4_colours(MX4Rows.empty(4, 48, "mxfp4", "meta"), meta(big + 4, 4), [[0.0, 0.0, 0.0]], 3)


def test_table_gradient_of_larger_gradient_buffers(monkeypatch):
    """backward() takes gradient buffers with room for more Gaussians than the render's; so does the table."""
    from types import SimpleNamespace
    seen = []
    monkeypatch.setattr(gc, "table_gradient", lambda g, *a: seen.append((g.shape, a[5].shape)))
    table = gc.SHTable(torch.zeros(2, 3, 4), torch.ones(6, dtype=torch.int32))
    for room, n in ((9, 6), (6, 6), (6, 9)):
        table.gradient(SimpleNamespace(sh_coeffs_grads=torch.zeros(room, 3, 4)),
                       SimpleNamespace(fgidx_to_gidx=torch.zeros(n, dtype=torch.int32), device_counts=torch.zeros(4, dtype=torch.int32)))
    assert seen == [((6, 3, 4), (6,)), ((6, 3, 4), (6,)), ((6, 3, 4), (9,))]


def test_calls_need_cuda_tensors_of_the_right_kind():
    t, i = torch.zeros(4, 48), torch.ones(3, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        gc.table_lookup(t, i)
    with pytest.raises(ValueError, match="int32"):
        gc.table_lookup(t, i.long())
    with pytest.raises(ValueError, match="int32"):
        gc.table_gradient(t, i, 4, fgidx_to_gidx=i.long())
    with pytest.raises(ValueError, match="CUDA"):
        gc.table_gradient(t, i, 4)
    with pytest.raises(ValueError, match="CUDA"):
        gc.mx4_quantise(t)
    with pytest.raises(ValueError, match="CUDA"):
        gc.mx4_dequantise(MX4Rows.empty(4, 48, "mxfp4", "cpu"))
    with pytest.raises(ValueError, match="positions"):
        gc.mx4_colours(MX4Rows.empty(4, 48, "mxfp4", "cpu"), torch.zeros(4, 4), [0.0, 0.0, 0.0], 3)
    with pytest.raises(ValueError):
        gc.SHTable(torch.zeros(4, 3, 5), i)
    with pytest.raises(ValueError):
        gc.fit_table(torch.zeros(4, 3, 16), 0)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_fit_table_refuses_what_has_no_mean(bad):
    """One coefficient that is not finite would make its row's mean NaN, the nearest row of every Gaussian
    after that, and so the whole table."""
    sh = torch.randn(50, 3, 4, generator=torch.Generator().manual_seed(1))
    sh[7, 1, 2] = bad
    with pytest.raises(ValueError, match="finite"):
        gc.fit_table(sh, 5)
    with pytest.raises(ValueError, match="float32"):
        gc.fit_table(sh.half(), 5)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("table", [False, True])
def test_compressed_model_file_round_trip(tmp_path, fmt, table):
    gen = torch.Generator().manual_seed(1)
    n, rows = 9, 4 if table else 9
    byte = lambda *s: torch.randint(0, 256, s, generator=gen, dtype=torch.uint8)  # noqa: E731
    sh = MX4Rows(byte(rows, 14), byte(rows, 2 if fmt == "nvfp4" else 1),
                 torch.tensor([0.3]) if fmt == "nvfp4" else None, 27, fmt)
    idx = torch.randint(0, 6, (n,), generator=gen, dtype=torch.int32) if table else None
    g = CompressedGaussiansVector(torch.randn(n, 4, generator=gen), torch.randn(n, 6, generator=gen), sh, idx)
    io.save_compressed(tmp_path / "m.npz", g)
    b = io.load_compressed(tmp_path / "m.npz")
    assert (b.sh.format, b.sh.dim, b.sh_degree) == (fmt, 27, 2)
    for x, y in ((g.means_opacities, b.means_opacities), (g.covariances, b.covariances), (sh.codes, b.sh.codes),
                 (sh.scales, b.sh.scales)):
        assert torch.equal(x, y)
    assert (b.indices is None) == (not table) and (not table or torch.equal(b.indices, idx))
    assert (b.sh.tensor_scale is None) == (fmt == "mxfp4")


def test_compressed_model_file_refusals(tmp_path):
    import numpy as np
    np.savez(tmp_path / "x.npz", a=np.zeros(3))
    with pytest.raises(ValueError, match="not a compressed"):
        io.load_compressed(tmp_path / "x.npz")
    with pytest.raises(ValueError, match="npz"):
        scripts.compress(tmp_path / "m.ply", tmp_path / "m.ply", device="cpu")


def test_a_table_trainer_holds_no_moments_of_the_gaussians_own_coefficients(monkeypatch):
    """Its optimizers are the geometry's and the table's: nothing of n x 48 moments, nor statistics for a
    densification that never happens, is allocated on the way there."""
    from gs3d import training
    from gs3d.optimizer import AdamMoments
    from gs3d.scene import SceneSpec, look_at_camera, synthetic_gaussians
    g = synthetic_gaussians(SceneSpec(20, "uniform:1", -3.5, 0.4), 2)
    cam = look_at_camera(96, 64, 60.0, (0, 0.4, 2.5))
    args = (g, gc.SHTable(torch.zeros(4, 3, 16), torch.ones(20, dtype=torch.int32)), [cam], [torch.rand(96, 64, 3)],
            training.RenderOptions.for_camera(cam, 3), training.Tiling.for_camera(cam),
            training.TrainingOptions(scene_radius=2.5))
    made, zeros = [], AdamMoments.zeros
    monkeypatch.setattr(AdamMoments, "zeros", lambda n, degree, device: made.append((n, degree)) or zeros(n, degree, device))
    monkeypatch.setattr(training.adc_mod.AdcBuffers, "create", lambda *a: pytest.fail("statistics"))
    tr = training.TableTrainer(*args)
    assert made == [(20, 0), (4, 3)]
    assert tr.optimizer.moments.n == 20 and tr.table_optimizer.moments.n == 4 and not tr.rebuild_sh_grads
    with pytest.raises(ValueError, match="rebuild_sh_grads"):
        training.TableTrainer(*args, rebuild_sh_grads=True)
    assert not training.TableTrainer(*args, rebuild_sh_grads=False).rebuild_sh_grads
