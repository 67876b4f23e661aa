"""SH coefficients in fewer bytes (no counterpart in the reference, which keeps 3 (d+1)^2 floats per
Gaussian): rows shared through a table, with the table's gradient for fine-tuning, and rows in
microscaled 4-bit floating point, with the colours a render takes from them. All through libgs3d.so.

    table_lookup / table_gradient ....... out[i] = scale * table[indices[i]], and its gradient
    mx4_tensor_scale / mx4_quantise /
    mx4_dequantise ...................... rows <-> 4-bit elements with block scales (MX4Rows)
    mx4_colours ......................... colours of Gaussians with 4-bit rows from given cameras
    SHTable, fit_table .................. a model's table and its 1-based row per Gaussian
    compress ............................ a CompressedGaussiansVector for gs3d.render

Every call runs on `stream` (default: the current stream of its tensors' device), allocates what it
returns and its workspace there, and does not synchronise; it can be captured into a CUDA graph."""
from __future__ import annotations

import ctypes as C
import functools
from dataclasses import dataclass

import numpy as np
import torch

from . import _abi
from .structs import (MX4_FORMATS, CompressedGaussiansVector, GaussiansVector, MX4Rows,
                      RenderOnlyGaussiansVector)

_TYPES = {torch.float32: _abi.GS3D_F32, torch.float16: _abi.GS3D_F16, torch.bfloat16: _abi.GS3D_BF16}


def _rows_c(t: torch.Tensor, what: str) -> _abi.RowsC:
    """gs3d_rows of a (rows, ...) tensor whose trailing axes are contiguous."""
    kind = _TYPES.get(t.dtype)
    if kind is None:
        raise ValueError(f"{what}: {t.dtype} is not float32, float16 or bfloat16")
    shape = t.shape
    if len(shape) < 2:
        raise ValueError(f"{what}: need (rows, ...), got shape {tuple(shape)}")
    rows, dim = shape[0], shape[1]
    for size in shape[2:]:
        dim *= size
    if dim > _abi.GS3D_MAX_ROW_DIM:  # the C field has 32 bits and would take the low ones
        raise ValueError(f"{what}: {dim} elements a row (at most {_abi.GS3D_MAX_ROW_DIM})")
    if t.is_contiguous():
        return _abi.RowsC(rows, dim, dim, kind, t.data_ptr())
    expect = 1
    for size, st in zip(reversed(shape[1:]), reversed(t.stride()[1:])):
        if size != 1 and st != expect:
            raise ValueError(f"{what}: the elements of a row must be contiguous")
        expect *= size
    stride = t.stride(0) if rows > 1 else dim
    if stride < dim:
        raise ValueError(f"{what}: rows overlap (row stride {stride}, {dim} elements)")
    return _abi.RowsC(rows, stride, dim, kind, t.data_ptr())


def _row_bytes(r: _abi.RowsC) -> tuple[int, int, int, int]:
    """First byte, byte behind the last, stride and length of the rows (of rows without gaps: one row)."""
    e = 4 if r.type == _abi.GS3D_F32 else 2
    begin, stride, size = r.data or 0, r.row_stride * e, r.dim * e
    end = begin + (r.rows - 1) * stride + size if r.rows > 0 else begin
    if r.rows > 1 and stride == size:
        stride = size = end - begin
    return begin, end, stride, size


def _rows_meet(a: tuple[int, int, int, int], b: tuple[int, int, int, int]) -> bool:
    """Whether rows (of _row_bytes) are known to share bytes: exactly, but for rows with gaps of
    different strides, which may lie between one another's."""
    (a0, a1, sa, la), (b0, b1, sb, lb) = a, b
    if a0 == a1 or b0 == b1 or a0 >= b1 or b0 >= a1:
        return False
    if a1 - a0 == la:  # a is one range: the first row of b that ends behind its start
        return b0 + max(0, -((b0 + lb - 1 - a0) // sb)) * sb < a1
    if b1 - b0 == lb:
        return a0 + max(0, -((a0 + la - 1 - b0) // sa)) * sa < b1
    if sa != sb:
        return False
    d = (b0 - a0) % sa
    return d < la or sa - d < lb


def _check_apart(out: _abi.RowsC, x: tuple[int, int, int, int], what: str) -> None:
    if _rows_meet(_row_bytes(out), x):
        raise ValueError(f"out overlaps {what}")


def _check_device(first: torch.Tensor, *others) -> torch.device:
    device = first.device
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, not {device}")
    for t in others:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {device} and {t.device}")
    return device


def _check_indices(t: torch.Tensor | None, what: str = "indices") -> None:
    if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous()):
        raise ValueError(f"{what} must be a contiguous (n,) int32 tensor (1-based)")


def _enter(device: torch.device, stream: torch.cuda.Stream | None):
    """(raw stream, context): makes the tensors' device and the call's stream current, so that what the
    call allocates belongs to that stream; context None where they are already. These calls can cost
    less on the GPU than their host side, so the raw handle is asked for without a Stream object."""
    index = device.index
    if stream is None:
        if index == torch.cuda.current_device():
            return torch._C._cuda_getCurrentRawStream(index), None
        context = torch.cuda.device(device)
    elif stream.device != device:
        raise ValueError(f"stream on {stream.device} for tensors on {device}")
    else:
        context = torch.cuda.stream(stream)
    context.__enter__()
    return torch._C._cuda_getCurrentRawStream(index), context


def _leave(context) -> None:
    if context is not None:
        context.__exit__(None, None, None)


@functools.lru_cache(maxsize=256)
def _gradient_workspace_bytes(grad_rows: int, table_rows: int, dim: int) -> int:
    nbytes = C.c_size_t(0)
    _abi.check(_abi.lib().gs3d_table_gradient_workspace_size(grad_rows, table_rows, dim, C.byref(nbytes)))
    return nbytes.value


# -- tables -----------------------------------------------------------------------------------
def table_lookup(table: torch.Tensor, indices: torch.Tensor, scale: float = 1.0,
                 dtype: torch.dtype | None = None, out: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """out[i] = scale * table[indices[i] - 1]: the rows of `table` ((rows, ...), float32, float16 or
    bfloat16) for 1-based int32 `indices`; an index outside 1 .. rows gives zeros. Products are
    fp32, rounded once to `dtype` (default: the table's). `out` ((n, ...), apart from the table) is
    filled in place."""
    _check_indices(indices)
    device = _check_device(table, indices, out)
    t = _rows_c(table, "table")
    shape = (indices.shape[0], *table.shape[1:])
    handle, context = _enter(device, stream)
    try:
        given = out is not None
        if not given:
            out = table.new_empty(shape, dtype=dtype)
        elif out.shape != shape or (dtype is not None and out.dtype != dtype):
            raise ValueError(f"out {tuple(out.shape)} {out.dtype} for a lookup of {shape} {dtype or out.dtype}")
        o = _rows_c(out, "out")
        if given:
            _check_apart(o, _row_bytes(t), "the table")
        _abi.check(_abi.lib().gs3d_table_lookup(t, indices.data_ptr(), scale, o, handle))
    finally:
        _leave(context)
    return out


def table_gradient(grads: torch.Tensor, indices: torch.Tensor, nb_rows: int, scale: float = 1.0,
                   out: torch.Tensor | None = None, accumulate: bool = False,
                   fgidx_to_gidx: torch.Tensor | None = None,
                   device_counts: torch.Tensor | None = None,
                   stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The gradient of table_lookup for a table of `nb_rows` rows: float32 rows out[k] = scale * sum
    of grads[f] over the rows f with index k + 1, summed in an order fixed by the indices.
    `fgidx_to_gidx`: row f of `grads` belongs to filtered Gaussian f (as in
    FilteredGaussiansGradients.sh_coeffs_grads) and has index indices[fgidx_to_gidx[f] - 1];
    `device_counts`: only the first device_counts[0] rows take part. `accumulate`: add to `out`
    (apart from `grads`)."""
    _check_indices(indices)
    _check_indices(fgidx_to_gidx, "fgidx_to_gidx")
    device = _check_device(grads, indices, fgidx_to_gidx, device_counts, out)
    g = _rows_c(grads, "grads")
    if fgidx_to_gidx is not None and fgidx_to_gidx.shape[0] < g.rows:
        raise ValueError(f"{fgidx_to_gidx.shape[0]} fgidx_to_gidx entries for {g.rows} rows")
    if device_counts is not None and (device_counts.dtype != torch.int32 or device_counts.numel() < 1):
        raise ValueError("device_counts must hold int32 counts")
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    shape = (int(nb_rows), *grads.shape[1:])
    handle, context = _enter(device, stream)
    try:
        given = out is not None
        if not given:
            out = grads.new_empty(shape, dtype=torch.float32)
        elif out.shape != shape or out.dtype != torch.float32:
            raise ValueError(f"out {tuple(out.shape)} {out.dtype} for a float32 table gradient of {shape}")
        o = _rows_c(out, "out")
        if given:
            _check_apart(o, _row_bytes(g), "grads")
        nbytes = _gradient_workspace_bytes(g.rows, o.rows, g.dim)
        ws = grads.new_empty(nbytes, dtype=torch.uint8) if nbytes else None
        _abi.check(_abi.lib().gs3d_table_gradient(
            g, indices.data_ptr(), indices.shape[0],
            None if fgidx_to_gidx is None else fgidx_to_gidx.data_ptr(),
            None if device_counts is None else device_counts.data_ptr(), scale, o,
            _abi.GS3D_TABLE_ACCUMULATE if accumulate else 0, ws.data_ptr() if nbytes else None, nbytes,
            handle))
    finally:
        _leave(context)
    return out


# -- 4-bit rows -------------------------------------------------------------------------------
def mx4_tensor_scale(x: torch.Tensor, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """(1,) float32: max(largest finite |x| * (1 / 2688), 2^-100), reciprocal and product in float32: the
    nvfp4 tensor scale with which the block scales of `x` ((rows, ...)) use their range. At most one unit in
    the last place from the quotient by 2688 rounded once."""
    device = _check_device(x)
    c = _rows_c(x, "x")
    handle, context = _enter(device, stream)
    try:
        scale = x.new_empty(1, dtype=torch.float32)
        _abi.check(_abi.lib().gs3d_mx4_tensor_scale(c, scale.data_ptr(), handle))
    finally:
        _leave(context)
    return scale


def mx4_quantise(x: torch.Tensor, format: str = "nvfp4", tensor_scale: torch.Tensor | None = None,
                 stream: torch.cuda.Stream | None = None) -> MX4Rows:
    """The rows of `x` ((rows, ...), float32, float16 or bfloat16) as 4-bit elements with block
    scales (gs3d_mx4_quantise). `tensor_scale` (nvfp4): (1,) float32 on the device, from 2^-100 to
    the largest float32 / 2688, which the rows keep (not a copy); None: mx4_tensor_scale(x)."""
    device = _check_device(x, tensor_scale)
    c = _rows_c(x, "x")
    handle, context = _enter(device, stream)
    try:
        if format == "nvfp4":
            if tensor_scale is None:
                tensor_scale = x.new_empty(1, dtype=torch.float32)
                _abi.check(_abi.lib().gs3d_mx4_tensor_scale(c, tensor_scale.data_ptr(), handle))
            elif tensor_scale.numel() != 1 or tensor_scale.dtype != torch.float32:
                raise ValueError("the tensor scale is (1,) float32")
        elif tensor_scale is not None:
            raise ValueError(f"{format} rows have no tensor scale")
        q = MX4Rows.empty_beside(x, c.rows, c.dim, format, tensor_scale)
        _abi.check(_abi.lib().gs3d_mx4_quantise(c, q.to_c(), handle))
    finally:
        _leave(context)
    return q


def mx4_dequantise(rows: MX4Rows, dtype: torch.dtype = torch.float32, out: torch.Tensor | None = None,
                   stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """The values `rows` stand for as (rows, dim) `dtype`, or into `out` ((rows, ...) of dim elements)."""
    device = _check_device(rows.codes, out)
    handle, context = _enter(device, stream)
    try:
        given = out is not None
        if not given:
            out = rows.codes.new_empty((rows.rows, rows.dim), dtype=dtype)
        o = _rows_c(out, "out")
        if given:
            for t, what in ((rows.codes, "the codes"), (rows.scales, "the scales")):
                begin, size = t.data_ptr(), t.numel()
                _check_apart(o, (begin, begin + size, size, size), what)
        _abi.check(_abi.lib().gs3d_mx4_dequantise(rows.to_c(), o, handle))
    finally:
        _leave(context)
    return out


def mx4_colours(rows: MX4Rows, means: torch.Tensor, positions, sh_degree: int,
                indices: torch.Tensor | None = None, out: torch.Tensor | None = None,
                stream: torch.cuda.Stream | None = None) -> torch.Tensor:
    """Colours of n Gaussians seen from the cameras at `positions` ((views, 3) float32, host): a
    (views, n, 4) float32 tensor, the fourth value 0 (the rows render_given_colour takes with
    shard_rows = n, n_ranks = 1). `means`: (n, 4) float32, the first three the mean; Gaussian i has
    SH row i of `rows`, or row indices[i] (1-based)."""
    pos = np.ascontiguousarray(positions, dtype=np.float32)
    if pos.ndim != 2 or pos.shape[1] != 3:
        raise ValueError(f"positions must be (views, 3), got {pos.shape}")
    _check_indices(indices)
    n = means.shape[0]
    if n >= 1 << 31:  # the C argument has 32 bits and would take the low ones
        raise ValueError(f"{n} Gaussians (below 2^31)")
    device = _check_device(rows.codes, means, indices, out)
    if means.shape != (n, 4) or means.dtype != torch.float32 or not means.is_contiguous():
        raise ValueError("means must be a contiguous (n, 4) float32 tensor")
    if indices is not None and indices.shape[0] != n:
        raise ValueError(f"{indices.shape[0]} indices for {n} Gaussians")
    shape = (pos.shape[0], n, 4)
    handle, context = _enter(device, stream)
    try:
        if out is None:
            out = means.new_empty(shape)
        elif out.shape != shape or out.dtype != torch.float32 or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous float32 tensor of shape {shape}")
        _abi.check(_abi.lib().gs3d_mx4_colours(
            rows.to_c(), int(sh_degree), None if indices is None else indices.data_ptr(),
            means.data_ptr(), n, pos.__array_interface__["data"][0], pos.shape[0], out.data_ptr(), n, handle))
    finally:
        _leave(context)
    return out


# -- models -----------------------------------------------------------------------------------
@dataclass
class SHTable:
    """SH coefficients shared by Gaussians: Gaussian i has scale * coeffs[indices[i] - 1].
    `coeffs`: (rows, 3, (d+1)^2) float32, float16 or bfloat16; `indices`: (n,) int32, 1-based."""

    coeffs: torch.Tensor
    indices: torch.Tensor
    scale: float = 1.0

    def __post_init__(self):
        if self.coeffs.dim() != 3 or self.coeffs.shape[1] != 3 or self.coeffs.shape[2] not in (1, 4, 9, 16):
            raise ValueError(f"coeffs must be (rows, 3, (d+1)^2), got {tuple(self.coeffs.shape)}")
        _check_indices(self.indices)

    @property
    def rows(self) -> int:
        return self.coeffs.shape[0]

    def expand(self, out: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """(n, 3, (d+1)^2) float32 SH coefficients, e.g. into a GaussiansVector's sh_coeffs."""
        return table_lookup(self.coeffs, self.indices, self.scale, torch.float32, out, stream)

    def gradient(self, fgradients, buffers, out: torch.Tensor | None = None, accumulate: bool = False,
                 stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """Gradient of `coeffs` from the SH gradients of backward() (FilteredGaussiansGradients and
        the RenderBuffers of its render). Above the render's SH degree backward() leaves the gradients as they
        were (zeros in fresh buffers), and those are what is summed there. Gradient buffers may hold more
        Gaussians than the render's; their further rows belong to none."""
        grads, f2g = fgradients.sh_coeffs_grads, buffers.fgidx_to_gidx
        return table_gradient(grads[:f2g.shape[0]], self.indices, self.rows, self.scale, out, accumulate, f2g,
                              buffers.device_counts, stream)

    def to(self, device) -> "SHTable":
        return SHTable(self.coeffs.to(device), self.indices.to(device), self.scale)


def fit_table(sh_coeffs: torch.Tensor, nb_rows: int, iterations: int = 10, seed: int = 0) -> SHTable:
    """A table of (at most) `nb_rows` rows for `sh_coeffs` ((n, 3, order) finite float32 on a CUDA device)
    by Lloyd's algorithm: rows start as a random choice of the Gaussians' coefficients, then every
    Gaussian takes its nearest row and every row the mean of its Gaussians (rows without any keep
    their value). A one-off preparation: the distances are torch products, in chunks."""
    n = sh_coeffs.shape[0]
    if n < 1 or nb_rows < 1:
        raise ValueError(f"a table of {nb_rows} rows for {n} Gaussians")
    if sh_coeffs.dtype != torch.float32 or not bool(torch.isfinite(sh_coeffs).all()):
        raise ValueError("the coefficients must be finite float32 values")
    x = sh_coeffs.reshape(n, -1)
    gen = torch.Generator().manual_seed(int(seed))
    pick = torch.randperm(n, generator=gen)[:nb_rows].to(x.device)
    centres = x[pick].clone()
    rows = centres.shape[0]
    chunk = max(1, (1 << 28) // rows)
    indices = torch.empty(n, dtype=torch.int32, device=x.device)
    for it in range(max(1, int(iterations)) + 1):
        half = 0.5 * (centres * centres).sum(dim=1)
        for a in range(0, n, chunk):
            b = min(n, a + chunk)
            indices[a:b] = (torch.addmm(half, x[a:b], centres.t(), alpha=-1.0).argmin(dim=1) + 1).to(torch.int32)
        if it == max(1, int(iterations)):
            break
        sums = table_gradient(x, indices, rows)
        members = torch.bincount(indices.long(), minlength=rows + 1)[1:, None]
        centres = torch.where(members > 0, sums / members.clamp(min=1), centres)
    return SHTable(centres.reshape(rows, *sh_coeffs.shape[1:]).contiguous(), indices)


def compress(gaussians, format: str = "nvfp4", table: SHTable | None = None) -> CompressedGaussiansVector:
    """A model for rendering with its SH coefficients in 4 bits: every Gaussian's own row, or with
    `table` the table's rows (times its scale) and its indices. `gaussians`: GaussiansVector or
    RenderOnlyGaussiansVector on a CUDA device."""
    ro = (RenderOnlyGaussiansVector.from_trainable(gaussians) if isinstance(gaussians, GaussiansVector)
          else gaussians)
    if table is None:
        return CompressedGaussiansVector(ro.means_opacities, ro.covariances,
                                         mx4_quantise(ro.sh_coeffs, format))
    rows = table_lookup(table.coeffs, torch.arange(1, table.rows + 1, dtype=torch.int32,
                                                   device=table.coeffs.device), table.scale, torch.float32)
    return CompressedGaussiansVector(ro.means_opacities, ro.covariances, mx4_quantise(rows, format),
                                     table.indices)


__all__ = ["MX4_FORMATS", "MX4Rows", "SHTable", "CompressedGaussiansVector", "compress", "fit_table",
           "mx4_colours", "mx4_dequantise", "mx4_quantise", "mx4_tensor_scale", "table_gradient",
           "table_lookup"]
