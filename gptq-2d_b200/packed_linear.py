"""Products with a rounded matrix in packed codes, and low-rank adapters of many requests beside them.

``packed_linear`` multiplies activations by the matrix that ``packed_codes.pack_codes`` stored: the codes are what is read, half a byte per weight, and
``(code + qmin - zero_point) * scale`` is formed inside the product.  The requests of a batch may each have a low-rank adapter of their own beside the
shared matrix (``LowRankAdapters``); a token names its adapter by number.  CUDA only, like the rest of the package; no gradients.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple

import torch

import _abi


class LowRankAdapters(NamedTuple):
    """``scaling[i] * up[i] @ down[i]`` for every adapter: ``down [adapters, rank, n]``, ``up [adapters, m, rank]`` in the activations' type, ``scaling [adapters]``
    float32 or None (1).  ``rank`` is a multiple of 8 up to 64; adapters of smaller rank are padded with zeros."""

    down: torch.Tensor
    up: torch.Tensor
    scaling: torch.Tensor | None = None


_HALF = {torch.float16: _abi.FP16, torch.bfloat16: _abi.BF16}
_WORKSPACE: dict[tuple, int] = {}  # bytes by sizes


def _parameter(t, m: int, n: int, name: str, device):
    """A scale or zero point: one value, one per row, or one per row and group of columns; with its strides over rows and groups, and how many groups."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.get_device() != device.index:
        t = torch.as_tensor(t, dtype=torch.float32, device=device)
    shape = t.shape
    assert len(shape) <= 2, f"{name} must be one value, one per row, or one per row and group of columns"
    rows, groups = (1, 1, *shape)[-2:]
    strides = (0, 0, *t.stride())[-2:]
    assert rows == m or rows == 1, f"{name} must have one row or one for each of the {m} rows of codes"
    assert groups == 1 or (groups > 1 and n % groups == 0 and n // groups % 64 == 0), f"{name}: groups must divide the {n} columns into multiples of 64"
    return t, strides[0] if rows > 1 else 0, strides[1] if groups > 1 else 0, groups


def packed_linear(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor, *, qmin: float, bits: int = 4,
                  adapters: LowRankAdapters | None = None, adapter_index: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T [..., m]`` for ``x [..., n]`` (float16 or bfloat16, CUDA) and the matrix ``W [m, n]`` whose 4-bit codes are ``codes`` (uint8 ``[m, n / 2]`` from
    ``pack_codes``, ``n`` a multiple of 32), ``W = (code + qmin - zero_point) * scale``.

    ``scale`` and ``zero_point`` are one value, ``[m, 1]``, or ``[m, groups]`` with equal groups of columns, each a multiple of 64 wide (float32; where both have groups,
    the same number).  Zero points are meant to be integers: with many tokens ``code + qmin - zero_point`` is rounded to x's type, exact up to 256 (bfloat16) or 2048 (float16).
    With ``adapters``, ``adapter_index`` (int32, one per token, in the order of ``x``'s leading dimensions) says whose adapter is added to a token's result; an index outside
    the adapters' range means none.  Sums are float32, results are rounded once to x's type.  ``out`` may be given as a contiguous ``[..., m]`` tensor, which must not
    overlap the inputs."""
    assert bits == 4, "only codes of 4 bits can be multiplied with"
    device, dtype, shape = x.device, x.dtype, x.shape
    index = device.index
    assert x.is_cuda, "the product with packed codes requires CUDA tensors (there is no CPU path)"
    half = _HALF.get(dtype)
    assert half is not None and len(shape) >= 1, "expected float16 or bfloat16 activations [..., n]"
    assert codes.dim() == 2 and codes.dtype == torch.uint8 and codes.is_contiguous() and codes.get_device() == index, "expected contiguous uint8 codes on the activations' device"
    n, (m, row_bytes), codes_at = shape[-1], codes.shape, codes.data_ptr()
    assert n > 0 and n % 32 == 0, "the number of columns must be a multiple of 32"
    assert row_bytes >= n // 2 and row_bytes % 16 == 0 and codes_at % 16 == 0, "rows of codes must hold n entries and be 16-byte aligned"
    rows = x if len(shape) == 2 else x.detach().reshape(-1, n)
    row_stride, last = rows.stride()
    tokens = rows.shape[0]
    # rows that lie over one another (one row for every token, windows of a longer one) are copied: the tiles' copies need rows that stand apart
    if last != 1 or row_stride % 8 or rows.data_ptr() % 16 or (row_stride < n and tokens > 1):
        rows = rows.detach().clone(memory_format=torch.contiguous_format)
        row_stride = n
    scale, scale_row, scale_group, groups = _parameter(scale, m, n, "scale", device)
    zero, zero_row, zero_group, zero_groups = _parameter(zero_point, m, n, "zero_point", device)
    assert groups == zero_groups or groups == 1 or zero_groups == 1, "scale and zero_point must have the same groups"
    count = rank = down_at = up_at = scaling_at = index_at = 0
    if adapters is not None:
        down, up, scaling = adapters
        assert adapter_index is not None, "adapters need an adapter_index"
        assert down.dim() == 3 and up.dim() == 3, "expected down [adapters, rank, n] and up [adapters, m, rank]"
        count, rank, _ = down.shape
        assert down.shape == (count, rank, n) and up.shape == (count, m, rank), "expected down [adapters, rank, n] and up [adapters, m, rank]"
        assert rank % 8 == 0 and 0 < rank <= 64, "the rank must be a multiple of 8, at most 64"
        assert down.dtype == dtype and up.dtype == dtype and down.get_device() == index and up.get_device() == index, "the adapters must have the activations' type and device"
        down_at, up_at = down.data_ptr(), up.data_ptr()
        assert down.is_contiguous() and up.is_contiguous() and not (down_at | up_at) & 15, "the adapters must be contiguous and 16-byte aligned"
        assert adapter_index.dtype == torch.int32 and adapter_index.get_device() == index and adapter_index.numel() == tokens and adapter_index.is_contiguous(), "expected a contiguous int32 adapter index per token"
        index_at = adapter_index.data_ptr()
        if scaling is not None:
            assert scaling.shape == (count,) and scaling.dtype == torch.float32 and scaling.get_device() == index and scaling.is_contiguous(), "expected contiguous float32 scaling [adapters]"
            scaling_at = scaling.data_ptr()
        if count == 0:
            rank = 0
    else:
        assert adapter_index is None, "an adapter_index needs adapters"
    if out is None:
        out = torch.empty((*shape[:-1], m), dtype=dtype, device=device)
    else:
        assert out.shape == (*shape[:-1], m) and out.dtype == dtype and out.get_device() == index and out.is_contiguous(), "out must be a contiguous tensor of x's type [..., m]"
    if tokens == 0 or m == 0:
        return out
    lib = _abi.library()
    fields = (half, bits, m, n, tokens, rows.data_ptr(), row_stride, codes_at, row_bytes, max(groups, zero_groups), scale.data_ptr(), scale_row, scale_group,
              zero.data_ptr(), zero_row, zero_group, float(qmin), count, rank, 0, down_at, up_at, scaling_at, index_at, out.data_ptr(), m)
    sizes = (m, n, tokens, rank, count)
    need = _WORKSPACE.get(sizes)
    if need is None:
        size = ctypes.c_size_t()
        _abi.check(lib.g2d_linear_workspace_bytes(_abi.LINEAR_DESC.pack(*fields, 0, 0, 0), ctypes.byref(size)), "g2d_linear_workspace_bytes")
        if len(_WORKSPACE) > 4096:
            _WORKSPACE.clear()
        need = _WORKSPACE[sizes] = size.value
    workspace = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    desc = _abi.LINEAR_DESC.pack(*fields, workspace.data_ptr() if need else 0, need, _abi.status_word(device).data_ptr())
    with _abi.on_device(index):
        status = lib.g2d_packed_linear(desc, _abi.raw_stream(index))
    if status:
        _abi.check(status, "g2d_packed_linear")
    return out
