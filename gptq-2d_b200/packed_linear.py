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


def _parameter(t, m: int, n: int, name: str, device):
    """A scale or zero point: one value, one per row, or one per row and group of columns; with its strides over rows and groups, and how many groups."""
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or t.device != device:
        t = torch.as_tensor(t, dtype=torch.float32, device=device)
    assert t.dim() <= 2, f"{name} must be one value, one per row, or one per row and group of columns"
    rows, groups = (1, 1, *t.shape)[-2:]
    strides = (0, 0, *t.stride())[-2:]
    assert rows in (1, m), f"{name} must have one row or one for each of the {m} rows of codes"
    assert groups == 1 or (n % groups == 0 and n // groups % 64 == 0), f"{name}: groups must divide the {n} columns into multiples of 64"
    return t, strides[0] if rows > 1 else 0, strides[1] if groups > 1 else 0, groups


@torch.no_grad()
def packed_linear(x: torch.Tensor, codes: torch.Tensor, scale: torch.Tensor, zero_point: torch.Tensor, *, qmin: float, bits: int = 4,
                  adapters: LowRankAdapters | None = None, adapter_index: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``x @ W.T [..., m]`` for ``x [..., n]`` (float16 or bfloat16, CUDA) and the matrix ``W [m, n]`` whose 4-bit codes are ``codes`` (uint8 ``[m, n / 2]`` from
    ``pack_codes``, ``n`` a multiple of 32), ``W = (code + qmin - zero_point) * scale``.

    ``scale`` and ``zero_point`` are one value, ``[m, 1]``, or ``[m, groups]`` with equal groups of columns, each a multiple of 64 wide (float32; where both have groups,
    the same number).  Zero points are meant to be integers: with many tokens ``code + qmin - zero_point`` is rounded to x's type, exact up to 256 (bfloat16) or 2048 (float16).
    With ``adapters``, ``adapter_index`` (int32, one per token, in the order of ``x``'s leading dimensions) says whose adapter is added to a token's result; an index outside
    the adapters' range means none.  Sums are float32, results are rounded once to x's type.  ``out`` may be given as a contiguous ``[..., m]`` tensor."""
    assert bits == 4, "only codes of 4 bits can be multiplied with"
    assert x.is_cuda, "the product with packed codes requires CUDA tensors (there is no CPU path)"
    assert x.dim() >= 1 and x.dtype in (torch.float16, torch.bfloat16), "expected float16 or bfloat16 activations [..., n]"
    assert codes.dim() == 2 and codes.dtype == torch.uint8 and codes.is_contiguous() and codes.device == x.device, "expected contiguous uint8 codes on the activations' device"
    device, n, (m, row_bytes) = x.device, x.size(-1), codes.shape
    assert n > 0 and n % 32 == 0, "the number of columns must be a multiple of 32"
    assert row_bytes >= n // 2 and row_bytes % 16 == 0 and codes.data_ptr() % 16 == 0, "rows of codes must hold n entries and be 16-byte aligned"
    shape = (*x.shape[:-1], m)
    rows = x if x.dim() == 2 else x.reshape(-1, n)
    if rows.stride(1) != 1 or rows.stride(0) % 8 or rows.data_ptr() % 16:
        rows = rows.clone(memory_format=torch.contiguous_format)
    tokens = rows.size(0)
    scale, scale_row, scale_group, groups = _parameter(scale, m, n, "scale", device)
    zero, zero_row, zero_group, zero_groups = _parameter(zero_point, m, n, "zero_point", device)
    assert groups == zero_groups or groups == 1 or zero_groups == 1, "scale and zero_point must have the same groups"
    desc = _abi.LinearDesc()
    desc.half, desc.bits, desc.m, desc.n, desc.tokens = _abi.half_code(x.dtype), bits, m, n, tokens
    desc.x, desc.x_stride, desc.codes, desc.row_bytes, desc.groups = rows.data_ptr(), rows.stride(0), codes.data_ptr(), row_bytes, max(groups, zero_groups)
    desc.scale, desc.scale_row_stride, desc.scale_group_stride = scale.data_ptr(), scale_row, scale_group
    desc.zero, desc.zero_row_stride, desc.zero_group_stride, desc.qmin = zero.data_ptr(), zero_row, zero_group, float(qmin)
    if adapters is not None:
        down, up, scaling = adapters
        assert adapter_index is not None, "adapters need an adapter_index"
        count, rank = down.shape[:2]
        assert down.shape == (count, rank, n) and up.shape == (count, m, rank), "expected down [adapters, rank, n] and up [adapters, m, rank]"
        assert rank % 8 == 0 and 0 < rank <= 64, "the rank must be a multiple of 8, at most 64"
        assert down.dtype == x.dtype and up.dtype == x.dtype and down.device == device and up.device == device, "the adapters must have the activations' type and device"
        assert down.is_contiguous() and up.is_contiguous() and down.data_ptr() % 16 == 0 and up.data_ptr() % 16 == 0, "the adapters must be contiguous and 16-byte aligned"
        assert adapter_index.dtype == torch.int32 and adapter_index.device == device and adapter_index.numel() == tokens and adapter_index.is_contiguous(), "expected a contiguous int32 adapter index per token"
        if scaling is not None:
            assert scaling.shape == (count,) and scaling.dtype == torch.float32 and scaling.device == device and scaling.is_contiguous(), "expected contiguous float32 scaling [adapters]"
            desc.scaling = scaling.data_ptr()
        if count > 0:
            desc.adapters, desc.rank, desc.down, desc.up, desc.index = count, rank, down.data_ptr(), up.data_ptr(), adapter_index.data_ptr()
    else:
        assert adapter_index is None, "an adapter_index needs adapters"
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=device)
    else:
        assert out.shape == shape and out.dtype == x.dtype and out.device == device and out.is_contiguous(), "out must be a contiguous tensor of x's type [..., m]"
    if out.numel() == 0:
        return out
    desc.out, desc.out_stride, desc.status = out.data_ptr(), m, _abi.status_word(device).data_ptr()
    lib = _abi.library()
    need = ctypes.c_size_t()
    _abi.check(lib.g2d_linear_workspace_bytes(ctypes.byref(desc), ctypes.byref(need)), "g2d_linear_workspace_bytes")
    if need.value:
        workspace = torch.empty(need.value, dtype=torch.uint8, device=device)
        desc.workspace, desc.workspace_bytes = workspace.data_ptr(), need.value
    with torch.cuda.device(device):
        _abi.check(lib.g2d_packed_linear(ctypes.byref(desc), _abi.stream_of(x)), "g2d_packed_linear")
    return out
