"""Keys and values in packed 4-bit codes, and attention over them.

Every row (the values of one token and one kv head) is rounded under its own abs-max scale, as ``int_abs_max_quantizer_*`` rounds a row of a
super-entry to the codes -8..7 with an fp16 scale, and stored as ``packed_codes.pack_codes`` stores a row with ``qmin=-8, bits=4``: ``head_dim / 2``
bytes of codes and 2 bytes of scale, 3.9 times less than 16-bit values at ``head_dim = 128``.

The cache is paged.  A step's tokens belong to sequences: sequence ``b`` has the tokens ``offsets[b]:offsets[b + 1]`` of the step (without
``offsets`` every sequence has the same number of them) and holds ``lengths[b]`` positions, this step's tokens being the last; position ``p`` lies in
page ``page_table[b, p // page_size]``.  These three are read on the device, so a captured graph follows them.  What they say is never
trusted with an address: positions beyond the table and page numbers outside the cache are absent (not written, read as zeros, seen by no query).
Offsets are meant to ascend: where they do
not, a token may be that of two sequences, and its row is either's (or, where that makes more work than can be counted, all results are NaN and
``check_status`` reports it).  Pages may be shared for reading; two tokens of a step that go to the same place leave the row of either, or a mixture.
CUDA only, like the rest of the package; no gradients.
"""
from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

import _abi

_HALF = {torch.float16: _abi.FP16, torch.bfloat16: _abi.BF16}
_WORKSPACE: dict[int, int] = {}  # bytes by head_dim


class _Tensors(NamedTuple):
    k_codes: torch.Tensor
    k_scale: torch.Tensor
    v_codes: torch.Tensor
    v_scale: torch.Tensor


class PackedCache(_Tensors):
    """Codes ``uint8 [pages, kv_heads, page_size, head_dim / 2]`` and scales ``float16 [pages, kv_heads, page_size]`` of keys and of values, contiguous on one CUDA
    device; ``page_size`` a power of two from 16 up, ``head_dim`` 64 or 128.  Checked when it is made."""

    def __new__(cls, k_codes, k_scale, v_codes, v_scale):
        device = k_codes.device
        assert k_codes.is_cuda, "the packed cache requires CUDA tensors (there is no CPU path)"
        assert k_codes.dim() == 4 and k_codes.dtype == torch.uint8 and v_codes.dtype == torch.uint8 and v_codes.shape == k_codes.shape, "expected uint8 codes of keys and values of one shape [pages, kv_heads, page_size, head_dim / 2]"
        assert k_scale.dtype == torch.float16 and v_scale.dtype == torch.float16, "expected float16 scales"
        assert k_scale.shape == k_codes.shape[:3] and v_scale.shape == k_codes.shape[:3], "expected a scale per page, kv head and place"
        self = super().__new__(cls, k_codes, k_scale, v_codes, v_scale)
        assert all(t.is_contiguous() and t.device == device and t.data_ptr() % 16 == 0 for t in self), "the cache's tensors must be contiguous, 16-byte aligned and on one device"
        pages, kv_heads, page_size, half_dim = k_codes.shape
        _check_layout(page_size, 2 * half_dim)
        assert kv_heads > 0, "expected at least one kv head"
        self.layout = (2 * half_dim, page_size, kv_heads, pages)
        return self

    @classmethod
    def _make(cls, tensors):  # what _replace goes through: checked as well
        return cls(*tensors)


def _check_layout(page_size: int, head_dim: int) -> None:
    assert head_dim in (64, 128), "head_dim must be 64 or 128"
    assert page_size >= 16 and page_size & (page_size - 1) == 0, "page_size must be a power of two, at least 16"


def new_packed_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, device) -> PackedCache:
    """An empty cache (all codes and scales zero)."""
    _check_layout(page_size, head_dim)
    codes = lambda: torch.zeros(pages, kv_heads, page_size, head_dim // 2, dtype=torch.uint8, device=device)  # noqa: E731
    scale = lambda: torch.zeros(pages, kv_heads, page_size, dtype=torch.float16, device=device)  # noqa: E731
    return PackedCache(codes(), scale(), codes(), scale())


def _cache_fields(cache: PackedCache, dtype, tokens: int, page_table, lengths, offsets):
    """Checks what says where the step's tokens are; returns the device and the fields of ``g2d_cache_desc``."""
    assert isinstance(cache, PackedCache), "expected a PackedCache"
    head_dim, page_size, kv_heads, pages = cache.layout
    k_codes, k_scale, v_codes, v_scale = cache
    device = k_codes.device
    index = device.index
    half = _HALF.get(dtype)
    assert half is not None, "expected float16 or bfloat16 values"
    assert page_table.dim() == 2 and page_table.dtype == torch.int32 and page_table.get_device() == index, "expected an int32 page table [batch, pages per sequence] on the cache's device"
    batch, width = page_table.shape
    table_stride, last = page_table.stride()
    assert last == 1 or width <= 1, "the rows of the page table must be contiguous"
    assert lengths.shape == (batch,) and lengths.dtype == torch.int32 and lengths.get_device() == index and lengths.is_contiguous(), "expected contiguous int32 lengths [batch] on the cache's device"
    if offsets is None:
        assert tokens == 0 or (batch > 0 and tokens % batch == 0), "without offsets every sequence has the same number of tokens"
        offsets_at = 0
    else:
        assert offsets.shape == (batch + 1,) and offsets.dtype == torch.int32 and offsets.get_device() == index and offsets.is_contiguous(), "expected contiguous int32 offsets [batch + 1] on the cache's device"
        offsets_at = offsets.data_ptr()
    return device, (half, head_dim, page_size, kv_heads, pages, batch, width, table_stride, tokens, k_codes.data_ptr(), k_scale.data_ptr(), v_codes.data_ptr(), v_scale.data_ptr(),
                    page_table.data_ptr(), lengths.data_ptr(), offsets_at)


def _rows(x: torch.Tensor, device, heads: int, dim: int, what: str) -> torch.Tensor:
    """``x [tokens, heads, dim]`` as the kernels read it: any strides of tokens and heads that keep 16-byte vectors whole, else a copy."""
    assert x.get_device() == device.index, f"{what} must be on the cache's device"
    assert x.dim() == 3 and x.shape[1:] == (heads, dim), f"expected {what} [tokens, {heads}, {dim}]"
    token, head, last = x.stride()
    if last != 1 or token % 8 or head % 8 or x.data_ptr() % 16:
        x = x.detach().clone(memory_format=torch.contiguous_format)
    return x


def append_packed(cache: PackedCache, k: torch.Tensor, v: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
    """Round the step's keys and values ``[tokens, kv_heads, head_dim]`` (float16 or bfloat16; strided views, such as parts of a fused projection, are
    read in place) and write them into the cache, in place.  ``lengths`` counts the step's tokens already.  A row with an infinity, a NaN or a
    magnitude whose scale a half cannot hold (491400 and more) reads back as NaN, and makes NaN every query that sees it."""
    assert k.dtype == v.dtype and k.dim() == 3 and k.shape == v.shape, "expected keys and values of one shape and type"
    device, fields = _cache_fields(cache, k.dtype, k.shape[0], page_table, lengths, offsets)
    k, v = _rows(k, device, fields[3], fields[1], "keys"), _rows(v, device, fields[3], fields[1], "values")
    index = device.index
    with _abi.on_device(index):
        status = _abi.library().g2d_cache_append(_abi.CACHE_DESC.pack(*fields), k.data_ptr(), *k.stride()[:2], v.data_ptr(), *v.stride()[:2], _abi.raw_stream(index))
    if status:
        _abi.check(status, "g2d_cache_append")


def read_packed(cache: PackedCache, page_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor | None = None, *, tokens: int,
                dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values ``[tokens, kv_heads, head_dim]`` that the cache holds for the last tokens of every sequence, ``offsets`` saying how many (all of them, where
    they add up to ``lengths``).  Rows of no sequence, and positions that the cache does not hold, are zeros."""
    device, fields = _cache_fields(cache, dtype, tokens, page_table, lengths, offsets)
    k = (torch.empty if fields[5] else torch.zeros)((tokens, fields[3], fields[1]), dtype=dtype, device=device)
    v = (torch.empty_like if fields[5] else torch.zeros_like)(k)
    index = device.index
    with _abi.on_device(index):
        status = _abi.library().g2d_cache_read(_abi.CACHE_DESC.pack(*fields), k.data_ptr(), v.data_ptr(), _abi.raw_stream(index))
    if status:
        _abi.check(status, "g2d_cache_read")
    return k, v


def attend_packed(q: torch.Tensor, cache: PackedCache, page_table: torch.Tensor, lengths: torch.Tensor, offsets: torch.Tensor | None = None, *,
                  scale: float | None = None, causal: bool = True, softcap: float = 0.0, slopes: torch.Tensor | None = None,
                  prefix: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of the step's queries ``q [tokens, heads, head_dim]`` (float16 or bfloat16) over the cache: ``[tokens, heads, head_dim]`` in q's type.

    ``heads`` is a multiple of the cache's kv heads; query head ``h`` reads kv head ``h // (heads // kv_heads)``.  The scores are ``scale * q . k`` (``1 /
    sqrt(head_dim)`` by default), with ``softcap > 0`` then ``softcap * tanh(score / softcap)``, with ``slopes`` (float32 ``[heads]``) then
    ``+ slopes[h] * (j - p)`` for a query at position p and a key at j.  A query sees its sequence's keys up to its own position, and those before
    ``prefix[b]`` (int32 ``[batch]``) wherever it stands; with ``causal=False`` all of them.  A query that sees no key gets zeros.  Rows of ``out`` that belong
    to no sequence are left as they are (zeros, without ``out``); ``out`` must not overlap the inputs.  What a step appends has to be in the cache before: call
    ``append_packed`` first."""
    assert q.dim() == 3, "expected queries [tokens, heads, head_dim]"
    dtype = q.dtype
    tokens, heads, _ = q.shape
    device, fields = _cache_fields(cache, dtype, tokens, page_table, lengths, offsets)
    head_dim, kv_heads = fields[1], fields[3]
    assert heads > 0 and heads % kv_heads == 0, "the number of heads must be a multiple of the cache's kv heads"
    q = _rows(q, device, heads, head_dim, "queries")
    assert math.isfinite(softcap) and softcap >= 0, "softcap must be finite and not negative"
    scale = 1 / math.sqrt(head_dim) if scale is None else float(scale)
    assert math.isfinite(scale), "scale must be finite"
    slopes_at = prefix_at = 0
    if slopes is not None:
        assert slopes.shape == (heads,) and slopes.dtype == torch.float32 and slopes.get_device() == device.index and slopes.is_contiguous(), "expected contiguous float32 slopes [heads] on the cache's device"
        slopes_at = slopes.data_ptr()
    if prefix is not None:
        assert prefix.shape == lengths.shape and prefix.dtype == torch.int32 and prefix.get_device() == device.index and prefix.is_contiguous(), "expected a contiguous int32 prefix [batch] on the cache's device"
        prefix_at = prefix.data_ptr()
    clear = out is None
    if clear:
        out = (torch.empty_like if fields[5] else torch.zeros_like)(q, memory_format=torch.contiguous_format)
    else:
        assert out.shape == q.shape and out.dtype == dtype and out.get_device() == device.index and out.is_contiguous() and out.data_ptr() % 16 == 0, "out must be a contiguous, 16-byte aligned tensor like q"
    if tokens == 0:
        return out
    lib, index = _abi.library(), device.index
    fields = (*fields, heads, bool(causal), scale, float(softcap), clear, 0, q.data_ptr(), *q.stride()[:2], out.data_ptr(), slopes_at, prefix_at)
    need = _WORKSPACE.get(head_dim)
    if need is None:
        size = ctypes.c_size_t()
        _abi.check(lib.g2d_attend_workspace_bytes(_abi.ATTEND_DESC.pack(*fields, 0, 0, 0), ctypes.byref(size)), "g2d_attend_workspace_bytes")
        need = _WORKSPACE[head_dim] = size.value
    workspace = torch.empty(need, dtype=torch.uint8, device=device)
    desc = _abi.ATTEND_DESC.pack(*fields, workspace.data_ptr(), need, _abi.status_word(device).data_ptr())
    with _abi.on_device(index):
        status = lib.g2d_cache_attend(desc, _abi.raw_stream(index))
    if status:
        _abi.check(status, "g2d_cache_attend")
    return out
