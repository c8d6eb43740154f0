"""More of what the packed product, the packed cache and attention over it refuse, as far as that shows without a GPU."""
import pytest
import torch
from test_packed_serving_cpu import LINEAR, half_of, lib, refused  # noqa: F401


@pytest.mark.parametrize("tokens, n", [(17, 64), (64, 64), (65, 64), (300, 64), (2, 32832)])
@pytest.mark.parametrize("x_stride", [0, 8, 56, -64])
def test_rows_of_activations_that_overlap_are_refused_by_tiles(lib, x_stride, tokens, n):  # noqa: F811
    """A stride of 0 must never reach a tensor map, where it would stand for rows one after the other."""
    import _abi

    fields = {**half_of(LINEAR), "tokens": tokens, "n": n, "row_bytes": -(-n // 32) * 16, "x_stride": x_stride, "workspace": 256, "bytes": 1 << 40}
    assert refused(lib.g2d_packed_linear(_abi.LINEAR_DESC.pack(*fields.values()), 0))


def test_caches_made_from_parts_are_checked():
    """``_make``, and ``_replace`` through it, check what they are given as the constructor does."""
    import packed_cache as C

    tensors = [torch.zeros(2, 1, 16, 32, dtype=torch.uint8), torch.zeros(2, 1, 16, dtype=torch.float16)] * 2
    with pytest.raises(AssertionError, match="CUDA"):
        C.PackedCache._make(tensors)


def test_the_library_has_one_description_of_each_descriptor():
    """A mirror of a descriptor beside the packed formats would have to be kept like them, and nothing uses one."""
    import _abi

    assert not any(hasattr(_abi, name) for name in ("CacheDesc", "AttendDesc", "LinearDesc"))
