"""What the packed product, the packed cache and attention over it refuse, as far as that shows without a GPU: the Python checks of tensors that are on the host,
and the status codes of the C entry points, which look at a descriptor before they touch the device."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

HERE = os.path.dirname(os.path.abspath(__file__))


def test_tensors_on_the_host_are_refused():
    import packed_cache as C
    import packed_linear as L

    with pytest.raises(AssertionError, match="CUDA"):
        L.packed_linear(torch.zeros(1, 64, dtype=torch.float16), torch.zeros(8, 32, dtype=torch.uint8), torch.ones(8, 1), torch.zeros(8, 1), qmin=-8)
    with pytest.raises(AssertionError, match="CUDA"):
        C.new_packed_cache(2, 16, 1, 64, "cpu")
    with pytest.raises(AssertionError, match="PackedCache"):
        C.attend_packed(torch.zeros(1, 1, 64), (None,) * 4, torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32))


@pytest.mark.parametrize("page_size, head_dim", [(8, 64), (24, 64), (0, 64), (16, 96), (16, 256), (16, 0)])
def test_layouts_of_the_cache_that_are_refused(page_size, head_dim):
    import packed_cache as C

    with pytest.raises(AssertionError):
        C.new_packed_cache(2, page_size, 1, head_dim, "cpu")


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_descriptors_have_the_sizes_of_the_header(tmp_path):
    import _abi

    source, program = tmp_path / "sizes.c", tmp_path / "sizes"
    source.write_text('#include <stdio.h>\n#include "gptq2d_b200.h"\nint main(void) { printf("%zu %zu %zu\\n", sizeof(g2d_cache_desc), sizeof(g2d_attend_desc), sizeof(g2d_linear_desc)); return 0; }\n')
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(HERE, "..", "include"), str(source), "-o", str(program)], check=True)
    sizes = [int(x) for x in subprocess.run([str(program)], check=True, capture_output=True, text=True).stdout.split()]
    assert sizes == [_abi.CACHE_DESC.size, _abi.ATTEND_DESC.size, _abi.LINEAR_DESC.size]


# ---- the C entry points: descriptors as the header lays them out, addresses that nothing reads ----
CACHE = dict(half=0, head_dim=64, page_size=16, kv_heads=2, pages=4, batch=1, width=2, table_stride=2, tokens=1, k=256, ks=256, v=256, vs=256, table=256, lengths=256, offsets=0)
ATTEND = dict(heads=4, causal=1, scale=1.0, softcap=0.0, clear=0, reserved=0, q=256, q_token=256, q_head=64, out=256, slopes=0, prefix=0, workspace=0, bytes=0, status=0)
LINEAR = dict(half=0, bits=4, m=64, n=64, tokens=1, x=256, x_stride=64, codes=256, row_bytes=32, groups=1, scale=256, scale_row=1, scale_group=0, zero=256, zero_row=1, zero_group=0, qmin=-8.0, adapters=0,
              rank=0, reserved=0, down=0, up=0, scaling=0, index=0, out=256, out_stride=64, workspace=0, bytes=0, status=0)


def refused(status):
    """A reason of the entry point's own, not what the missing device would give."""
    return status in (-1, -2, -3, -5)


@pytest.fixture(scope="module")
def lib():
    import _abi

    if not os.path.exists(_abi.LIBRARY_PATH):
        pytest.skip("the CUDA library is not built")
    return _abi.library()


def half_of(defaults):
    import _abi

    return {**defaults, "half": _abi.FP16}


@pytest.mark.parametrize("change", [dict(half=99), dict(head_dim=96), dict(head_dim=32), dict(page_size=8), dict(page_size=24), dict(page_size=1 << 21), dict(kv_heads=0), dict(pages=-1), dict(batch=-1),
                                    dict(tokens=-1), dict(width=-1), dict(tokens=3, batch=2), dict(k=0), dict(vs=8), dict(lengths=0), dict(table=0), dict(table_stride=-2), dict(tokens=1 << 31), dict(kv_heads=1 << 17),
                                    dict(batch=0)])
def test_cache_descriptors_that_are_refused(lib, change):
    import _abi

    desc = _abi.CACHE_DESC.pack(*{**half_of(CACHE), **change}.values())
    assert refused(lib.g2d_cache_append(desc, 256, 128, 64, 256, 128, 64, 0))
    assert refused(lib.g2d_cache_read(desc, 256, 256, 0))
    size = ctypes.c_size_t()
    assert refused(lib.g2d_attend_workspace_bytes(_abi.ATTEND_DESC.pack(*{**half_of(CACHE), **change}.values(), *ATTEND.values()), ctypes.byref(size)))


def test_keys_and_values_that_are_refused(lib):
    import _abi

    desc = _abi.CACHE_DESC.pack(*half_of(CACHE).values())
    assert refused(lib.g2d_cache_append(desc, 0, 128, 64, 256, 128, 64, 0))
    assert refused(lib.g2d_cache_append(desc, 258, 128, 64, 256, 128, 64, 0))
    assert refused(lib.g2d_cache_append(desc, 256, 127, 64, 256, 128, 64, 0))
    assert refused(lib.g2d_cache_append(desc, 256, 128, 64, 256, 128, 63, 0))
    assert refused(lib.g2d_cache_read(desc, 256, 8, 0))
    empty = _abi.CACHE_DESC.pack(*{**half_of(CACHE), "tokens": 0}.values())
    assert lib.g2d_cache_append(empty, 0, 0, 0, 0, 0, 0, 0) == 0 and lib.g2d_cache_read(empty, 0, 0, 0) == 0


@pytest.mark.parametrize("change", [dict(heads=0), dict(heads=5), dict(softcap=-1.0), dict(softcap=float("nan")), dict(q=0), dict(q=264), dict(out=0), dict(q_token=257), dict(q_head=4), dict(workspace=0),
                                    dict(workspace=264), dict(bytes=1), dict(reserved=1)])
def test_attention_that_is_refused(lib, change):
    import _abi

    size = ctypes.c_size_t()
    fields = {**ATTEND, "workspace": 256}
    assert lib.g2d_attend_workspace_bytes(_abi.ATTEND_DESC.pack(*half_of(CACHE).values(), *fields.values()), ctypes.byref(size)) == 0 and size.value > 0
    fields["bytes"] = size.value
    assert refused(lib.g2d_cache_attend(_abi.ATTEND_DESC.pack(*half_of(CACHE).values(), *{**fields, **change}.values()), 0))
    assert lib.g2d_cache_attend(_abi.ATTEND_DESC.pack(*{**half_of(CACHE), "tokens": 0}.values(), *fields.values()), 0) == 0


def test_attention_whose_work_cannot_be_counted(lib):
    import _abi

    cache = {**half_of(CACHE), "tokens": 1 << 20, "batch": 1, "width": 1 << 24, "page_size": 1024, "table_stride": 1 << 24}
    fields = {**ATTEND, "workspace": 256, "bytes": 1 << 40, "heads": 64}
    assert refused(lib.g2d_cache_attend(_abi.ATTEND_DESC.pack(*cache.values(), *fields.values()), 0))


@pytest.mark.parametrize("change", [dict(half=99), dict(bits=3), dict(bits=8), dict(n=48), dict(n=0), dict(row_bytes=31), dict(row_bytes=16), dict(rank=4), dict(rank=72), dict(rank=-8), dict(groups=0), dict(groups=2),
                                    dict(m=-1), dict(tokens=-1), dict(adapters=-1), dict(x=0), dict(x=264), dict(x_stride=63), dict(codes=0), dict(codes=260), dict(scale=0), dict(zero=0), dict(out=0), dict(out=257),
                                    dict(out_stride=63), dict(m=1 << 31), dict(tokens=1 << 31), dict(rank=8, adapters=2), dict(rank=8, adapters=2, down=256, up=256, index=0), dict(reserved=1)])
def test_products_that_are_refused(lib, change):
    import _abi

    fields = {**half_of(LINEAR), **change}
    if "rank" in change:
        fields.update(workspace=256, bytes=1 << 30)
    assert refused(lib.g2d_packed_linear(_abi.LINEAR_DESC.pack(*fields.values()), 0))


@pytest.mark.parametrize("tokens", [1, 16, 17, 64, 65, 2000])
@pytest.mark.parametrize("m, n", [(64, 64), (28672, 4096), (1, 32)])
def test_workspaces_of_products(lib, m, n, tokens):
    """What the library asks for covers the adapters' inner values, is refused when it is smaller, and is the same for descriptors without addresses."""
    import _abi

    size = ctypes.c_size_t()
    fields = {**half_of(LINEAR), "m": m, "n": n, "tokens": tokens, "row_bytes": -(-n // 32) * 16, "x_stride": n, "out_stride": m, "rank": 16, "adapters": 3, "down": 256, "up": 256, "index": 256}
    assert lib.g2d_linear_workspace_bytes(_abi.LINEAR_DESC.pack(*fields.values()), ctypes.byref(size)) == 0
    assert size.value >= tokens * (2 * 64 * 2 + 4)
    assert refused(lib.g2d_packed_linear(_abi.LINEAR_DESC.pack(*{**fields, "workspace": 256, "bytes": size.value - 1}.values()), 0))
    assert refused(lib.g2d_packed_linear(_abi.LINEAR_DESC.pack(*{**fields, "workspace": 0, "bytes": size.value}.values()), 0))
