"""Corners of the packed product, the packed cache and attention over it: forms of their inputs that calls allow and that are easily got wrong.  Plain formulas in
64 bits and tolerances are those of the files that test the operators one by one."""
import pytest
import torch
from test_gpu_packed_linear import Problem

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("adapters", [0, 3])
@pytest.mark.parametrize("tokens", [1, 2, 16, 17, 64, 65, 300])
def test_one_row_for_every_token(tokens, adapters, dtype):
    """An expanded row is what its copies are, to the last bit."""
    p = Problem(200, 256, tokens, dtype, adapters=adapters, rank=8)
    row = p.x[:1].clone()
    p.x = row.repeat(tokens, 1)
    want = p.check()
    p.x = row.expand(tokens, 256)
    assert p.x.stride(0) == 0 or tokens == 1
    assert torch.equal(p.run(), want)
    p.x = row[0].expand(1, tokens, 256)  # and with leading dimensions
    assert torch.equal(p.run()[0], want)


@pytest.mark.parametrize("tokens", [3, 16, 17, 130])
@pytest.mark.parametrize("step", [8, 24, 248])
def test_windows_of_a_longer_row(step, tokens):
    p = Problem(130, 256, tokens, torch.float16, adapters=2, rank=8)
    long = (0.3 + torch.randn(256 + step * tokens, generator=torch.Generator(device="cuda").manual_seed(tokens), device="cuda")).half()
    windows = long.as_strided((tokens, 256), (step, 1))
    p.x = windows.clone(memory_format=torch.contiguous_format)
    want = p.check()
    p.x = windows
    assert torch.equal(p.run(), want)


@pytest.mark.parametrize("tokens", [1, 2, 16])
def test_one_long_row_for_every_token(tokens):
    """Rows that go by tiles whatever the number of tokens."""
    p = Problem(70, 32800, tokens, torch.bfloat16)
    row = p.x[:1].clone()
    p.x = row.repeat(tokens, 1)
    want = p.check()
    p.x = row.expand(tokens, 32800)
    assert torch.equal(p.run(), want)
    p.x = row.as_strided((1, 32800), (8, 1))
    assert torch.equal(p.run(), want[:1])
