"""Corners of the packed product, the packed cache and attention over it: forms of their inputs that calls allow and that are easily got wrong.  Plain formulas in
64 bits and tolerances are those of the files that test the operators one by one."""
import pytest
import torch
from test_gpu_packed_cache import Batch
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


@pytest.mark.parametrize("options", [{}, {"softcap": 30.0}, {"softcap": 1e4}, {"slopes": True}, {"softcap": 5.0, "slopes": True}])
@pytest.mark.parametrize("queries", [1, 4, 12, 100])
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_key_that_is_not_finite_makes_nan_what_sees_it(dtype, head_dim, queries, options):
    """An infinity among appended keys, a row whose scale is beyond a half's range, and infinite scales over any codes: NaN for every query that sees
    the key, with few rows and with many, capped or not; no trace for those that do not."""
    import packed_cache as C

    length, bad = 150, 150 - 1 - queries // 2  # of the last `queries` positions half come after the bad one, or are it
    batch = Batch([(length, length)] * 24, 2, head_dim, 32, dtype, fill=False)
    k, v = batch.randn(batch.tokens, 2, head_dim), batch.randn(batch.tokens, 2, head_dim)
    q = batch.randn(24 * queries, 8, head_dim)
    if options.get("slopes"):
        options = {**options, "slopes": torch.linspace(-0.01, 0.1, 8, device="cuda")}
    run = lambda: C.attend_packed(q, batch.cache, batch.table, batch.lengths, **options).view(24, queries, 8, head_dim)  # noqa: E731
    C.append_packed(batch.cache, k, v, batch.table, batch.lengths, batch.offsets)
    clean = run()
    assert clean.isfinite().all()
    blind = queries - (length - bad)  # queries before the bad position
    spoiled = k.view(24, length, 2, head_dim)
    row = spoiled[:, bad].clone()

    def seen_and_unseen():
        got = run()
        assert got[:, blind:].isnan().all() and torch.equal(got[:, :blind], clean[:, :blind])

    for value in [float("inf"), -float("inf")] + ([1e6, -3e38] if dtype == torch.bfloat16 else []):
        spoiled[:, bad, :, 5] = value
        C.append_packed(batch.cache, k, v, batch.table, batch.lengths, batch.offsets)
        seen_and_unseen()
        spoiled[:, bad] = row
    C.append_packed(batch.cache, k, v, batch.table, batch.lengths, batch.offsets)
    pages = batch.table[:, bad // 32].long()
    for value in (float("inf"), -float("inf"), float("nan")):
        batch.cache.k_scale[pages, :, bad % 32] = value
        seen_and_unseen()
