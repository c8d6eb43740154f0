"""Corners of the packed product, the packed cache and attention over it: forms of their inputs that calls allow and that are easily got wrong.  Plain formulas in
64 bits and tolerances are those of the files that test the operators one by one."""
import pytest
import torch
from test_gpu_packed_cache import Batch, assert_near, reference, rounded
from test_gpu_packed_linear import Problem

pytestmark = pytest.mark.gpu

# What a result of the attention may be off beside its own rounding, of the largest |v| that its row sees: each product of an exponential and a value's scale is rounded to fp16, by half a step, which is
# 2^-11 of a value just above a power of two (finfo(float16).eps / 2), and 2^-16 for exponentials, scores and sums in fp32.
NEAR = 2.0 ** -11 + 2.0 ** -16


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


def guarded(shape, dtype, fill, room=4096):
    """A tensor in the middle of a larger one, and what lies around it."""
    n = torch.Size(shape).numel()
    whole = torch.full((n + 2 * room,), fill, dtype=dtype, device="cuda")
    return whole[room:room + n].view(shape), (whole[:room], whole[room + n:])


@pytest.mark.parametrize("heads, tokens", [(2, 6), (8, 40), (2, 300)])
@pytest.mark.parametrize("which", ["beyond both ends", "descending", "all behind", "empty", "overlapping"])
def test_wild_offsets_touch_nothing_else(which, heads, tokens):
    """Whatever the offsets say: rows and cache rows outside what they leave after they are brought into range stay as they were, with few rows and with tiles."""
    import gptq_2d
    import packed_cache as C

    offsets = {"beyond both ends": [-7, 3, 900], "descending": [5, 2, 1], "all behind": [900, 901, 1 << 30], "empty": [3, 3, 3], "overlapping": [0, tokens, 0, tokens]}[which]
    count = len(offsets) - 1
    batch = Batch([(400, 1)] * count, 1, 64, 16, torch.float16)
    q, k = batch.randn(tokens, heads, 64), batch.randn(tokens, 1, 64)
    device = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    pieces = []  # (first, last) of each sequence's tokens as they are brought into range
    for b in range(count):
        lo = min(max(offsets[b], 0), tokens)
        pieces.append((lo, min(max(offsets[b + 1], lo), tokens)))
    out, around = guarded((tokens, heads, 64), torch.float16, 7.0)
    C.attend_packed(q, batch.cache, batch.table, batch.lengths, device, out=out)
    gptq_2d.check_status()
    torch.cuda.synchronize()
    assert all((side == 7).all() for side in around)
    mine = torch.zeros(tokens, dtype=torch.bool, device="cuda")
    for lo, hi in pieces:
        mine[lo:hi] = True
    assert (out[~mine] == 7).all() and not (out[mine] == 7).all(-1).any()
    if which == "beyond both ends":
        for b, (lo, hi) in enumerate(pieces):
            alone = C.attend_packed(q[lo:hi], batch.cache, batch.table[b:b + 1], batch.lengths[b:b + 1])
            assert (out[lo:hi].float() - alone.float()).abs().max() <= 2 * 8.4 * (2.0 ** -11 + 2.0 ** -11 + 2.0 ** -16)  # cut otherwise, so summed otherwise: both as near as they have to be (see `NEAR`), |v| <= 8 * 1.05
    before = [t.clone() for t in batch.cache]
    C.append_packed(batch.cache, k, k, batch.table, batch.lengths, device)
    places = torch.zeros(batch.cache.k_scale.shape, dtype=torch.bool, device="cuda")
    for b, (lo, hi) in enumerate(pieces):
        for p in range(400 - (hi - lo), 400):
            places[int(batch.table[b, p // 16]), :, p % 16] = True
    for old, new in zip(before, batch.cache):
        assert torch.equal(old[~places].view(torch.uint8), new[~places].view(torch.uint8))
    got = C.read_packed(batch.cache, batch.table, batch.lengths, device, tokens=tokens, dtype=torch.float16)
    torch.cuda.synchronize()
    gptq_2d.check_status()
    if which != "overlapping":
        assert not got[0][~mine].any() and got[0][mine].any(-1).all()


@pytest.mark.parametrize("heads, tokens, step, page_size, width", [(1, 65536, 65536, 4096, 2040), (8, 64, 8, 1 << 20, 680)])
def test_offsets_that_make_more_work_than_can_be_counted(heads, tokens, step, page_size, width):
    """Overlapping sequences whose units pass 32 bits, of tiles and of few rows: refused on the device, at once."""
    import gptq_2d
    import packed_cache as C

    batch = 4096 if step == tokens else 64
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda").expand(batch, width)  # no page is there
    offsets = torch.tensor([step * (b % (tokens // step + 1)) for b in range(batch + 1)], dtype=torch.int32, device="cuda")
    lengths = torch.full((batch,), 2 ** 31 - 1, dtype=torch.int32, device="cuda")
    cache = C.PackedCache(*(torch.zeros(0, 1, page_size, *rest, dtype=dtype, device="cuda") for dtype, rest in ((torch.uint8, (32,)), (torch.float16, ())) * 2))
    q = torch.ones(tokens, heads, 64, dtype=torch.float16, device="cuda")
    gptq_2d.check_status()
    out, around = guarded(q.shape, torch.float16, 7.0)
    C.attend_packed(q, cache, table, lengths, offsets, out=out)
    with pytest.raises(RuntimeError):
        gptq_2d.check_status()
    assert out.isnan().all() and all((side == 7).all() for side in around)
    gptq_2d.check_status()
    assert not C.attend_packed(q[:8], cache, table[:1], torch.full_like(lengths[:1], 100)).any()  # and the next call is sound
    gptq_2d.check_status()


POWERS = [-118, -100, -80, -73, -62, -50, -30, -13, -12, -11, 0, 40, 63, 64, 65, 71, 72, 73, 90, 110]


@pytest.mark.parametrize("adapters", [0, 2])
@pytest.mark.parametrize("groups, n", [(1, 1280), (5, 320), (1, 4096)])
@pytest.mark.parametrize("tokens", [1, 8, 16, 20])
def test_bf16_activations_of_any_magnitude(tokens, groups, n, adapters):
    """Tokens each of a size of their own, from near the smallest normal numbers to near the largest."""
    p = Problem(130, n, tokens, torch.bfloat16, groups=groups, adapters=adapters, rank=8)
    x = p.x.float()
    for first in range(0, len(POWERS), tokens):
        powers = torch.tensor([POWERS[(first + t) % len(POWERS)] for t in range(tokens)], device="cuda").float()
        p.x = (x * torch.exp2(powers)[:, None]).bfloat16()
        p.check()


@pytest.mark.parametrize("tokens", [1, 5, 16])
@pytest.mark.parametrize("low, high", [(-100, 0), (-70, 70), (-126, -90), (0, 100), (-133, 0)])
def test_bf16_activations_of_mixed_magnitudes(low, high, tokens):
    """Columns of very different sizes: in halves (other CTAs' columns), in turn, a single large one, and zeros."""
    p = Problem(200, 2048, tokens, torch.bfloat16)
    x = p.x.float()
    small, large = (x * 2.0 ** low).bfloat16(), (x * 2.0 ** high).bfloat16()
    k = torch.arange(2048, device="cuda")
    for pick in (k < 1024, k >= 1024, k % 2 == 0, k == 77, k < 0):
        p.x = torch.where(pick, large, small)
        p.check()
        p.x = torch.where(pick, large, torch.zeros_like(small))
        p.check()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m, n, groups", [(130, 96, 1), (200, 320, 5), (70, 4096, 1), (257, 2048, 16)])
@pytest.mark.parametrize("tokens", [1, 4, 9, 16, 17, 80])
def test_infinite_activations(tokens, m, n, groups, dtype):
    """Infinities, or NaN where a weight is zero or they have both signs: as a product with the unpacked matrix has them, however many tokens there are."""
    inf = float("inf")
    p = Problem(m, n, tokens, dtype, groups)
    clean, x = p.check(), p.x.clone()
    field = torch.stack((p.codes & 15, p.codes >> 4), -1).flatten(1).double()
    wide = lambda t: t.double().repeat_interleave(n // groups, 1)  # noqa: E731
    w = (field + p.qmin - wide(p.zero)) * wide(p.scale)
    some = 7 % tokens
    for spots in ([(0, 5, inf)], [(0, n - 1, -inf)], [(some, 3, inf), (some, n // 2, -inf), (some, n - 2, inf)], [(0, 31, inf), (0, 32, inf)], [(0, 8, inf), (0, 9, float("nan"))],
                  [(t, (37 * t) % n, inf if t % 3 else -inf) for t in range(tokens)]):
        p.x = x.clone()
        want, touched = torch.zeros(tokens, m, dtype=torch.float64, device="cuda"), set()
        for token, k, value in spots:
            p.x[token, k] = value
            want[token] += w[:, k] * value
            touched.add(token)
        got = p.run()
        for token in range(tokens):
            assert torch.equal(got[token], clean[token]) if token not in touched else torch.equal(got[token].double().nan_to_num(nan=1.0), want[token].nan_to_num(nan=1.0)), (spots, token)
    p.x = x.fill_(float("nan"))
    assert p.run().isnan().all()


@pytest.mark.parametrize("m, n, tokens, adapters, rank", [(5100, 1056, 600, 3, 8), (4097, 1440, 513, 7, 40), (2300, 3104, 300, 0, 8), (20000, 480, 1025, 5, 64), (4096, 2048, 2300, 2, 16)])
def test_pairs_of_ctas(m, n, tokens, adapters, rank):
    """Tiles by two CTAs, whose slots chunks and adapters take in turn: any number of both, the last rows and tokens in either CTA, the same from cold caches."""
    for dtype, groups in ((torch.float16, 1), (torch.bfloat16, n // 32 if n % 64 else n // 64)):
        p = Problem(m, n, tokens, dtype, groups=groups if n // groups % 64 == 0 else 1, adapters=adapters, rank=rank)
        first = p.check()
        flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
        for i in range(3):
            flush.fill_(i)
            assert torch.equal(p.run(), first)


@pytest.mark.parametrize("width", [512, 528, 1024, 1040, 2048, 2064])
@pytest.mark.parametrize("queries, heads", [(1, 8), (4, 32)])
@pytest.mark.parametrize("count", [23, 24, 37, 38, 49, 50, 74, 75])
def test_either_side_of_whole_items(count, queries, heads, width):
    """Items cut evenly and items whole to each CTA: 92 to 300 of them on tables of 512 to 2064 positions."""
    import packed_cache as C

    lengths = [width if b == 0 else max((53 * b) % width, queries) for b in range(count)]
    batch = Batch([(n, queries) for n in lengths], 4, 64, 16, torch.bfloat16, seed=count)
    q = batch.randn(count * queries, heads, 64)
    got = C.attend_packed(q, batch.cache, batch.table, batch.lengths)
    want = reference(batch, q)
    assert_near(got, *want)
    wide = torch.cat((batch.table, torch.full((count, 300), -1, dtype=torch.int32, device="cuda")), 1)  # the same sequences in a table for longer ones
    assert_near(C.attend_packed(q, batch.cache, wide, batch.lengths), *want)
    assert_near(C.attend_packed(q, batch.cache, wide[:, :batch.table.shape[1]], batch.lengths), *want)


def test_caches_made_from_others():
    """A cache with some of its tensors replaced works like one that was made of them."""
    import packed_cache as C

    batch = Batch([(100, 3), (40, 1)], 2, 64, 16, torch.float16)
    q = batch.randn(4, 4, 64)
    want = C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets)
    other = batch.cache._replace(k_codes=batch.cache.k_codes.clone(), v_scale=batch.cache.v_scale.clone())
    assert isinstance(other, C.PackedCache) and torch.equal(C.attend_packed(q, other, batch.table, batch.lengths, batch.offsets), want)
    with pytest.raises(AssertionError):
        batch.cache._replace(k_scale=batch.cache.k_scale.float())


@pytest.mark.parametrize("queries", [1, 6, 90])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_queries_of_any_strides(head_dim, queries):
    """Heads before tokens, one head or one token for all, parts of something wider, windows that overlap, rows off 16 bytes: as their copies, to the last bit."""
    import packed_cache as C

    batch = Batch([(200, queries)] * 3, 2, head_dim, 16, torch.bfloat16)
    tokens, heads = batch.tokens, 8
    base = batch.randn(tokens + 4, heads + 4, 2 * head_dim + 8)
    flat = batch.randn(tokens * heads * head_dim + 64 * heads + head_dim)
    forms = [base[:tokens, :heads, :head_dim].transpose(0, 1).contiguous().transpose(0, 1), base[:tokens, :1, :head_dim].expand(tokens, heads, head_dim), base[:1, :heads, :head_dim].expand(tokens, heads, head_dim),
             base[2:2 + tokens, 3:3 + heads, 16:16 + head_dim], base[:tokens, :heads, 1:1 + head_dim], flat.as_strided((tokens, heads, head_dim), (8, 64, 1)),
             base[:tokens, :heads, :head_dim].transpose(1, 2).contiguous().transpose(1, 2)]
    for q in forms:
        plain = q.clone(memory_format=torch.contiguous_format)
        want = C.attend_packed(plain, batch.cache, batch.table, batch.lengths)
        assert_near(want, *reference(batch, plain))
        assert torch.equal(C.attend_packed(q, batch.cache, batch.table, batch.lengths), want)
        assert torch.equal(C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets), C.attend_packed(plain, batch.cache, batch.table, batch.lengths, batch.offsets))


@pytest.mark.parametrize("scale", [0.0, -0.2, 1e-30, 3.0])
@pytest.mark.parametrize("queries", [1, 5, 70])
def test_scales_of_any_sign(queries, scale):
    batch = Batch([(150, queries), (queries, queries)], 1, 64, 16, torch.float16)
    q = 0.3 * batch.randn(batch.tokens, 4, 64)
    import packed_cache as C

    for options in ({}, {"softcap": 3.0}, {"slopes": torch.linspace(-0.05, 0.05, 4, device="cuda")}):
        assert_near(C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets, scale=scale, **options), *reference(batch, q, scale=scale, **options))


def test_a_single_row_of_activations():
    """``x [n]``: ``[m]``."""
    p = Problem(70, 96, 1, torch.bfloat16, adapters=1, rank=8)
    p.index.fill_(0)
    want = p.check()
    p.x = p.x[0]
    assert torch.equal(p.run(), want[0])


@pytest.mark.parametrize("options", [{}, {"softcap": 20.0}, {"prefix": True}])
@pytest.mark.parametrize("queries", [4, 12, 33, 128, 300])
@pytest.mark.parametrize("small, large", [(1e-4, 6e4), (0.01, 6e4), (1e-4, 60.0), (1.0, 1.0)])
def test_hidden_values_of_any_size_leave_no_trace(small, large, queries, options):
    """Values far larger than those that a row sees, among the keys that the mask hides from it: the row is as near as if they were not there, that is, by the largest value that it sees
    (`NEAR`; and 2^-31 of the largest that is seen)."""
    import packed_cache as C

    group = 2 if queries > 12 else 4
    if queries <= 12 and large > 2.0 ** 26 * small * 0.05:
        small = large * 2.0 ** -26 / 0.05  # few rows: the documented distance (scales are 0.05 and more times `small`)
    batch = Batch([(queries, queries), (queries + 37, queries)], 1, 64, 16, torch.float16, seed=queries)
    scale = batch.cache.v_scale
    there = ~scale.isnan()
    scale[there] = (scale[there].float() * small).half()
    spots = {}  # every fifth position or so, from the middle of the queries on
    for b, (length, _) in enumerate(batch.sequences):
        spots[b] = list(range(length - queries // 2, length, 5))
        for p in spots[b]:
            scale[int(batch.table[b, p // 16]), :, p % 16] = large
    q = batch.randn(batch.tokens, group, 64)
    if options.get("prefix"):
        options = {"prefix": torch.tensor([2, queries], dtype=torch.int32, device="cuda")}
    got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets, **options)
    want, _ = reference(batch, q, **options)
    size = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    for b, (length, _) in enumerate(batch.sequences):
        largest = batch.values(b)[1].abs().amax((0, 2))
        for i in range(queries):
            visible = max(length - queries + i + 1, int(options["prefix"][b]) if options else 0) if "prefix" in options else length - queries + i + 1
            size[b * queries + i] = largest[:visible].max()
    bound = 2.0 ** -11 * want.abs() + NEAR * size[..., None] + 2.0 ** -25  # the last: half a step among the subnormal halves
    # a value from 65520 on, half a step above the largest half, rounds to infinity: 8 * 6e4 is one
    infinite = got.isinf() & (want.abs() + bound >= 65520) & (got.sign() == want.sign())
    gap = (got.double() - want).abs().masked_fill(infinite, 0.0)
    assert bool((gap <= bound).all()), float((gap / bound).max())


@pytest.mark.parametrize("heads, kv_heads", [(33, 1), (64, 1), (65, 1), (128, 1), (160, 1), (256, 2), (71, 71)])
@pytest.mark.parametrize("queries", [1, 2])
def test_groups_of_any_size(queries, heads, kv_heads):
    """Single queries whose heads alone make a tile, groups that divide its rows and groups that do not."""
    import packed_cache as C

    batch = Batch([(300, queries), (31, queries), (129, queries)], kv_heads, 64, 32, torch.float16)
    q = batch.randn(batch.tokens, heads, 64)
    for offsets in (None, batch.offsets):
        assert_near(C.attend_packed(q, batch.cache, batch.table, batch.lengths, offsets), *reference(batch, q))


@pytest.mark.parametrize("queries", [1, 5, 80])
def test_caches_beyond_4_gb(queries):
    """Pages whose codes begin behind the first 2^32 bytes are written, read and attended to like the first ones."""
    import packed_cache as C

    pages, kv_heads, page_size = 66000, 8, 128
    big = C.new_packed_cache(pages, page_size, kv_heads, 128, "cuda")
    assert big.k_codes.numel() > 2 ** 32
    small = C.new_packed_cache(8, page_size, kv_heads, 128, "cuda")
    batch = Batch([(300, 300), (150, 150)], kv_heads, 128, page_size, torch.bfloat16, fill=False)
    k, v, q = batch.randn(450, kv_heads, 128), batch.randn(450, kv_heads, 128), batch.randn(2 * queries, 16, 128)
    table = torch.tensor([[7, 1, 3], [2, 0, 6]], dtype=torch.int32, device="cuda")
    results = []
    for cache, shift in ((small, 0), (big, pages - 8)):
        where = table + shift
        C.append_packed(cache, k, v, where, batch.lengths, batch.offsets)
        results.append((C.attend_packed(q, cache, where, batch.lengths), *C.read_packed(cache, where, batch.lengths, batch.offsets, tokens=450, dtype=torch.bfloat16)))
    assert all(torch.equal(x, y) for x, y in zip(*results))
    assert torch.equal(results[0][1], rounded(k)[0].bfloat16())
    assert not any(t[:pages - 8].any() for t in big)


@pytest.mark.parametrize("tokens", [2, 20, 300])
def test_matrices_beyond_4_gb(tokens):
    """The last rows of a matrix of more than 2^32 bytes of codes."""
    import packed_linear as L

    m, n, tail = 264000, 32768, 700
    p = Problem(tail, n, tokens, torch.float16)
    codes = torch.zeros(m, n // 2, dtype=torch.uint8, device="cuda")
    assert codes.numel() > 2 ** 32
    codes[-tail:], scale, zero = p.codes, torch.ones(m, 1, device="cuda"), torch.full((m, 1), -8.0, device="cuda")  # of zeros above: code 0, zero point -8, so 0
    scale[-tail:], zero[-tail:] = p.scale, p.zero
    got = L.packed_linear(p.x, codes, scale, zero, qmin=p.qmin)
    want, slack = p.reference()
    bound = 2.0 ** -11 * want.abs() * (1 + 2.0 ** -8) + slack + 2.0 ** -14
    assert bool(((got[:, -tail:].double() - want).abs() <= bound).all())
    # x times zero weights: what two sums of n terms, each lost to 2^-23 of 16 |x| a step, may leave
    assert bool((got[:, :-tail].double().abs() <= (n / 16 + 16) * 2.0 ** -23 * 16 * p.x.double().abs().sum(1, keepdim=True)).all())


@pytest.mark.parametrize("queries", [1, 5, 100])
@pytest.mark.parametrize("length", [3000, 30000, 200000])
def test_slopes_of_either_sign_over_long_distances(length, queries):
    """Biases of tens of thousands where the keys that count are far from the query."""
    import packed_cache as C

    batch = Batch([(length, queries)], 1, 64, 128, torch.float16)
    q = batch.randn(queries, 4, 64)
    slopes = torch.tensor([-0.5, 0.5, -0.01, 0.0], device="cuda")
    for options in ({}, {"softcap": 30.0}, {"prefix": torch.full((1,), length - 10, dtype=torch.int32, device="cuda")}):
        got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, slopes=slopes, **options)
        want, size = reference(batch, q, slopes=slopes, **options)
        gap = (got.double() - want).abs() / (2.0 ** -11 * want.abs() + NEAR * size[..., None])
        assert bool((gap <= 1).all()), float(gap.max())


def test_calls_from_several_threads():
    """Host threads with streams of their own, each with calls of all kinds at once: bit for bit what one thread alone gets."""
    import threading

    import gptq_2d
    import packed_cache as C

    def work(seed):
        problems = [Problem(700, 512, t, torch.float16, adapters=4, rank=8, seed=seed) for t in (1, 30, 90, 600)]
        batch = Batch([(400, 1)] * 5 + [(300, 200)], 2, 64, 16, torch.float16, seed=seed)
        q, k = batch.randn(batch.tokens, 8, 64), batch.randn(batch.tokens, 2, 64)
        return problems, batch, q, k

    def run(state):
        problems, batch, q, k = state
        out = [p.run() for p in problems]
        C.append_packed(batch.cache, k, k, batch.table, batch.lengths, batch.offsets)
        out.append(C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets, softcap=20.0))
        return out + list(C.read_packed(batch.cache, batch.table, batch.lengths, batch.offsets, tokens=batch.tokens, dtype=torch.float16))

    states = [work(seed) for seed in range(4)]
    want = [run(state) for state in states]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def loop(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = run(states[i])
                torch.cuda.current_stream().synchronize()
        except BaseException as error:  # a thread's failure is the test's
            errors.append(error)

    threads = [threading.Thread(target=loop, args=(i,)) for i in range(4)]
    for thread in threads:
        thread.start()
    for thread in threads:
        thread.join()
    assert not errors
    gptq_2d.check_status()
    for mine, alone in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(mine, alone))
