"""The packed cache and attention over it, against plain formulas in 64 bits.

Tolerances, derived before the first run.  A result is one rounding of the exact value (half a step of its type, ``eps / 2`` relative) plus what the kernel loses
on the way: each product of an exponential with a value's scale is rounded to 11 bits (2^-12 relative, so at most 2^-12 of the sum of |p v| / sum p,
which the largest |v| of the row's keys bounds), the exponentials themselves are good to 2^-20 for scores of the sizes here, and fp32 sums add less.
So |got - want| <= eps / 2 |want| + (2^-12 + 2^-16) max |v| is asserted, entry by entry, with the 2^-16 for all the rest.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


def unpacked(codes, scale):
    """float64 values [.., places, head_dim] of codes and scales, by their definition."""
    fields = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).double() - 8
    return fields * scale.double()[..., None]


def rounded(x):
    """Codes' values of rows under their abs-max scales, in 64 bits."""
    x = x.double()
    scale = (x.abs().amax(-1, keepdim=True) / 7.5).float().half().double()
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return torch.clamp(torch.round(x / scale), -8, 7) * scale, scale.squeeze(-1)


class Batch:
    """Sequences of (length, queries) in a cache with shuffled pages; pages that no sequence has are left with codes and scales of NaN."""

    def __init__(self, sequences, kv_heads, head_dim, page_size, dtype, seed=0, fill=True, spare=2):
        import packed_cache as C

        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.sequences, self.kv_heads, self.head_dim, self.page_size, self.dtype, self.gen = sequences, kv_heads, head_dim, page_size, dtype, gen
        width = max([1] + [-(-length // page_size) for length, _ in sequences])
        pages = width * len(sequences) + spare
        self.cache = C.new_packed_cache(pages, page_size, kv_heads, head_dim, "cuda")
        for t in (self.cache.k_scale, self.cache.v_scale):
            t.fill_(float("nan"))
        for t in (self.cache.k_codes, self.cache.v_codes):
            t.random_(0, 256, generator=gen)
        order = torch.randperm(pages, generator=gen, device="cuda")
        self.table = order[: width * len(sequences)].to(torch.int32).view(len(sequences), width).contiguous()
        self.lengths = torch.tensor([length for length, _ in sequences], dtype=torch.int32, device="cuda")
        self.offsets = torch.tensor([0] + [q for _, q in sequences], device="cuda").cumsum(0).to(torch.int32)
        self.tokens = sum(q for _, q in sequences)
        if fill:
            for name in ("k", "v"):
                codes, scale = getattr(self.cache, name + "_codes"), getattr(self.cache, name + "_scale")
                for b, (length, _) in enumerate(sequences):
                    for p in range(0, length, page_size):
                        page, here = int(self.table[b, p // page_size]), min(page_size, length - p)
                        scale[page, :, :here] = (0.05 + torch.rand(kv_heads, here, generator=gen, device="cuda")).half()

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda").to(self.dtype)

    def values(self, b):
        """Keys and values [kv_heads, length, head_dim] of a sequence, float64."""
        length = self.sequences[b][0]
        pages = self.table[b].long()
        whole = lambda codes, scale: unpacked(codes[pages], scale[pages]).transpose(0, 1).reshape(self.kv_heads, -1, self.head_dim)[:, :length]  # noqa: E731
        return whole(self.cache.k_codes, self.cache.k_scale), whole(self.cache.v_codes, self.cache.v_scale)


def reference(batch, q, scale=None, causal=True, softcap=0.0, slopes=None, prefix=None):
    """float64 results, and the largest |v| that each row's tolerance goes by."""
    heads, group = q.size(1), q.size(1) // batch.kv_heads
    scale = batch.head_dim ** -0.5 if scale is None else scale
    out, size = torch.zeros(q.shape, dtype=torch.float64, device="cuda"), torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    at = 0
    for b, (length, queries) in enumerate(batch.sequences):
        if queries and length:
            k, v = (x.repeat_interleave(group, 0) for x in batch.values(b))
            u = scale * q[at:at + queries].double().transpose(0, 1) @ k.transpose(1, 2)
            if softcap:
                u = softcap * torch.tanh(u / softcap)
            p = torch.arange(length - queries, length, device="cuda")[:, None]
            j = torch.arange(length, device="cuda")[None]
            if slopes is not None:
                u = u + slopes.double()[:, None, None] * (j - p)
            if causal:
                hidden = (j > p) & (j >= (0 if prefix is None else int(prefix[b])))
                u = u.masked_fill(hidden, -math.inf)
            w = torch.softmax(u, -1)
            w = torch.where(torch.isnan(w), torch.zeros_like(w), w) if causal else w
            out[at:at + queries] = (w @ v).transpose(0, 1)
            size[at:at + queries] = v.abs().amax((1, 2))[None]
        at += queries
    return out, size


def assert_near(got, want, size):
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + (2.0 ** -12 + 2.0 ** -16) * size[..., None] + torch.finfo(got.dtype).smallest_normal
    gap = (got.double() - want).abs()
    assert bool((gap <= bound).all()), f"off by {float((gap / bound).max()):.2f} of the bound"


def attend(batch, q, uniform=False, **options):
    import gptq_2d
    import packed_cache as C

    got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, None if uniform else batch.offsets, **options)
    gptq_2d.check_status()
    want, size = reference(batch, q, **{k: v for k, v in options.items() if k != "out"})
    assert_near(got, want, size)
    return got


# ---- writing and reading -----------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("head_dim, kv_heads, page_size", [(64, 1, 16), (128, 8, 64), (64, 5, 128), (128, 3, 32)])
@pytest.mark.parametrize("sequences", [[(1, 1)], [(70, 70), (0, 0), (33, 1), (129, 64)], [(16, 16), (17, 17), (15, 15)]])
def test_append_and_read(sequences, head_dim, kv_heads, page_size, dtype):
    import packed_cache as C

    batch = Batch(sequences, kv_heads, head_dim, page_size, dtype, fill=False)
    k, v = batch.randn(batch.tokens, kv_heads, head_dim), batch.randn(batch.tokens, kv_heads, head_dim)
    k[0], v[-1] = 0, 2.0 ** -20  # a row of zeros; scales among the subnormal halves
    before = [t.clone() for t in batch.cache]
    C.append_packed(batch.cache, k, v, batch.table, batch.lengths, batch.offsets)
    got = C.read_packed(batch.cache, batch.table, batch.lengths, batch.offsets, tokens=batch.tokens, dtype=dtype)
    for x, y in zip((k, v), got):
        assert torch.equal(y, rounded(x)[0].to(dtype))
    # nothing but the step's rows has changed
    at, mine = 0, torch.zeros(batch.cache.k_scale.shape, dtype=torch.bool, device="cuda")
    for b, (length, queries) in enumerate(sequences):
        for p in range(length - queries, length):
            mine[int(batch.table[b, p // page_size]), :, p % page_size] = True
    for old, new in zip(before, batch.cache):
        assert torch.equal(old[~mine].view(torch.uint8), new[~mine].view(torch.uint8))


def test_append_agrees_with_the_packages_quantizer():
    import packed_cache as C
    import packed_codes
    import quantizer_int

    batch = Batch([(96, 96)], 2, 128, 32, torch.bfloat16, fill=False)
    k, v = batch.randn(96, 2, 128), batch.randn(96, 2, 128)
    C.append_packed(batch.cache, k, v, batch.table, batch.lengths, batch.offsets)
    rows = k.float().reshape(-1, 128)
    scale = quantizer_int.int_abs_max_scale_cuda(rows, qmin=-8, qmax=7, dtype=torch.float16)
    codes = packed_codes.pack_codes(torch.clamp(torch.round(rows / scale), -8, 7) * scale, scale, torch.zeros(1, 1, device="cuda"), qmin=-8, bits=4)
    pages = batch.table[0].long()
    assert torch.equal(batch.cache.k_codes[pages].transpose(1, 2).reshape(-1, 64), codes)
    assert torch.equal(batch.cache.k_scale[pages].transpose(1, 2).reshape(-1).float(), scale.flatten())


def test_rows_that_are_not_finite_read_as_nan():
    import packed_cache as C

    batch = Batch([(20, 20)], 1, 64, 16, torch.float16, fill=False)
    k, v = batch.randn(20, 1, 64), batch.randn(20, 1, 64)
    k[3, 0, 7], v[5, 0, 63], v[6, 0, 0] = float("inf"), float("nan"), -float("inf")
    C.append_packed(batch.cache, k, v, batch.table, batch.lengths, batch.offsets)
    gk, gv = C.read_packed(batch.cache, batch.table, batch.lengths, batch.offsets, tokens=20, dtype=torch.float16)
    assert gk[3].isnan().all() and gv[5].isnan().all() and gv[6].isnan().all()
    gk[3], gv[5], gv[6] = 0, 0, 0
    assert gk.isfinite().all() and gv.isfinite().all()


def test_strided_keys_and_values_are_read_in_place():
    import packed_cache as C

    batch = Batch([(40, 40), (21, 9)], 4, 128, 16, torch.bfloat16, fill=False)
    qkv = batch.randn(batch.tokens, 12 + 4 + 4, 128)
    k, v = qkv[:, 12:16], qkv[:, 16:]
    odd = torch.empty(batch.tokens * 4 * 128 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(batch.tokens, 4, 128).copy_(k)  # two bytes off
    for keys in (k, odd, k.transpose(1, 2).contiguous().transpose(1, 2)):
        C.append_packed(batch.cache, keys, v, batch.table, batch.lengths, batch.offsets)
        gk, gv = C.read_packed(batch.cache, batch.table, batch.lengths, batch.offsets, tokens=batch.tokens, dtype=torch.bfloat16)
        assert torch.equal(gk, rounded(k)[0].bfloat16()) and torch.equal(gv, rounded(v)[0].bfloat16())
        batch.cache.k_codes.zero_()


# ---- attention ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("heads, kv_heads", [(1, 1), (8, 8), (8, 1), (28, 4), (12, 1), (40, 2)])
def test_one_query_per_sequence(heads, kv_heads, head_dim, dtype):
    batch = Batch([(1, 1), (63, 1), (64, 1), (65, 1), (200, 1), (1000, 1)], kv_heads, head_dim, 32, dtype)
    q = batch.randn(batch.tokens, heads, head_dim)
    a = attend(batch, q, uniform=True)
    assert torch.equal(a, attend(batch, q))


@pytest.mark.parametrize("page_size", [16, 32, 64, 128, 1024])
@pytest.mark.parametrize("causal", [True, False])
def test_pages_and_ragged_queries(page_size, causal):
    batch = Batch([(130, 3), (0, 0), (5, 5), (300, 0), (77, 20), (1030, 2), (64, 64)], 2, 128, page_size, torch.float16)
    attend(batch, batch.randn(batch.tokens, 8, 128), causal=causal)


@pytest.mark.parametrize("queries, length", [(1, 1), (2, 2), (5, 300), (17, 17), (64, 64), (65, 700), (130, 131), (257, 1000), (513, 513)])
@pytest.mark.parametrize("heads, kv_heads, head_dim", [(4, 4, 64), (8, 2, 128), (5, 1, 128)])
def test_prompts(queries, length, heads, kv_heads, head_dim):
    batch = Batch([(length, queries)] * 2, kv_heads, head_dim, 16, torch.bfloat16, seed=queries)
    attend(batch, batch.randn(batch.tokens, heads, head_dim), uniform=True)


@pytest.mark.parametrize("queries", [1, 3, 200])
@pytest.mark.parametrize("options", [{"softcap": 2.0}, {"slopes": True}, {"softcap": 30.0, "slopes": True}, {"prefix": True}, {"prefix": True, "slopes": True, "softcap": 5.0}, {"scale": 0.3}])
def test_options(options, queries):
    batch = Batch([(300, queries), (queries, queries), (257, queries)], 2, 128, 32, torch.float16)
    options = dict(options)
    if options.get("slopes"):
        options["slopes"] = torch.linspace(-0.01, 0.5, 6, device="cuda")
    if options.get("prefix"):
        options["prefix"] = torch.tensor([150, 100000, -5], dtype=torch.int32, device="cuda")
    attend(batch, batch.randn(batch.tokens, 6, 128), uniform=True, **options)


def test_long_sequences_and_many():
    """Work that is split over many warps, sequences of very different lengths, more sequences than a warp looks at once."""
    lengths = [40000, 1, 0, 777] + [5 * i for i in range(60)]
    batch = Batch([(n, min(n, 1)) for n in lengths], 2, 64, 64, torch.float16)
    attend(batch, batch.randn(batch.tokens, 8, 64))


def test_a_sharp_maximum_anywhere():
    """One key that takes nearly all of the weight, in every block of a long sequence, and scores far below zero everywhere else."""
    length = 700
    batch = Batch([(length, 1)] * 8, 1, 64, 64, torch.float16)
    batch.cache.k_codes.fill_(0x88)  # all keys zero
    q = torch.full((8, 1, 64), 4.0, device="cuda", dtype=torch.float16)
    for b in range(8):
        p = 97 * b + 5
        batch.cache.k_codes[int(batch.table[b, p // 64]), 0, p % 64] = 0xff
    attend(batch, q, uniform=True)
    attend(batch, -q, uniform=True)


def test_values_of_very_different_scales():
    batch = Batch([(500, 1), (130, 2)], 1, 128, 16, torch.bfloat16)
    scale = batch.cache.v_scale
    ok = ~scale.isnan()
    scale[ok] = (scale[ok].float() * torch.exp2(torch.randint(-22, 12, (int(ok.sum()),), generator=batch.gen, device="cuda").float())).half()
    attend(batch, batch.randn(3, 4, 128))
    scale[ok] = 0
    got = attend(batch, batch.randn(3, 4, 128))
    assert not got.any()


def test_what_is_masked_may_be_anything():
    """Infinite and NaN scales at positions that a query does not see leave no trace; seen ones make the row NaN."""
    import packed_cache as C

    batch = Batch([(100, 4)], 1, 64, 16, torch.float16)
    q = batch.randn(4, 2, 64)
    clean = attend(batch, q)
    page = int(batch.table[0, 99 // 16])
    for bad in (float("inf"), float("nan"), -float("inf")):
        batch.cache.v_scale[page, 0, 99 % 16] = bad
        got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets)
        assert torch.equal(got[:3], clean[:3]) and not got[3].isfinite().any()
    batch.cache.v_scale[page, 0, 99 % 16] = 1
    batch.cache.k_scale[page, 0, 99 % 16] = float("nan")
    got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets)
    assert torch.equal(got[:3], clean[:3]) and got[3].isnan().all()


def test_queries_without_keys_and_rows_of_no_sequence():
    import packed_cache as C

    batch = Batch([(0, 0), (3, 3), (40, 2)], 2, 64, 16, torch.float16)
    lengths = torch.tensor([0, 1, 40], dtype=torch.int32, device="cuda")  # two of the three queries stand before the first position
    offsets = torch.tensor([2, 2, 5, 7], dtype=torch.int32, device="cuda")
    q = batch.randn(10, 4, 64)
    out = torch.full((10, 4, 64), 7.0, dtype=torch.float16, device="cuda")
    got = C.attend_packed(q, batch.cache, batch.table, lengths, offsets, out=out)
    assert got is out and (out[:2] == 7).all() and (out[7:] == 7).all()
    assert not out[2:4].any() and out[4].any() and out[5:7].any()
    assert not C.attend_packed(q, batch.cache, batch.table, lengths, offsets)[7:].any()
    k = batch.randn(10, 2, 64)
    before = batch.cache.k_codes.clone()
    C.append_packed(batch.cache, k, k, batch.table, lengths, offsets)
    changed = (before != batch.cache.k_codes).any(-1).nonzero().tolist()
    assert len(changed) <= 3 * 2  # position 0 of the second sequence, 38 and 39 of the third, in two heads


def test_absent_pages():
    """Page numbers outside the cache and lengths beyond the table: nothing is read or written there, the rest is as it should be."""
    import packed_cache as C

    batch = Batch([(200, 1), (90, 1)], 1, 64, 16, torch.float16)
    q = batch.randn(2, 4, 64)
    table = batch.table.clone()
    table[0, 3], table[0, 7], table[1, 0] = -1, 10 ** 6, 2 ** 31 - 1
    got = C.attend_packed(q, batch.cache, table, batch.lengths, None)
    holes = [[3, 7], [0]]
    for b in range(2):
        k, v = batch.values(b)
        keep = torch.ones(k.size(1), dtype=torch.bool, device="cuda")
        for page in holes[b]:
            keep[16 * page:16 * page + 16] = False
        u = q[b].double() @ k[0].t() / 8
        want = torch.softmax(u[:, keep], -1) @ v[0][keep]
        assert_near(got[b], want, torch.full((4,), float(v.abs().max()), dtype=torch.float64, device="cuda"))
    # longer than the table says: the positions that exist
    lengths = torch.tensor([13 * 16 + 1000, 90], dtype=torch.int32, device="cuda")
    before = [t.clone() for t in batch.cache]
    C.append_packed(batch.cache, q[:, :1], q[:, :1], table, torch.tensor([13 * 16 + 1000, -4], dtype=torch.int32, device="cuda"))
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, batch.cache))
    gk, _ = C.read_packed(batch.cache, table, lengths, tokens=2, dtype=torch.float16)
    assert not gk[0].any() and gk[1].any()


def test_wild_offsets_stay_in_bounds():
    import packed_cache as C

    batch = Batch([(100, 1), (50, 1)], 1, 64, 16, torch.float16)
    q = batch.randn(6, 2, 64)
    for offsets in ([5, 2, 900], [-7, 3, 2], [0, 6, 6], [6, 6, 6]):
        got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        assert got.shape == q.shape


def test_streams_and_graphs():
    import packed_cache as C

    batch = Batch([(500, 1), (700, 1)], 2, 128, 64, torch.bfloat16)
    q, out = batch.randn(2, 16, 128), torch.empty(2, 16, 128, dtype=torch.bfloat16, device="cuda")
    k, v = batch.randn(2, 2, 128), batch.randn(2, 2, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())

    def step():
        C.append_packed(batch.cache, k, v, batch.table, batch.lengths)
        C.attend_packed(q, batch.cache, batch.table, batch.lengths, out=out)

    with torch.cuda.stream(side):
        step()
    graphs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()]
    for graph in graphs:
        with torch.cuda.graph(graph):
            step()
    batch.lengths += 1  # the next position: a captured step follows what is on the device
    batch.sequences = [(501, 1), (701, 1)]
    q.copy_(batch.randn(2, 16, 128))
    for graph in graphs * 2:
        graph.replay()
    want, size = reference(batch, q)
    assert_near(out, want, size)
    assert torch.equal(out, C.attend_packed(q, batch.cache, batch.table, batch.lengths))


def test_results_do_not_depend_on_the_run():
    batch = Batch([(3000, 1), (100, 1), (9000, 1)], 4, 128, 16, torch.float16)
    q = batch.randn(3, 32, 128)
    first = attend(batch, q)
    for _ in range(5):
        assert torch.equal(first, attend(batch, q))
