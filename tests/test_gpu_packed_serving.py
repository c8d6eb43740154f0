"""The packed product with adapters, the packed cache and attention over it, run together as a serving loop runs them, and what a loop does to them: workspaces
that hold anything, several streams, graphs that are replayed, batches of decoding and prompt sequences.  Each operator's result is held against its plain formula in
64 bits for the inputs that it got, to the tolerances derived in the two files that test them one by one."""
import pytest
import torch
from test_gpu_packed_cache import Batch, assert_near, reference, rounded
from test_gpu_packed_linear import Problem

pytestmark = pytest.mark.gpu


def litter():
    """What was freed last, and what a call without a workspace of its own gets next, is full of large numbers."""
    for size in (1 << 12, 1 << 16, 1 << 20, 3 << 20, 10 << 20, 40 << 20):
        blocks = [torch.full((size,), 0x7f, dtype=torch.uint8, device="cuda") for _ in range(3)]
        del blocks


class Layer:
    """One attention block: fused projection with adapters, cache, attention, output projection with adapters."""

    def __init__(self, hidden, heads, kv_heads, head_dim, dtype, pages=64, page_size=16, adapters=3, rank=8):
        import packed_cache as C
        import packed_linear as L

        self.heads, self.kv_heads, self.head_dim, self.dtype = heads, kv_heads, head_dim, dtype
        wide = (heads + 2 * kv_heads) * head_dim
        self.gen = torch.Generator(device="cuda").manual_seed(hidden + heads)
        randn = lambda *shape: torch.randn(*shape, generator=self.gen, device="cuda")  # noqa: E731
        self.weights = []
        for m, n in ((wide, hidden), (hidden, heads * head_dim)):
            codes = torch.randint(0, 256, (m, n // 2), generator=self.gen, device="cuda", dtype=torch.uint8)
            scale = (0.5 + torch.rand(m, 1, generator=self.gen, device="cuda")) / (5 * n ** 0.5)
            own = L.LowRankAdapters((randn(adapters, rank, n) / n ** 0.5).to(dtype), (0.3 * randn(adapters, m, rank)).to(dtype))
            self.weights.append((codes, scale, torch.zeros(m, 1, device="cuda"), own))
        self.cache = C.new_packed_cache(pages, page_size, kv_heads, head_dim, "cuda")

    def project(self, which, x, index):
        import packed_linear as L

        codes, scale, zero, adapters = self.weights[which]
        return L.packed_linear(x, codes, scale, zero, qmin=-8, adapters=adapters, adapter_index=index)

    def step(self, x, index, table, lengths, offsets):
        import packed_cache as C

        h, k = self.heads, self.kv_heads
        qkv = self.project(0, x, index).view(x.shape[0], h + 2 * k, self.head_dim)
        q, keys, values = qkv[:, :h], qkv[:, h:h + k], qkv[:, h + k:]
        C.append_packed(self.cache, keys, values, table, lengths, offsets)
        o = C.attend_packed(q, self.cache, table, lengths, offsets)
        return qkv, o, self.project(1, o.flatten(1), index)

    def check_product(self, which, x, index, got):
        p = Problem.__new__(Problem)
        p.qmin, p.x, p.index = -8, x, index
        p.codes, p.scale, p.zero, p.adapters = self.weights[which]
        want, slack = p.reference()
        bound = torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + slack + torch.finfo(got.dtype).smallest_normal
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_a_prompt_and_decoding_steps(head_dim, dtype):
    import gptq_2d

    layer = Layer(256, 8, 2, head_dim, dtype)
    lengths = [70, 1, 33, 19]
    held = [None] * len(lengths)  # the rounded keys and values so far, by sequence
    table = torch.randperm(64, generator=layer.gen, device="cuda")[:32].to(torch.int32).view(4, 8).contiguous()
    for queries in ([70, 1, 33, 19], [1, 1, 1, 1], [0, 2, 1, 0], [1, 0, 16, 1]):
        if held[0] is not None:
            lengths = [n + q for n, q in zip(lengths, queries)]
        tokens = sum(queries)
        offsets = torch.tensor([0] + queries, device="cuda").cumsum(0).to(torch.int32)
        x = torch.randn(tokens, 256, generator=layer.gen, device="cuda").to(dtype)
        index = torch.randint(-1, 4, (tokens,), generator=layer.gen, device="cuda", dtype=torch.int32)
        litter()
        qkv, o, y = layer.step(x, index, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), offsets)
        gptq_2d.check_status()
        layer.check_product(0, x, index, qkv.flatten(1))
        layer.check_product(1, o.flatten(1), index, y)
        at = 0
        for b, q in enumerate(queries):
            new = [rounded(qkv[at:at + q, 8 + 2 * i:10 + 2 * i])[0].transpose(0, 1) for i in range(2)]
            held[b] = new if held[b] is None else [torch.cat((old, rows), 1) for old, rows in zip(held[b], new)]
            at += q
        batch = type("Held", (), {"sequences": list(zip(lengths, queries)), "kv_heads": 2, "head_dim": head_dim, "values": lambda self, b: held[b]})()
        assert all(held[b][0].shape[1] == n for b, n in enumerate(lengths))
        assert_near(o, *reference(batch, qkv[:, :8]))


def test_a_captured_step_follows_the_lengths():
    """Decoding steps from one graph, the lengths counted up on the device, give bit for bit what eager calls give."""
    results = []
    for captured in (False, True):
        layer = Layer(128, 4, 4, 64, torch.float16)
        table = torch.arange(12, dtype=torch.int32, device="cuda").view(3, 4).flip(1).contiguous()
        lengths, one = torch.tensor([0, 14, 31], dtype=torch.int32, device="cuda"), torch.ones(3, dtype=torch.int32, device="cuda")
        x, index = torch.zeros(3, 128, dtype=torch.float16, device="cuda"), torch.tensor([2, 9, 0], dtype=torch.int32, device="cuda")
        steps = torch.randn(5, 3, 128, generator=layer.gen, device="cuda").half()

        def step():
            lengths.add_(one)
            return layer.step(x, index, table, lengths, None)[2]

        if captured:
            step()  # set up, then as if it had not been
            lengths.copy_(torch.tensor([0, 14, 31], dtype=torch.int32))
            layer.cache.k_codes.zero_(), layer.cache.v_codes.zero_(), layer.cache.k_scale.zero_(), layer.cache.v_scale.zero_()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        for row in steps:
            x.copy_(row)
            if captured:
                graph.replay()
            else:
                out = step()
            results.append(out.clone())
    for eager, replayed in zip(results[:5], results[5:]):
        assert torch.equal(eager, replayed)


@pytest.mark.parametrize("sequences", [[(300, 1)] * 40, [(300, 1)] * 40 + [(900, 500)], [(700, 300), (5, 1), (0, 0), (257, 257)], [(64, 9)] * 9, [(2000, 70), (100, 1)], [(0, 0)] * 33 + [(40, 40)]])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_decoding_and_prompts_in_one_batch(sequences, head_dim):
    """Sequences by rows and by tiles in one call, each kind the larger part; more than a warp looks at once; workspaces full of large numbers."""
    import gptq_2d
    import packed_cache as C

    batch = Batch(sequences, 2, head_dim, 32, torch.float16)
    q = batch.randn(batch.tokens, 8, head_dim)
    want, size = reference(batch, q)
    for _ in range(2):
        litter()
        got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets)
        assert_near(got, want, size)
    # rows of no sequence, before and behind: zeros in a new tensor, as they were in a given one
    wide = torch.cat((q[:1], q, q[:2]))
    offsets = batch.offsets + 1
    litter()
    got = C.attend_packed(wide, batch.cache, batch.table, batch.lengths, offsets)
    assert not got[:1].any() and not got[-2:].any()
    assert_near(got[1:-2], want, size)
    out = torch.full_like(wide, 3.0)
    C.attend_packed(wide, batch.cache, batch.table, batch.lengths, offsets, out=out)
    assert (out[:1] == 3).all() and (out[-2:] == 3).all() and torch.equal(out[1:-2], got[1:-2])
    litter()
    k, v = C.read_packed(batch.cache, batch.table, batch.lengths, offsets, tokens=wide.shape[0], dtype=torch.float16)
    assert not k[:1].any() and not k[-2:].any() and not v[:1].any() and not v[-2:].any()
    gptq_2d.check_status()


@pytest.mark.parametrize("softcap", [1e-25, 1e-3, 63.0, 65.0, 1000.0, 1e6, 1e12, 1e31])
@pytest.mark.parametrize("queries", [1, 3, 100])
def test_caps_of_any_size(queries, softcap):
    """From caps that leave no score to caps far above all of them."""
    import packed_cache as C

    batch = Batch([(300, queries)] * 2, 1, 64, 32, torch.float16)
    q = 4 * batch.randn(batch.tokens, 4, 64)
    assert_near(C.attend_packed(q, batch.cache, batch.table, batch.lengths, softcap=softcap), *reference(batch, q, softcap=softcap))


@pytest.mark.parametrize("rows", [31, 32, 33, 63, 64, 65, 66])
@pytest.mark.parametrize("batch_size", [1, 70])
def test_either_side_of_the_line_between_rows_and_tiles(rows, batch_size):
    batch = Batch([(90 + rows, rows)] * batch_size, 1, 64, 16, torch.bfloat16)
    q = batch.randn(batch.tokens, 1, 64)
    import packed_cache as C

    assert_near(C.attend_packed(q, batch.cache, batch.table, batch.lengths), *reference(batch, q))


@pytest.mark.parametrize("m, n, tokens, adapters, rank", [(19200, 256, 128, 3, 16), (20480, 2048, 200, 2, 8), (20000, 1984, 150, 0, 8), (19328, 192, 64, 40, 64), (300, 4096, 33, 5, 24), (9600, 64, 50, 2, 8),
                                                          (5000, 4096, 700, 4, 32), (4000, 512, 100, 40, 16), (4096, 320, 250, 30, 8), (9000, 1024, 256, 24, 16)])
def test_whole_rounds_of_tiles_and_tiles_that_are_cut(m, n, tokens, adapters, rank):
    litter()
    Problem(m, n, tokens, torch.float16, adapters=adapters, rank=rank).check()
    litter()
    Problem(m, n, tokens, torch.bfloat16, groups=1 if n % 128 else n // 64, adapters=adapters, rank=rank).check()


@pytest.mark.parametrize("tokens", [1, 9, 16])
@pytest.mark.parametrize("n", [32768, 32800, 65536])
def test_rows_that_are_longer_than_shared_memory(n, tokens):
    Problem(70, n, tokens, torch.bfloat16, adapters=3, rank=8).check()
    if n % 128 == 0:
        Problem(70, n, tokens, torch.float16, groups=n // 64).check()


def test_two_streams_at_once():
    import gptq_2d
    import packed_cache as C

    problems = [Problem(2048, 2048, t, torch.float16, adapters=4, seed=t) for t in (1, 40, 300)]
    batches = [Batch([(900, 1)] * 6, 4, 128, 64, torch.float16, seed=3), Batch([(600, 200), (50, 1)], 4, 128, 64, torch.float16, seed=4)]
    queries = [b.randn(b.tokens, 16, 128) for b in batches]
    calls = [p.run for p in problems] + [lambda b=b, q=q: C.attend_packed(q, b.cache, b.table, b.lengths, b.offsets) for b, q in zip(batches, queries)]
    alone = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i] += [call() for call in (calls if i else calls[::-1])]
    torch.cuda.synchronize()
    gptq_2d.check_status()
    for i in range(2):
        for k, result in enumerate(got[i]):
            want = alone[k % 5] if i else alone[4 - k % 5]
            assert torch.equal(result, want)


def test_two_graphs_that_are_replayed_at_once():
    """Each graph has workspaces of its own."""
    import packed_cache as C

    problems = [Problem(1024, 2048, 48, torch.bfloat16, adapters=6, seed=s) for s in (1, 2)]
    batch = Batch([(400, 1)] * 5, 2, 64, 16, torch.bfloat16)
    queries = [batch.randn(5, 8, 64) for _ in range(2)]
    run = lambda i: (problems[i].run(), C.attend_packed(queries[i], batch.cache, batch.table, batch.lengths))  # noqa: E731
    alone = [run(i) for i in range(2)]
    graphs, outs = [], []
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(i))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, alone):
        assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("queries", ["prompts", "drafts"])
def test_cold_caches_change_nothing(queries, head_dim):
    """Keys, values and scales that come late in any order: what was pushed out of the caches in between gives the same results bit for bit."""
    import gptq_2d
    import packed_cache as C

    sequences = [(2500, 1500), (1801, 700), (900, 900), (2000, 70)] if queries == "prompts" else [(3000, 4), (1, 1), (2222, 7)] * 8
    batch = Batch(sequences, 4, head_dim, 64, torch.float16)
    q = batch.randn(batch.tokens, 16, head_dim)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    first = None
    for i in range(16):
        flush.fill_(i)
        got = C.attend_packed(q, batch.cache, batch.table, batch.lengths, batch.offsets, causal=i % 2 == 0)
        if i < 2:
            assert_near(got, *reference(batch, q, causal=i == 0))
            first = (first or []) + [got]
        assert torch.equal(got, first[i % 2])
    gptq_2d.check_status()


@pytest.mark.parametrize("tokens", [3, 16, 50, 120, 400])
@pytest.mark.parametrize("groups", [1, 32])
def test_products_from_cold_caches_are_the_same(groups, tokens):
    p = Problem(5000, 2048, tokens, torch.bfloat16, groups=groups, adapters=6, rank=16)
    flush = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
    first = p.check()
    for i in range(8):
        flush.fill_(i)
        assert torch.equal(p.run(), first)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("queries, heads", [(1, 8), (3, 8), (16, 4), (2, 32)])
@pytest.mark.parametrize("width", [1, 64, 65, 130, 511, 512, 513, 2048])
def test_short_tables(width, queries, heads, head_dim):
    """Sequences of all lengths that a short table holds, more items than SMs and fewer; queries before the first position."""
    import packed_cache as C

    for count in (1, 25, 90):
        lengths = [width if b == 0 else (37 * b) % (width + 1) for b in range(count)]
        batch = Batch([(max(n, 1), 1) for n in lengths], 4, head_dim, 16, torch.float16, seed=width)
        batch.sequences = [(n, queries) for n in lengths]
        q = batch.randn(count * queries, heads, head_dim)
        litter()
        got = C.attend_packed(q, batch.cache, batch.table, torch.tensor(lengths, dtype=torch.int32, device="cuda"))
        assert_near(got, *reference(batch, q))
