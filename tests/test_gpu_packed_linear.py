"""Products with packed codes and low-rank adapters beside them, against plain formulas in 64 bits.

Tolerances, derived before the first run.  A result is rounded once: ``eps / 2 |y|``.  The sums are float32 on the tensor cores, which may truncate: a product of
sixteen terms loses at most 2^-23 of the running sum, which sum_k 16 s |x_k| bounds (codes are summed as 0 .. 15 or as -8 .. 7, the rest of (code + qmin - zero) s x
being smaller for the zero points here), and a chain has n / 16 of them; the joins of partial sums add less than 16 more.  The inner values of the adapters are
fp32 sums of n terms (n / 16 + 16 steps of 2^-23 again, of sum |down x|), held to 2^-16 of the token's largest; the outer sums have 64 terms at most (2^-17).
"""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALVES = [torch.float16, torch.bfloat16]


class Problem:
    def __init__(self, m, n, tokens, dtype, groups=1, adapters=0, rank=16, qmin=-8, seed=0, scaling=True):
        import packed_linear as L

        gen = torch.Generator(device="cuda").manual_seed(seed + m + n + tokens)
        rand = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
        randn = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
        self.qmin = qmin
        self.codes = torch.randint(0, 256, (m, n // 2), generator=gen, device="cuda", dtype=torch.uint8)
        self.scale = 0.01 + 0.02 * rand(m, groups)
        self.zero = torch.randint(0, 16, (m, groups), generator=gen, device="cuda").float() + (qmin + 0.0)
        self.x = (0.3 + randn(tokens, n)).to(dtype)
        self.adapters = self.index = None
        if adapters:
            self.adapters = L.LowRankAdapters((randn(adapters, rank, n) / n ** 0.5).to(dtype), randn(adapters, m, rank).to(dtype), 0.5 + rand(adapters) if scaling else None)
            self.index = torch.randint(-1, adapters + 1, (tokens,), generator=gen, device="cuda", dtype=torch.int32)  # both ends out of range

    def reference(self):
        m, n = self.codes.shape[0], self.x.shape[1]
        groups = max(self.scale.shape[1], self.zero.shape[1])
        wide = lambda t: t.double().expand(m, groups).repeat_interleave(n // groups, 1)  # noqa: E731
        field = torch.stack((self.codes & 15, self.codes >> 4), -1).flatten(1).double()[:, :n]
        w, x = (field + self.qmin - wide(self.zero)) * wide(self.scale), self.x.double()
        steps = (n / 16 + 16) * 2.0 ** -23
        y, slack = x @ w.t(), steps * (x.abs() @ (16 * wide(self.scale)).t())
        if self.adapters:
            down, up, scaling = (t if t is None else t.double() for t in self.adapters)
            for i in range(down.shape[0]):
                mine = (self.index == i).nonzero().flatten()
                f = 1.0 if scaling is None else scaling[i]
                inner, lost = x[mine] @ down[i].t(), steps * (x[mine].abs() @ down[i].abs().t())
                y[mine] += f * inner @ up[i].t()
                lost = lost + 2.0 ** -16 * inner.abs().amax(1, keepdim=True)
                slack[mine] += f * ((lost + 2.0 ** -17 * inner.abs()) @ up[i].abs().t())
        return y, slack

    def run(self, **options):
        import packed_linear as L

        return L.packed_linear(self.x, self.codes, self.scale, self.zero, qmin=self.qmin, adapters=self.adapters, adapter_index=self.index, **options)

    def check(self, **options):
        import gptq_2d

        got = self.run(**options)
        gptq_2d.check_status()
        want, slack = self.reference()
        bound = torch.finfo(got.dtype).eps / 2 * want.abs() * (1 + 2.0 ** -8) + slack + torch.finfo(got.dtype).smallest_normal
        gap = (got.double() - want).abs()
        assert bool((gap <= bound).all()), f"off by {float((gap / bound).max()):.2f} of the bound"
        return got


TOKENS = [1, 2, 7, 8, 9, 16, 17, 33, 64, 65, 130, 257]


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("m, n, groups", [(1, 32, 1), (130, 96, 1), (257, 512, 4), (64, 320, 5), (1000, 2048, 1), (515, 1280, 10)])
def test_product(m, n, groups, tokens, dtype):
    Problem(m, n, tokens, dtype, groups).check()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("tokens", TOKENS)
@pytest.mark.parametrize("adapters, rank", [(1, 8), (5, 16), (40, 64), (3, 24)])
def test_adapters(adapters, rank, tokens, dtype):
    Problem(300, 608, tokens, dtype, adapters=adapters, rank=rank, scaling=adapters != 3).check()


@pytest.mark.parametrize("tokens", [3, 700])
def test_tokens_of_a_prompt_stand_together(tokens):
    p = Problem(384, 1024, tokens, torch.bfloat16, groups=8, adapters=4, rank=32)
    p.index = (torch.arange(tokens, device="cuda") * 5 // tokens - 1).to(torch.int32)
    p.check()


@pytest.mark.parametrize("m, n, tokens", [(8192, 4096, 5), (3, 8192, 16), (4100, 28672, 12), (700, 16384, 300)])
def test_sizes_of_real_layers(m, n, tokens):
    Problem(m, n, tokens, torch.float16, adapters=3).check()


@pytest.mark.parametrize("tokens", [4, 100])
def test_shapes_of_the_parameters(tokens):
    p = Problem(96, 256, tokens, torch.float16, groups=2)
    scale, zero = p.scale, p.zero
    for s, z in ((scale[:, :1], zero[:, :1]), (scale[:1, :1], zero[:1, :1]), (scale, zero[:1, :1]), (scale[:, :1], zero), (scale[:1], zero[:1])):
        p.scale, p.zero = s, z
        p.check()
    p.scale, p.zero = scale.half(), zero.double()
    p.check()
    p.scale, p.zero = scale[0, 0].view(1, 1), torch.zeros(1, 1, device="cuda")
    import packed_linear as L

    assert torch.equal(p.run(), L.packed_linear(p.x, p.codes, float(scale[0, 0]), 0.0, qmin=p.qmin))


@pytest.mark.parametrize("tokens", [6, 90])
def test_strides_and_leading_dimensions(tokens):
    import packed_linear as L

    p = Problem(200, 128, tokens, torch.bfloat16, adapters=2, rank=8)
    want = p.check()
    whole = torch.zeros(tokens, 3 * 128 + 8, dtype=torch.bfloat16, device="cuda")
    for first in (0, 8, 136, 129):  # rows of a wider tensor; the last off by two bytes
        p.x = whole[:, first:first + 128].copy_(p.x.clone())
        assert torch.equal(p.run(), want)
    p.x = p.x.t().contiguous().t()
    assert torch.equal(p.run(), want)
    p.x = p.x.contiguous().view(2, tokens // 2, 128)
    out = torch.empty(2, tokens // 2, 200, dtype=torch.bfloat16, device="cuda")
    assert p.run(out=out) is out and torch.equal(out.view(tokens, 200), want)
    padded = torch.randint(0, 256, (200, 96), device="cuda", dtype=torch.uint8)  # rows longer than their entries
    padded[:, :64] = p.codes
    assert torch.equal(L.packed_linear(p.x, padded, p.scale, p.zero, qmin=p.qmin, adapters=p.adapters, adapter_index=p.index), out)


@pytest.mark.parametrize("tokens", [2, 150])
def test_agrees_with_unpacked_codes(tokens):
    """What pack_codes stored, multiplied: the same matrix as unpack_codes gives back."""
    import packed_codes
    import packed_linear as L
    import quantizer_int

    gen = torch.Generator(device="cuda").manual_seed(3)
    w = 0.02 * torch.randn(300, 512, generator=gen, device="cuda")
    scale, zero = quantizer_int.int_abs_max_scale_triton(w, qmin=-8, qmax=7, dtype=torch.float16), torch.zeros(1, 1, device="cuda")
    codes = packed_codes.pack_codes(torch.clamp(torch.round(w / scale), -8, 7) * scale, scale, zero, qmin=-8, bits=4)
    x = torch.randn(tokens, 512, generator=gen, device="cuda").half()
    dense = packed_codes.unpack_codes(codes, scale, zero, qmin=-8, bits=4, n=512)
    want = x.double() @ dense.double().t()
    got = L.packed_linear(x, codes, scale, zero, qmin=-8).double()
    assert bool(((got - want).abs() <= 2.0 ** -11 * want.abs() + 48 * 2.0 ** -23 * (x.double().abs() @ (16 * scale.double().expand(300, 512)).t()) + 2.0 ** -24).all())


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("tokens", [5, 80])
def test_small_and_large_activations(tokens, dtype):
    p = Problem(130, 256, tokens, dtype, adapters=2, rank=8)
    p.x = (p.x.float() * torch.exp2(torch.linspace(-12, 6, tokens, device="cuda"))[:, None]).to(dtype)
    p.check()


@pytest.mark.parametrize("tokens", [5, 80])
def test_what_is_not_finite_stays_in_its_row(tokens):
    """An infinite activation or a NaN in a request's adapter reaches the results of that token, or of that adapter's tokens, alone."""
    p = Problem(130, 256, tokens, torch.float16, adapters=3, rank=8)
    p.index = (torch.arange(tokens, device="cuda") % 3).to(torch.int32)
    clean = p.check()
    p.x[1, 7] = float("inf")
    got = p.run()
    assert not got[1].isfinite().any() and torch.equal(got[2:], clean[2:]) and torch.equal(got[0], clean[0])
    p.x[1, 7] = 0
    clean = p.check()
    p.adapters.up[2, 5, 3] = float("nan")
    got = p.run()
    mine = p.index == 2
    assert got[mine, 5].isnan().all()
    got[mine, 5] = clean[mine, 5]
    assert torch.equal(got, clean)
    p.adapters.up[2, 5, 3] = 0
    p.adapters.down[2, 1, 1] = float("inf")
    got = p.run()
    assert not got[mine].isfinite().all(1).any() and torch.equal(got[~mine], clean[~mine])


@pytest.mark.parametrize("tokens", [3, 20, 200])
def test_streams_graphs_and_repeats(tokens):
    p = Problem(500, 1024, tokens, torch.bfloat16, adapters=5)
    out = p.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(p.run(), out)
    static = torch.empty_like(out)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph in graphs:
        with torch.cuda.graph(graph):
            p.run(out=static)
    p.x.copy_(p.x.flip(0))
    p.index.copy_(p.index.flip(0))
    for graph in graphs * 2:
        static.zero_()
        graph.replay()
        assert torch.equal(static, out.flip(0))


def test_empty():
    p = Problem(40, 64, 1, torch.float16, adapters=1)
    p.x, p.index = p.x[:0], p.index[:0]
    assert p.run().shape == (0, 40)
    p = Problem(40, 64, 3, torch.float16, adapters=2)
    p.index.fill_(-1)
    import packed_linear as L

    none = L.LowRankAdapters(p.adapters.down[:0], p.adapters.up[:0], None)
    assert torch.equal(p.run(), L.packed_linear(p.x, p.codes, p.scale, p.zero, qmin=-8, adapters=none, adapter_index=p.index))
