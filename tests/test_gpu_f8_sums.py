"""How the products of 8-bit floating point are summed: exactly, in FP32, unless a handle was told F8_SUMS_FAST.

Among every eight K-values two products are 2^14 and -2^14, the others below 2 and multiples of 2^-3.  All partial sums of a block, in
whatever order, are multiples of 2^-3 up to 16 2^14, which FP32 holds (21 bits), and scales are powers of two: the result is that of
FP64, rounded once to its type.  Sums that cut the eight products to multiples of 2^-13 of the largest lose the small ones."""
import pytest
import torch

from test_gpu_f8 import F8, OUTS, blocks, code, run, run_gated
from test_gpu_grouped import offsets_of, spans, type_code

pytestmark = pytest.mark.gpu

SIZES = [[1], [3, 0, 14], [40, 50, 0, 63], [130, 0, 257], [256, 300]]
SHAPES = [(256, 512), (128, 1280), (144, 400), (131, 333), (16, 128), (67, 40)]


def operands(seed, m, n, k, groups, op, f8, matrices=1):
    """(matrices as they are stored, scales, the same [groups, m, k] in FP64) of each, (tokens, scales, [n, k] in FP64)"""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def pick(values, *shape):
        return torch.tensor(values, device="cuda")[torch.randint(len(values), shape, generator=g, device="cuda")]
    large = torch.zeros(k, dtype=torch.bool, device="cuda")
    sign = torch.zeros(k, device="cuda")
    for at in range(0, k - 7, 8):  # (where among the eight: any places)
        two = torch.randperm(8, generator=g, device="cuda")[:2] + at
        large[two], sign[two[0]], sign[two[1]] = True, 1.0, -1.0
    x = torch.where(large, 64.0 * sign, pick([1.0, -1.0, 0.5, 1.25, -0.75], n, k))
    xs = 2.0 ** pick([-3.0, 0.0, 2.0], n, blocks(k))
    ws = []
    for _ in range(matrices):
        w = torch.where(large, 256.0, pick([1.0, 0.5, 1.5, -1.0], groups, m, k))
        s = 2.0 ** pick([-6.0, -5.0, -2.0], groups, blocks(m), blocks(k))
        wide = w.double() * s.double().repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :m, :k]
        stored, stored_s = (w, s) if op == "T" else (w.transpose(1, 2).contiguous(), s.transpose(1, 2).contiguous())
        ws.append((stored.to(F8["e4m3"]).view(torch.uint8).contiguous(), stored_s, wide))
    return ws, (x.to(F8[f8]).view(torch.uint8).contiguous(), xs, x.double() * xs.double().repeat_interleave(128, 1)[:, :k])


def product(cg, handle, op, m, k, sizes, f8, out):
    """(the library's, FP64's)"""
    n, groups = sum(sizes), len(sizes)
    ((w, ws, wide),), (x, xs, tokens) = operands(1, m, n, k, groups, op, f8)
    c = torch.full((n, m), 7.0, device="cuda", dtype=out)
    assert handle.gemm_f8(cg.OP_T if op == "T" else cg.OP_N, m, n, k, w, k if op == "T" else m, m * k, cg.R_8F_E4M3, ws, ws[0].numel(), x, k,
                          code(cg, f8), xs, c, m, type_code(cg, out), offsets_of(sizes), groups) == 0
    torch.cuda.synchronize()
    want = torch.zeros(n, m, device="cuda", dtype=torch.float64)
    for g, (lo, hi) in enumerate(spans(sizes)):
        want[lo:hi] = tokens[lo:hi] @ wide[g].t().contiguous()
    return c, want


def gated(cg, handle, m, k, sizes, f8, out):
    """(the library's, from FP64's projections: RELU and one product, in FP32)"""
    n, groups = sum(sizes), len(sizes)
    ((a, sa, wa), (b, sb, wb)), (x, xs, tokens) = operands(2, m, n, k, groups, "T", f8, 2)
    c = torch.full((n, m), 7.0, device="cuda", dtype=out)
    assert handle.gemm_gated_f8(cg.RELU, m, n, k, a, b, k, m * k, cg.R_8F_E4M3, sa, sb, sa[0].numel(), x, k, code(cg, f8), xs, c, m,
                                type_code(cg, out), offsets_of(sizes), groups) == 0
    torch.cuda.synchronize()
    g, u = (torch.zeros(n, m, device="cuda", dtype=torch.float64) for _ in range(2))
    for i, (lo, hi) in enumerate(spans(sizes)):
        g[lo:hi], u[lo:hi] = tokens[lo:hi] @ wa[i].t().contiguous(), tokens[lo:hi] @ wb[i].t().contiguous()
    return c, g.float().clamp(min=0) * u.float()


@pytest.mark.parametrize("cls", [None, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("f8", F8)
def test_sums_are_exact(cg, handle, f8, op, cls, monkeypatch):
    """Whichever kernel takes the call, and whatever the result's type."""
    if cls is not None:
        monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for i, (m, k) in enumerate(SHAPES):
        for j, sizes in enumerate(SIZES):
            out = OUTS[(i + j) % 3]
            got, want = product(cg, handle, op, m, k, sizes, f8, out)
            assert torch.equal(got, want.to(out)), (m, k, sizes, out)
            if op == "T":
                got, want = gated(cg, handle, m, k, sizes, f8, out)
                assert torch.equal(got, want.to(out)), ("gated", m, k, sizes, out)


def test_a_token_by_itself_and_among_others(cg, handle):
    """The same bits where the sums are exact."""
    for n in (1, 20, 60, 300):
        got, want = product(cg, handle, "T", 256, 512, [n], "e4m3", torch.bfloat16)
        assert torch.equal(got, want.to(torch.bfloat16))


@pytest.mark.parametrize("dtype", OUTS, ids=str)
def test_a_served_block(cg, handle, dtype):
    """F8GatedExperts against FP64 on the same FP8 values, the hidden ones rounded to the layer's type and quantised again as the layer
    does.  Projections off by 2^-21 of their size turn one hidden value in 2^18 by a step of E4M3, 2^-3 of it: 2^-12 of the result's
    norm, twice that allowed, beside the result's own rounding."""
    from cumpsgemm_amd import experts, gated as layers
    count, n, inner, f, m = 2, 1500, 768, 1024, 512
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(count, 2 * f, inner, generator=g, device="cuda") * inner ** -0.5
    v = torch.randn(count, m, f, generator=g, device="cuda") * f ** -0.5
    x = torch.randn(n, inner, generator=g, device="cuda").to(dtype)
    e = torch.randint(count, (n,), generator=g, device="cuda")
    before = handle.stream
    handle.set_stream(torch.cuda.current_stream())
    layer = layers.GatedExperts(handle, w.to(dtype), v.to(dtype)).to_f8()
    got = layer.forward(x, e).double()

    def values(q, s, rows):
        return q.float().double() * s.double().repeat_interleave(rows, -2).repeat_interleave(128, -1)[..., :q.shape[-2], :q.shape[-1]]
    tokens = values(*experts._tokens_to_f8(handle, x), 1)
    gate_up = values(layer.gate_up.view(2 * count, f, inner), layer.gate_up_scale.view(2 * count, *layer.gate_up_scale.shape[2:]), 128)
    down = values(layer.down, layer.down_scale, 128)
    h = torch.empty(n, f, device="cuda", dtype=dtype)
    for i in range(count):
        a, b = (tokens[e == i] @ p.t().contiguous() for p in (gate_up[2 * i], gate_up[2 * i + 1]))
        h[e == i] = (a * torch.sigmoid(a) * b).to(dtype)
    hidden = values(*experts._tokens_to_f8(handle, h), 1)
    want = torch.empty(n, m, device="cuda", dtype=torch.float64)
    for i in range(count):
        want[e == i] = hidden[e == i] @ down[i].t().contiguous()
    handle.set_stream(before)
    rounding, size = float((want.to(dtype).double() - want).norm()), float(want.norm())
    assert float((got - want).norm()) <= (rounding ** 2 + (2.0 ** -11 * size) ** 2) ** 0.5


@pytest.fixture
def fast(cg, handle):
    assert handle.set_f8_sums(cg.F8_SUMS_FAST) == 0
    yield handle
    assert handle.set_f8_sums(cg.F8_SUMS_FP32) == 0


@pytest.mark.parametrize("cls", [None, 0, 1, 2, 3, 4])
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("f8", F8)
def test_fast_sums(cg, fast, f8, op, cls, monkeypatch):
    """Within the bounds of sums that are cut (test_gpu_f8.py), in every tile."""
    if cls is not None:
        monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for m, k, sizes, out in ((512, 512, [300, 0, 257], torch.bfloat16), (272, 144, [9, 33], torch.float16), (128, 1280, [40, 200], torch.float32),
                             (71, 53, [40, 3], torch.bfloat16), (301, 1021, [130, 0, 257], torch.float32), (1, 1, [1], torch.bfloat16)):
        run(cg, fast, op, m, k, sizes, f8, out)
        if op == "T":
            run_gated(cg, fast, "SILU", m, k, sizes, f8, out)


def test_the_choice_is_the_handles(cg, fast, monkeypatch):
    """FAST cuts (in 128 x 128 tiles; a call of this size would be left to those of 32 tokens, which do not), from the call on that sets it
    to the one that ends it; gated blocks with results in FP32 and FP16 stay exact."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", "1")
    shape = ("T", 512, 512, [600, 700], "e4m3")
    got, want = product(cg, fast, *shape, torch.float32)
    assert not torch.equal(got, want.float())
    assert torch.equal(gated(cg, fast, *shape[1:], torch.float32)[0], gated(cg, fast, *shape[1:], torch.float32)[1])
    other = cg.Handle(stream=torch.cuda.current_stream())
    torch.cuda.synchronize()
    assert torch.equal(product(cg, other, *shape, torch.float32)[0], want.float())
    other.close()
    assert fast.set_f8_sums(cg.F8_SUMS_FP32) == 0
    assert torch.equal(product(cg, fast, *shape, torch.float32)[0], want.float())


def test_a_graph_keeps_the_sums_it_was_captured_with(cg, torch_gpu, monkeypatch):
    """Two graphs of one handle, one with each; replayed in turn after the setting has changed, with eager calls between them."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", "1")
    m, k, n = 256, 512, 300
    ((w, ws, wide),), (x, xs, tokens) = operands(5, m, n, k, 1, "T", "e4m3")
    want = (tokens @ wide[0].t().contiguous()).float()
    h, side = cg.Handle(), torch.cuda.Stream()
    h.set_stream(side)

    def call(c):
        assert h.gemm_f8(cg.OP_T, m, n, k, w, k, 0, cg.R_8F_E4M3, ws, 0, x, k, cg.R_8F_E4M3, xs, c, m, cg.R_32F) == 0
    graphs, eager = [], torch.empty(n, m, device="cuda")
    torch.cuda.synchronize()
    for sums in (cg.F8_SUMS_FAST, cg.F8_SUMS_FP32):
        assert h.set_f8_sums(sums) == 0
        with torch.cuda.stream(side):
            call(eager)
        torch.cuda.synchronize()
        graph, c = torch.cuda.CUDAGraph(), torch.empty(n, m, device="cuda")
        with torch.cuda.graph(graph, stream=side):
            call(c)
        graphs.append((graph, c, eager.clone()))
    assert torch.equal(graphs[1][2], want) and not torch.equal(graphs[0][2], want)
    for _ in range(3):
        for graph, c, result in graphs:
            c.fill_(7.0)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                call(eager)
            torch.cuda.synchronize()
            assert torch.equal(c, result) and torch.equal(eager, want)
    h.close()
