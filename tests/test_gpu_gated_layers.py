"""The layers of cumpsgemm_amd/gated.py and the FP8 layer of cumpsgemm_amd/experts.py on the GPU: whole steps, streams other than
the handle's, graphs, dropped tokens, sizes beyond 32 bits."""
import pytest
import torch

from cumpsgemm_amd import experts, gated

pytestmark = pytest.mark.gpu

COUNT, OUT, F, INNER, TOKENS = 6, 136, 144, 200, 300


def data(seed, dtype, tokens=TOKENS):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(tokens, INNER, generator=g, device="cuda").to(dtype), torch.randint(COUNT, (tokens,), generator=g, device="cuda"),
            torch.randn(tokens, OUT, generator=g, device="cuda").to(dtype))


def step(layer, served, plain, x, e, dy):
    y, saved = layer.forward(x, e)
    return (y, *layer.backward(saved, dy), served.forward(x, e), plain.forward(x, e))


@pytest.fixture
def layers(cg, torch_gpu):
    h = cg.Handle(stream=torch.cuda.current_stream())

    def make(dtype, act=cg.SILU):
        g = torch.Generator(device="cuda").manual_seed(1)
        w = torch.randn(COUNT, 2 * F, INNER, generator=g, device="cuda") * INNER ** -0.5
        v = torch.randn(COUNT, OUT, F, generator=g, device="cuda") * F ** -0.5
        layer = gated.GatedExperts(h, w.to(dtype), v.to(dtype), activation=act)
        return layer, layer.to_f8(), experts.Experts(h, w.to(dtype)).to_f8()
    yield h, make
    torch.cuda.synchronize()
    h.close()


def relative(got, want):
    return float((got.double() - want).norm() / want.norm())


@pytest.mark.parametrize("act", ["SILU", "GELU", "GELU_TANH", "RELU"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_a_step(cg, layers, dtype, act):
    """Roundings are independent: in FP32 2^-21 of a product's size and 2^-23 sqrt(K) of the sums', in 16 bits up to four roundings of
    half a step on the way.  FP8: three roundings to 2^-4 / sqrt(3) of a value, or less."""
    layer, served, plain = layers[1](dtype, getattr(cg, act))
    x, e, dy = data(2, dtype)
    got = step(layer, served, plain, x, e, dy)
    want = gated.gated_reference(layer.gate_up, layer.down, x, e, dy, getattr(cg, act))
    bar = {torch.float32: 2 * (2.0 ** -21 + 2.0 ** -23 * TOKENS ** 0.5), torch.float16: 4 * 2.0 ** -11, torch.bfloat16: 4 * 2.0 ** -8}[dtype]
    for name, a, b in zip(("y", "dx", "d_gate_up", "d_down"), got, want):
        assert relative(a, b) <= bar, (name, relative(a, b))
    assert relative(got[4], want[0]) <= 0.1
    dz = torch.zeros(TOKENS, 2 * F, device="cuda")
    assert relative(got[5], experts.reference(layer.gate_up, x, e, dz)[0]) <= 0.05


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_on_another_stream_than_the_handles(layers, dtype):
    """The tokens are written on that stream, behind other work; then the handle's own stream has the next step."""
    h, make = layers
    all_of_them = make(dtype)
    x, e, dy = data(2, dtype)
    want = step(*all_of_them, x, e, dy)
    torch.cuda.synchronize()
    own, side, busy = h.stream, torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    late = [torch.full_like(x, float("nan")), torch.zeros_like(e), torch.full_like(dy, float("nan"))]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            busy = busy @ busy * 2.0 ** -6
        for to, t in zip(late, (x, e, dy)):
            to.copy_(t)
        got = step(*all_of_them, *late)
        assert h.stream == own
    side.synchronize()
    again = step(*all_of_them, x, e, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("tokens", [3, TOKENS])
def test_in_a_graph(layers, dtype, tokens):
    """Two graphs of one handle, captured on a stream that is not the handle's; replays in turn take the tokens and experts of the
    time, with eager steps between them."""
    h, make = layers
    all_of_them = make(dtype)
    side = torch.cuda.Stream()
    graphs = []
    for seed in (3, 13):
        buffers = data(seed, dtype, tokens)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            step(*all_of_them, *buffers)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = step(*all_of_them, *buffers)
        graphs.append((graph, buffers, got))
    for seed in (4, 5, 6, 4):
        for graph, buffers, got in graphs:
            for to, t in zip(buffers, data(seed, dtype, tokens)):
                to.copy_(t)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want = step(*all_of_them, *buffers)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_dropped_tokens_are_zeros_and_count_for_nothing(layers, dtype):
    """Numbers below 0 and beyond the last expert, their tokens NaN and infinities: as if those tokens were not there, in memory that
    held NaN before."""
    all_of_them = layers[1](dtype)
    x, _, dy = data(8, dtype)
    e = torch.randint(-2, COUNT + 3, (TOKENS,), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    kept = (e >= 0) & (e < COUNT)
    alone = step(*all_of_them, x[kept], e[kept], dy[kept])
    x[~kept], dy[~kept] = float("nan"), float("inf")
    torch.full((64 << 20,), float("nan"), device="cuda")  # (what the results' memory held before)
    got = step(*all_of_them, x, e, dy)
    for i in (0, 1, 4, 5):
        assert not got[i][~kept].any()
        assert relative(got[i][kept], alone[i].double()) <= 2.0 ** -6  # (another number of tokens may take other tiles)
    for i in (2, 3):
        assert relative(got[i], alone[i].double()) <= 2.0 ** -6


def test_gradients_against_differences(layers):
    """The step's gradients along a random direction against central differences of sum(y dy), in FP32: results of about 200 products
    are off by 2^-20 of their size; the step of 2^-7 leaves its square times a third derivative, below one half for SiLU of inputs
    whose projections change by about one."""
    layer, *_ = layers[1](torch.float32)
    x, e, dy = data(5, torch.float32)
    _, saved = layer.forward(x, e)
    dx, da, db = layer.backward(saved, dy)
    g = torch.Generator(device="cuda").manual_seed(6)
    for which, grad in enumerate((dx, da, db)):
        move = torch.randn(grad.shape, generator=g, device="cuda") * (1.0 if which == 0 else 0.07)
        step = 2.0 ** -7

        def loss(sign):
            args = [x, layer.gate_up, layer.down]
            args[which] = args[which] + sign * step * move
            other = gated.GatedExperts(layer.handle, args[1], args[2])
            return (other.forward(args[0], e)[0].double() * dy.double())
        terms = (loss(1) - loss(-1)) / (2 * step)
        want, got = float(terms.sum()), float((grad.double() * move.double()).sum())
        size = float(loss(0).abs().sum())
        assert abs(got - want) <= step ** 2 * float(terms.abs().sum()) + 2.0 ** -20 * size / step, (which, got, want)


def test_the_command(torch_gpu):
    """In FP32 2^-21 of a product's size and 2^-23 sqrt(K) of the sums', a few of each on the way; in BF16 up to four roundings."""
    for shape in ((1000, 512, 768, 8), (37, 100, 33, 5), (3, 256, 64, 16)):
        errors = gated.main(shape)
        for name, e in errors.items():
            bar = 0.1 if name.startswith("8-bit") else 4 * 2.0 ** -8 if name.startswith("BF16") else 2 * (2.0 ** -21 + 2.0 ** -23 * max(shape) ** 0.5)
            assert 0 <= e <= bar, (name, e, bar)
        assert len(errors) == 9


def test_offsets_past_32_bits(cg, handle):
    """Tokens and gradients whose elements lie beyond 2^32 bytes and 2^31 elements from the first."""
    n, m, k = 70000, 128, 128
    ld = 33000  # 70000 * 33000 = 2.3e9 elements
    w = torch.randn(2, m, k, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(torch.bfloat16) * k ** -0.5
    x = torch.empty(n * ld, device="cuda", dtype=torch.bfloat16)
    xv = torch.as_strided(x, (n, k), (ld, 1))
    xv.copy_(torch.randn(n, k, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda"))
    y = torch.full((n * ld,), 7.0, device="cuda", dtype=torch.bfloat16)
    yv = [torch.as_strided(y, (n, m), (ld, 1), at) for at in (0, 512, 1024)]
    off = torch.tensor([0, 100, n], dtype=torch.int32, device="cuda")
    assert handle.gemm_gated(cg.OP_T, cg.SILU, m, n, k, w, w, k, m * k, x, ld, yv[0], ld, yv[1], yv[2], ld, off, 2, cg.FP16TC, cg.R_16BF) == 0
    rows = torch.tensor([0, 99, 100, 40000, 65100, n - 1], device="cuda")
    group = (rows >= 100).long()
    g = torch.stack([w[a].double() @ xv[r].double() for a, r in zip(group, rows)])
    for v, want in zip(yv, (g * torch.sigmoid(g) * g, g, g)):
        # (a rounding to 2^-8 of up to 30, and 2^-24 K S of the sums)
        assert float((v[rows].double() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
    d = [torch.as_strided(y, (n, m), (ld, 1), at) for at in (2048, 2560)]
    assert handle.gemm_gated_backward(cg.OP_N, cg.SILU, k, n, m, w, k, m * k, x, ld, yv[1], yv[2], ld, d[0], d[1], ld, None, 0, off, 2, cg.FP16TC,
                                      cg.R_16BF) == 0
    dh = torch.stack([xv[r].double() @ w[a].double() for a, r in zip(group, rows)])
    z = yv[1][rows].double()
    s = torch.sigmoid(z)
    for v, want in zip(d, (dh * z * s * (1 + z * (1 - s)), dh * z * s)):
        assert float((v[rows].double() - want).abs().max()) <= 2.0 ** -7 * float(want.abs().max())
    assert float(y[200]) == 7.0 and float(y[700]) == 7.0 and float(y[-1]) == 7.0
    # FP8: 2^32 bytes
    q = torch.empty(n * 2 * ld, device="cuda", dtype=torch.uint8)
    s = torch.empty(n, 1, device="cuda")
    assert handle.quantize_f8(k, n, x, ld, 0, cg.R_16BF, 1, q, 2 * ld, 0, cg.R_8F_E4M3, s) == 0
    wq, ws = torch.empty(2, m, k, device="cuda", dtype=torch.uint8), torch.empty(2, 1, 1, device="cuda")
    assert handle.quantize_f8(k, m, w, k, m * k, cg.R_16BF, 128, wq, k, m * k, cg.R_8F_E4M3, ws, 2) == 0
    assert handle.gemm_f8(cg.OP_T, m, n, k, wq, k, m * k, cg.R_8F_E4M3, ws, 1, q, 2 * ld, cg.R_8F_E4M3, s, yv[0], ld, cg.R_16BF, off, 2) == 0
    # (E4M3's roundings, 2^-4 of each value at most, are independent over 128 products)
    assert float((yv[0][rows].double() - g).norm() / g.norm()) <= 0.08


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("cls", ["1", "3"])
def test_leading_dimensions_beyond_32_bits_of_a_tile(cg, handle, op, cls, monkeypatch):
    """FP32 and FP8 matrices whose tiles span more bytes than the kernels' 32-bit offsets reach."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", cls)
    g = torch.Generator(device="cuda").manual_seed(1)
    m, k, n = (40, 48, 20) if op == "T" else (48, 40, 20)
    rows, cols = (m, k) if op == "T" else (k, m)
    ld = (1 << 21) + 64 if op == "T" else (1 << 23) + 64  # a step's rows: 256 of K-contiguous ones, 64 lines else
    buf = torch.empty(2 * rows * ld, device="cuda")
    w = torch.as_strided(buf, (2, rows, cols), (rows * ld, ld, 1))
    w.copy_(torch.randn(2, rows, cols, generator=g, device="cuda") * k ** -0.5)
    x = torch.randn(n, k, generator=g, device="cuda")
    y, z = torch.empty(n, m, device="cuda"), torch.empty(2, n, m, device="cuda")
    o = cg.OP_T if op == "T" else cg.OP_N
    assert handle.gemm_gated(o, cg.SILU, m, n, k, buf, w[1], ld, 0, x, k, y, m, z[0], z[1], m, None, 1, cg.TF32TCEC, cg.R_32F) == 0
    wide = w.double() if op == "T" else w.double().transpose(1, 2)
    a, b = (x.double() @ t.t().contiguous() for t in wide)
    for got, want in ((z[0], a), (z[1], b), (y, a * torch.sigmoid(a) * b)):
        assert relative(got, want) <= 2.0 ** -20
    d = torch.empty(2, n, m, device="cuda")
    assert handle.gemm_gated_backward(o, cg.SILU, m, n, k, buf, ld, 0, x, k, z[0], z[1], m, d[0], d[1], m, None, 0, None, 1, cg.TF32TCEC, cg.R_32F) == 0
    s = torch.sigmoid(z[0].double())
    assert relative(d[1], a * z[0].double() * s) <= 2.0 ** -20
    del buf, w
    ld8 = (1 << 23) + 64 if op == "T" else (1 << 24) + 64
    q = torch.empty(rows * ld8, device="cuda", dtype=torch.uint8)
    v = torch.as_strided(q, (rows, cols), (ld8, 1))
    v.copy_(torch.randn(rows, cols, generator=g, device="cuda").to(torch.float8_e4m3fn).view(torch.uint8))
    xq = x.to(torch.float8_e4m3fn)
    ws, xs = torch.ones(1, device="cuda"), torch.ones(n, device="cuda")
    assert handle.gemm_f8(o, m, n, k, q, ld8, 0, cg.R_8F_E4M3, ws, 0, xq, k, cg.R_8F_E4M3, xs, y, m, cg.R_32F) == 0
    wide = v.contiguous().view(torch.float8_e4m3fn).float().double()
    want = xq.float().double() @ (wide.t().contiguous() if op == "T" else wide)
    assert relative(y, want) <= 2.0 ** -13
