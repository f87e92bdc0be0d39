"""The layers of cumpsgemm_amd/experts.py on streams other than the handle's, inside a graph, and with small gradients."""
import pytest
import torch

from cumpsgemm_amd import experts
from test_gpu_grouped import check

pytestmark = pytest.mark.gpu

COUNT, OUT, INNER, TOKENS = 6, 136, 200, 300


def data(seed, dtype):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(TOKENS, INNER, generator=g, device="cuda").to(dtype), torch.randint(COUNT, (TOKENS,), generator=g, device="cuda"),
            torch.randn(TOKENS, OUT, generator=g, device="cuda").to(dtype))


def step(layer, served, x, e, dy):
    y, saved = layer.forward(x, e)
    return (y, *layer.backward(saved, dy), served.forward(x, e))


@pytest.fixture
def layers(cg, torch_gpu):
    h = cg.Handle(stream=torch.cuda.current_stream())

    def make(dtype):
        w = torch.randn(COUNT, OUT, INNER, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").to(dtype)
        layer = experts.Experts(h, w)
        return layer, layer.to_int8()
    yield h, make
    torch.cuda.synchronize()
    h.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_on_another_stream_than_the_handles(layers, dtype):
    """The tokens are written on that stream, behind other work; then the handle's own stream has the next step."""
    h, make = layers
    layer, served = make(dtype)
    x, e, dy = data(2, dtype)
    want = step(layer, served, x, e, dy)
    torch.cuda.synchronize()
    own, side, busy = h.stream, torch.cuda.Stream(), torch.randn(4096, 4096, device="cuda")
    late = [torch.full_like(x, float("nan")), torch.zeros_like(e), torch.full_like(dy, float("nan"))]
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            busy = busy @ busy * 2.0 ** -6
        for to, t in zip(late, (x, e, dy)):
            to.copy_(t)
        got = step(layer, served, *late)
        assert h.stream == own
    side.synchronize()
    again = step(layer, served, x, e, dy)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, again))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_in_a_graph(layers, dtype):
    """Captured on a stream that is not the handle's; replays take the tokens and experts of the time."""
    h, make = layers
    layer, served = make(dtype)
    buffers = data(3, dtype)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        step(layer, served, *buffers)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        got = step(layer, served, *buffers)
    for seed in (4, 5, 6, 4):
        for to, t in zip(buffers, data(seed, dtype)):
            to.copy_(t)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = step(layer, served, *buffers)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("scale", [1.0, 1e-6, 1e-9, 1e-20, 1e6])
def test_small_and_large_gradients_keep_their_digits(layers, scale):
    """Expert by expert, under the bounds of test_gpu_grouped.py, which go by the sizes of the sums."""
    layer, _ = layers[1](torch.float32)
    x, e, dy = data(7, torch.float32)
    dy = dy * scale
    dx, dw = layer.backward(layer.forward(x, e)[1], dy)
    for g in range(COUNT):
        xs, ds, w = x[e == g].double(), dy[e == g].double(), layer.weights[g].double()
        check(dx[e == g], ds @ w, ds.abs() @ w.abs(), "TF32TCEC", OUT, torch.float32)
        dst = ds.t().contiguous()
        check(dw[g], dst @ xs, dst.abs() @ xs.abs(), "TF32TCEC", len(xs), torch.float32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
def test_dropped_tokens_are_zeros_and_count_for_nothing(layers, dtype):
    """Numbers below 0 and beyond the last expert, their tokens NaN and infinities: as if those tokens were not there."""
    layer, served = layers[1](dtype)
    x, _, dy = data(8, dtype)
    e = torch.randint(-2, COUNT + 3, (TOKENS,), generator=torch.Generator(device="cuda").manual_seed(9), device="cuda")
    kept = (e >= 0) & (e < COUNT)
    served_alone = served.forward(x[kept], e[kept])
    x[~kept], dy[~kept] = float("nan"), float("inf")
    torch.full((64 << 20,), float("nan"), device="cuda")  # (what the results' memory held before)
    y, dx, dw, y8 = step(layer, served, x, e, dy)
    assert (y[~kept] == 0).all() and (dx[~kept] == 0).all() and (y8[~kept] == 0).all()
    assert torch.equal(y8[kept], served_alone)  # (sums of integers: any kernel's)
    forward, gradients = ("FP16TCEC", "TF32TCEC") if dtype == torch.float32 else ("f16", "f16") if dtype == torch.float16 else ("bf16", "bf16")
    for g in range(COUNT):
        xs, ds, w = x[e == g].double(), dy[e == g].double(), layer.weights[g].double()
        wt, dst = w.t().contiguous(), ds.t().contiguous()
        check(y[e == g], xs @ wt, xs.abs() @ wt.abs(), forward, INNER, dtype)
        check(dx[e == g], ds @ w, ds.abs() @ w.abs(), gradients, OUT, dtype)
        check(dw[g], dst @ xs, dst.abs() @ xs.abs(), gradients, len(xs), torch.float32)
