"""What the layers of cumpsgemm_amd/experts.py refuse, and what they make of tokens, types and streams, on the CPU: in the
handle's place stands one that computes the products from the addresses, types and sizes that it is given, as the library does."""
import itertools

import pytest
import torch

import cumpsgemm_amd as cg
from cumpsgemm_amd import experts

TYPES = [torch.float32, torch.float16, torch.bfloat16]


class CpuHandle:
    """The library's calls on tensors in host memory.  Reading or writing past the end of one raises (as_strided does)."""
    TYPES = {cg.R_32F: torch.float32, cg.R_16F: torch.float16, cg.R_16BF: torch.bfloat16}

    def __init__(self):
        self.calls, self.modes, self.stream, self.streams = 0, [], "its own", []

    def set_stream(self, stream):
        self.stream = stream
        return 0

    @staticmethod
    def memory(t, dtype, shape, strides):
        """What lies at t's address, as `dtype`."""
        flat = torch.as_strided(t, (t.untyped_storage().nbytes() // t.element_size() - t.storage_offset(),), (1,)).view(dtype)
        return torch.as_strided(flat, shape, strides)

    @staticmethod
    def spans(offsets, groups, count):
        for g in range(groups):
            lo = min(max(int(offsets[g]), 0), count)
            yield g, lo, max(lo, min(int(offsets[g + 1]), count))

    def gemm_grouped(self, op, m, n, k, alpha, a, lda, stridea, b, ldb, beta, c, ldc, offsets, groups, mode, type_ab, type_c):
        self.calls += 1
        self.streams.append(self.stream)
        self.modes.append(("columns", mode))
        rows, cols = (k, m) if op == cg.OP_N else (m, k)
        a = self.memory(a, self.TYPES[type_ab], (groups, rows, cols), (stridea, lda, 1))
        b = self.memory(b, self.TYPES[type_ab], (n, k), (ldb, 1))
        c = self.memory(c, self.TYPES[type_c], (n, m), (ldc, 1))
        for g, lo, hi in self.spans(offsets, groups, n):
            y = alpha * (b[lo:hi].double() @ (a[g] if op == cg.OP_N else a[g].t()).double())
            c[lo:hi] = (y if beta == 0 else y + beta * c[lo:hi].double()).to(c.dtype)
        return 0

    def gemm_grouped_k(self, m, n, k, alpha, a, lda, b, ldb, beta, c, ldc, stridec, offsets, groups, mode, type_ab, type_c):
        self.calls += 1
        self.streams.append(self.stream)
        self.modes.append(("over k", mode))
        a = self.memory(a, self.TYPES[type_ab], (k, m), (lda, 1))
        b = self.memory(b, self.TYPES[type_ab], (k, n), (ldb, 1))
        c = self.memory(c, self.TYPES[type_c], (groups, n, m), (stridec, ldc, 1))
        for g, lo, hi in self.spans(offsets, groups, k):
            y = alpha * (b[lo:hi].t().double() @ a[lo:hi].double())
            c[g] = (y if beta == 0 else y + beta * c[g].double()).to(c.dtype)
        return 0

    def quantize_i8(self, k, n, x, ldx, type_x, q, ldq, scale):
        self.calls += 1
        self.streams.append(self.stream)
        x = self.memory(x, self.TYPES[type_x], (n, k), (ldx, 1)).double()
        q, scale = self.memory(q, torch.int8, (n, k), (ldq, 1)), self.memory(scale, torch.float32, (n,), (1,))
        scale.copy_(x.abs().amax(1) / 127 if k else 0)
        q.copy_(torch.round(torch.nan_to_num(x / scale[:, None])).clamp(-127, 127))
        return 0

    def gemm_i8(self, m, n, k, a, lda, stridea, scale_a, b, ldb, scale_b, c, ldc, type_c, offsets, groups):
        self.calls += 1
        self.streams.append(self.stream)
        a = self.memory(a, torch.int8, (groups, m, k), (stridea, lda, 1))
        b = self.memory(b, torch.int8, (n, k), (ldb, 1))
        scale_a = self.memory(scale_a, torch.float32, (groups, m), (m, 1))
        scale_b = self.memory(scale_b, torch.float32, (n,), (1,))
        c = self.memory(c, self.TYPES[type_c], (n, m), (ldc, 1))
        for g, lo, hi in self.spans(offsets, groups, n):
            y = b[lo:hi].double() @ a[g].t().double()
            c[lo:hi] = (y * scale_a[g].double() * scale_b[lo:hi, None].double()).to(c.dtype)
        return 0


@pytest.fixture
def handle(monkeypatch):
    # (host memory takes the place of the GPU's)
    monkeypatch.setattr(experts, "_stream_of", lambda t: "torch's", raising=False)
    return CpuHandle()


def layer_of(handle, dtype=torch.float32, shape=(3, 5, 7), tokens=11, **how):
    """(layer, x, experts, dy)"""
    g = torch.Generator().manual_seed(1)
    count, out, inner = shape
    return (experts.Experts(handle, torch.randn(*shape, generator=g).to(dtype), **how), torch.randn(tokens, inner, generator=g).to(dtype),
            torch.randint(count, (tokens,), generator=g), torch.randn(tokens, out, generator=g).to(dtype))


def int8_layer(handle, shape=(3, 5, 7)):
    g = torch.Generator().manual_seed(2)
    return experts.Int8Experts(handle, torch.randint(-127, 128, shape, generator=g).to(torch.int8), torch.rand(shape[:2], generator=g))


def close(got, want, dtype):
    # (one rounding of the result: the products here are computed in 64 bits)
    bound = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}[dtype]
    return got.shape == want.shape and bool(((got.double() - want).abs() <= bound * want.abs().clamp(min=2.0 ** -14)).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_step_as_the_handle_sees_it(handle, dtype):
    layer, x, e, dy = layer_of(handle, dtype)
    y, saved = layer.forward(x, e)
    dx, dw = layer.backward(saved, dy)
    want = experts.reference(layer.weights, x, e, dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == torch.float32
    assert close(y, want[0], dtype) and close(dx, want[1], dtype) and close(dw, want[2], torch.float32)


def refused(handle, call, *args, **kwargs):
    """ValueError, and nothing was launched."""
    before = handle.calls
    with pytest.raises(ValueError):
        call(*args, **kwargs)
    return handle.calls == before


@pytest.mark.parametrize("weights,tokens", [p for p in itertools.product(TYPES + [torch.float64], repeat=2) if p[0] != p[1]], ids=str)
def test_types_that_differ(handle, weights, tokens):
    """One type goes to the library for all operands: FP32 tokens would have 16-bit weights read past their end."""
    if weights == torch.float64:
        with pytest.raises(ValueError):
            layer_of(handle, weights)
        return
    layer, x, e, dy = layer_of(handle, weights)
    _, saved = layer.forward(x, e)
    assert refused(handle, layer.forward, x.to(tokens), e)
    assert refused(handle, layer.backward, saved, dy.to(tokens))
    assert refused(handle, layer.backward, (saved[0].to(tokens), *saved[1:]), dy)


def test_types_of_the_layer_in_8_bits(handle):
    layer, x, e, _ = layer_of(handle)
    q = int8_layer(handle)
    for weights, scale in ((q.weights.to(torch.uint8), q.scale), (q.weights.float(), q.scale), (q.weights, q.scale.double()), (q.weights, q.scale.half())):
        with pytest.raises(ValueError):
            experts.Int8Experts(handle, weights, scale)
    for dtype in (torch.float64, torch.int8, torch.int32):
        assert refused(handle, q.forward, x.to(dtype), e)


def shapes_beside(t):
    """t with one feature, one row fewer and one more, transposed, in one dimension and in three."""
    rows, cols = t.shape
    return [t[:, :-1], torch.cat([t, t[:, :1]], 1), t[:-1], torch.cat([t, t[:1]]), t.t(), t[0], t.reshape(rows, cols, 1), t[:, :0]]


def test_shapes_that_do_not_belong_together(handle):
    """Tokens with fewer features than the weights would be read past their end, and so on."""
    layer, x, e, dy = layer_of(handle)
    _, saved = layer.forward(x, e)
    for t in shapes_beside(x):
        assert refused(handle, layer.forward, t, e)
        assert refused(handle, int8_layer(handle).forward, t, e)
        if t.dim() != 2 or t.shape[1] != x.shape[1]:
            assert refused(handle, layer.backward, (t, *saved[1:]), dy)
    for t in shapes_beside(dy):
        assert refused(handle, layer.backward, saved, t)
    for t in (e[:-1], torch.cat([e, e[:1]]), e[:, None], e[:0]):
        assert refused(handle, layer.forward, x, t)
        assert refused(handle, int8_layer(handle).forward, x, t)
    # what another layer's forward saved
    for shape in ((4, 5, 7), (2, 5, 7), (3, 5, 8)):
        other, ox, oe, _ = layer_of(handle, shape=shape)
        assert refused(handle, layer.backward, other.forward(ox, oe)[1], dy)


def test_shapes_of_weights(handle):
    q = int8_layer(handle)
    for w in (torch.zeros(5, 7), torch.zeros(3, 5, 7, 1), torch.zeros(7)):
        for make in (lambda: experts.Experts(handle, w), lambda: experts.Int8Experts(handle, w.to(torch.int8), q.scale)):
            with pytest.raises(ValueError):
                make()
    for scale in (q.scale[:2], q.scale[:, :4], q.scale.t(), q.scale.reshape(-1), torch.rand(3, 5, 1)):
        with pytest.raises(ValueError):
            experts.Int8Experts(handle, q.weights, scale)


def test_no_tokens(handle):
    layer, x, e, dy = layer_of(handle, tokens=0)
    y, saved = layer.forward(x, e)
    dx, dw = layer.backward(saved, dy)
    assert y.shape == dy.shape and dx.shape == x.shape and (dw == 0).all()


def test_layouts(handle):
    """Views: transposed, every other row or column, broadcast."""
    layer, x, e, dy = layer_of(handle)
    q = int8_layer(handle)
    y, saved = layer.forward(x, e)
    dx, dw = layer.backward(saved, dy)
    y8 = q.forward(x, e)

    def views(t):
        wide = torch.zeros(*t.shape[:-1], 2 * t.shape[-1], dtype=t.dtype)
        wide[..., ::2] = t
        yield wide[..., ::2]
        yield t.transpose(-1, -2).contiguous().transpose(-1, -2)
        yield torch.cat([torch.zeros_like(t), t])[len(t):]

    for w, w8, s8, vx, ve, vdy in zip(views(layer.weights), views(q.weights), views(q.scale), views(x), [e.repeat_interleave(2)[::2]] * 3, views(dy)):
        again = experts.Experts(handle, w)
        vy, vsaved = again.forward(vx, ve)
        assert torch.equal(vy, y) and all(torch.equal(a, b) for a, b in zip(again.backward(vsaved, vdy), (dx, dw)))
        assert torch.equal(experts.Int8Experts(handle, w8, s8).forward(vx, ve), y8)
    one = x[:1].expand(11, 7)
    assert torch.equal(layer.forward(one, e)[0], layer.forward(one.clone(), e)[0])
    assert torch.equal(layer.backward(saved, dy[:1].expand(11, 5))[0], layer.backward(saved, dy[:1].repeat(11, 1))[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_dw_is_fp32_contiguous_and_as_large_as_the_weights(handle, dtype):
    """It is written as such: a 16-bit one, as the grad of 16-bit weights is, was written past its end."""
    layer, x, e, dy = layer_of(handle, dtype)
    _, saved = layer.forward(x, e)
    _, once = layer.backward(saved, dy)
    for dw in ([torch.zeros(3, 5, 7, dtype=t) for t in (torch.float16, torch.bfloat16, torch.float64)] +
               [torch.zeros(3, 5, 6), torch.zeros(2, 5, 7), torch.zeros(3, 7, 5), torch.zeros(15, 7), torch.zeros(3, 5, 7, 1),
                torch.zeros(3, 7, 5).transpose(1, 2), torch.zeros(3, 5, 14)[..., ::2], torch.zeros(1, 5, 7).expand(3, 5, 7)]):
        assert refused(handle, layer.backward, saved, dy, dw)
        assert (dw == 0).all()
    dw = torch.ones(3, 5, 7)
    assert layer.backward(saved, dy, dw)[1] is dw and close(dw, 1 + experts.reference(layer.weights, x, e, dy)[2], torch.float32)
    layer.backward(saved, dy, torch.cat([dw, dw])[3:])  # (behind other tensors' gradients)


def test_every_call_is_on_torchs_stream(handle):
    """... and the handle on its own again, whatever happens in between."""
    layer, x, e, dy = layer_of(handle)
    _, saved = layer.forward(x, e)
    layer.backward(saved, dy)
    layer.to_int8().forward(x, e)
    assert handle.streams == ["torch's"] * 6 and handle.stream == "its own"
    handle.gemm_grouped = lambda *args: cg.STATUS_INVALID_VALUE
    with pytest.raises(RuntimeError):
        layer.forward(x, e)
    assert handle.stream == "its own"


def test_weights_on_the_host():
    """(Without the fixture: the library would be given host memory's addresses.)"""
    handle = CpuHandle()
    layer, x, e, dy = layer_of(handle)
    saved = (x, torch.arange(11), torch.tensor([0, 11, 11, 11], dtype=torch.int32))
    for call in (lambda: layer.forward(x, e), lambda: layer.backward(saved, dy), layer.to_int8, lambda: int8_layer(handle).forward(x, e)):
        assert refused(handle, call)


def test_the_handle_knows_its_stream(cg):
    class Stream:
        cuda_stream = 4096
    h = cg.Handle.__new__(cg.Handle)
    h._h = None  # (no handle: the library refuses the call)
    h._L = cg.lib()
    assert h.stream == 0
    for stream, want in ((Stream(), 4096), (8192, 8192), (None, 0), (0, 0)):
        h.set_stream(stream)
        assert h.stream == want


def test_tensors_on_two_devices(handle):
    """(torch itself indexes one device's tensor by another's, and the offsets would be host memory.)"""
    layer, x, e, dy = layer_of(handle)
    q = int8_layer(handle)
    _, saved = layer.forward(x, e)
    for t in ((x.to("meta"), e), (x, e.to("meta")), (x.to("meta"), e.to("meta"))):
        assert refused(handle, layer.forward, *t)
        assert refused(handle, q.forward, *t)
    assert refused(handle, layer.backward, saved, dy.to("meta"))
    assert refused(handle, layer.backward, saved, dy, torch.zeros(3, 5, 7, device="meta"))
    for i in range(3):
        assert refused(handle, layer.backward, tuple(t.to("meta") if i == j else t for j, t in enumerate(saved)), dy)
    with pytest.raises(ValueError):
        experts.Int8Experts(handle, q.weights, q.scale.to("meta"))
    with pytest.raises(ValueError):
        experts.Int8Experts(handle, q.weights.to("meta"), q.scale)


def test_what_forward_saved_holds_the_types_that_the_library_reads(handle):
    layer, x, e, dy = layer_of(handle)
    grouped, order, offsets = layer.forward(x, e)[1]
    assert refused(handle, layer.backward, (grouped, order, offsets.long()), dy)
    assert refused(handle, layer.backward, (grouped, order.bool(), offsets), dy)


@pytest.fixture
def memory_in_use():
    """torch.empty gives NaN (and the largest integers) instead of whatever lies there."""
    before = torch.utils.deterministic.fill_uninitialized_memory, torch.are_deterministic_algorithms_enabled()
    torch.utils.deterministic.fill_uninitialized_memory = True
    torch.use_deterministic_algorithms(True)
    assert torch.isnan(torch.empty(3)).all()
    yield
    torch.utils.deterministic.fill_uninitialized_memory = before[0]
    torch.use_deterministic_algorithms(before[1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("numbers", [[-1, 0, 3, 1, -5, 2, 2, 7, 0, 1, -1], [-1] * 11, [3] * 11, [-1, 1 << 40, -(1 << 40), 0, 0, 0, 0, 0, 0, 0, 2]], ids=str)
def test_tokens_of_no_expert(handle, memory_in_use, dtype, numbers):
    """Zeros for them, whatever they hold, and nothing of them in the weights' gradient."""
    layer, x, _, dy = layer_of(handle, dtype)
    e = torch.tensor(numbers)
    kept = (e >= 0) & (e < 3)
    want = experts.reference(layer.weights, x[kept], e[kept], dy[kept])
    x[~kept], dy[~kept] = float("nan"), float("inf")
    y, saved = layer.forward(x, e)
    dx, dw = layer.backward(saved, dy)
    assert close(y[kept], want[0], dtype) and close(dx[kept], want[1], dtype) and close(dw, want[2], torch.float32)
    assert (y[~kept] == 0).all() and (dx[~kept] == 0).all()
    y8 = layer.to_int8().forward(x, e)
    assert (y8[~kept] == 0).all() and torch.isfinite(y8).all()


@pytest.mark.parametrize("count", [2, 127, 128, 129, 255, 256, 300, 40000])
@pytest.mark.parametrize("dtype", [torch.bool, torch.uint8, torch.int8, torch.int16, torch.int32, torch.int64], ids=str)
def test_expert_numbers_of_any_integer_type(dtype, count):
    """As many experts as the numbers' type holds, and more: `count` itself is beyond it then."""
    most = min(count, 2 if dtype == torch.bool else torch.iinfo(dtype).max + 1)
    e = torch.randint(most, (200,), generator=torch.Generator().manual_seed(count))
    e[:2] = torch.tensor([0, most - 1])
    order, offsets = experts.group_by_expert(e.to(dtype), count)
    want = torch.cat([torch.zeros(1, dtype=torch.int64), torch.bincount(e, minlength=count).cumsum(0)])
    assert torch.equal(order, torch.argsort(e, stable=True)) and torch.equal(offsets, want.to(torch.int32))


def test_modes(handle):
    """The gradients' operands keep FP32's range unless another mode is asked for."""
    layer, x, e, dy = layer_of(handle)
    layer.backward(layer.forward(x, e)[1], dy)
    assert handle.modes == [("columns", cg.FP16TCEC), ("columns", cg.TF32TCEC), ("over k", cg.TF32TCEC)]
    layer, *_ = layer_of(handle, mode=cg.TF32TC, gradient_mode=cg.FP16TC)
    layer.backward(layer.forward(x, e)[1], dy)
    assert handle.modes[3:] == [("columns", cg.TF32TC), ("columns", cg.FP16TC), ("over k", cg.FP16TC)]
