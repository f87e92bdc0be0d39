"""The layers of cumpsgemm_amd/gated.py and the FP8 layer of cumpsgemm_amd/experts.py on the CPU: in the handle's place stands one
that computes the products from the addresses, types and sizes that it is given, as the library does."""
import math

import pytest
import torch

import cumpsgemm_amd as cg
from cumpsgemm_amd import experts, gated
from test_experts_arguments import TYPES, CpuHandle, memory_in_use, refused, shapes_beside  # noqa: F401 (a fixture)

ACTS = [cg.SILU, cg.GELU, cg.GELU_TANH, cg.RELU]
STEP = {torch.float32: 2.0 ** -23, torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7}


def act_of(act, g):
    """act(g) and its derivative"""
    if act == cg.SILU:
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == cg.GELU:
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == cg.GELU_TANH:
        t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)
    return g.clamp(min=0), (g > 0).double()


class GatedHandle(CpuHandle):
    F8 = {cg.R_8F_E4M3: (torch.float8_e4m3fn, 448.0), cg.R_8F_E5M2: (torch.float8_e5m2, 57344.0)}

    def begin(self, name, mode=None):
        self.calls += 1
        self.streams.append(self.stream)
        self.modes.append((name, mode))

    def gemm_gated(self, op, act, m, n, k, gate, up, lda, stridea, b, ldb, c, ldc, z_gate=None, z_up=None, ldz=0, offsets=None, groups=1, mode=0, type=0):
        self.begin("gated", mode)
        if n == 0:
            return 0
        t = self.TYPES[type]
        rows, cols = (k, m) if op == cg.OP_N else (m, k)
        w = [self.memory(a, t, (groups, rows, cols), (stridea, lda, 1)).double() for a in (gate, up)]
        b, c = self.memory(b, t, (n, k), (ldb, 1)).double(), self.memory(c, t, (n, m), (ldc, 1))
        z = [self.memory(a, t, (n, m), (ldz, 1)) for a in (z_gate, z_up)] if z_gate is not None else None
        for g, lo, hi in self.spans(offsets, groups, n):
            p = [b[lo:hi] @ (a[g] if op == cg.OP_N else a[g].t()) for a in w]
            c[lo:hi] = (act_of(act, p[0])[0] * p[1]).to(t)
            if z is not None:
                z[0][lo:hi], z[1][lo:hi] = p[0].to(t), p[1].to(t)
        return 0

    def gemm_gated_backward(self, op, act, m, n, k, a, lda, stridea, b, ldb, z_gate, z_up, ldz, d_gate, d_up, ldd, c=None, ldc=0, offsets=None, groups=1,
                            mode=0, type=0):
        self.begin("backward", mode)
        if n == 0:
            return 0
        t = self.TYPES[type]
        rows, cols = (k, m) if op == cg.OP_N else (m, k)
        a, b = self.memory(a, t, (groups, rows, cols), (stridea, lda, 1)).double(), self.memory(b, t, (n, k), (ldb, 1)).double()
        z, d = ([self.memory(x, t, (n, m), (ld, 1)) for x in (u, v)] for u, v, ld in ((z_gate, z_up, ldz), (d_gate, d_up, ldd)))
        c = None if c is None else self.memory(c, t, (n, m), (ldc, 1))
        for g, lo, hi in self.spans(offsets, groups, n):
            x = b[lo:hi] @ (a[g] if op == cg.OP_N else a[g].t())
            gate, up = z[0][lo:hi].double(), z[1][lo:hi].double()
            y, slope = act_of(act, gate)
            d[0][lo:hi], d[1][lo:hi] = (x * up * slope).to(t), (x * y).to(t)
            if c is not None:
                c[lo:hi] = (y * up).to(t)
        return 0

    @staticmethod
    def wide(scale, rows, cols, block_rows):
        return scale.double().repeat_interleave(block_rows, -2).repeat_interleave(128, -1)[..., :rows, :cols]

    def quantize_f8(self, k, n, x, ldx, stridex, type_x, block_n, q, ldq, strideq, type_q, scale, batch=1):
        self.begin("quantize")
        dtype, most = self.F8[type_q]
        x = self.memory(x, self.TYPES[type_x], (batch, n, k), (stridex, ldx, 1)).double()
        q = self.memory(q, dtype, (batch, n, k), (strideq, ldq, 1))
        nb, kb = -(-n // block_n), -(-k // 128)
        scale = self.memory(scale, torch.float32, (batch, nb, kb), (nb * kb, kb, 1))
        full = torch.zeros(batch, nb * block_n, kb * 128, dtype=torch.float64)
        full[:, :n, :k] = x.abs()
        scale.copy_(full.view(batch, nb, block_n, kb, 128).amax((2, 4)) / most)
        q.copy_(torch.nan_to_num(x / self.wide(scale, n, k, block_n)).clamp(-most, most).float().to(dtype))
        return 0

    def values(self, a, type, scale, stride_scale, groups, rows, cols, stride, ld, block_rows):
        a = self.memory(a, self.F8[type][0], (groups, rows, cols), (stride, ld, 1)).float().double()
        rb, cb = -(-rows // block_rows), -(-cols // 128)
        return a * self.wide(self.memory(scale, torch.float32, (groups, rb, cb), (stride_scale, cb, 1)), rows, cols, block_rows)

    def gemm_f8(self, op, m, n, k, a, lda, stridea, type_a, scale_a, stridescale, b, ldb, type_b, scale_b, c, ldc, type_c=0, offsets=None, groups=1):
        self.begin("f8")
        rows, cols = (k, m) if op == cg.OP_N else (m, k)
        a = self.values(a, type_a, scale_a, stridescale, groups, rows, cols, stridea, lda, 128)
        b = self.values(b, type_b, scale_b, 0, 1, n, k, 0, ldb, 1)[0]
        c = self.memory(c, self.TYPES[type_c], (n, m), (ldc, 1))
        for g, lo, hi in self.spans(offsets, groups, n):
            c[lo:hi] = (b[lo:hi] @ (a[g] if op == cg.OP_N else a[g].t())).to(c.dtype)
        return 0

    def gemm_gated_f8(self, act, m, n, k, gate, up, lda, stridea, type_a, scale_gate, scale_up, stridescale, b, ldb, type_b, scale_b, c, ldc, type_c=0,
                      offsets=None, groups=1):
        self.begin("gated f8")
        w = [self.values(a, type_a, s, stridescale, groups, m, k, stridea, lda, 128) for a, s in ((gate, scale_gate), (up, scale_up))]
        b = self.values(b, type_b, scale_b, 0, 1, n, k, 0, ldb, 1)[0]
        c = self.memory(c, self.TYPES[type_c], (n, m), (ldc, 1))
        for g, lo, hi in self.spans(offsets, groups, n):
            p = [b[lo:hi] @ a[g].t() for a in w]
            c[lo:hi] = (act_of(act, p[0])[0] * p[1]).to(c.dtype)
        return 0


@pytest.fixture
def handle(monkeypatch):
    # (host memory takes the place of the GPU's)
    monkeypatch.setattr(experts, "_stream_of", lambda t: "torch's")
    return GatedHandle()


def layer_of(handle, dtype=torch.float32, shape=(3, 5, 6, 7), tokens=11, **how):
    """(layer, x, experts, dy); shape: experts, features out, features of the block, features in"""
    g = torch.Generator().manual_seed(1)
    count, out, f, inner = shape
    return (gated.GatedExperts(handle, torch.randn(count, 2 * f, inner, generator=g).to(dtype), torch.randn(count, out, f, generator=g).to(dtype), **how),
            torch.randn(tokens, inner, generator=g).to(dtype), torch.randint(count, (tokens,), generator=g), torch.randn(tokens, out, generator=g).to(dtype))


def near(got, want, dtype):
    """Each of up to four tensors on the way is rounded once, and what they are off by grows by less than their size, about ten
    features' products of a few units: 4 * 10 * 4 half steps."""
    return got.shape == want.shape and float((got.double() - want).abs().max()) <= 80 * STEP[dtype] * (1 + float(want.abs().max()))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_step_as_the_handle_sees_it(handle, dtype, act):
    layer, x, e, dy = layer_of(handle, dtype, activation=act)
    y, saved = layer.forward(x, e)
    got = (y, *layer.backward(saved, dy))
    want = gated.gated_reference(layer.gate_up, layer.down, x, e, dy, act)
    assert [t.dtype for t in got] == [dtype, dtype, torch.float32, torch.float32]
    assert all(near(a, b, dtype) for a, b in zip(got, want))


def test_gradients_are_added(handle):
    layer, x, e, dy = layer_of(handle)
    _, saved = layer.forward(x, e)
    _, a, b = layer.backward(saved, dy)
    da, db = torch.ones_like(a), torch.ones_like(b)
    _, ga, gb = layer.backward(saved, dy, da, db)
    assert ga is da and gb is db
    assert torch.allclose(da, 1 + a) and torch.allclose(db, 1 + b)
    for bad in (da.double(), da[:, :-1], da.transpose(1, 2), torch.zeros(3, 12, 14)[..., ::2]):
        assert refused(handle, layer.backward, saved, dy, bad)
    for bad in (db.half(), db[:2], torch.zeros(3, 6, 5).transpose(1, 2)):
        assert refused(handle, layer.backward, saved, dy, None, bad)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_serving_in_f8(handle, dtype):
    """As the handle sees it: off by the roundings to E4M3 of what went in (2^-4 each, three deep)."""
    for shape in ((3, 5, 6, 7), (2, 130, 140, 150)):
        layer, x, e, dy = layer_of(handle, dtype, shape)
        scaled = gated.GatedExperts(handle, layer.gate_up * shape[3] ** -0.5, layer.down * shape[2] ** -0.5)
        want = gated.gated_reference(scaled.gate_up, scaled.down, x, e, dy)[0]
        got = scaled.to_f8().forward(x, e)
        assert got.dtype == dtype and float((got.double() - want).norm()) <= 0.15 * float(want.norm())
        plain = experts.Experts(handle, layer.down * shape[2] ** -0.5)
        h = torch.randn(11, shape[2], generator=torch.Generator().manual_seed(3)).to(dtype)
        want = experts.reference(plain.weights, h, e, dy)[0]
        assert float((plain.to_f8().forward(h, e).double() - want).norm()) <= 0.08 * float(want.norm())


def test_types_and_shapes(handle):
    layer, x, e, dy = layer_of(handle)
    _, saved = layer.forward(x, e)
    served, plain = layer.to_f8(), experts.Experts(handle, layer.down).to_f8()
    for t in shapes_beside(x):
        assert refused(handle, layer.forward, t, e) and refused(handle, served.forward, t, e)
    for t in shapes_beside(dy):
        assert refused(handle, layer.backward, saved, t)
    for t in (e[:-1], torch.cat([e, e[:1]]), e[:, None]):
        assert refused(handle, layer.forward, x, t) and refused(handle, served.forward, x, t) and refused(handle, plain.forward, x[:, :6], t)
    for dtype in (torch.float16, torch.float64, torch.int8):
        assert refused(handle, layer.forward, x.to(dtype), e) and refused(handle, layer.backward, saved, dy.to(dtype))
        assert refused(handle, layer.backward, (saved[0].to(dtype), *saved[1:]), dy) and refused(handle, layer.backward, (saved[0], saved[1].to(dtype), *saved[2:]), dy)
    for dtype in (torch.float64, torch.int32):
        assert refused(handle, served.forward, x.to(dtype), e) and refused(handle, plain.forward, x[:, :6].to(dtype), e)
    assert refused(handle, layer.backward, (saved[0], saved[1][:, :-1], *saved[2:]), dy)
    assert refused(handle, layer.backward, (*saved[:3], saved[3].long()), dy) and refused(handle, layer.backward, (*saved[:2], saved[2].int(), saved[3]), dy)
    for i in range(4):
        assert refused(handle, layer.backward, tuple(t.to("meta") if i == j else t for j, t in enumerate(saved)), dy)
    assert refused(handle, layer.forward, x.to("meta"), e.to("meta")) and refused(handle, layer.backward, saved, dy.to("meta"))
    w, v = layer.gate_up, layer.down
    for bad in ((w[:, :-1], v), (w[0], v), (w, v[0]), (w, v[:2]), (w, v[..., :-1]), (w, v.half()), (w.double(), v.double()), (w, v.to("meta")),
                (w[:, :-2], v)):
        with pytest.raises(ValueError):
            gated.GatedExperts(handle, *bad)
    for act in (4, -1, "silu"):
        with pytest.raises(ValueError):
            gated.GatedExperts(handle, w, v, activation=act)
        with pytest.raises(ValueError):
            gated.F8GatedExperts(handle, served.gate_up, served.gate_up_scale, served.down, served.down_scale, activation=act)
    q, s, p, r = served.gate_up, served.gate_up_scale, served.down, served.down_scale
    for bad in ((q.float(), s, p, r), (q, s.double(), p, r), (q, s[:, :1], p, r), (q, s, p.float(), r), (q, s, p[..., :-1], r), (q, s, p, r[:2]),
                (q[:, :-1], s, p, r), (q, s, p.to("meta"), r), (q, s.to("meta"), p, r)):
        with pytest.raises(ValueError):
            gated.F8GatedExperts(handle, *bad)
    for bad in ((p.float(), r), (p, r.double()), (p, r[:2]), (p[0], r), (p, r.to("meta"))):
        with pytest.raises(ValueError):
            experts.F8Experts(handle, *bad)


def test_streams_modes_and_hosts(handle):
    layer, x, e, dy = layer_of(handle)
    layer.backward(layer.forward(x, e)[1], dy)
    assert handle.modes == [("gated", cg.FP16TCEC), ("columns", cg.FP16TCEC), ("backward", cg.TF32TCEC), ("columns", cg.TF32TCEC), ("over k", cg.TF32TCEC),
                            ("over k", cg.TF32TCEC)]
    layer.to_f8().forward(x, e)
    experts.Experts(handle, layer.down).to_f8().forward(x[:, :6], e)
    assert handle.streams == ["torch's"] * len(handle.streams) and handle.stream == "its own"
    handle.gemm_gated = lambda *args: cg.STATUS_INVALID_VALUE
    with pytest.raises(RuntimeError):
        layer.forward(x, e)
    assert handle.stream == "its own"


def test_weights_on_the_host():
    """(Without the fixture: the library would be given host memory's addresses.)"""
    handle = GatedHandle()
    layer, x, e, dy = layer_of(handle)
    saved = (x, torch.zeros(11, 12), torch.arange(11), torch.tensor([0, 11, 11, 11], dtype=torch.int32))
    for call in (lambda: layer.forward(x, e), lambda: layer.backward(saved, dy), layer.to_f8, experts.Experts(handle, layer.down).to_f8):
        assert refused(handle, call)


def test_layouts_and_no_tokens(handle):
    layer, x, e, dy = layer_of(handle)
    y, saved = layer.forward(x, e)
    want = (y, *layer.backward(saved, dy))
    w, v = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (layer.gate_up, layer.down))
    again = gated.GatedExperts(handle, w, v)
    y, saved = again.forward(torch.stack([x, x], 2)[..., 0], e.repeat_interleave(2)[::2])
    assert all(torch.equal(a, b) for a, b in zip((y, *again.backward(saved, dy.t().contiguous().t())), want))
    layer, x, e, dy = layer_of(handle, tokens=0)
    y, saved = layer.forward(x, e)
    dx, da, db = layer.backward(saved, dy)
    assert y.shape == dy.shape and dx.shape == x.shape and not da.any() and not db.any()
    assert layer.to_f8().forward(x, e).shape == y.shape


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("numbers", [[-1, 0, 3, 1, -5, 2, 2, 7, 0, 1, -1], [-1] * 11, [3] * 11], ids=str)
def test_tokens_of_no_expert(handle, memory_in_use, dtype, numbers):  # noqa: F811
    """Zeros for them, whatever they hold, and nothing of them in the matrices' gradients."""
    layer, x, _, dy = layer_of(handle, dtype)
    e = torch.tensor(numbers)
    kept = (e >= 0) & (e < 3)
    want = gated.gated_reference(layer.gate_up, layer.down, x[kept], e[kept], dy[kept])
    x[~kept], dy[~kept] = float("nan"), float("inf")
    y, saved = layer.forward(x, e)
    dx, da, db = layer.backward(saved, dy)
    assert near(da, want[2], dtype) and near(db, want[3], dtype) and not y[~kept].any() and not dx[~kept].any()
    if kept.any():
        assert near(y[kept], want[0], dtype) and near(dx[kept], want[1], dtype)
    for served in (layer.to_f8(), ):
        y8 = served.forward(x, e)
        assert not y8[~kept].any() and torch.isfinite(y8).all()
    y8 = experts.Experts(handle, layer.gate_up).to_f8().forward(x, e)
    assert not y8[~kept].any() and torch.isfinite(y8).all()
