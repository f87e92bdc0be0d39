"""Gated blocks and their gradients (gemm_gated, gemm_gated_backward) against the formulas in FP64.

Bounds, by element.  A sum G of K products with S = sum |a| |b| is off by eG = (split + (K + 2) 2^-24) S (test_gpu_grouped.py).
act has slopes of at most 1.13, so act(G) U is off by 1.13 eG |U| + |act(G)| eU, by eG eU, and by what act itself is off: its
factor s or P, at most 1, by the roundings of its argument, of the exponential, the sum and the quotient, 2^-21 together (the
largest y s(1 - s) and y P' are below a quarter and a half, and the argument has at most four roundings of 2^-24), hence
|x| 2^-21.  Of the slope, s + x s(1 - s) y', the second part is off by |x y'| 2^-21, y' <= 1.6 + 0.22 x^2: in all at most
2^-20 (1 + |x|)^3.  A result is rounded once, to half a step of its type."""
import itertools
import math

import pytest
import torch

from test_gpu_grouped import KINDS, ROUND, SPLIT, dtype_of, mode_of, offsets_of, randn, spans, type_code

pytestmark = pytest.mark.gpu

ACTS = ["SILU", "GELU", "GELU_TANH", "RELU"]


def act_of(act, g):
    """act(g) and its derivative in FP64"""
    if act == "SILU":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    if act == "GELU":
        p = torch.special.ndtr(g)
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "GELU_TANH":
        t = torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * math.sqrt(2 / math.pi) * (1 + 0.134145 * g * g)
    return g.clamp(min=0), (g > 0).double()


def filled(n, ld, cols, dtype, values=None, fill=float("nan")):
    """(buffer of n rows of ld, view of its first `cols` columns)"""
    buf = torch.full((n * ld + 8,), fill, device="cuda", dtype=dtype)
    view = torch.as_strided(buf, (n, cols), (ld, 1))
    if values is not None:
        view.copy_(values)
    return buf, view


def untouched(buf, view, n, fill):
    """Nothing but the first n rows of the view was written."""
    view[:n] = fill
    return bool((buf == fill).all()) if fill == fill else bool(torch.isnan(buf).all())


def near(name, got, want, bound, dtype):
    bound = bound + ROUND[dtype] * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 1e-30)
    got = got.double()
    assert torch.isfinite(got).all(), name
    worst = float(((got - want).abs() / bound).max()) if got.numel() else 0.0
    assert worst <= 1.0, (name, worst)


def matrices(kind, op, m, k, groups, layout, pad, seed):
    """Two matrices for each group: (address of one, of the other, lda, stride, the two as [groups, m, k] in FP64)."""
    dt = dtype_of(kind)
    r, c = (m, k) if op == "T" else (k, m)
    apart, lda, stride = {
        "separate": (groups * r * (c + pad) + 40, c + pad, r * (c + pad)),
        "stacked": (r * (c + pad), c + pad, 2 * r * (c + pad)),        # one behind the other in each group
        "reversed": (-r * (c + pad), c + pad, 2 * r * (c + pad)),      # the other one first
        "interleaved": (c + pad, 2 * (c + pad), 2 * r * (c + pad)),    # row by row
    }[layout]
    room = max(abs(apart) if layout == "separate" else 0, 0) + 2 * groups * stride + 8
    buf = torch.full((room,), float("nan"), device="cuda", dtype=dt)
    at = r * (c + pad) if layout == "reversed" else 0
    views = [torch.as_strided(buf, (groups, r, c), (stride, lda, 1), at), torch.as_strided(buf, (groups, r, c), (stride, lda, 1), at + apart)]
    for i, v in enumerate(views):
        v.copy_(randn(seed + i, groups, r, c) * k ** -0.5)
    wide = [v.double() if op == "T" else v.double().transpose(1, 2) for v in views]
    es = buf.element_size()
    return buf, buf.data_ptr() + at * es, buf.data_ptr() + (at + apart) * es, lda, stride, wide


def sums(w, x, sizes, m):
    """w[group] x for each token, and the same of the magnitudes"""
    y = torch.zeros(len(x), m, device="cuda", dtype=torch.float64)
    s = torch.zeros_like(y)
    for g, (lo, hi) in enumerate(spans(sizes)):
        right = w[g].t().contiguous()
        y[lo:hi] = x[lo:hi].double() @ right
        s[lo:hi] = x[lo:hi].double().abs() @ right.abs()
    return y, s


def run_forward(cg, handle, kind, op, act, m, k, sizes, keep=True, layout="stacked", pads=(0, 0, 0, 0), extra=0, dense=False):
    dt = dtype_of(kind)
    n, groups = sum(sizes), len(sizes)
    hold, gate, up, lda, stride, w = matrices(kind, op, m, k, groups, layout, pads[0], 1)
    ldb, ldc, ldz = k + pads[1], m + pads[2], m + pads[3]
    b_buf, b = filled(n, ldb, k, dt, randn(3, n, k))
    outs = [filled(n + extra, ld, m, dt, None, 7.0) for ld in (ldc, ldz, ldz)]
    z = (outs[1][0], outs[2][0]) if keep else (None, None)
    st = handle.gemm_gated(cg.OP_T if op == "T" else cg.OP_N, getattr(cg, act), m, n, k, gate, up, lda, stride, b_buf, ldb, outs[0][0], ldc,
                           *z, ldz, None if dense else offsets_of(sizes), groups, mode_of(cg, kind), type_code(cg, dt))
    assert st == 0
    torch.cuda.synchronize()
    (g, sg), (u, su) = (sums(x, b, sizes, m) for x in w)
    unit = SPLIT[kind] + (k + 2) * 2.0 ** -24
    eg, eu = unit * sg, unit * su
    a, _ = act_of(act, g)
    near("result", outs[0][1][:n], a * u, 1.13 * eg * u.abs() + a.abs() * eu + 1.13 * eg * eu + g.abs() * 2.0 ** -21 * (u.abs() + eu), dt)
    if keep:
        near("gate", outs[1][1][:n], g, eg, dt)
        near("up", outs[2][1][:n], u, eu, dt)
    got = [v[:n].clone() for _, v in outs]
    for i, (buf, v) in enumerate(outs):
        assert untouched(buf, v, n if keep or i == 0 else 0, 7.0), "written outside the results"
    return got


def run_backward(cg, handle, kind, op, act, m, k, sizes, result=True, in_place=False, pads=(0, 0, 0, 0), extra=0, dense=False, stacked=False):
    dt = dtype_of(kind)
    n, groups = sum(sizes), len(sizes)
    r, c = (m, k) if op == "T" else (k, m)
    lda, ldb, ldc, ldz = c + pads[0], k + pads[1], m + pads[2], (2 * m if stacked else m) + pads[3]
    ldd = ldz if in_place else ldz + pads[2]
    a_buf = torch.full((groups * r * lda + 8,), float("nan"), device="cuda", dtype=dt)
    av = torch.as_strided(a_buf, (groups, r, c), (r * lda, lda, 1))
    av.copy_(randn(1, groups, r, c) * k ** -0.5)
    w = av.double() if op == "T" else av.double().transpose(1, 2)
    b_buf, b = filled(n, ldb, k, dt, randn(2, n, k))
    z0, z1 = randn(3, n, m, dtype=dt) * 2, randn(4, n, m, dtype=dt)
    fill = 7.0
    outs = []
    zs = [filled(n + extra, ldz, m, dt, None, fill) for _ in range(2)]
    for (_, v), x in zip(zs, (z0, z1)):
        v[:n].copy_(x)
    ds = zs if in_place else [filled(n + extra, ldd, m, dt, None, fill) for _ in range(2)]
    outs = ds + [filled(n + extra, ldc, m, dt, None, fill)]
    if stacked and not in_place:  # both in one tensor, as one product behind them wants it
        one = torch.full(((n + extra) * ldd + 8,), fill, device="cuda", dtype=dt)
        views = [torch.as_strided(one, (n + extra, m), (ldd, 1), at) for at in (0, m)]
        outs = [(one, views[0]), (one, views[1]), outs[2]]
    st = handle.gemm_gated_backward(cg.OP_T if op == "T" else cg.OP_N, getattr(cg, act), m, n, k, a_buf, lda, r * lda, b_buf, ldb, zs[0][0],
                                    zs[1][0], ldz, outs[0][1], outs[1][1], ldd, outs[2][0] if result else None, ldc,
                                    None if dense else offsets_of(sizes), groups, mode_of(cg, kind), type_code(cg, dt))
    assert st == 0
    torch.cuda.synchronize()
    d, s = sums(w, b, sizes, m)
    ed = (SPLIT[kind] + (k + 2) * 2.0 ** -24) * s
    g, u = z0.double(), z1.double()
    a, slope = act_of(act, g)
    ea, es = g.abs() * 2.0 ** -21, 2.0 ** -20 * (1 + g.abs()) ** 3
    # (two roundings of the products to FP32)
    near("d_gate", outs[0][1][:n], d * u * slope, u.abs() * (ed * (slope.abs() + es) + d.abs() * es) + 2.0 ** -22 * (d * u * slope).abs(), dt)
    near("d_up", outs[1][1][:n], d * a, ed * (a.abs() + ea) + d.abs() * ea + 2.0 ** -22 * (d * a).abs(), dt)
    if result:
        near("result", outs[2][1][:n], a * u, u.abs() * ea + 2.0 ** -22 * (a * u).abs(), dt)
    got = [v[:n].clone() for _, v in outs]
    if stacked and not in_place:
        outs[1][1][:n] = fill
    for i, (buf, v) in enumerate(outs):
        assert untouched(buf, v, n if result or i < 2 else 0, fill), "written outside the results"
    return got


SIZES = [[1], [5, 0, 3], [0, 0, 17, 1, 0], [130, 0, 64, 7, 255], [1] * 70 + [0] * 70 + [3]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}t")
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_forward(cg, handle, kind, op, sizes):
    # aligned, then sizes that no chunk or tile divides
    for (m, k), act in zip(((256, 192), (136, 72), (67, 33), (1, 1), (7, 20)), ACTS + ["SILU"]):
        run_forward(cg, handle, kind, op, act, m, k, sizes)


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}t")
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_backward(cg, handle, kind, op, sizes):
    for (m, k), act in zip(((256, 192), (136, 72), (67, 33), (1, 1), (7, 20)), ACTS + ["SILU"]):
        run_backward(cg, handle, kind, op, act, m, k, sizes)


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_larger_tiles(cg, handle, kind, op):
    for m, k, sizes, act in ((520, 320, [700, 0, 300, 257], "SILU"), (300, 1000, [256, 255, 0, 513], "GELU"),
                             (264, 40, [50, 90, 47, 60], "GELU_TANH"), (261, 129, [60, 45, 70], "RELU")):
        run_forward(cg, handle, kind, op, act, m, k, sizes)
        run_backward(cg, handle, kind, op, act, m, k, sizes)


@pytest.mark.parametrize("cls", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_every_tile(cg, handle, kind, op, cls, monkeypatch):
    """Every tile, whichever the choice would take: whole ones, ones that end inside the matrix, few tokens."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for (m, k, sizes), act in itertools.product(((512, 256, [300, 0, 257]), (200, 136, [9, 33]), (71, 53, [40, 3])), ("SILU", "GELU")):
        run_forward(cg, handle, kind, op, act, m, k, sizes)
        run_backward(cg, handle, kind, op, act, m, k, sizes)


@pytest.mark.parametrize("cls", [1, 2])
@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_lines_that_begin_inside_words(cg, handle, kind, cls, monkeypatch):
    """Matrices stored along their rows, of odd and even lengths and distances, over many steps."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for m, k, sizes, pad in ((301, 1003, [130, 0, 257], 0), (300, 704, [40, 1], 1), (129, 577, [33], 2), (8, 321, [5, 60], 0), (15, 640, [70], 0)):
        for layout in ("separate", "stacked", "reversed", "interleaved"):
            run_forward(cg, handle, kind, "N", "SILU", m, k, sizes, layout=layout, pads=(pad, 0, 0, 0))


@pytest.mark.parametrize("layout", ["separate", "stacked", "reversed", "interleaved"])
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", ["FP16TCEC", "f16", "bf16"])
def test_where_the_matrices_lie(cg, handle, kind, op, layout):
    for pads in ((0, 0, 0, 0), (8, 16, 8, 24), (1, 3, 5, 7)):
        for keep, m, k, sizes in ((True, 144, 104, [3, 0, 9, 1]), (False, 144, 104, [70, 0, 90, 61]), (True, 320, 64, [300, 1, 280])):
            run_forward(cg, handle, kind, op, "SILU", m, k, sizes, keep, layout, pads, extra=3)


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", ["TF32TCEC", "f16", "bf16"])
def test_gradients_in_place_and_strided(cg, handle, kind, op):
    for pads in ((0, 0, 0, 0), (8, 16, 8, 24), (1, 3, 5, 7)):
        for m, k, sizes in ((144, 104, [3, 0, 9, 1]), (144, 104, [70, 0, 90, 61]), (320, 64, [300, 1, 280])):
            run_backward(cg, handle, kind, op, "GELU", m, k, sizes, True, False, pads, extra=3)
            run_backward(cg, handle, kind, op, "GELU", m, k, sizes, False, True, pads, extra=3)
            run_backward(cg, handle, kind, op, "SILU", m, k, sizes, True, False, pads, extra=3, stacked=True)


@pytest.mark.parametrize("kind", ["FP16TCEC", "bf16"])
def test_a_dense_block(cg, handle, kind):
    for n in (1, 37, 300):
        run_forward(cg, handle, kind, "T", "SILU", 264, 136, [n], dense=True)
        run_backward(cg, handle, kind, "N", "SILU", 264, 136, [n], dense=True)


@pytest.mark.parametrize("kind", ["FP16TCEC", "f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_no_features(cg, handle, kind, act):
    """k = 0: both projections are zero."""
    dt = dtype_of(kind)
    c, z, d = (torch.full((n, 5, 8), 7.0, device="cuda", dtype=dt) for n in (1, 2, 2))
    assert handle.gemm_gated(cg.OP_T, getattr(cg, act), 8, 5, 0, None, None, 0, 0, None, 0, c, 8, z[0], z[1], 8, None, 1, mode_of(cg, kind),
                             type_code(cg, dt)) == 0
    assert not c.any() and not z.any()
    z = randn(1, 2, 5, 8, dtype=dt)
    assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), 8, 5, 0, None, 0, 0, None, 0, z[0], z[1], 8, d[0], d[1], 8, None, 0, None, 1,
                                      mode_of(cg, kind), type_code(cg, dt)) == 0
    assert not d.any()


@pytest.mark.parametrize("act", ACTS)
def test_extreme_projections(cg, handle, act):
    """Values far out on both sides, and what is no number: as the formulas say."""
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20.0, -20.0, 90.0, -90.0, 1e30, -1e30, float("inf"), float("nan")], device="cuda")
    w = g[None, :, None].contiguous()  # one feature in: G = g, U = 1
    one = torch.ones(1, len(g), 1, device="cuda")
    c, zg, zu = (torch.empty(1, len(g), device="cuda") for _ in range(3))
    x = torch.ones(1, 1, device="cuda")
    assert handle.gemm_gated(cg.OP_T, getattr(cg, act), len(g), 1, 1, w, one, 1, len(g), x, 1, c, len(g), zg, zu, len(g), None, 1, cg.TF32TCEC, cg.R_32F) == 0
    # (an infinity is not split: what it multiplies is NaN)
    want = act_of(act, torch.where(g.abs() < 1e29, g, float("nan")).double())[0]
    finite = torch.isfinite(want)
    assert bool((c[0].double()[finite] - want[finite]).abs().max() <= 2.0 ** -20 * 90) and bool(torch.isnan(c[0][10:]).all())
    if act in ("SILU", "RELU"):  # (the cubes and squares of the others overflow on the way to the same limits)
        assert float(c[0, 8]) == float(zg[0, 8]) and float(c[0, 9]) == 0.0
    z = torch.cat([g[:10], torch.tensor([float("inf"), float("nan")], device="cuda")])[None].contiguous()
    d0, d1 = torch.empty_like(z), torch.empty_like(z)
    assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), len(g), 1, 1, one, 1, len(g), x, 1, z, torch.ones_like(z), len(g), d0, d1, len(g),
                                      None, 0, None, 1, cg.TF32TCEC, cg.R_32F) == 0
    a, slope = act_of(act, z.double())
    inside = z[0].abs() <= 90
    assert bool((d0.double() - slope)[0][inside].abs().max() <= 2.0 ** -14) and bool((d1.double() - a)[0][inside].abs().max() <= 2.0 ** -20 * 90)
    assert bool(torch.isnan(d1[0, 11]))


@pytest.mark.parametrize("kind", ["TF32TCEC", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_gradients_far_out(cg, handle, act, kind):
    """From 200 on an activation is G or 0 and its slope 1 or 0, also where squares and cubes of G are infinite."""
    dt = dtype_of(kind)
    z = torch.tensor([200.0, -200.0, 1e4, -1e4, 1e18, -1e18, 1e20, -1e20, 1e38, -1e38], device="cuda").to(dt)[None].contiguous()
    m = z.shape[1]
    w, one, x = torch.ones(1, m, 1, device="cuda", dtype=dt), torch.ones_like(z), torch.ones(1, 1, device="cuda", dtype=dt)
    d = torch.full((3, 1, m), 7.0, device="cuda", dtype=dt)
    assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), m, 1, 1, w, 1, m, x, 1, z, one, m, d[0], d[1], m, d[2], m, None, 1,
                                      mode_of(cg, kind), type_code(cg, dt)) == 0
    assert torch.equal(d[0], (z > 0).to(dt)) and torch.equal(d[1], z.clamp(min=0)) and torch.equal(d[2], d[1])


def test_the_gradient_is_that_of_differences(cg, handle):
    """d_gate and d_up against central differences of the block's result, in FP32: a step of 2^-6 in G leaves a third derivative,
    at most 1.2 for SiLU, and two results that are off by 2^-21 each."""
    m, k, n = 24, 16, 6
    w2, dy = randn(1, 1, m, k) * k ** -0.5, randn(2, n, k)
    z = randn(3, 2, n, m)
    d = torch.empty(2, n, m, device="cuda")
    for act in ("SILU", "GELU", "GELU_TANH"):
        assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), m, n, k, w2, k, m * k, dy, k, z[0], z[1], m, d[0], d[1], m, None, 0, None, 1,
                                          cg.TF32TCEC, cg.R_32F) == 0

        def result(gate, up):  # of the block, by the library: one feature in
            out = torch.empty(1, n * m, device="cuda")
            assert handle.gemm_gated(cg.OP_T, getattr(cg, act), n * m, 1, 1, gate.reshape(1, -1, 1).contiguous(), up.reshape(1, -1, 1).contiguous(), 1,
                                     n * m, torch.ones(1, 1, device="cuda"), 1, out, n * m, None, None, 0, None, 1, cg.TF32TCEC, cg.R_32F) == 0
            return out.view(n, m).double()
        step = 2.0 ** -6
        dh = dy.double() @ w2[0].double().t().contiguous()
        by_gate = (result(z[0] + step, z[1]) - result(z[0] - step, z[1])) / (2 * step) * dh
        by_up = (result(z[0], z[1] + step) - result(z[0], z[1] - step)) / (2 * step) * dh
        size = 1 + z.double().abs().max()
        bound = (step ** 2 * 1.2 / 6 + 2.0 ** -20 * size / step) * size * dh.abs() + 1e-6
        assert bool(((d[0].double() - by_gate).abs() <= bound).all()) and bool(((d[1].double() - by_up).abs() <= bound).all())


def test_results_repeat(cg, handle):
    for kind in ("FP16TCEC", "bf16"):
        x = [run_forward(cg, handle, kind, "T", "SILU", 300, 200, [100, 0, 60]) for _ in range(2)]
        assert all(torch.equal(p, q) for p, q in zip(*x))
        x = [run_backward(cg, handle, kind, "N", "SILU", 300, 200, [100, 0, 60]) for _ in range(2)]
        assert all(torch.equal(p, q) for p, q in zip(*x))


def test_offsets_out_of_range_stay_inside(cg, handle):
    """As the other products: nothing outside the operands is read or written."""
    m, k, n = 72, 40, 50
    w, x = randn(1, 2, 3, m, k, dtype=torch.bfloat16), randn(2, n, k, dtype=torch.bfloat16)
    buf = torch.full((n + 2, m), 7.0, device="cuda", dtype=torch.bfloat16)
    for off in ([-5, 20, 10, 99], [60, 70, 80, 90], [2 ** 31 - 1, -2 ** 31, 0, 50]):
        assert handle.gemm_gated(cg.OP_T, cg.SILU, m, n, k, w[0], w[1], k, m * k, x, k, buf[1:], m, None, None, 0,
                                 torch.tensor(off, dtype=torch.int32, device="cuda"), 3, cg.FP16TC, cg.R_16BF) == 0
        torch.cuda.synchronize()
        assert bool((buf[0] == 7).all()) and bool((buf[n + 1] == 7).all())
