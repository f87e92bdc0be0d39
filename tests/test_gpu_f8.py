"""Products of 8-bit floating point with scales for blocks of 128 (gemm_f8, gemm_gated_f8, quantize_f8) against the formulas in
FP64.

Bounds, by element, in terms of S = sum |a| |b| with their scales: of eight neighbouring products the matrix cores cut all but
the largest to multiples of 2^-13 of its power of two, 7 2^-13 of it at most; a block's sixteen sums are cut to 2^-23 and the
blocks' sums, scaled, are rounded like any FP32 sum: (K + 16) 2^-23.  A result is rounded once.  Over a whole matrix the cuts are
independent: 2^-13 of S.  Gated blocks as in test_gpu_gated.py, with the fast exponential for all types: 2^-20 in place of
2^-21."""
import math

import numpy as np
import pytest
import torch

from test_gpu_gated import act_of, filled, near, untouched
from test_gpu_grouped import ROUND, offsets_of, randn, spans, type_code

pytestmark = pytest.mark.gpu

F8 = {"e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
MOST = {"e4m3": 448.0, "e5m2": 57344.0}
OUTS = [torch.bfloat16, torch.float16, torch.float32]


def code(cg, f8):
    return {"e4m3": cg.R_8F_E4M3, "e5m2": cg.R_8F_E5M2}[f8]


def blocks(n):
    return -(-n // 128)


def unit(k):
    return 7 * 2.0 ** -13 + (k + 16) * 2.0 ** -23


def f8_bytes(seed, *shape, f8):
    """Values of all sizes that the type has, as tensors' bytes: normal ones, and some of the smallest and largest."""
    x = randn(seed, *shape) * (MOST[f8] / 4 if f8 == "e4m3" else 1000)
    pick = torch.rand(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    x = torch.where(pick < 0.05, x * 2.0 ** -12, x).clamp(-MOST[f8], MOST[f8])
    return x.to(F8[f8]).view(torch.uint8)


def scales(seed, *shape):
    return 2.0 ** (randn(seed, *shape) * 2) * 0.01


def strided(values, ld, groups=1, stride=None, f8="e4m3"):
    """Bytes [groups, rows, cols] in rows of ld bytes whose rest are NaN: (buffer, stride)"""
    g, r, c = values.shape
    stride = stride or r * ld
    buf = torch.full((g * stride + 16,), 0x7f, device="cuda", dtype=torch.uint8)
    torch.as_strided(buf, (g, r, c), (stride, ld, 1)).copy_(values)
    return buf, stride


def weights(seed, m, k, groups, op, pad=0, scale_pad=0):
    """(bytes, lda, stride, scales, stride of the scales, values [groups, m, k] in FP64)"""
    r, c = (m, k) if op == "T" else (k, m)
    q = f8_bytes(seed, groups, r, c, f8="e4m3")
    buf, stride = strided(q, c + pad)
    per = blocks(r) * blocks(c)
    s = torch.full((groups * (per + scale_pad),), float("nan"), device="cuda")
    sv = torch.as_strided(s, (groups, blocks(r), blocks(c)), (per + scale_pad, blocks(c), 1))
    sv.copy_(scales(seed + 1, groups, blocks(r), blocks(c)))
    wide = q.view(torch.float8_e4m3fn).float().double() * sv.double().repeat_interleave(128, 1).repeat_interleave(128, 2)[:, :r, :c]
    return buf, c + pad, stride, s, per + scale_pad, wide if op == "T" else wide.transpose(1, 2)


def tokens(seed, n, k, f8, pad=0):
    q = f8_bytes(seed, 1, n, k, f8=f8)
    buf, _ = strided(q, k + pad, f8=f8)
    s = scales(seed + 1, n, blocks(k))
    return buf, s, q[0].view(F8[f8]).float().double() * s.double().repeat_interleave(128, 1)[:, :k]


def sums(w, x, sizes, m):
    y = torch.zeros(len(x), m, device="cuda", dtype=torch.float64)
    s = torch.zeros_like(y)
    for g, (lo, hi) in enumerate(spans(sizes)):
        right = w[g].t().contiguous()
        y[lo:hi], s[lo:hi] = x[lo:hi] @ right, x[lo:hi].abs() @ right.abs()
    return y, s


def run(cg, handle, op, m, k, sizes, f8="e4m3", out=torch.float32, pads=(0, 0, 0, 0), extra=0, dense=False):
    n, groups = sum(sizes), len(sizes)
    a, lda, stride, sa, ss, w = weights(1, m, k, groups, op, pads[0], pads[3])
    b, sb, x = tokens(5, n, k, f8, pads[1])
    ldc = m + pads[2]
    c_buf, c = filled(n + extra, ldc, m, out, None, 7.0)
    st = handle.gemm_f8(cg.OP_T if op == "T" else cg.OP_N, m, n, k, a, lda, stride, cg.R_8F_E4M3, sa, ss, b, k + pads[1], code(cg, f8), sb, c_buf,
                        ldc, type_code(cg, out), None if dense else offsets_of(sizes), groups)
    assert st == 0
    torch.cuda.synchronize()
    y, s = sums(w, x, sizes, m)
    if out == torch.float16:  # (beyond its range: infinities on both sides)
        inside = y.abs() + unit(k) * s < 65504
        got = torch.where(inside, c[:n].double(), 0.0)
        y, s = torch.where(inside, y, 0.0), torch.where(inside, s, 0.0)
    else:
        got = c[:n].double()
    near("product", got, y, unit(k) * s, out)
    if got.numel() > 256:
        bar = 2.0 ** -13 + 2 * ROUND[out] + 2 * 2.0 ** -23 * np.sqrt(k + 1)
        assert float((got - y).norm()) <= bar * float(s.norm())
    keep = c[:n].clone()
    assert untouched(c_buf, c, n, 7.0), "written outside the results"
    return keep


def run_gated(cg, handle, act, m, k, sizes, f8="e4m3", out=torch.float32, pads=(0, 0, 0, 0), extra=0):
    n, groups = sum(sizes), len(sizes)
    gate, lda, stride, sg, ss, w0 = weights(1, m, k, groups, "T", pads[0], pads[3])
    up, _, _, su, _, w1 = weights(11, m, k, groups, "T", pads[0], pads[3])
    sg, su, w0, w1 = sg / 64, su / 64, w0 / 64, w1 / 64  # (projections of a few units)
    b, sb, x = tokens(5, n, k, f8, pads[1])
    sb, x = sb / 1024, x / 1024
    c_buf, c = filled(n + extra, m + pads[2], m, out, None, 7.0)
    st = handle.gemm_gated_f8(getattr(cg, act), m, n, k, gate, up, lda, stride, cg.R_8F_E4M3, sg, su, ss, b, k + pads[1], code(cg, f8), sb, c_buf,
                              m + pads[2], type_code(cg, out), offsets_of(sizes), groups)
    assert st == 0
    torch.cuda.synchronize()
    (g, eg), (u, eu) = (sums(w, x, sizes, m) for w in (w0, w1))
    eg, eu = unit(k) * eg, unit(k) * eu
    a, _ = act_of(act, g)
    bound = 1.13 * eg * u.abs() + a.abs() * eu + 1.13 * eg * eu + (g.abs() + eg) * 2.0 ** -20 * (u.abs() + eu)
    got, want = c[:n].double(), a * u
    if out == torch.float16:
        inside = want.abs() + bound < 65504
        got, want, bound = (torch.where(inside, t, 0.0) for t in (got, want, bound))
    near("result", got, want, bound, out)
    keep = c[:n].clone()
    assert untouched(c_buf, c, n, 7.0), "written outside the results"
    return keep


SIZES = [[1], [5, 0, 3], [0, 0, 17, 1, 0], [130, 0, 64, 7, 255], [1] * 70 + [0] * 70 + [3]]
# aligned, blocks that are not whole, sizes that no chunk divides, less than a chunk
SHAPES = [(256, 256), (144, 208), (128, 384), (67, 33), (130, 129), (1, 1), (7, 20), (20, 7)]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}t")
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("f8", F8)
def test_products(cg, handle, f8, op, sizes):
    for i, (m, k) in enumerate(SHAPES):
        run(cg, handle, op, m, k, sizes, f8, OUTS[i % 3])


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}t")
@pytest.mark.parametrize("f8", F8)
def test_gated(cg, handle, f8, sizes):
    for i, (m, k) in enumerate(SHAPES):
        run_gated(cg, handle, ["SILU", "GELU", "GELU_TANH", "RELU"][i % 4], m, k, sizes, f8, OUTS[i % 3])


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("f8", F8)
def test_larger_tiles(cg, handle, f8, op):
    for (m, k, sizes), out in zip(((528, 640, [700, 0, 300, 257]), (304, 1000, [256, 255, 0, 513]), (264, 144, [50, 90, 47, 60]),
                                   (261, 129, [60, 45, 70]), (1024, 2048, [300, 40])), OUTS + OUTS):
        run(cg, handle, op, m, k, sizes, f8, out)
        if op == "T":
            run_gated(cg, handle, "SILU", m, k, sizes, f8, out)


@pytest.mark.parametrize("cls", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("f8", F8)
def test_every_tile(cg, handle, f8, op, cls, monkeypatch):
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for m, k, sizes in ((512, 512, [300, 0, 257]), (272, 144, [9, 33]), (128, 1280, [40, 200]), (71, 53, [40, 3]), (256, 16, [130])):
        run(cg, handle, op, m, k, sizes, f8)
        if op == "T":
            run_gated(cg, handle, "SILU", m, k, sizes, f8, torch.bfloat16)


@pytest.mark.parametrize("cls", [1, 2])
@pytest.mark.parametrize("op", ["T", "N"])
def test_any_alignment_over_many_steps(cg, handle, op, cls, monkeypatch):
    """Steps that are whole and the last one, lines shorter and a little longer than a chunk."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for m, k, sizes in ((301, 1021, [130, 0, 257]), (7, 520, [40]), (16, 385, [5, 60]), (17, 384, [70]), (130, 640, [33, 1])):
        run(cg, handle, op, m, k, sizes, "e4m3", torch.bfloat16, (1, 3, 5, 7), extra=2)
        run(cg, handle, op, m, k, sizes, "e5m2", torch.float32)
        if op == "T":
            for out in OUTS:
                run_gated(cg, handle, "SILU", m, k, sizes, "e4m3", out, (1, 3, 5, 7))


@pytest.mark.parametrize("pads", [(16, 32, 8, 5), (1, 3, 5, 7), (16, 0, 4, 0)])
@pytest.mark.parametrize("op", ["T", "N"])
def test_strides(cg, handle, op, pads):
    for m, k, sizes in ((144, 112, [3, 0, 9, 1]), (144, 400, [70, 0, 90, 61]), (320, 256, [300, 1, 280])):
        run(cg, handle, op, m, k, sizes, "e4m3", torch.bfloat16, pads, extra=3)
        if op == "T":
            run_gated(cg, handle, "SILU", m, k, sizes, "e4m3", torch.bfloat16, pads, extra=3)


def test_one_matrix_for_all(cg, handle):
    for n in (1, 37, 300):
        for op in "TN":
            run(cg, handle, op, 272, 144, [n], out=torch.bfloat16, dense=True)


def test_no_features(cg, handle):
    c = torch.full((5, 8), 7.0, device="cuda")
    assert handle.gemm_f8(cg.OP_T, 8, 5, 0, None, 0, 0, cg.R_8F_E4M3, None, 0, None, 0, cg.R_8F_E4M3, None, c, 8, cg.R_32F, None, 1) == 0
    assert not c.any()
    c.fill_(7.0)
    assert handle.gemm_gated_f8(cg.SILU, 8, 5, 0, None, None, 0, 0, cg.R_8F_E4M3, None, None, 0, None, 0, cg.R_8F_E4M3, None, c, 8, cg.R_32F, None, 1) == 0
    assert not c.any()


def test_what_is_no_number_stays_with_its_token(cg, handle):
    """A token whose block has no scale, and one with a NaN among its values: NaN throughout, and nothing of it in the others."""
    for n in (3, 100, 400):
        m, k = 256, 512
        a, lda, stride, sa, ss, w = weights(1, m, k, 1, "T")
        b, sb, x = tokens(5, n, k, "e4m3")
        sb[1, 2] = float("nan")
        b[2 * k + 300] = 0x7f
        c = torch.empty(n, m, device="cuda")
        assert handle.gemm_f8(cg.OP_T, m, n, k, a, lda, stride, cg.R_8F_E4M3, sa, ss, b, k, cg.R_8F_E4M3, sb, c, m, cg.R_32F, None, 1) == 0
        bad = torch.isnan(c)
        assert bool(bad[1:3].all()) and int(bad.sum()) == 2 * m


# ---- quantisation ----

def rounded(v, f8):
    """v in FP64 to the nearest value of the type, ties to even"""
    bits, least = (4, -6) if f8 == "e4m3" else (3, -14)
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=least).double() - (bits - 1))
    return torch.round(v / step) * step


def quantised(cg, handle, x, f8, block_n, pads=(0, 0)):
    """x: [batch, n, k].  (values as FP64, scales)"""
    batch, n, k = x.shape
    ldx, ldq = k + pads[0], k + pads[1]
    x_buf = torch.full((batch * n * ldx + 8,), float("nan"), device="cuda", dtype=x.dtype)
    torch.as_strided(x_buf, (batch, n, k), (n * ldx, ldx, 1)).copy_(x)
    q_buf = torch.full((batch * n * ldq + 8,), 0x55, device="cuda", dtype=torch.uint8)
    q = torch.as_strided(q_buf, (batch, n, k), (n * ldq, ldq, 1))
    nb = n if block_n == 1 else blocks(n)
    s_buf = torch.full((batch * nb * blocks(k) + 3,), 7.0, device="cuda")
    assert handle.quantize_f8(k, n, x_buf, ldx, n * ldx, type_code(cg, x.dtype), block_n, q_buf, ldq, n * ldq, code(cg, f8), s_buf, batch) == 0
    torch.cuda.synchronize()
    assert bool((s_buf[-3:] == 7).all())
    got, s = q.clone().view(F8[f8]).float().double(), s_buf[:-3].view(batch, nb, blocks(k)).clone()
    q.fill_(0x55)
    assert bool((q_buf == 0x55).all()), "written outside the results"
    return got, s


def peaks(x, block_n):
    """The largest magnitude of each block: as the scales lie, and for each value."""
    batch, n, k = x.shape
    rows = n if block_n == 1 else blocks(n)
    full = torch.zeros(batch, rows * block_n, blocks(k) * 128, device="cuda", dtype=torch.float64)
    full[:, :n, :k] = x.double().abs()
    p = full.view(batch, rows, block_n, blocks(k), 128).amax((2, 4))
    return p, p.repeat_interleave(block_n, 1).repeat_interleave(128, 2)[:, :n, :k]


@pytest.mark.parametrize("block_n", [1, 128])
@pytest.mark.parametrize("f8", F8)
@pytest.mark.parametrize("dtype", OUTS, ids=str)
def test_quantize(cg, handle, dtype, f8, block_n):
    for (batch, n, k), pads in (((1, 300, 1024), (0, 0)), ((1, 1, 1), (0, 0)), ((3, 130, 200), (0, 0)), ((2, 5, 129), (3, 5)), ((1, 77, 136), (8, 8)),
                                ((1, 2000, 384), (0, 0))):
        x = (randn(1, batch, n, k) * 10.0 ** randn(2, batch, n, 1)).to(dtype)
        got, s = quantised(cg, handle, x, f8, block_n, pads)
        p, each = peaks(x, block_n)
        assert torch.equal(s, (p / MOST[f8]).float())
        y = (x * MOST[f8]).double() if dtype == torch.float32 else x.double() * MOST[f8]
        v = torch.where(each > 0, y / each, 0.0)
        want = rounded(v, f8)
        if dtype == torch.float32:  # (a quotient nearer to half way than FP32 tells may go either way)
            other = torch.where(got < v, rounded(v * (1 - 2.0 ** -22), f8), rounded(v * (1 + 2.0 ** -22), f8))
            off = got != want
            assert torch.equal(torch.where(off, other, got), got) and int(off.sum()) <= 3
        else:
            assert torch.equal(got, want)


@pytest.mark.parametrize("k", [520, 515])
@pytest.mark.parametrize("dtype", OUTS, ids=str)
def test_quantize_many(cg, handle, dtype, k):
    """So many tokens that a thread has several blocks, an odd number of them: as a thousand tokens at a time."""
    x = (randn(1, 1, 9001, k) * 10.0 ** randn(2, 1, 9001, 1)).to(dtype)
    got, s = quantised(cg, handle, x, "e4m3", 1)
    for at in range(0, 9001, 1000):
        part, t = quantised(cg, handle, x[:, at:at + 1000].contiguous(), "e4m3", 1)
        assert torch.equal(got[:, at:at + 1000], part) and torch.equal(s[:, at:at + 1000], t)


@pytest.mark.parametrize("block_n", [1, 128])
@pytest.mark.parametrize("f8", F8)
def test_quantize_extremes(cg, handle, f8, block_n):
    """Blocks of zeros, with an infinity or a NaN, of the largest and the smallest numbers: each by itself."""
    special = [0.0, float("inf"), -float("inf"), float("nan"), 3.4e38, 1e-30, 1e-37, 1e-40, 1e-45, 1.0]
    x = randn(1, len(special), 2, 256).clamp(-2, 2)
    for i, v in enumerate(special):
        x[i, :, :128] = x[i, :, :128] * 0.4 * v if math.isfinite(v) else x[i, :, :128]
        x[i, 1, 77] = v
        x[i, 0, 78] = v if math.isfinite(v) else 1.0
    got, s = quantised(cg, handle, x, f8, block_n)
    p, each = peaks(torch.nan_to_num(x, posinf=0.0, neginf=0.0), block_n)
    for i, v in enumerate(special):
        rows = slice(0, 2) if block_n == 128 else slice(1, 2)  # (of what is not finite)
        if not math.isfinite(v):
            assert bool(torch.isnan(s[i, rows if block_n == 1 else slice(0, 1), 0]).all()) and not got[i, rows, :128].any()
        elif v == 0.0 or abs(v) < 1e-42:
            assert not s[i, :, 0].any() and not got[i, :, :128].any()
        else:
            want = p[i, :, 0] / MOST[f8]
            assert bool(((s[i, :, 0].double() - want).abs() <= 2.0 ** -24 * want + 2.0 ** -150).all())
            t = got[i, :, :128] / MOST[f8] * each[i, :, :128]
            least = 2.0 ** (-10 if f8 == "e4m3" else -17) / MOST[f8]
            bound = (2.0 ** (-4 if f8 == "e4m3" else -3) + 2.0 ** -22) * x[i, :, :128].double().abs() + least * each[i, :, :128] + 2.0 ** -149
            assert bool(((t - x[i, :, :128].double()).abs() <= bound).all()), v
        assert bool((s[i, :, 1] > 0).all()) and float(got[i, :, 128:].abs().max()) == MOST[f8]


def test_a_layer_from_its_tensors(cg, handle):
    """Quantised tokens times quantised matrices, the whole way: off by the roundings to E4M3, half a step of 2^-3 each."""
    n, m, k = 70, 256, 640
    x, w = randn(1, n, k, dtype=torch.bfloat16), randn(2, m, k, dtype=torch.bfloat16)
    q, s = torch.empty(n, k, device="cuda", dtype=torch.uint8), torch.empty(n, blocks(k), device="cuda")
    wq, ws = torch.empty(m, k, device="cuda", dtype=torch.uint8), torch.empty(blocks(m), blocks(k), device="cuda")
    c = torch.empty(n, m, device="cuda")
    assert handle.quantize_f8(k, n, x, k, 0, cg.R_16BF, 1, q, k, 0, cg.R_8F_E4M3, s) == 0
    assert handle.quantize_f8(k, m, w, k, 0, cg.R_16BF, 128, wq, k, 0, cg.R_8F_E4M3, ws) == 0
    assert handle.gemm_f8(cg.OP_T, m, n, k, wq, k, 0, cg.R_8F_E4M3, ws, 0, q, k, cg.R_8F_E4M3, s, c, m, cg.R_32F) == 0
    size = x.double().abs() @ w.double().abs().t().contiguous()
    want = x.double() @ w.double().t().contiguous()
    # (a value below 2^-6 of 448ths is off by 2^-10 of them: 2^-19 of its block's largest, at most 8 here, on either side)
    step = 2 * 2.0 ** -4 + 2.0 ** -8 + 7 * 2.0 ** -13
    bound = step * size + 2.0 ** -10 / 448 * 8 * (x.double().abs().sum(1, keepdim=True) + w.double().abs().sum(1)[None] + 1)
    assert bool(((c.double() - want).abs() <= bound).all())
    assert float((c.double() - want).norm()) <= 2.0 ** -4 * float(want.norm())


def test_results_repeat(cg, handle):
    for sizes in ([3, 1], [100, 0, 60], [300, 300]):
        x = [run(cg, handle, "T", 304, 640, sizes, out=torch.bfloat16) for _ in range(2)]
        y = [run_gated(cg, handle, "SILU", 304, 640, sizes, out=torch.bfloat16) for _ in range(2)]
        assert torch.equal(*x) and torch.equal(*y)


def test_offsets_out_of_range_stay_inside(cg, handle):
    m, k, n = 72, 144, 50
    a, lda, stride, sa, ss, w = weights(1, m, k, 3, "T")
    b, sb, x = tokens(5, n, k, "e4m3")
    buf = torch.full((n + 2, m), 7.0, device="cuda")
    for off in ([-5, 20, 10, 99], [60, 70, 80, 90], [2 ** 31 - 1, -2 ** 31, 0, 50]):
        assert handle.gemm_f8(cg.OP_T, m, n, k, a, lda, stride, cg.R_8F_E4M3, sa, ss, b, k, cg.R_8F_E4M3, sb, buf[1:], m, cg.R_32F,
                              torch.tensor(off, dtype=torch.int32, device="cuda"), 3) == 0
        torch.cuda.synchronize()
        assert bool((buf[0] == 7).all()) and bool((buf[n + 1] == 7).all())
