"""Experts' products (gemm_grouped, gemm_grouped_k, gemm_i8, quantize_i8) against the formulas in FP64.

Bounds, by element, in terms of S = sum |a| |b| of its products: FP32 sums of K products are off by at most K 2^-24 S;
the splits leave 2^-21 (FP16TCEC, bf16x3: two terms of 11 bits, three of 8, products of the smallest dropped), 2^-10
(FP16TC: one term of 11 bits) or 2^-14 (bf16x2) of each product; a result in FP16 / BF16 is rounded once, to 2^-11 / 2^-8.
Over a whole matrix the roundings are independent: 2^-24 sqrt(K), twice over, in place of K 2^-24."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = ["FP16TCEC", "TF32TCEC", "FP16TC", "TF32TC", "f16", "bf16"]
SPLIT = {"FP16TCEC": 2.0 ** -21, "TF32TCEC": 2.0 ** -21, "FP16TC": 2.0 ** -10, "TF32TC": 2.0 ** -14, "f16": 0.0, "bf16": 0.0}
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16}


def dtype_of(kind):
    return DTYPE.get(kind, torch.float32)


def type_code(cg, dtype):
    return {torch.float32: cg.R_32F, torch.float16: cg.R_16F, torch.bfloat16: cg.R_16BF}[dtype]


def mode_of(cg, kind):
    return getattr(cg, kind, cg.AUTO)  # (16-bit operands: the mode is not looked at)


def offsets_of(sizes):
    return torch.tensor(np.concatenate([[0], np.cumsum(sizes)]), dtype=torch.int32, device="cuda")


def randn(seed, *shape, dtype=torch.float32):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(*shape, generator=g, device="cuda").to(dtype)


def rows(tensor_rows, ld, seed, dtype, fill=float("nan")):
    """[rows, cols] values inside rows of ld elements whose rest is `fill`: (flat buffer, view of the values)."""
    r, cols = tensor_rows
    buf = torch.full((r * ld + 8,), fill, device="cuda", dtype=dtype)
    view = buf[:r * ld].view(r, ld)[:, :cols]
    view.copy_(randn(seed, r, cols, dtype=dtype))
    return buf, view


def check(got, want, size, kind, k, out_dtype):
    """got, want, size (sum of |a||b|, with |beta c|): same shape; want and size in FP64."""
    got = got.double()
    assert torch.isfinite(got).all()
    d = (got - want).abs()
    bound = (SPLIT[kind] + (k + 2) * 2.0 ** -24) * size + ROUND[out_dtype] * want.abs() + 1e-30
    if out_dtype == torch.float16:
        bound = bound + 2.0 ** -25  # (subnormal results)
    worst = float((d / bound).max()) if d.numel() else 0.0
    assert worst <= 1.0, worst
    if d.numel() > 256:
        bar = SPLIT[kind] + 2 * 2.0 ** -24 * np.sqrt(k + 1) + 2 * ROUND[out_dtype]
        assert float(d.norm()) <= bar * float(size.norm()), (float(d.norm() / size.norm()), bar)


def spans(sizes):
    at = np.concatenate([[0], np.cumsum(sizes)])
    return list(zip(at[:-1].tolist(), at[1:].tolist()))


def run_columns(cg, handle, kind, op, m, k, sizes, alpha=1.0, beta=0.0, pads=(0, 0, 0, 0), out=None, extra_columns=0, c_fill=None):
    """One call; returns (C's columns, expected, sizes of the sums) and checks everything that must not change."""
    dt = dtype_of(kind)
    od = out or dt
    n, groups = int(np.sum(sizes)), len(sizes)
    ar, ac = (m, k) if op == "T" else (k, m)
    lda, ldb, ldc = ac + pads[0], k + pads[1], m + pads[2]
    stride = ar * lda + pads[3]
    a_buf = torch.full((groups * stride + 8,), float("nan"), device="cuda", dtype=dt)
    a = torch.as_strided(a_buf, (groups, ar, ac), (stride, lda, 1))
    a.copy_(randn(1, groups, ar, ac, dtype=dt))
    b_buf, b = rows((n, k), ldb, 2, dt)
    c_buf, c = rows((n + extra_columns, m), ldc, 3, od, 7.0)
    if c_fill is not None:
        c.fill_(c_fill)
    before = c_buf.clone()
    old = c[:n].double().clone()
    st = handle.gemm_grouped(cg.OP_T if op == "T" else cg.OP_N, m, n, k, alpha, a_buf, lda, stride, b_buf, ldb, beta,
                             c_buf, ldc, offsets_of(sizes), groups, mode_of(cg, kind), type_code(cg, dt), type_code(cg, od))
    assert st == 0
    want = torch.empty(n, m, device="cuda", dtype=torch.float64)
    size = torch.empty_like(want)
    for g, (lo, hi) in enumerate(spans(sizes)):
        w = a[g].double() if op == "N" else a[g].double().t().contiguous()
        want[lo:hi] = alpha * (b[lo:hi].double() @ w)
        size[lo:hi] = abs(alpha) * (b[lo:hi].double().abs() @ w.abs())
    if beta != 0:
        want += beta * old
        size += (beta * old).abs()
    torch.cuda.synchronize()
    got = c[:n].clone()
    c[:n] = 0
    keep = before.clone()
    torch.as_strided(keep, (n, m), (ldc, 1)).zero_()
    assert torch.equal(c_buf.view(torch.uint8), keep.view(torch.uint8)), "written outside the results"
    return got, want, size


SIZES = [
    [1], [5, 0, 3], [0, 0, 17, 1, 0], [130, 0, 64, 7, 255], [513, 300, 1, 0, 400], [1] * 70 + [0] * 70 + [3], [0] * 65 + [33],
]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}t")
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_columns(cg, handle, kind, op, sizes):
    # aligned, then sizes that no chunk or tile divides
    for m, k in ((256, 192), (136, 72), (67, 33), (1, 1)):
        dt = dtype_of(kind)
        got, want, size = run_columns(cg, handle, kind, op, m, k, sizes)
        check(got, want, size, kind, k, dt)


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_columns_larger_tiles(cg, handle, kind, op):
    for m, k, sizes in ((520, 320, [700, 0, 300, 257]), (300, 1000, [256, 255, 0, 513]), (512, 64, [64, 60, 40]),
                        (264, 40, [50, 90, 47, 60]), (261, 129, [60, 45, 70])):
        got, want, size = run_columns(cg, handle, kind, op, m, k, sizes)
        check(got, want, size, kind, k, dtype_of(kind))


@pytest.mark.parametrize("pads", [(8, 16, 8, 64), (1, 3, 5, 7), (4, 0, 4, 0)])
@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", KINDS)
def test_columns_strides_alpha_beta(cg, handle, kind, op, pads):
    for sizes in ([3, 0, 9, 1], [70, 0, 90, 61], [300, 1, 280]):
        got, want, size = run_columns(cg, handle, kind, op, 144, 104, sizes, alpha=-1.5, beta=0.5, pads=pads, extra_columns=3)
        check(got, want, size, kind, 104, dtype_of(kind))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_columns_of_16_bit_operands_in_fp32(cg, handle, kind):
    for m, k, sizes in ((256, 128, [4, 0, 20]), (257, 65, [150, 1])):
        got, want, size = run_columns(cg, handle, kind, "T", m, k, sizes, beta=-0.25, out=torch.float32)
        check(got, want, size, kind, k, torch.float32)


@pytest.mark.parametrize("op", ["T", "N"])
@pytest.mark.parametrize("kind", ["FP16TCEC", "bf16"])
def test_columns_beta_zero_reads_no_c_and_no_neighbour(cg, handle, kind, op):
    """C full of NaN, NaN beside every operand's values and in another group's matrix and tokens."""
    got, want, size = run_columns(cg, handle, kind, op, 136, 40, [5, 0, 40, 300], pads=(8, 8, 0, 8), c_fill=float("nan"))
    check(got, want, size, kind, 40, dtype_of(kind))
    dt = dtype_of(kind)
    m, k, sizes = 136, 40, [20, 30, 25]
    a = randn(1, 3, m, k, dtype=dt)
    a[1] = float("nan")
    b = randn(2, 75, k, dtype=dt)
    b[20:50] = float("inf")
    c = torch.full((75, m), float("nan"), device="cuda", dtype=dt)
    at = a if op == "T" else a.transpose(1, 2).contiguous()
    assert handle.gemm_grouped(cg.OP_T if op == "T" else cg.OP_N, m, 75, k, 1.0, at, k if op == "T" else m, m * k, b, k, 0.0, c,
                               m, offsets_of(sizes), 3, mode_of(cg, kind), type_code(cg, dt), type_code(cg, dt)) == 0
    assert torch.isnan(c[20:50]).all()
    for g, lo, hi in ((0, 0, 20), (2, 50, 75)):
        want = b[lo:hi].double() @ a[g].double().t().contiguous()
        check(c[lo:hi], want, b[lo:hi].double().abs() @ a[g].double().abs().t().contiguous(), kind, k, dt)


def run_over_k(cg, handle, kind, m, n, sizes, alpha=1.0, beta=0.0, pads=(0, 0, 0, 0), out=None, before_rows=0):
    dt = dtype_of(kind)
    od = out or dt
    k, groups = int(np.sum(sizes)), len(sizes)
    lda, ldb, ldc = m + pads[0], n + pads[1], m + pads[2]
    stride = ldc * n + pads[3]
    a_buf, a = rows((k, m), lda, 1, dt)
    b_buf, b = rows((k, n), ldb, 2, dt)
    c_buf = torch.full((groups * stride + 8,), 7.0, device="cuda", dtype=od)
    c = torch.as_strided(c_buf, (groups, n, m), (stride, ldc, 1))
    c.copy_(randn(3, groups, n, m, dtype=od) if beta != 0 else torch.full((groups, n, m), float("nan"), device="cuda"))
    before, old = c_buf.clone(), c.double().clone()
    st = handle.gemm_grouped_k(m, n, k, alpha, a_buf, lda, b_buf, ldb, beta, c_buf, ldc, stride, offsets_of(sizes), groups,
                               mode_of(cg, kind), type_code(cg, dt), type_code(cg, od))
    assert st == 0
    want = torch.zeros(groups, n, m, device="cuda", dtype=torch.float64)
    size = torch.zeros_like(want)
    for g, (lo, hi) in enumerate(spans(sizes)):
        bt = b[lo:hi].double().t().contiguous()
        want[g] = alpha * (bt @ a[lo:hi].double())
        size[g] = abs(alpha) * (bt.abs() @ a[lo:hi].double().abs())
    if beta != 0:
        want += beta * old
        size += (beta * old).abs()
    torch.cuda.synchronize()
    got = c.clone()
    c.zero_()
    torch.as_strided(before, (groups, n, m), (stride, ldc, 1)).zero_()
    assert torch.equal(c_buf.view(torch.uint8), before.view(torch.uint8)), "written outside the results"
    return got, want, size


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}g{sum(s)}t")
@pytest.mark.parametrize("kind", KINDS)
def test_over_k(cg, handle, kind, sizes):
    for m, n in ((128, 136), (72, 33), (1, 1)):
        got, want, size = run_over_k(cg, handle, kind, m, n, sizes)
        check(got, want, size, kind, max(sizes), dtype_of(kind))
        for g, s in enumerate(sizes):
            if s == 0:
                assert (got[g] == 0).all()


@pytest.mark.parametrize("kind", KINDS)
def test_over_k_tiles_strides_alpha_beta(cg, handle, kind):
    for m, n, sizes, pads in ((520, 264, [300, 0, 65], (8, 16, 8, 64)), (259, 131, [77, 300], (1, 3, 5, 7)),
                              (2048, 2048, [70, 33, 0, 128], (0, 0, 0, 0)), (2056, 1048, [40, 7, 1, 0, 64, 3, 9], (0, 0, 0, 0))):
        got, want, size = run_over_k(cg, handle, kind, m, n, sizes, alpha=0.75, beta=1.0, pads=pads)
        check(got, want, size, kind, max(sizes), dtype_of(kind))


@pytest.mark.parametrize("parts", [2, 3, 16])
@pytest.mark.parametrize("kind", KINDS)
def test_over_k_in_parts(cg, torch_gpu, kind, parts, monkeypatch):
    """K of every group in parts that are added in order: groups shorter than their parts, and the same bits each time."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_KSPLIT", str(parts))
    h = cg.Handle(stream=torch.cuda.current_stream())
    for m, n, sizes, pads in ((264, 136, [300, 0, 65, 1], (0, 0, 0, 0)), (67, 33, [1000], (1, 3, 5, 7))):
        runs = [run_over_k(cg, h, kind, m, n, sizes, alpha=0.75, beta=0.5, pads=pads) for _ in range(2)]
        check(*runs[0], kind, max(sizes), dtype_of(kind))
        assert torch.equal(runs[0][0], runs[1][0]) and h.workspace_size() > 0
    h.close()


def test_over_k_takes_parts_where_tiles_are_few(cg, torch_gpu):
    h = cg.Handle(stream=torch.cuda.current_stream())
    for kind in ("FP16TCEC", "bf16"):
        got, want, size = run_over_k(cg, h, kind, 256, 256, [4000, 96])
        check(got, want, size, kind, 4000, dtype_of(kind))
    assert h.workspace_size() > 0
    h.close()


@pytest.mark.parametrize("cls", [0, 1, 2, 3])
@pytest.mark.parametrize("kind", KINDS + ["i8"])
def test_every_kernel_at_sizes_that_it_would_not_be_chosen_for(cg, handle, kind, cls, monkeypatch):
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    for m, k, sizes in ((264, 200, [1, 0, 300, 33, 129, 257]), (520, 64, [17, 65, 191]), (72, 1000, [20])):
        if kind == "i8":
            run_i8(cg, handle, m, k // 16 * 16, sizes, torch.float32)
            continue
        for op in "TN":
            got, want, size = run_columns(cg, handle, kind, op, m, k, sizes, alpha=1.5, beta=0.5)
            check(got, want, size, kind, k, dtype_of(kind))
        got, want, size = run_over_k(cg, handle, kind, m, 136, sizes)
        check(got, want, size, kind, max(sizes), dtype_of(kind))


@pytest.mark.parametrize("kind", ["f16", "bf16"])
def test_over_k_accumulates_in_fp32(cg, handle, kind):
    got, want, size = run_over_k(cg, handle, kind, 136, 72, [100, 0, 31], beta=1.0, out=torch.float32)
    check(got, want, size, kind, 100, torch.float32)


@pytest.mark.parametrize("kind", ["FP16TCEC", "TF32TCEC", "f16", "bf16"])
def test_over_k_another_groups_nan_stays_there(cg, handle, kind):
    """Groups that end inside a K-step: the neighbour's tokens are infinities and NaN."""
    dt, (m, n), sizes = dtype_of(kind), (136, 128), [37, 50, 45, 0, 3]
    k = sum(sizes)
    a, b = randn(1, k, m, dtype=dt), randn(2, k, n, dtype=dt)
    a[37:87] = float("nan")
    b[37:87] = float("inf")
    c = torch.empty(5, n, m, device="cuda", dtype=dt)
    assert handle.gemm_grouped_k(m, n, k, 1.0, a, m, b, n, 0.0, c, m, m * n, offsets_of(sizes), 5, mode_of(cg, kind),
                                 type_code(cg, dt), type_code(cg, dt)) == 0
    assert torch.isnan(c[1]).all() and (c[3] == 0).all()
    for g, (lo, hi) in enumerate(spans(sizes)):
        if g in (0, 2, 4):
            bt = b[lo:hi].double().t().contiguous()
            check(c[g], bt @ a[lo:hi].double(), bt.abs() @ a[lo:hi].double().abs(), kind, hi - lo, dt)


def randint8(seed, *shape, lo=-127):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randint(lo, 128, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.int8)


def run_i8(cg, handle, m, k, sizes, od, pads=(0, 0, 0, 0), dense=False, lo=-127):
    n, groups = int(np.sum(sizes)), len(sizes)
    lda, ldb, ldc = k + pads[0], k + pads[1], m + pads[2]
    stride = m * lda + pads[3]
    a_buf = torch.full((groups * stride + 16,), 99, device="cuda", dtype=torch.int8)
    a = torch.as_strided(a_buf, (groups, m, k), (stride, lda, 1))
    a.copy_(randint8(1, groups, m, k, lo=lo))
    b_buf = torch.full((n * ldb + 16,), 99, device="cuda", dtype=torch.int8)
    b = torch.as_strided(b_buf, (n, k), (ldb, 1))
    b.copy_(randint8(2, n, k, lo=lo))
    sa, sb = randn(3, groups, m).abs() * 0.01 + 1e-3, randn(4, n).abs() * 0.01 + 1e-3
    c_buf = torch.full((n * ldc + 8,), float("nan"), device="cuda", dtype=od)
    c = torch.as_strided(c_buf, (n, m), (ldc, 1))
    st = handle.gemm_i8(m, n, k, a_buf, lda, stride, sa, b_buf, ldb, sb, c_buf, ldc, type_code(cg, od),
                        None if dense else offsets_of(sizes), groups)
    assert st == 0
    want = torch.empty(n, m, device="cuda", dtype=torch.float64)
    for g, (lo_, hi) in enumerate(spans(sizes)):
        want[lo_:hi] = (b[lo_:hi].double() @ a[g].double().t().contiguous()) * sa[g].double() * sb[lo_:hi, None].double()
    d, tol = (c.double() - want).abs(), (4 * 2.0 ** -24 + ROUND[od]) * want.abs()  # exact sums; converted, scaled twice, rounded
    if od == torch.float16:
        tol = tol + 2.0 ** -25
    assert (d <= tol).all(), float((d / (tol + 1e-30)).max())
    rest = torch.ones(c_buf.numel(), dtype=torch.bool, device="cuda")
    torch.as_strided(rest, (n, m), (ldc, 1)).fill_(False)
    assert torch.isnan(c_buf[rest]).all()


@pytest.mark.parametrize("od", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("sizes", SIZES + [[700, 0, 300, 257], [50, 90, 47, 60]], ids=lambda s: f"{len(s)}g{sum(s)}t")
def test_i8(cg, handle, sizes, od):
    for m, k in ((256, 192), (136, 80), (67, 33), (1, 1)):
        run_i8(cg, handle, m, k, sizes, od)
    run_i8(cg, handle, 144, 112, sizes, od, pads=(16, 32, 8, 64))
    run_i8(cg, handle, 144, 112, sizes, od, pads=(1, 2, 3, 5))


@pytest.mark.parametrize("n", [1, 2, 3, 15, 16, 17, 33, 64, 100, 129, 300, 600])
def test_i8_one_matrix(cg, handle, n):
    for m, k in ((512, 1024), (1000, 1040), (515, 777)):
        run_i8(cg, handle, m, k, [n], torch.bfloat16, dense=True)


def test_i8_longest_sum_of_extremes(cg, handle):
    """k = 131071, all values -128: a sum of 2^31 - 16384, one FP32 rounding, and the next k is refused."""
    k = 131071
    for m, n in ((4, 3), (130, 140)):
        a = torch.full((m, k + 1), -128, device="cuda", dtype=torch.int8)
        b = torch.full((n, k + 1), -128, device="cuda", dtype=torch.int8)
        one, c = torch.ones(max(m, n), device="cuda"), torch.empty(n, m, device="cuda")
        assert handle.gemm_i8(m, n, k, a, k + 1, 0, one, b, k + 1, one, c, m) == 0
        assert (c == np.float32(k * 16384)).all()
        assert handle.gemm_i8(m, n, k + 1, a, k + 1, 0, one, b, k + 1, one, c, m) == cg.STATUS_INVALID_VALUE


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("k", [1, 7, 8, 100, 1024, 4096, 8192, 8200, 20001])
def test_quantize(cg, handle, dtype, k):
    """Scale and integers are those of FP32 division, to the last bit."""
    n = 9
    for pad in (0, 8, 3):
        x = randn(k, n, k + pad, dtype=dtype)
        x[:, k:] = float("nan")
        x[1] = 0
        x[2, :k] *= 1e-4
        x[3, k // 2] = 200.0
        q = torch.full((n, k + pad), 55, device="cuda", dtype=torch.int8)
        s = torch.empty(n, device="cuda")
        assert handle.quantize_i8(k, n, x, k + pad, type_code(cg, dtype), q, k + pad, s) == 0
        xf = x[:, :k].float().cpu().numpy()
        peak = np.abs(xf).max(axis=1)
        scale = peak / np.float32(127)
        want = np.rint(np.divide(xf * np.float32(127), peak[:, None], out=np.zeros_like(xf), where=peak[:, None] != 0))
        if dtype != torch.float32:  # the formula in 64 bits: 16-bit values times 127 are exact, and so are their ties
            x64 = xf.astype(np.float64)
            assert np.array_equal(want, np.rint(np.divide(x64 * 127, peak[:, None], out=np.zeros_like(x64), where=peak[:, None] != 0)))
        assert np.array_equal(s.cpu().numpy(), scale)
        assert np.array_equal(q[:, :k].cpu().numpy(), want.astype(np.int8))
        assert (q[:, k:] == 55).all()
        # in 64 bits: half a step, and what the scale's own rounding adds
        off = np.abs(xf.astype(np.float64) - want * scale[:, None].astype(np.float64))
        assert (off <= scale[:, None] * (0.5 + 127 * 2.0 ** -23)).all()


def test_quantize_without_a_scale(cg, handle):
    """Infinities and NaN take their column with them and no other; the smallest numbers have a scale of zero or a subnormal one."""
    k = 16
    x = randn(1, 7, k)
    x[1, 3], x[2, 5], x[3, 0] = float("inf"), float("nan"), -float("inf")
    x[4] = 1e-45
    x[5] = 0
    x[5, 2] = -3e-43  # (214 of the smallest numbers: a scale of 2 of them, 107 steps)
    q, s = torch.full((7, k), 55, device="cuda", dtype=torch.int8), torch.empty(7, device="cuda")
    assert handle.quantize_i8(k, 7, x, k, cg.R_32F, q, k, s) == 0
    for j in (1, 2, 3):
        assert torch.isnan(s[j]) and (q[j] == 0).all()
    assert s[4] == 0 and (q[4] == 0).all()
    assert s[5] > 0 and q[5, 2] == -107 and q[5].abs().sum() == 107
    for j in (0, 6):
        assert torch.isfinite(s[j]) and q[j].abs().max() == 127
    x = randn(2, 2, k)
    x[0] *= 1e37
    x[0, 7], x[1] = 3.4e38, x[1] * 1e-37
    assert handle.quantize_i8(k, 2, x, k, cg.R_32F, q, k, s) == 0
    x64 = x.double()
    peak = x64.abs().amax(1, keepdim=True)
    assert torch.equal(q[:2].double(), torch.round(x64 * 127 / peak)) and torch.isfinite(s[:2]).all()


def test_nothing_to_do(cg, handle):
    off = offsets_of([2, 0])
    a, b = randn(1, 2, 8, 8), randn(2, 2, 8)
    c = torch.full((2, 8), 3.0, device="cuda")
    args = (a, 8, 64, b, 8)
    for m, n, g in ((0, 2, 2), (8, 0, 2), (8, 2, 0)):
        assert handle.gemm_grouped(cg.OP_T, m, n, 8, 1.0, *args, 0.0, c, 8, off, g, cg.FP16TCEC) == 0
        assert handle.gemm_grouped_k(m, n, 2, 1.0, a, 8, b, 8, 0.0, c, 8, 64, off, g, cg.FP16TCEC) == 0
    assert (c == 3).all()
    # k = 0: A and B are not looked at
    assert handle.gemm_grouped(cg.OP_T, 8, 2, 0, 1.0, None, 0, 0, None, 0, 0.5, c, 8, off, 2, cg.FP16TCEC) == 0
    assert (c == 1.5).all()
    big = torch.full((2, 8, 8), 2.0, device="cuda")
    assert handle.gemm_grouped_k(8, 8, 0, 1.0, None, 0, None, 0, 2.0, big, 8, 64, offsets_of([0, 0]), 2, cg.TF32TCEC) == 0
    assert (big == 4).all()
    h = torch.full((2, 8), 2.0, device="cuda")
    one = torch.ones(16, device="cuda")
    assert handle.gemm_i8(8, 2, 0, None, 0, 0, one, None, 0, one, h, 8) == 0
    assert (h == 0).all()
    s = torch.full((2,), 9.0, device="cuda")
    assert handle.quantize_i8(0, 2, None, 0, cg.R_32F, None, 0, s) == 0 and (s == 0).all()
    assert handle.quantize_i8(4, 0, None, 4, cg.R_32F, None, 4, None) == 0


def test_offsets_of_any_value_stay_inside(cg, handle):
    """Out of range or out of order: nothing outside the operands is touched, the rows of sound groups are right."""
    for kind in ("FP16TCEC", "bf16"):
        dt, m, k, n = dtype_of(kind), 128, 64, 40
        a, b = randn(1, 5, m, k, dtype=dt), randn(2, n, k, dtype=dt)
        c = torch.full((n + 4, m), 7.0, device="cuda", dtype=dt)
        for off in ([0, 10, 5, -3, 1 << 30, 40], [-5, 100, 100, 7, 3, 2], [2147483647, -2147483648, 0, 0, 0, 0]):
            o = torch.tensor(off, dtype=torch.int32, device="cuda")
            assert handle.gemm_grouped(cg.OP_T, m, n, k, 1.0, a, k, m * k, b, k, 0.0, c, m, o, 5, mode_of(cg, kind),
                                       type_code(cg, dt), type_code(cg, dt)) == 0
            g = torch.full((5, k, m + 8), 7.0, device="cuda", dtype=dt)
            assert handle.gemm_grouped_k(m, k, n, 1.0, torch.zeros(n, m, device="cuda", dtype=dt), m, b, k, 0.0, g, m + 8,
                                         k * (m + 8), o, 5, mode_of(cg, kind), type_code(cg, dt), type_code(cg, dt)) == 0
            torch.cuda.synchronize()
            assert (c[n:] == 7).all() and (g[:, :, m:] == 7).all() and (g[:, :, :m] == 0).all()
        # columns of no group keep their values
        c.fill_(7.0)
        o = torch.tensor([5, 9, 9, 9, 9, 30], dtype=torch.int32, device="cuda")
        assert handle.gemm_grouped(cg.OP_T, m, n, k, 1.0, a, k, m * k, b, k, 0.0, c, m, o, 5, mode_of(cg, kind),
                                   type_code(cg, dt), type_code(cg, dt)) == 0
        assert (c[:5] == 7).all() and (c[30:] == 7).all()
        for gi, lo, hi in ((0, 5, 9), (4, 9, 30)):
            w = a[gi].double().t().contiguous()
            check(c[lo:hi], b[lo:hi].double() @ w, b[lo:hi].double().abs() @ w.abs(), kind, k, dt)


def test_refusals(cg, handle):
    bad = cg.STATUS_INVALID_VALUE
    off, a, b, c = offsets_of([4, 4]), randn(1, 2, 8, 8), randn(2, 8, 8), torch.full((8, 8), 3.0, device="cuda")

    def columns(op=cg.OP_T, m=8, n=8, k=8, a=a, lda=8, b=b, ldb=8, c=c, ldc=8, off=off, g=2, mode=cg.FP16TCEC, t=cg.R_32F, tc=cg.R_32F):
        return handle.gemm_grouped(op, m, n, k, 1.0, a, lda, 64, b, ldb, 0.0, c, ldc, off, g, mode, t, tc)

    def over_k(m=8, n=8, k=8, a=a, lda=8, b=b, ldb=8, c=c, ldc=8, stride=64, off=off, g=1, mode=cg.FP16TCEC, t=cg.R_32F, tc=cg.R_32F):
        return handle.gemm_grouped_k(m, n, k, 1.0, a, lda, b, ldb, 0.0, c, ldc, stride, off, g, mode, t, tc)

    for f in (columns, over_k):
        for change in (dict(a=None), dict(b=None), dict(c=None), dict(off=None), dict(lda=7), dict(ldb=7), dict(ldc=7),
                       dict(m=1 << 31), dict(n=1 << 31), dict(k=1 << 31), dict(g=1 << 31), dict(mode=cg.AUTO),
                       dict(mode=cg.FP16TCEC_SCALING), dict(mode=cg.CUBLAS), dict(mode=99), dict(t=cg.R_8I), dict(t=5),
                       dict(tc=cg.R_16F), dict(t=cg.R_16F, tc=cg.R_16BF), dict(t=cg.R_16BF, tc=cg.R_16F)):
            assert f(**change) == bad, change
    assert columns(op=7) == bad and columns(op=cg.OP_N, m=9, ldc=9) == bad
    assert over_k(stride=63, g=2) == bad
    i8, one = torch.zeros(64, device="cuda", dtype=torch.int8), torch.ones(16, device="cuda")

    def ints(m=8, n=8, k=8, a=i8, lda=8, sa=one, b=i8, ldb=8, sb=one, c=c, ldc=8, tc=cg.R_32F, off=None, g=1):
        return handle.gemm_i8(m, n, k, a, lda, 64, sa, b, ldb, sb, c, ldc, tc, off, g)

    for change in (dict(a=None), dict(b=None), dict(c=None), dict(sa=None), dict(sb=None), dict(lda=7), dict(ldb=7), dict(ldc=7),
                   dict(g=2), dict(tc=cg.R_8I), dict(k=131072, lda=131072, ldb=131072), dict(m=1 << 31), dict(n=1 << 31)):
        assert ints(**change) == bad, change
    q = torch.zeros(64, device="cuda", dtype=torch.int8)

    def quant(k=8, n=8, x=b, ldx=8, t=cg.R_32F, q=q, ldq=8, s=one):
        return handle.quantize_i8(k, n, x, ldx, t, q, ldq, s)

    for change in (dict(x=None), dict(q=None), dict(s=None), dict(ldx=7), dict(ldq=7), dict(t=cg.R_8I), dict(k=1 << 31), dict(n=1 << 31)):
        assert quant(**change) == bad, change
    L = cg.lib()
    assert L.cuMpSGEMM_gemm_grouped(None, cg.OP_T, 8, 8, 8, None, None, 8, 64, None, 8, None, None, 8, None, 2, 1, 0, 0) == bad
    assert L.cuMpSGEMM_gemm_grouped_k(None, 8, 8, 8, None, None, 8, None, 8, None, None, 8, 64, None, 2, 1, 0, 0) == bad
    assert L.cuMpSGEMM_gemm_i8(None, 8, 8, 8, None, 8, 64, None, None, 8, None, None, 8, 0, None, 1) == bad
    assert L.cuMpSGEMM_quantize_i8(None, 8, 8, None, 8, 0, None, 8, None) == bad
    torch.cuda.synchronize()
    assert (c == 3).all()


@pytest.mark.parametrize("kind", ["FP16TCEC", "bf16"])
def test_gradients_match_the_formulas_and_differences(cg, handle, kind):
    """Loss = sum over tokens of <r, W_g x>, r fixed: dL/dx = W_g^T r, dL/dW_g = sum r x^T, taken by autograd in FP64 and by
    differences of the forward product, which is linear in x and in W: a step of any size gives the derivative, up to
    the rounding of the two products."""
    dt, (m, k), sizes = dtype_of(kind), (96, 72), [30, 0, 41, 1]
    n, G, off = sum(sizes), len(sizes), offsets_of(sizes)
    w, x, r = randn(1, G, m, k, dtype=dt), randn(2, n, k, dtype=dt), randn(3, n, m, dtype=dt)
    t, mode = type_code(cg, dt), mode_of(cg, kind)
    dx, dw = torch.empty_like(x), torch.empty(G, m, k, device="cuda")
    assert handle.gemm_grouped(cg.OP_N, k, n, m, 1.0, w, k, m * k, r, m, 0.0, dx, k, off, G, mode, t, t) == 0
    # dW_g stored as W_g is, k contiguous: C_g = sum over tokens of x r^T, k x m
    assert handle.gemm_grouped_k(k, m, n, 1.0, x, k, r, m, 0.0, dw, k, m * k, off, G, mode, t, cg.R_32F) == 0
    w64, x64 = w.double().requires_grad_(), x.double().requires_grad_()
    loss = sum(((x64[lo:hi] @ w64[g].t()) * r[lo:hi].double()).sum() for g, (lo, hi) in enumerate(spans(sizes)))
    loss.backward()
    size_x, size_w = torch.empty_like(x64), torch.zeros_like(w64)
    for g, (lo, hi) in enumerate(spans(sizes)):
        size_x[lo:hi] = r[lo:hi].double().abs() @ w[g].double().abs()
        size_w[g] = r[lo:hi].double().abs().t() @ x[lo:hi].double().abs()
    check(dx, x64.grad, size_x.detach(), kind, m, dt)
    check(dw, w64.grad, size_w.detach(), kind, max(sizes), torch.float32)

    def forward(w, x):
        y = torch.empty(n, m, device="cuda")
        assert handle.gemm_grouped(cg.OP_T, m, n, k, 1.0, w, k, m * k, x, k, 0.0, y, m, off, G, mode, t, cg.R_32F) == 0
        return y.double()

    y0 = forward(w, x)
    for token, i in ((0, 0), (35, 71), (71, 40)):
        x1 = x.clone()
        x1[token, i] = x[token, i] + 4
        step = float(x1[token, i].double() - x[token, i].double())
        diff = float(((forward(w, x1) - y0) * r.double()).sum()) / step
        err = (SPLIT[kind] + (k + 2) * 2.0 ** -24) * float(r[token].double().abs().sum()) * 4 * np.sqrt(k) * 4
        assert abs(diff - float(dx[token, i])) <= err + ROUND[dt] * abs(diff)
    for g, i, j in ((0, 5, 6), (2, 95, 71), (3, 0, 0)):
        w1 = w.clone()
        w1[g, i, j] = w[g, i, j] + 4
        step = float(w1[g, i, j].double() - w[g, i, j].double())
        diff = float(((forward(w1, x) - y0) * r.double()).sum()) / step
        lo, hi = spans(sizes)[g]
        err = (SPLIT[kind] + (k + 2) * 2.0 ** -24) * float(r[lo:hi, i].double().abs().sum()) * 4 * np.sqrt(k) * 4
        assert abs(diff - float(dw[g, i, j])) <= err


def test_repeats_bit_for_bit_and_on_another_stream(cg, torch_gpu):
    h = cg.Handle()
    side = torch.cuda.Stream()
    for kind, m, k, sizes in (("FP16TCEC", 200, 300, [70, 3, 0, 90]), ("bf16", 512, 512, [3, 1, 9, 2]), ("f16", 136, 1000, [300, 20])):
        dt = dtype_of(kind)
        n, G, off = sum(sizes), len(sizes), offsets_of(sizes)
        w, x = randn(1, G, m, k, dtype=dt), randn(2, n, k, dtype=dt)
        ys = [torch.empty(n, m, device="cuda", dtype=dt) for _ in range(3)]
        gs = [torch.empty(G, k, m, device="cuda", dtype=dt) for _ in range(3)]
        torch.cuda.synchronize()
        for i, s in enumerate((torch.cuda.current_stream(), side, side)):
            h.set_stream(s)
            t = type_code(cg, dt)
            assert h.gemm_grouped(cg.OP_T, m, n, k, 1.0, w, k, m * k, x, k, 0.0, ys[i], m, off, G, mode_of(cg, kind), t, t) == 0
            assert h.gemm_grouped_k(m, k, n, 1.0, ys[i], m, x, k, 0.0, gs[i], m, m * k, off, G, mode_of(cg, kind), t, t) == 0
        torch.cuda.synchronize()
        for i in (1, 2):
            assert torch.equal(ys[0], ys[i]) and torch.equal(gs[0], gs[i])
    h.close()


def test_graph_replays_take_the_offsets_of_the_time(cg, torch_gpu):
    m, k, n, G = 256, 192, 96, 6
    w, x = randn(1, G, m, k), randn(2, n, k)
    w8, sw = randint8(3, G, m, k), randn(4, G, m).abs()
    q, sx = torch.empty(n, k, device="cuda", dtype=torch.int8), torch.empty(n, device="cuda")
    off = offsets_of([16] * 6)
    y, g, z = torch.empty(n, m, device="cuda"), torch.empty(G, k, m, device="cuda"), torch.empty(n, m, device="cuda")
    h = cg.Handle()

    def calls(y, g, z):
        assert h.gemm_grouped(cg.OP_T, m, n, k, 1.0, w, k, m * k, x, k, 0.0, y, m, off, G, cg.FP16TCEC) == 0
        assert h.gemm_grouped_k(m, k, n, 1.0, y, m, x, k, 0.0, g, m, m * k, off, G, cg.TF32TCEC) == 0
        assert h.quantize_i8(k, n, x, k, cg.R_32F, q, k, sx) == 0
        assert h.gemm_i8(m, n, k, w8, k, m * k, sw, q, k, sx, z, m, cg.R_32F, off, G) == 0

    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        h.set_stream(side)
        calls(y, g, z)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            calls(y, g, z)
    for sizes in ([16] * 6, [96, 0, 0, 0, 0, 0], [0, 1, 50, 0, 44, 1], [16] * 6):
        off.copy_(offsets_of(sizes))
        x.copy_(randn(sum(i * s for i, s in enumerate(sizes)), n, k))
        for t in (y, g, z):
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        eager = [torch.empty_like(t) for t in (y, g, z)]
        with torch.cuda.stream(side):
            calls(*eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((y, g, z), eager))
    h.close()


@pytest.mark.parametrize("kind", ["FP16TCEC", "bf16"])
def test_offsets_past_32_bits(cg, handle, kind):
    """Matrices, tokens and results more than 2^32 bytes and elements apart."""
    dt, m, k, sizes = dtype_of(kind), 64, 64, [2, 0, 3]
    t, far = type_code(cg, dt), (1 << 31) + 64
    buf = torch.empty(2 * far + m * k, device="cuda", dtype=dt)
    w = torch.as_strided(buf, (3, m, k), (far, k, 1))
    w.copy_(randn(1, 3, m, k, dtype=dt))
    x = randn(2, 5, k, dtype=dt)
    off = offsets_of(sizes)
    y = torch.empty(5, m, device="cuda", dtype=dt)
    for op, a64 in ((cg.OP_T, w.double().transpose(1, 2).contiguous()), (cg.OP_N, w.double())):
        assert handle.gemm_grouped(op, m, 5, k, 1.0, buf, 64, far, x, k, 0.0, y, m, off, 3, mode_of(cg, kind), t, t) == 0
        for g, (lo, hi) in enumerate(spans(sizes)):
            check(y[lo:hi], x[lo:hi].double() @ a64[g], x[lo:hi].double().abs() @ a64[g].abs(), kind, k, dt)
    # results of the groups, as far apart
    r = randn(3, 5, m, dtype=dt)
    assert handle.gemm_grouped_k(m, k, 5, 1.0, r, m, x, k, 0.0, buf, 64, far, off, 3, mode_of(cg, kind), t, t) == 0
    for g, (lo, hi) in enumerate(spans(sizes)):
        bt = x[lo:hi].double().t().contiguous()
        check(w[g], bt @ r[lo:hi].double(), bt.abs() @ r[lo:hi].double().abs(), kind, hi - lo, dt)
    # tokens and their results, far apart: leading dimensions of 2^30
    ld = (1 << 30) + 8
    xb = torch.as_strided(buf, (4, k), (ld, 1))
    xb.copy_(x[:4])
    yb = torch.empty(3 * ld + m, device="cuda", dtype=dt)
    w1 = randn(5, 2, m, k, dtype=dt)
    assert handle.gemm_grouped(cg.OP_T, m, 4, k, 1.0, w1, k, m * k, buf, ld, 0.0, yb, ld, offsets_of([1, 3]), 2,
                               mode_of(cg, kind), t, t) == 0
    y4 = torch.as_strided(yb, (4, m), (ld, 1))
    for g, lo, hi in ((0, 0, 1), (1, 1, 4)):
        a64 = w1[g].double().t().contiguous()
        check(y4[lo:hi], x[lo:hi].double() @ a64, x[lo:hi].double().abs() @ a64.abs(), kind, k, dt)
    assert handle.gemm_grouped_k(m, k, 4, 1.0, buf, ld, x, k, 0.0, yb, m, m * k, offsets_of([1, 3]), 2, mode_of(cg, kind), t, t) == 0
    c = yb[:2 * m * k].view(2, k, m)
    for g, lo, hi in ((0, 0, 1), (1, 1, 4)):
        bt = x[lo:hi].double().t().contiguous()
        check(c[g], bt @ x[lo:hi].double(), bt.abs() @ x[lo:hi].double().abs(), kind, hi - lo, dt)
