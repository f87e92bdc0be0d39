"""Values of gated blocks where their activations' arguments are large: results in FP32 to a few units in the last place, gradients at
infinity."""
import pytest
import torch

from test_gpu_gated import ACTS
from test_gpu_grouped import dtype_of, mode_of, type_code

pytestmark = pytest.mark.gpu


def tail(act, g):
    """act(g) in FP64, without 1 - erf"""
    return g / (1 + torch.exp(-g)) if act == "SILU" else g * 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)


@pytest.fixture(params=["F8_SUMS_FP32", "F8_SUMS_FAST"])
def sums(cg, handle, request):
    assert handle.set_f8_sums(getattr(cg, request.param)) == 0
    yield request.param
    assert handle.set_f8_sums(cg.F8_SUMS_FP32) == 0


@pytest.mark.parametrize("cls", ["1", "2", "3", "4"])
@pytest.mark.parametrize("act", ["SILU", "GELU"])
def test_fp32_results_of_f8_blocks(cg, handle, act, sums, cls, monkeypatch):
    """One feature: G = w s, w E4M3 and s, the scale of the gate's matrix, of six bits, so that G and, for GELU, its square are exact, and
    U = 1.  What is left: the exponential, its argument and its correction 2^-23 each, the polynomial 2^-24 and nine roundings of 2^-24, quotient and
    products three more, 2^-20 together, of the value itself.  (The hardware's exponential rounds an argument of 70 log2 e to
    2^-18 alone.)"""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", cls)
    w = (torch.arange(-12, -3, device="cuda") if act == "GELU" else torch.arange(-80, -3, 4, device="cuda")).to(torch.float8_e4m3fn)
    m, n = len(w), 33
    one = torch.ones(m, 1, device="cuda").to(torch.float8_e4m3fn)
    x = torch.ones(n, 1, device="cuda").to(torch.float8_e4m3fn)
    s = 0.75 + torch.arange(n, device="cuda").float() / 64
    got, want = torch.empty(n, m, device="cuda"), torch.empty(n, m, device="cuda", dtype=torch.float64)
    scale_one, xs = torch.ones(1, device="cuda"), torch.ones(n, device="cuda")
    rows = torch.empty(n, m, device="cuda")
    for j in range(n):
        assert handle.gemm_gated_f8(getattr(cg, act), m, n, 1, w, one, 1, m, cg.R_8F_E4M3, s[j:j + 1], scale_one, 1, x, 1, cg.R_8F_E4M3, xs, rows, m,
                                    cg.R_32F, None, 1) == 0
        assert torch.equal(rows, rows[:1].expand(n, m))
        got[j], want[j] = rows[0], tail(act, w.double() * s[j].double())
    # (the factor of G, below 2^-126 from G = -87.3 on, is no normal number then, and the hardware's reciprocal makes it zero: G 2^-126)
    bound = 2.0 ** -20 * want.abs() + 2.0 ** -126 * (w.double()[None] * s.double()[:, None]).abs()
    assert float(((got.double() - want).abs() / bound).max()) <= 1.0


@pytest.mark.parametrize("cls", ["1", "3"])
@pytest.mark.parametrize("kind", ["FP16TCEC", "TF32TCEC", "f16", "bf16"])
@pytest.mark.parametrize("act", ACTS)
def test_the_gradient_at_infinity(cg, handle, act, kind, cls, monkeypatch):
    """A projection that was stored as an infinity (in FP16, one beyond 65504) has the value and slope that any large one has: itself and 1,
    or 0 and 0; one that is no number has none.  D = 2, U = 3."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", cls)
    dt = dtype_of(kind)
    z = torch.tensor([1.0, float("inf"), 3e4, float("nan"), 100.0, -float("inf"), -3e4], device="cuda").to(dt)[None].contiguous()
    m = z.shape[1]
    w, x, up = torch.ones(1, m, 1, device="cuda", dtype=dt), torch.full((1, 1), 2.0, device="cuda", dtype=dt), torch.full_like(z, 3.0)
    d = torch.full((3, 1, m), 7.0, device="cuda", dtype=dt)
    assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), m, 1, 1, w, 1, m, x, 1, z, up, m, d[0], d[1], m, d[2], m, None, 1,
                                      mode_of(cg, kind), type_code(cg, dt)) == 0
    assert d[0, 0, [1, 2, 4]].tolist() == [6.0, 6.0, 6.0]
    assert d[1, 0, 1] == float("inf") and d[2, 0, 1] == float("inf")
    assert not d[:, 0, 5:].any()
    assert bool(torch.isnan(d[1:, 0, 3]).all()) and (act == "RELU" or bool(torch.isnan(d[0, 0, 3])))


@pytest.mark.parametrize("act", ACTS)
def test_a_projection_beyond_fp16(cg, handle, act):
    """G = 2^17, U = 2^-3 in FP16: the result is 2^14, G is stored as an infinity, and its gradient is D U.  G = -2^17: zeros."""
    w = torch.tensor([[[2.0 ** 9]], [[2.0 ** -11]]], device="cuda", dtype=torch.float16)
    x, one = torch.full((1, 1), 2.0 ** 8, device="cuda", dtype=torch.float16), torch.ones(1, 1, 1, device="cuda", dtype=torch.float16)
    c, z = torch.empty(1, 1, device="cuda", dtype=torch.float16), torch.empty(2, 1, 1, device="cuda", dtype=torch.float16)
    assert handle.gemm_gated(cg.OP_T, getattr(cg, act), 1, 1, 1, w[0], w[1], 1, 1, x, 1, c, 1, z[0], z[1], 1, None, 1, cg.FP16TC, cg.R_16F) == 0
    assert float(c) == 2.0 ** 14 and z.flatten().tolist() == [float("inf"), 0.125]
    d = torch.empty(2, 1, 1, device="cuda", dtype=torch.float16)
    assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), 1, 1, 1, one, 1, 1, x, 1, z[0], z[1], 1, d[0], d[1], 1, None, 0, None, 1, cg.FP16TC,
                                      cg.R_16F) == 0
    assert float(d[0]) == 32.0
    assert handle.gemm_gated(cg.OP_T, getattr(cg, act), 1, 1, 1, -w[0], w[1], 1, 1, x, 1, c, 1, z[0], z[1], 1, None, 1, cg.FP16TC, cg.R_16F) == 0
    assert float(c) == 0.0 and z.flatten().tolist() == [-float("inf"), 0.125]
    assert handle.gemm_gated_backward(cg.OP_T, getattr(cg, act), 1, 1, 1, one, 1, 1, x, 1, z[0], z[1], 1, d[0], d[1], 1, c, 1, None, 1, cg.FP16TC,
                                      cg.R_16F) == 0
    assert not d.any() and not c.any()
