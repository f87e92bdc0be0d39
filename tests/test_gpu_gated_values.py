"""Values of gated blocks where their activations' arguments are large: results in FP32 to a few units in the last place, gradients at
infinity."""
import math

import pytest
import torch

from test_gpu_gated import act_of

pytestmark = pytest.mark.gpu


def tail(act, g):
    """act(g) in FP64, without 1 - erf"""
    return g / (1 + torch.exp(-g)) if act == "SILU" else g * 0.5 * torch.special.erfc(-g * 0.5 ** 0.5)


@pytest.mark.parametrize("cls", ["1", "2", "3", "4"])
@pytest.mark.parametrize("sums", ["F8_SUMS_FP32", "F8_SUMS_FAST"])
@pytest.mark.parametrize("act", ["SILU", "GELU"])
def test_fp32_results_of_f8_blocks(cg, handle, act, sums, cls, monkeypatch):
    """One feature: G = w s, w E4M3 and s, the scale of the gate's matrix, of six bits, so that G and, for GELU, its square are exact, and U = 1.  What is left: the
    exponential, its argument and its correction 2^-23 each, the polynomial 2^-24 and nine roundings of 2^-24, quotient and
    products three more, 2^-20 together, of the value itself.  (The hardware's exponential rounds an argument of 70 log2 e to
    2^-18 alone.)"""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", cls)
    assert handle.set_f8_sums(getattr(cg, sums)) == 0
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
    assert handle.set_f8_sums(cg.F8_SUMS_FP32) == 0
    # (the factor of G, below 2^-126 from G = -87.3 on, is no normal number then, and the hardware's reciprocal makes it zero: G 2^-126)
    bound = 2.0 ** -20 * want.abs() + 2.0 ** -126 * (w.double()[None] * s.double()[:, None]).abs()
    assert float(((got.double() - want).abs() / bound).max()) <= 1.0
