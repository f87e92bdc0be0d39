"""How products of 8-bit floating point are summed, as far as it shows on the CPU: what the setting refuses, and the matrix
instructions of the kernels as compiled."""
import ctypes
import re

import pytest

import cumpsgemm_amd as cg
from cumpsgemm_amd import _lib
from test_grouped_kernel_code import k_loops, of_experts
from test_kernel_code import kernels  # noqa: F401 (a fixture)


@pytest.mark.parametrize("sums,status", [(0, 0), (1, 0), (2, 3), (-1, 3)])
def test_the_setting(sums, status):
    memory = ctypes.create_string_buffer(4096)
    h = cg.Handle.__new__(cg.Handle)
    h._L, h._h, h._addr, h.close = _lib.lib(), ctypes.c_void_p(ctypes.addressof(memory)), ctypes.addressof(memory), lambda: None
    assert (cg.F8_SUMS_FP32, cg.F8_SUMS_FAST) == (0, 1)
    assert h.set_f8_sums(sums) == status
    assert any(memory.raw) == (sums == 1)
    h._h = None
    assert h.set_f8_sums(sums) == cg.STATUS_INVALID_VALUE


def test_exact_kernels_multiply_in_bf16(kernels):  # noqa: F811
    """The last argument of a tile's type says whether its sums are exact: then no FP8 MFMA is in it, and else no other."""
    count = {"0": 0, "1": 0}
    for name, code in of_experts(kernels, "amd9f8_kernel").items():
        exact = re.search(r"8EpilogueE\dELb([01])E", name).group(1)
        f8, bf16 = (sum(what in t for t, _, _ in code) for what in ("f8f6f4", "v_mfma_f32_16x16x32_bf16"))
        assert (f8 == 0 and bf16 > 0) if exact == "1" else (f8 > 0 and bf16 == 0), name
        count[exact] += 1
    assert count["1"] >= 30 and count["0"] >= 20, count
    for name, code in of_experts(kernels, "f8_stream_kernel").items():
        assert not any("f8f6f4" in t for t, _, _ in code), name


def test_additions_are_among_the_mfmas(kernels):  # noqa: F811
    """FAST kernels: never four FP8 MFMAs in a row without a multiply-add, a loop's end and its beginning together too."""
    loops = 0
    for name, code in of_experts(kernels, "amd9f8_kernel").items():
        for body in k_loops(code):
            if not any(t.startswith("global_load_lds") for t in body) or not any("f8f6f4" in t for t in body):
                continue
            loops += 1
            row = longest = 0
            for t in body + body:
                row = row + 1 if "f8f6f4" in t else 0 if t.startswith("v_fma") else row
                longest = max(longest, row)
            assert longest <= 3, (name, longest)
    assert loops > 20


@pytest.mark.parametrize("ld", [0, 1, 16])
@pytest.mark.parametrize("op", [cg.OP_T, cg.OP_N])
@pytest.mark.parametrize("sums", [0, 1])
def test_more_tiles_than_a_launch_has_are_refused(sums, op, ld):
    """As an invalid value, whichever tiles the operands and sums can take; nothing is launched."""
    memory = ctypes.create_string_buffer(4096)
    h = cg.Handle.__new__(cg.Handle)
    h._L, h._h, h._addr, h.close = _lib.lib(), ctypes.c_void_p(ctypes.addressof(memory)), ctypes.addressof(memory), lambda: None
    assert h.set_f8_sums(sums) == 0
    most, p = (1 << 31) - 16, 0x1000
    a = dict(m=most, n=most, k=160, stridea=0, type_a=cg.R_8F_E4M3, stridescale=0, b=p, ldb=160 + ld, type_b=cg.R_8F_E4M3, scale_b=p, c=p, ldc=most)
    assert h.gemm_f8(op_a=op, a=p, lda=(160 if op == cg.OP_T else most) + ld, scale_a=p, **a) == cg.STATUS_INVALID_VALUE
    assert h.gemm_gated_f8(activation=cg.SILU, gate=p, up=p, lda=160 + ld, scale_gate=p, scale_up=p, **a) == cg.STATUS_INVALID_VALUE
