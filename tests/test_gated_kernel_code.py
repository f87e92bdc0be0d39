"""What the compiler made of the kernels of 8-bit floating point and of the gated blocks, read back from the built library."""
import re

from test_grouped_kernel_code import k_loops, of_experts
from test_kernel_code import kernels  # noqa: F401 (a fixture)


def test_no_scratch_in_the_loops_of_f8(kernels):  # noqa: F811
    all_of_them = {**of_experts(kernels, "amd9f8_kernel"), **of_experts(kernels, "f8_stream_kernel")}
    assert len(all_of_them) > 30 and all(k_loops(c) for c in all_of_them.values())
    bad = [n for n, c in all_of_them.items() if any("scratch_" in t for body in k_loops(c) for t in body)]
    assert not bad, bad


def test_loops_of_f8_that_load_to_lds_wait_once_a_step(kernels):  # noqa: F811
    """One wait for the loads in front of each barrier (at the end of K it is another one); and a step's additions are among its MFMAs,
    never four MFMAs in a row without one."""
    loops = 0
    for name, code in of_experts(kernels, "amd9f8_kernel").items():
        for body in k_loops(code):
            if not any(t.startswith("global_load_lds") for t in body):
                continue
            loops += 1
            barriers = sum(t.startswith("s_barrier") for t in body)
            waits = sum(bool(re.match(r"s_waitcnt .*vmcnt", t)) for t in body)
            assert barriers >= 1 and waits <= 2 * barriers, (name, barriers, waits)
            assert sum(t.startswith("v_fma") for t in body) >= 4 * sum("f8f6f4" in t for t in body), name
            row = longest = 0
            for t in body:
                row = row + 1 if "f8f6f4" in t else 0 if t.startswith("v_fma") else row
                longest = max(longest, row)
            assert longest <= 4, (name, longest)
    assert loops > 40


def test_no_packed_fp32(kernels):  # noqa: F811
    bad = [n for n, c in kernels.items() if ("f8_" in n or "quantize_f8" in n or "grouped_" in n) and
           any(t.startswith(("v_pk_fma_f32", "v_pk_mul_f32", "v_pk_add_f32")) for t, _, _ in c)]
    assert not bad, bad
