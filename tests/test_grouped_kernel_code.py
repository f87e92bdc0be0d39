"""What the compiler made of the kernels of experts' products, read back from the built library."""
import re

from test_kernel_code import kernels  # noqa: F401 (a fixture)


def of_experts(kernels, name="grouped_kernel"):
    return {n: c for n, c in kernels.items() if name in n}


def k_loops(code):
    """Innermost loops that load and multiply: their instructions.  (Spans that store results, and larger ones that begin or
    end inside a loop, are jumps back to code that the compiler has laid out ahead.)"""
    back = []
    for text, at, target in code:
        jump = re.match(r"s_branch (\d+)", text)
        if jump:
            target = at + 4 + 4 * (int(jump.group(1)) - (65536 if int(jump.group(1)) >= 32768 else 0))
        if target is not None and target <= at:
            back.append((target, at))
    found = []
    for lo, hi in sorted(back, key=lambda s: s[1] - s[0]):
        if any(lo <= b and a <= hi for a, b, _ in found):
            continue
        body = [t for t, a, _ in code if lo <= a <= hi]
        loads = any(t.startswith(("global_load", "buffer_load")) for t in body)
        if loads and any(t.startswith("v_mfma") for t in body) and not any(t.startswith("global_store") for t in body):
            found.append((lo, hi, body))
    return [body for _, _, body in found]


def test_no_scratch_in_the_loops(kernels):
    all_of_them = {**of_experts(kernels), **of_experts(kernels, "grouped_stream_kernel")}
    assert len(all_of_them) > 70 and all(k_loops(c) for c in all_of_them.values())
    bad = [n for n, c in all_of_them.items() if any("scratch_" in t for body in k_loops(c) for t in body)]
    assert not bad, bad


def test_loops_that_load_to_lds_wait_once_a_step(kernels):
    """One wait for the loads, the kernel's own, in front of each barrier (at the end of K it is another one); any more
    would be the compiler's, and for all loads."""
    loops = 0
    for name, code in of_experts(kernels).items():
        for body in k_loops(code):
            if not any(t.startswith("global_load_lds") for t in body):
                continue
            loops += 1
            barriers = sum(t.startswith("s_barrier") for t in body)
            waits = sum(bool(re.match(r"s_waitcnt .*vmcnt", t)) for t in body)
            assert barriers >= 1 and waits <= 2 * barriers, (name, barriers, waits)
    assert loops > 30
