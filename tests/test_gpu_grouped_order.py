"""Which tile a workgroup of gemm_grouped_k takes where groups are ranked by length, and quantize_i8 near ties.

Bounds as in test_gpu_grouped.py."""
import numpy as np
import pytest
import torch

from test_gpu_grouped import check, dtype_of, mode_of, offsets_of, randn, run_over_k, type_code

pytestmark = pytest.mark.gpu

# Results of 1032 x 1100: 81 tiles of 128, 25 - 45 of the larger ones; all groups' together are more than the CUs.
LENGTHS = {
    "even": [512] * 9,
    "two long ones": [2900, 3, 0, 1600, 1, 0, 64, 65, 130],
    "one has everything": [0, 0, 0, 0, 4700, 0, 0, 0, 0],
    "ascending": [8 * g * g for g in range(14)],
    "seventeen": [int(x) for x in np.random.RandomState(3).permutation([0, 1, 5, 40, 64, 100, 128, 129, 150, 160, 200, 250, 300, 320, 500, 600, 700])],
}


@pytest.mark.parametrize("sizes", LENGTHS.values(), ids=LENGTHS.keys())
@pytest.mark.parametrize("kind", ["FP16TCEC", "TF32TCEC", "bf16"])
@pytest.mark.parametrize("cls", [0, 1])
def test_every_tile_is_taken_once(cg, handle, kind, cls, sizes, monkeypatch):
    """beta = 1: a tile that two workgroups had would be added to twice."""
    monkeypatch.setenv("CUMPSGEMM_FORCE_TILE_CLASS", str(cls))
    monkeypatch.setenv("CUMPSGEMM_FORCE_KSPLIT", "1")
    got, want, size = run_over_k(cg, handle, kind, 1032, 1100, sizes, beta=1.0)
    check(got, want, size, kind, max(sizes), dtype_of(kind))


@pytest.mark.parametrize("groups", [64, 65, 70])
def test_many_groups(cg, handle, groups):
    rng = np.random.RandomState(groups)
    sizes = [int(x) for x in 150 * np.exp(0.8 * rng.randn(groups))]
    sizes[7] = 0
    for kind in ("FP16TCEC", "f16"):
        got, want, size = run_over_k(cg, handle, kind, 264, 300, sizes, beta=1.0)
        check(got, want, size, kind, max(sizes), dtype_of(kind))


def test_ranked_offsets_of_any_value_stay_inside(cg, handle):
    for kind in ("FP16TCEC", "bf16"):
        dt, m, n, k = dtype_of(kind), 1032, 1096, 2000
        a, b = torch.zeros(k, m, device="cuda", dtype=dt), randn(1, k, n, dtype=dt)
        for off in ([0, 900, 500, -3, 1 << 30, 2000, 7, 7, 7, 2100], [2147483647, -2147483648, 0, 0, 1999, 1, 2000, 0, 2000, 0]):
            c = torch.full((9, n, m + 8), 7.0, device="cuda", dtype=dt)
            assert handle.gemm_grouped_k(m, n, k, 1.0, a, m, b, n, 0.0, c, m + 8, n * (m + 8),
                                         torch.tensor(off, dtype=torch.int32, device="cuda"), 9, mode_of(cg, kind),
                                         type_code(cg, dt), type_code(cg, dt)) == 0
            torch.cuda.synchronize()
            assert (c[:, :, m:] == 7).all() and (c[:, :, :m] == 0).all()


def test_tokens_of_no_group_do_not_count(cg, handle):
    """Offsets that begin behind the first token and end before the last."""
    m, n, k, dt = 1032, 1096, 3000, torch.float32
    a, b = randn(1, k, m), randn(2, k, n)
    a[:200], b[2600:] = float("nan"), float("nan")
    off = [200, 900, 900, 1000, 1001, 1100, 1300, 2500, 2510, 2600]
    c = torch.empty(9, n, m, device="cuda")
    assert handle.gemm_grouped_k(m, n, k, 1.0, a, m, b, n, 0.0, c, m, m * n, torch.tensor(off, dtype=torch.int32, device="cuda"), 9,
                                 cg.FP16TCEC, cg.R_32F, cg.R_32F) == 0
    for g in range(9):
        x, y = a[off[g]:off[g + 1]].double(), b[off[g]:off[g + 1]].double().t().contiguous()
        check(c[g], y @ x, y.abs() @ x.abs(), "FP16TCEC", 1200, dt)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=str)
@pytest.mark.parametrize("columns", [3, 2100])
def test_quantize_every_16_bit_value_goes_where_64_bits_say(cg, handle, dtype, columns):
    """All values up to a maximum, for maxima over a power of two: ties go to the even integer."""
    every = torch.arange(65536, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
    every = every[torch.isfinite(every.float())]
    steps = 128 if dtype == torch.bfloat16 else 1024
    for step in range(0, steps, steps // 16 + 1):
        peak = torch.tensor(2.0 + 2.0 * step / steps, device="cuda").to(dtype)
        v = every[every.float().abs() <= peak.float()]
        k = 1000 if columns > 3 else v.numel() // 3
        v = v[torch.randperm(v.numel(), generator=torch.Generator().manual_seed(step)).cuda()][:columns * (k - 1)]
        n = v.numel() // (k - 1)
        x = torch.cat([v[:n * (k - 1)].view(n, k - 1), peak.expand(n, 1)], dim=1).contiguous()
        q, scale = torch.empty(n, k, device="cuda", dtype=torch.int8), torch.empty(n, device="cuda")
        assert handle.quantize_i8(k, n, x, k, type_code(cg, dtype), q, k, scale) == 0
        want = torch.round(x.double() * 127 / x.double().abs().amax(1, keepdim=True))
        assert torch.equal(q, want.to(torch.int8))


@pytest.mark.parametrize("k", [8, 500, 1024, 1032, 2048, 2056, 4096, 4104])
@pytest.mark.parametrize("n", [2047, 2048, 5000])
def test_quantize_with_any_number_of_waves(cg, handle, n, k):
    for dtype in (torch.float32, torch.bfloat16):
        x = randn(k, n, k, dtype=dtype)
        q, scale = torch.empty(n, k, device="cuda", dtype=torch.int8), torch.empty(n, device="cuda")
        assert handle.quantize_i8(k, n, x, k, type_code(cg, dtype), q, k, scale) == 0
        xs = x.double()
        # (divided on the CPU: torch multiplies by 1 / 127 on the GPU)
        assert np.array_equal(scale.cpu().numpy(), x.float().abs().amax(1).cpu().numpy() / np.float32(127))
        step = xs.abs().amax(1, keepdim=True) / 127
        # half a step, and the two roundings of a quotient of up to 127
        assert ((xs / step - q.double()).abs() <= 0.5 + 127 * 2.0 ** -23).all()
