"""The experts' layer of cumpsgemm_amd/experts.py: grouping on the CPU, the whole layer on the GPU."""
import numpy as np
import pytest
import torch

from cumpsgemm_amd import experts


@pytest.mark.parametrize("tokens,count", [(0, 3), (1, 1), (1, 5), (7, 3), (1000, 8), (64, 300)])
def test_grouping(tokens, count):
    e = torch.from_numpy(np.random.RandomState(tokens).randint(0, count, tokens))
    order, offsets = experts.group_by_expert(e, count)
    assert offsets.dtype == torch.int32 and len(offsets) == count + 1 and offsets[0] == 0 and offsets[-1] == tokens
    for g in range(count):
        mine = order[offsets[g]:offsets[g + 1]]
        assert torch.equal(mine, torch.nonzero(e == g)[:, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1000, 512, 768, 8), (37, 100, 33, 5), (3, 256, 64, 16)], ids=str)
def test_a_training_step_and_serving(torch_gpu, shape):
    """Roundings are independent: 2^-22 of a product's size and 2^-24 sqrt(K) of the sums' in FP32, 2^-8 / sqrt(3) in BF16.
    8-bit integers: a step is max / 127, off by a twelfth of its square on average, for tokens and channels alike: with a
    maximum below 6 standard deviations, 2 * (6 / 127)^2 / 12 is below 0.02^2."""
    errors = experts.main(shape)
    for name, e in errors.items():
        bar = 0.02 if name.startswith("8-bit") else 2.0 ** -8 if name in ("BF16 y", "BF16 dx") else 2.0 ** -21 + 2.0 ** -23 * max(shape) ** 0.5
        assert 0 <= e <= bar, (name, e, bar)
    assert len(errors) == 7


@pytest.mark.gpu
def test_gradients_of_the_weights_are_added(torch_gpu, cg):
    torch.manual_seed(0)
    h = cg.Handle(stream=torch.cuda.current_stream())
    for dtype in (torch.float32, torch.float16):
        layer = experts.Experts(h, torch.randn(4, 48, 64, device="cuda").to(dtype), cg.TF32TCEC)
        x, dy = torch.randn(50, 64, device="cuda").to(dtype), torch.randn(50, 48, device="cuda").to(dtype)
        e = torch.randint(3, (50,), device="cuda")  # (the last expert has no token)
        _, saved = layer.forward(x, e)
        _, dw = layer.backward(saved, dy)
        once = dw.clone()
        _, again = layer.backward(saved, dy, dw)
        assert again is dw and (once[3] == 0).all()
        # the second call adds in FP32 what the first stored: one rounding
        assert ((dw - 2 * once).abs() <= 2.0 ** -23 * dw.abs()).all()
    h.close()
