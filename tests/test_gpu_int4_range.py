"""Quantising weights near the largest value of their type."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("largest", [2.0 ** 100, 2.0 ** 126, 2.0 ** 127, 1.5 * 2.0 ** 127])
def test_a_range_wider_than_fp32_has_a_finite_scale(largest):
    import swiftrt_b200 as srt
    g = torch.Generator().manual_seed(3)
    w = ((torch.rand(64, 40, generator=g) * 2 - 1) * largest).to(torch.bfloat16)
    w[0], w[1] = largest, -largest
    q = srt.quantize_int4(w.cuda(), 32, True)
    scale = ((w.double().view(2, 32, 40).amax(1).clamp_min(0) - w.double().view(2, 32, 40).amin(1).clamp_max(0)) / 15).to(torch.bfloat16)
    assert torch.equal(q.scales.cpu(), scale)
    # half a step of its scale, at the ends up to a whole one (the zero point is rounded too), and the rounding of the scale and the result
    step = scale.double().repeat_interleave(32, 0)
    rounding = torch.finfo(torch.bfloat16).eps / 2
    assert bool(((q.dequantize().cpu().double() - w.double()).abs() <= step + 3 * rounding * w.double().abs()).all())
