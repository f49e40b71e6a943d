"""moe_decode near the ends of fp32: what the formula gives is finite, so the result is."""
import pytest
import torch

from tests.test_gpu_moe_decode import FORMATS, bound, far, layer, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [2.0 ** 61, 2.0 ** -61])
def test_results_near_the_ends(cuda_device, fmt, scale):
    """Rows of x of 2^61 have hidden values of 2^122 and results about as large; the sums before the weights' scales are up to 2^13
    times that.  (2^-61: silu(g) u is g u / 2 there, 2^-123 of the smallest normal numbers.)"""
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(4, 4, 256, 128, 128, fmt)
    x = (x.float().clamp(-4, 4) * torch.tensor([1.0, scale, 1.0, scale], device="cuda")[:, None]).bfloat16()
    want, got = layer(x, logits, w, 2), moe_decode(x, logits, w, 2)
    assert (want.abs() < torch.finfo(torch.float32).max / 16).all()
    for t in range(4):
        # 2^-149, the step of subnormal numbers, in each of 128 hidden values and in the result
        floor = 2.0 ** -149 * 128 / want[t].norm().item() if scale < 1 and t % 2 else 0.0
        assert torch.isfinite(got[t]).all() and far(got[t], want[t]) <= bound(fmt, x.dtype) + floor
