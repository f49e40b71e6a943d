"""moe_decode: a NaN among a token's logits is its result, whatever the others are; the other tokens do not see it."""
import pytest
import torch

from tests.test_gpu_moe_decode import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("E,D", [(10, 192), (40, 75), (300, 1032)])
def test_nan_logits(cuda_device, E, D, logits_dtype, out_dtype):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(8, E, 256, 128, D, "nvfp4", logits_dtype=logits_dtype)
    nan, inf = float("nan"), float("inf")
    logits[2] = -inf
    clean = moe_decode(x, logits, w, 4, out_dtype=out_dtype)
    logits[0] = nan                                          # nothing else
    logits[1], logits[1, E - 1] = -inf, nan                  # beside minus infinities
    logits[3, 0] = nan                                       # among finite ones
    logits[4, 1:], logits[4, 0] = nan, 0.5                   # one that can be chosen
    logits[5, 3:], logits[5, 1] = -inf, nan                  # fewer than k
    for renormalize in (True, False):
        got = moe_decode(x, logits, w, 4, renormalize=renormalize, out_dtype=out_dtype)
        for t in (0, 1, 3, 4, 5):
            assert torch.isnan(got[t]).all(), t
        assert not got[2].any()
    got = moe_decode(x, logits, w, 4, out_dtype=out_dtype)
    assert torch.isfinite(clean).all() and ((got[6:].double() - clean[6:].double()).norm() / clean[6:].double().norm()).item() <= 1e-5 + (
        0 if out_dtype == torch.float32 else 2.0 ** -8)      # sums split otherwise, and a bf16 rounding that this tips
