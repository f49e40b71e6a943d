"""moe_decode on fp32 activations: they, and the hidden activation after them, keep two 16-bit terms."""
import pytest
import torch

from tests.test_gpu_moe_decode import FORMATS, bound, far, layer, make

pytestmark = pytest.mark.gpu
SIZES = [(1, 8, 2, 256, 128, 256), (3, 4, 4, 384, 256, 200), (9, 6, 2, 640, 128, 264), (16, 8, 8, 256, 256, 128), (32, 33, 32, 128, 128, 48),
         (5, 1, 1, 1536, 1280, 56), (2, 64, 8, 2048, 768, 2048), (7, 3, 2, 288, 96, 50)]


def fp32_bound(fmt, K, H):
    """Relative error in the 2-norm.  A value is a f16 term (half a step: 2^-11 of it) and one of the rest (2^-11 of that, or 2^-25 where
    the rest is subnormal), so off by 2^-22 of itself and 2^-25 beside values around 1: 2^-21 leaves room for rows of smaller values.
    x, passed on by gate and up, and the hidden activation: 3.1 such roundings, as in `bound` (bf16 weights: two bf16 terms, 2^-16).
    Sums: the tensor cores cut each addition of 16 products off at 2^-23 of the partial sum at worst, two terms of K / 16 of them, then
    of H / 16."""
    return 3.1 * 2.0 ** (-16 if fmt == "bf16" else -21) + 2 * (K + H) / 16 * 2.0 ** -23


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,E,k,K,H,D", SIZES)
def test_layer(cuda_device, fmt, T, E, k, K, H, D):
    from dsl_tool_b200 import moe_decode
    if fmt == "fp8_block128" and (K % 128 or H % 128):
        K, H = 256, 128
    x, logits, w = make(T, E, K, H, D, fmt, dtype=torch.float32)
    want = layer(x, logits, w, k)
    got = moe_decode(x, logits, w, k)
    assert far(got, want) <= fp32_bound(fmt, K, H)
    assert torch.equal(moe_decode(x, logits, w, k), got)
    assert torch.equal(moe_decode(x, logits, w, k, out_dtype=torch.bfloat16), got.bfloat16())


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** -8, 2.0 ** 20, 2.0 ** 61])
def test_scale_of_the_rows(cuda_device, fmt, scale):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(6, 4, 256, 128, 128, fmt, dtype=torch.float32)
    x = x.clamp(-4, 4)
    x[1::2] *= scale
    want, got = layer(x, logits, w, 2), moe_decode(x, logits, w, 2)
    for t in range(6):
        assert torch.isfinite(got[t]).all() and far(got[t], want[t]) <= fp32_bound(fmt, 256, 128)


@pytest.mark.parametrize("fmt", FORMATS)
def test_special_values_stay_in_their_row(cuda_device, fmt):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(12, 3, 256, 128, 128, fmt, dtype=torch.float32)
    clean = moe_decode(x, logits, w, 2)
    x[2, 5], x[9, 0], x[4] = float("nan"), float("inf"), 0.0
    got = moe_decode(x, logits, w, 2)
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[9]).all() and not got[4].any()
    keep = [t for t in range(12) if t not in (2, 4, 9)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("fmt,K,H,T", [("fp8", 128, 20480, 5), ("int8", 32768, 32, 3), ("nvfp4", 14336, 128, 20), ("mxfp4", 64, 14336, 9),
                                       ("mxfp4", 32768, 64, 2), ("nvfp4", 36000, 32, 1)])
def test_rows_that_do_not_all_fit(cuda_device, fmt, K, H, T):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(T, 2, K, H, 64, fmt, dtype=torch.float32)
    assert far(moe_decode(x, logits, w, 2), layer(x, logits, w, 2)) <= fp32_bound(fmt, K, H)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4", "int8"])
@pytest.mark.parametrize("E,k,T", [(1024, 32, 32), (3, 1, 31), (2, 2, 4)])
def test_many_and_few_experts(cuda_device, fmt, E, k, T):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(T, E, 128, 32, 24, fmt, dtype=torch.float32)
    assert far(moe_decode(x, logits, w, k), layer(x, logits, w, k)) <= fp32_bound(fmt, 128, 32)


def test_sixteen_bit_activations_as_before(cuda_device):
    """The choice is the caller's, by the type of x: fp32 of bf16 values is nearer to 64 bits than the bf16 values are."""
    from dsl_tool_b200 import moe_decode
    for fmt in ("fp8", "nvfp4", "mxfp4"):
        x, logits, w = make(8, 8, 512, 256, 256, fmt)
        want = layer(x, logits, w, 2)
        short, full = moe_decode(x, logits, w, 2), moe_decode(x.float(), logits, w, 2)
        assert far(full, want) <= fp32_bound(fmt, 512, 256) < far(short, want) <= bound(fmt, x.dtype)
