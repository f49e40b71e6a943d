"""moe_forward with int8 experts: the activations are quantised from what they are, whatever their type, once per token."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _layer(T, E, K, H, D, dtype):
    from dsl_tool_b200 import MoEWeights
    g = torch.Generator(device="cuda").manual_seed(T)
    x = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    logits = torch.randn(T, E, generator=g, device="cuda")
    return x, logits, MoEWeights.pack(torch.randn(E, 2 * H, K, generator=g, device="cuda") * 0.1,
                                      torch.randn(E, D, H, generator=g, device="cuda") * 0.1, "int8")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,K,H,D", [(1, 6, 256, 128, 192), (37, 6, 272, 128, 192), (300, 5, 512, 144, 136)])
def test_rows_are_quantised_from_their_own_type(cuda_device, dtype, T, E, K, H, D):
    """One expert a token, so its weight is 1 and the result is the expert's row: the products of the expert-sorted rows, bit for
    bit (integer sums, the same roundings)."""
    from dsl_tool_b200 import linear, moe_forward
    x, logits, w = _layer(T, E, K, H, D, dtype)
    expert = logits.argmax(1)
    order = torch.sort(expert, stable=True)[1]
    offs = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offs[1:] = torch.bincount(expert, minlength=E).cumsum(0)
    h = linear(x[order], w.gate_up, expert_offsets=offs, activation="swiglu", out_dtype=torch.bfloat16)
    y = linear(h, w.down, expert_offsets=offs, out_dtype=torch.bfloat16)
    want = torch.empty_like(y)
    want[order] = y
    assert torch.equal(moe_forward(x, logits, w, 1, out_dtype=torch.bfloat16), want)


def test_a_token_has_one_scale_for_all_its_experts(cuda_device, monkeypatch):
    from dsl_tool_b200 import moe, moe_forward
    x, logits, w = _layer(20, 6, 256, 128, 192, torch.float32)
    rows = []
    monkeypatch.setattr(moe, "quantize_int8", lambda t, quantize=moe.quantize_int8: (rows.append(tuple(t.shape)), quantize(t))[1])
    moe_forward(x, logits, w, 3)
    assert rows == [(20, 256)]


def test_experts_of_two_ranks(cuda_device):
    """Every token has one expert, so one rank's share is the result and the other's is zero; rows of other ranks stay unwritten."""
    from dsl_tool_b200 import moe
    T, E, K, H, D = 50, 6, 256, 128, 192
    x, logits, whole = _layer(T, E, K, H, D, torch.float32)
    g = torch.Generator(device="cuda").manual_seed(T)
    torch.randn(T, K, generator=g, device="cuda"), torch.randn(T, E, generator=g, device="cuda")
    gu, dn = torch.randn(E, 2 * H, K, generator=g, device="cuda") * 0.1, torch.randn(E, D, H, generator=g, device="cuda") * 0.1
    shares = [moe.moe_partial(x, logits, moe.MoEWeights.pack(gu, dn, "int8", rank=r, world=2), 1) for r in range(2)]
    assert torch.equal(shares[0] + shares[1], moe.moe_partial(x, logits, whole, 1))
