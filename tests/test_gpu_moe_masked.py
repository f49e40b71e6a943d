"""Routing where a mask leaves a token fewer experts than it has slots: every slot gets one all the same, masked ones with weight 0, so
that no row of the plan stays unwritten."""
import numpy as np
import pytest
import torch

from tests.test_gpu_moe_decode import layer, make

pytestmark = pytest.mark.gpu
INF = float("inf")


def masked(logits, k):
    """A batch of logits (at least 9 rows) with masks of every kind."""
    E = logits.shape[1]
    low = torch.finfo(logits.dtype).min
    logits[1] = -INF                                  # nobody
    logits[2, 1:] = -INF                              # one, the first
    logits[3, :-1] = -INF                             # one, the last
    logits[4] = low                                   # all at the type's lowest value
    logits[5, : E // 2] = low
    logits[5, E // 2 + 1:] = -INF
    logits[6, ::2] = -INF
    logits[7, E // 3] = INF
    return logits


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("E,k", [(3, 3), (8, 5), (33, 32), (64, 8), (65, 8), (96, 32), (200, 20), (1024, 32)])
def test_route(cuda_device, E, k, renorm, dtype):
    from dsl_tool_b200.moe import route
    g = torch.Generator(device="cuda").manual_seed(E)
    logits = masked(torch.randn(20, E, generator=g, device="cuda").to(dtype), k)
    logits[9, E - 1] = float("nan")
    logits[10] = float("nan")
    logits[11, 1:] = float("nan")
    logits[11, 0] = -INF
    ids, w = route(logits, k, renorm)
    l = logits.double().cpu().numpy()
    want = np.argsort(-l, axis=1, kind="stable")[:, :k]          # NaN behind everything
    assert np.array_equal(ids.cpu().numpy(), want)
    nan = [9, 10, 11, 7]                                          # an infinity's softmax is NaN too
    assert torch.isnan(w[[9, 10, 11]]).all() and not w[1].any()
    rest = [t for t in range(20) if t not in nan and t != 1]
    p = torch.softmax(torch.from_numpy(l), 1).gather(1, torch.from_numpy(want))[rest]
    if renorm:
        p = p / p.sum(1, keepdim=True)
    got = w[rest].double().cpu()
    # fp32: expf off by 2 ulp, a sum over at most 1024 experts in 32 + 5 steps, a division, a second sum of 32 and a division
    assert ((got - p).abs() <= p * 2.0 ** -24 * (4 + 37 + 1 + 32 + 1 + 4) + 2.0 ** -126).all()


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4", "fp8", "fp8_block128", "int8", "bf16"])
@pytest.mark.parametrize("E", [8, 80])
def test_layer_has_no_stale_rows(cuda_device, fmt, E):
    """The hidden activation of every planned row is written, so what lay in memory before is in no scale and no result."""
    from dsl_tool_b200 import moe_forward
    x, logits, w = make(40, E, 256, 128, 192, fmt)
    logits = masked(logits, 5)
    logits[7, E // 3] = 0.0
    results = []
    for value in (float("nan"), 1e30, 0.0):
        poison = [torch.empty(n, device="cuda").fill_(value) for n in (1 << 22, 40 * 5 * 64, 40 * 5 * 128, 1 << 16, 40 * 5 * 256)]
        torch.cuda.synchronize()
        del poison
        results.append(moe_forward(x, logits, w, 5))
    assert torch.isfinite(results[0]).all() and not results[0][1].any()
    assert all(torch.equal(r, results[0]) for r in results)
    if fmt == "bf16":
        # bf16 hidden activation and expert results: half a step of 8 bits, 2^-8, each (their errors are independent: the norm's too)
        want = layer(x, logits, w, 5)
        assert ((results[0].double() - want).norm() / want.norm()).item() <= 2 * 2.0 ** -8


def test_plan_of_ids_without_an_expert(cuda_device):
    """An id outside the experts gets no row: -1."""
    from dsl_tool_b200 import moe
    ids = torch.tensor([[0, 7], [2, -1], [1, 0]], dtype=torch.int32, device="cuda")
    p = moe.plan(ids, torch.ones(3, 2, device="cuda"), 3)
    assert p.offsets.tolist() == [0, 2, 3, 4] and p.dest.tolist() == [0, -1, 3, -1, 2, 1]
