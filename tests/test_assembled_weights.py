"""Weights put together by hand in front of the calls that read them by pointer: what is not as pack_weight lays it out is refused, or
goes through the form that converts it.  The refusals run on the CPU: nothing is launched."""
from dataclasses import replace

import pytest
import torch

from dsl_tool_b200 import _lib, gemm_kernels, linear
from dsl_tool_b200.quantize import PackedWeight

N, K = 256, 512
FORMATS = ["fp8", "fp8_block128", "int8", "nvfp4", "mxfp4", "bf16"]


def packed(fmt, groups=2):
    """The tensors that pack_weight would make, with nothing in them."""
    if fmt == "bf16":
        return PackedWeight(fmt, torch.zeros((groups * N, K), dtype=torch.bfloat16), None, None, groups, N, K)
    if fmt == "int8":
        return PackedWeight(fmt, torch.zeros((groups * N, K), dtype=torch.int8), torch.ones(groups * N), None, groups, N, K)
    q = torch.zeros((groups * N, K // 2 if fmt.endswith("fp4") else K), dtype=torch.uint8)
    if fmt == "fp8":
        return PackedWeight(fmt, q, torch.ones(1), None, groups, N, K)
    if fmt == "fp8_block128":
        return PackedWeight(fmt, q, torch.ones((groups, N // 128, K // 128)), None, groups, N, K)
    sf = torch.zeros(groups * (N // 128) * (K // (16 if fmt == "nvfp4" else 32) // 4) * 512, dtype=torch.uint8)
    return PackedWeight(fmt, q, sf, torch.ones(1) if fmt == "nvfp4" else None, groups, N, K)


CHANGES = {
    "n too large": lambda w: replace(w, n=2 * w.n),
    "a row missing": lambda w: replace(w, q=w.q[:-1]),
    "columns apart": lambda w: replace(w, q=w.q.t().contiguous().t()),
    "wider elements": lambda w: replace(w, q=w.q.to(torch.float32)),
    "scales missing": lambda w: replace(w, scale=None),
    "scales too few": lambda w: replace(w, scale=w.scale.reshape(-1)[:-1]),
    "scales of another type": lambda w: replace(w, scale=w.scale.to(torch.float64)),
    "scales apart": lambda w: replace(w, scale=torch.stack((w.scale, w.scale), -1)[..., 0]),
    "scales elsewhere": lambda w: replace(w, scale=w.scale.to("meta")),
    "global scale missing": lambda w: replace(w, global_scale=None),
    "global scale of another type": lambda w: replace(w, global_scale=w.global_scale.double()),
}


def changed(fmt):
    for name, change in CHANGES.items():
        if ("scale" in name and fmt == "bf16") or ("global" in name and fmt != "nvfp4"):
            continue
        if name == "scales apart" and fmt == "fp8":          # one element is contiguous however it lies
            continue
        yield name, change(packed(fmt))


@pytest.mark.parametrize("fmt", FORMATS)
def test_descriptor_of_an_assembled_weight(fmt):
    assert gemm_kernels._new_weight_desc(packed(fmt)).n == N
    for name, w in changed(fmt):
        with pytest.raises(ValueError, match="not laid out as pack_weight"):
            gemm_kernels._new_weight_desc(w)
            pytest.fail(name)


@pytest.mark.parametrize("fmt", ["fp8", "fp8_block128", "int8"])
def test_quantised_activations_meet_only_packed_weights(fmt, monkeypatch):
    """`linear(act_scale=)` reads the weight by pointer: it refuses before anything is launched."""
    def launch(*args):
        raise AssertionError("launched")
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(gemm_kernels, "_run", launch)
    q = torch.zeros((4, K), dtype=torch.int8 if fmt == "int8" else torch.uint8)
    s = torch.ones({"fp8": (1,), "fp8_block128": (4, K // 128), "int8": (4,)}[fmt])
    offs = torch.tensor([0, 2, 4], dtype=torch.int32)
    with pytest.raises(AssertionError, match="launched"):
        linear(q, packed(fmt), act_scale=s, expert_offsets=offs)
    for name, w in changed(fmt):
        with pytest.raises(ValueError, match="not laid out as pack_weight"):
            linear(q, w, act_scale=s, expert_offsets=offs)
            pytest.fail(name)


def test_scales_of_quantised_activations_keep_their_order(monkeypatch):
    """[M, K/128] and nothing else of as many values: the transposed one is another scale for every element."""
    def launch(*args):
        raise AssertionError("launched")
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(gemm_kernels, "_run", launch)
    q, w = torch.zeros((8, K), dtype=torch.uint8), packed("fp8_block128", 1)
    for shape in ((K // 128, 8), (8 * (K // 128),), (2, 4, K // 128)):
        with pytest.raises(ValueError, match="act_scale must be"):
            linear(q, w, act_scale=torch.ones(shape))
    with pytest.raises(AssertionError, match="launched"):
        linear(q, w, act_scale=torch.ones((K // 128, 8)).t())


@pytest.mark.parametrize("fmt", FORMATS)
def test_kept_descriptor_follows_the_weight(fmt):
    """Another tensor in the weight, at whatever address, and other sizes are looked at again."""
    w = packed(fmt)
    d = gemm_kernels._weight_desc(w)
    assert gemm_kernels._weight_desc(w) is d
    whole = w.q
    w.q = whole[:-1]                                         # the same address, a row less
    with pytest.raises(ValueError, match="not laid out"):
        gemm_kernels._weight_desc(w)
    w.q = whole
    assert gemm_kernels._weight_desc(w).q == whole.data_ptr()
    w.n *= 2
    with pytest.raises(ValueError, match="not laid out"):
        gemm_kernels._weight_desc(w)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FORMATS)
def test_refused_or_converted(cuda_device, fmt):
    """`linear` on plain activations: the step-by-step form converts what only wants converting."""
    from dsl_tool_b200 import pack_weight
    g = torch.Generator(device="cuda").manual_seed(2)
    x = torch.randn(33, K, generator=g, device="cuda").bfloat16()
    w = pack_weight(torch.randn(N, K, generator=g, device="cuda") * 0.05, fmt)
    want = linear(x, w)
    if fmt != "bf16":
        assert torch.equal(linear(x, replace(w, q=w.q.t().contiguous().t())), want)
        with pytest.raises(ValueError, match="scale missing"):
            linear(x, replace(w, scale=None))
    if fmt in ("fp8", "fp8_block128", "int8"):
        assert torch.equal(linear(x, replace(w, scale=w.scale.double())), want)
    if fmt == "nvfp4":
        assert torch.equal(linear(x, replace(w, global_scale=w.global_scale.double())), want)
        with pytest.raises(ValueError, match="global_scale missing"):
            linear(x, replace(w, global_scale=None))
    with pytest.raises(ValueError):
        linear(x, replace(w, q=w.q[:-1]))


@pytest.mark.parametrize("fmt", ["fp8", "fp8_block128"])
@pytest.mark.parametrize("short", ["row_scale", "col_scale"])
def test_factors_of_the_epilogue_are_counted(fmt, short, monkeypatch):
    """One per token, one per output channel of every group: fewer would be read past their end."""
    monkeypatch.setattr(_lib, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "lib", lambda: None)
    monkeypatch.setattr(gemm_kernels, "_run", lambda *args: pytest.fail("launched"))
    q, w, offs = torch.zeros((4, K), dtype=torch.uint8), packed(fmt), torch.tensor([0, 2, 4], dtype=torch.int32)
    s = torch.ones((1,) if fmt == "fp8" else (4, K // 128))
    count = 4 if short == "row_scale" else 2 * N
    for factors in (torch.ones(count - 1), torch.ones(1), torch.ones(N)[:0]):
        with pytest.raises(ValueError, match=f"{short} must hold {count} values"):
            linear(q, w, act_scale=s, expert_offsets=offs, **{short: factors})
        with pytest.raises(ValueError, match=f"{short} must hold {count} values"):
            if fmt == "fp8":
                gemm_kernels.gemm_fp8_quantized(q, w.q, 1.0, 1.0, n=N, expert_offsets=offs, **{short: factors})
            else:
                gemm_kernels.gemm_fp8_groupwise_quantized(q, w.q, s, w.scale, n=N, sb_block=True, expert_offsets=offs, **{short: factors})
        with pytest.raises(ValueError, match=f"{short} must hold {count} values"):
            gemm_kernels._linear_one_call(torch.zeros((4, K)), w, torch.float32, offs, factors if short == "row_scale" else None,
                                          factors if short == "col_scale" else None, None, None)
