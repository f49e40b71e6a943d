"""Products and quantisers of no rows: an empty result, from every entry point and in every form of a call."""
import pytest
import torch

pytestmark = pytest.mark.gpu
N, K = 256, 512


def _w():
    return torch.randn(N, K, device="cuda") * 0.05


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_quantisers(cuda_device, dtype):
    from dsl_tool_b200 import quantize_fp4, quantize_fp8, quantize_int8
    x = torch.empty((0, K), dtype=dtype, device="cuda")
    for mode, shape in (("per_tensor", (1,)), ("groupwise", (0, K // 128)), ("block128", (0, K // 128))):
        q, s = quantize_fp8(x, mode)
        assert q.shape == (0, K) and s.shape == shape
    assert torch.equal(quantize_fp8(x)[1], quantize_fp8(torch.zeros((1, K), device="cuda"))[1])      # the scale of zeros
    assert quantize_fp8(x, scale=0.5)[1].item() == 0.5
    for fmt in ("nvfp4", "mxfp4"):
        q, sf, gs = quantize_fp4(x, fmt)
        zeros = quantize_fp4(torch.zeros((1, K), device="cuda"), fmt)
        assert q.shape == (0, K // 2) and (gs is None if fmt == "mxfp4" else torch.equal(gs, zeros[2]))
        offs = torch.zeros(4, dtype=torch.int32, device="cuda")
        q, sf, gs = quantize_fp4(x, fmt, group_offsets=offs)
        assert q.shape == (0, K // 2) and not sf.any()
    assert quantize_fp4(x, "nvfp4", global_scale=0.5)[2].item() == 0.5
    assert quantize_fp4(x, "nvfp4", global_scale="per_token")[2].shape == (0,)
    q, s = quantize_int8(x)
    assert q.shape == (0, K) and s.shape == (0,)


@pytest.mark.parametrize("layout", ["kn", "nk"])
def test_gemms_of_plain_operands(cuda_device, layout):
    from dsl_tool_b200 import bf16_gemm, fp4_gemm, fp8_gemm, int8_gemm
    w = _w()
    b = w.t().contiguous() if layout == "kn" else w
    for dtype in (torch.float32, torch.bfloat16):
        a = torch.empty((0, K), dtype=dtype, device="cuda")
        for mode in ("per_tensor", "groupwise", "block128"):
            assert fp8_gemm(a, b, mode=mode, b_layout=layout).shape == (0, N)
        for mx in (False, True):
            assert fp4_gemm(a, b, use_mxfp4=mx, b_layout=layout).shape == (0, N)
        assert int8_gemm(a, b, b_layout=layout).shape == (0, N)
        for c in (b, b.bfloat16()):
            assert bf16_gemm(a, c, b_layout=layout).shape == (0, N)


def test_gemms_of_quantised_operands(cuda_device):
    from dsl_tool_b200 import fp4_gemm, fp8_gemm, int8_gemm, quantize_fp4, quantize_fp8, quantize_int8
    w, x = _w(), torch.empty((0, K), device="cuda")
    for out in ("float32", "bfloat16"):
        q, s = quantize_fp8(x)
        qw, sw = quantize_fp8(w)
        for b, layout in ((qw, "nk"), (qw.t().contiguous(), "kn")):
            assert fp8_gemm(q, b, s, sw, b_layout=layout, out_dtype=out).shape == (0, N)
        q, s = quantize_fp8(x, "groupwise")
        qw, sw = quantize_fp8(w, "block128")
        assert fp8_gemm(q, qw, s, sw, mode="block128", b_layout="nk", out_dtype=out).shape == (0, N)
        per_column = torch.ones((K // 128, N), device="cuda")
        assert fp8_gemm(q, qw, s, per_column, mode="groupwise", b_layout="nk", out_dtype=out).shape == (0, N)
        for fmt in ("nvfp4", "mxfp4"):
            q, sf, gs = quantize_fp4(x, fmt)
            qw, sfw, gsw = quantize_fp4(w, fmt)
            assert fp4_gemm(q, qw, sf, sfw, format=fmt, b_layout="nk", global_scale_a=gs, global_scale_b=gsw, out_dtype=out).shape == (0, N)
        q, s = quantize_int8(x)
        qw, sw = quantize_int8(w)
        assert int8_gemm(q, qw, s, sw, b_layout="nk", out_dtype=out).shape == (0, N)


@pytest.mark.parametrize("fmt", ["fp8", "fp8_block128", "int8", "nvfp4", "mxfp4", "bf16"])
def test_linear_and_groups(cuda_device, fmt):
    from dataclasses import replace

    from dsl_tool_b200 import grouped_gemm, linear, pack_weight
    one, three = pack_weight(_w(), fmt), pack_weight(torch.randn(3, N, K, device="cuda"), fmt)
    offs = torch.zeros(4, dtype=torch.int32, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):                       # fp32 with a bf16 weight takes the step-by-step form
        x = torch.empty((0, K), dtype=dtype, device="cuda")
        assert linear(x, one).shape == (0, N)
        assert linear(x, three, expert_offsets=offs).shape == (0, N)
        name = {"fp8_block128": "fp8_groupwise"}.get(fmt, fmt)
        assert grouped_gemm(x, three, expert_offsets=offs, format=name).shape == (0, N)
        assert grouped_gemm(torch.empty((3, 0, K), dtype=dtype, device="cuda"), three, format=name).shape == (3, 0, N)
        if fmt != "bf16":                                               # a weight that goes step by step
            apart = replace(one, q=one.q.t().contiguous().t())
            assert linear(x, apart).shape == (0, N)
        if fmt in ("nvfp4", "fp8"):
            q, sf, gs = linear(x, one, out_dtype="nvfp4", out_global_scale=0.5)
            assert q.shape == (0, N // 2) and gs.item() == 0.5


def test_rows_of_nothing(cuda_device):
    """An int8 row without elements has the scale of a row of zeros."""
    from dsl_tool_b200 import quantize_int8
    for rows in (1, 5):
        q, s = quantize_int8(torch.empty((rows, 0), device="cuda"))
        assert q.shape == (rows, 0) and torch.equal(s, quantize_int8(torch.zeros((rows, 16), device="cuda"))[1])
