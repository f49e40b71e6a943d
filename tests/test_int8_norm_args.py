"""Argument checks of the int8 and norm entry points, and the container of an int8 weight.  CPU: nothing is launched."""
import ctypes

import pytest
import torch

from dsl_tool_b200 import _lib
from dsl_tool_b200.build import build_library
from dsl_tool_b200.quantize import PackedWeight
from dsl_tool_b200.weight_store import load_packed, save_packed


@pytest.fixture(scope="module")
def cdll():
    build_library()
    return _lib.lib()


def _buffer():
    raw = ctypes.create_string_buffer(4096 + 256)
    return raw, (ctypes.addressof(raw) + 255) // 256 * 256


def test_quant_int8_arguments(cdll):
    keep, p = _buffer()
    assert cdll.dsl_quant_int8(None, 0, 4, 16, p, p, None) == -1
    assert cdll.dsl_quant_int8(p, 0, 4, 16, None, p, None) == -1
    assert cdll.dsl_quant_int8(p, 3, 4, 16, p, p, None) == -4
    assert cdll.dsl_quant_int8(p, 0, 4, 24, p, p, None) == -2              # cols % 16
    assert cdll.dsl_quant_int8(p, 0, -1, 16, p, p, None) == -2
    assert cdll.dsl_quant_int8(p, 0, 1 << 31, 16, p, p, None) == -2
    assert cdll.dsl_quant_int8(p, 0, 4, 32784, p, p, None) == -6           # longer than a CTA holds
    assert cdll.dsl_quant_int8(p + 4, 0, 4, 16, p, p, None) == -3
    assert cdll.dsl_quant_int8(p, 0, 4, 16, p, p + 8, None) == -3
    assert cdll.dsl_quant_int8(p, 0, 0, 16, p, p, None) == 0               # nothing to do, nothing launched
    del keep


def test_rms_norm_arguments(cdll):
    keep, p = _buffer()

    def call(x=p, dtype=0, rows=4, cols=32, residual=None, gain=p, gain_dtype=0, fmt=1, sum_out=None, out=p, scale_out=p, scale_in=None):
        return cdll.dsl_rms_norm(x, dtype, rows, cols, residual, gain, gain_dtype, 1e-6, fmt, sum_out, out, scale_out, scale_in, None)
    assert call(x=None) == -1 and call(gain=None) == -1 and call(out=None) == -1
    assert call(residual=p) == -1                                          # a residual without a place for the sum
    assert call(scale_out=None) == -1 and call(fmt=2, scale_out=None) == -1
    assert call(fmt=3, scale_in=None) == -1
    assert call(dtype=3) == -4 and call(gain_dtype=-1) == -4 and call(fmt=4) == -4
    assert call(cols=40) == -2 and call(cols=0) == -2 and call(rows=-1) == -2
    assert call(cols=32784) == -6
    assert call(x=p + 8) == -3 and call(gain=p + 2) == -3 and call(out=p + 4) == -3
    assert call(residual=p + 4, sum_out=p) == -3 and call(residual=p, sum_out=p + 8) == -3
    assert call(rows=0) == 0
    del keep


def test_gemm_int8_arguments(cdll):
    keep, p = _buffer()
    ep = _lib.Epilogue()
    ref = ctypes.byref(ep)
    assert cdll.dsl_gemm_int8(p, p, p, 16, 4, 16, 32, None, 1, None, None, None) == -1
    assert cdll.dsl_gemm_int8(p, p, p, 16, 4, 16, 24, None, 1, ref, None, None) == -2      # K % 16
    assert cdll.dsl_gemm_int8(p, p, p, 8, 4, 16, 32, None, 1, ref, None, None) == -2       # ldc < N
    assert cdll.dsl_gemm_int8(p, p, p, 16, 4, 16, 131072, None, 1, ref, None, None) == -6  # sums could leave int32
    assert cdll.dsl_gemm_int8(p, p, p, 16, 4, 16, 32, p, 5000, ref, None, None) == -6
    ep.b_is_kn = 1
    assert cdll.dsl_gemm_int8(p, p, p, 16, 4, 16, 32, None, 1, ref, None, None) == -4      # K-major weights only
    ep.b_is_kn = 0
    assert cdll.dsl_gemm_int8(p, p, p, 16, 0, 16, 32, None, 1, ref, None, None) == 0
    w = _lib.Weight()
    w.format, w.groups, w.n, w.k, w.q, w.scale = _lib.W_INT8, 1, 16, 32, p, None
    assert cdll.dsl_linear(p, 0, 4, ctypes.byref(w), None, p, 4096, p, 16, ref, None, None) == -1
    assert cdll.dsl_linear_quantized(p, p, 4, ctypes.byref(w), None, p, 16, ref, None, None) == -1
    w.scale = p
    ep.row_scale = p
    assert cdll.dsl_linear_quantized(p, p, 4, ctypes.byref(w), None, p, 16, ref, None, None) == -4     # the slot is taken
    ep.row_scale = None
    assert cdll.dsl_linear_quantized(None, p, 4, ctypes.byref(w), None, p, 16, ref, None, None) == -1
    w.format = _lib.W_NVFP4
    assert cdll.dsl_linear_quantized(p, p, 4, ctypes.byref(w), None, p, 16, ref, None, None) == -4
    assert cdll.dsl_linear_scratch_bytes(_lib.W_INT8, 5, 64, 1) >= 5 * 64 + 5 * 4
    assert cdll.dsl_gemm_kn_served(_lib.OP_GEMM_INT8, 512, 512, 512, 1) == 0
    del keep


def test_int8_weight_round_trip_on_disk(tmp_path):
    w = PackedWeight("int8", torch.arange(-64, 64, dtype=torch.int8).reshape(4, 32), torch.tensor([0.5, 1.0, 2.0, 3.0]), None, 2, 2, 32, True)
    save_packed(tmp_path / "w.bin", w)
    r = load_packed(tmp_path / "w.bin", device="cpu")
    assert (r.format, r.groups, r.n, r.k, r.gate_up_interleaved, r.global_scale) == ("int8", 2, 2, 32, True, None)
    assert r.q.dtype == torch.int8 and torch.equal(r.q, w.q) and torch.equal(r.scale, w.scale)


def test_assembled_int8_weight_is_looked_at():
    from dsl_tool_b200.gemm_kernels import _new_weight_desc
    q, s = torch.zeros((4, 32), dtype=torch.int8), torch.ones(4)
    assert _new_weight_desc(PackedWeight("int8", q, s, None, 1, 4, 32)).format == _lib.W_INT8
    for bad_q, bad_s in ((q.view(torch.uint8), s), (q[:3], s), (q, None), (q, s[:3]), (q, s.double()), (q.t().contiguous().t(), s)):
        with pytest.raises(ValueError, match="int8 weight"):
            _new_weight_desc(PackedWeight("int8", bad_q, bad_s, None, 1, 4, 32))


def test_registered_with_the_dispatcher():
    from dsl_tool_b200.dispatcher import KernelDispatcher
    info = KernelDispatcher().kernel_info("gemm.int8_gemm", "cuda")
    assert {"A", "B", "scale_a", "scale_b", "b_layout", "out_dtype"} <= set(info["input_schema"])


def test_moe_decode_arguments(cdll):
    keep, p = _buffer()

    def weight(fmt, n, k, groups=4, q=p, scale=p, gs=p):
        w = _lib.Weight()
        w.format, w.groups, w.n, w.k, w.q, w.scale, w.global_scale = fmt, groups, n, k, q, scale, gs
        return w

    def need(gu, dn, tokens=2, k=2, x_dtype=_lib.BF16):
        return cdll.dsl_moe_decode_scratch_bytes(ctypes.byref(gu), ctypes.byref(dn), tokens, k, x_dtype)

    def call(gu, dn, tokens=2, k=2, x=p, x_dtype=_lib.BF16, logits=p, l_dtype=0, scratch=p, nbytes=1 << 30, out=p, o_dtype=0):
        return cdll.dsl_moe_decode(x, x_dtype, logits, l_dtype, tokens, k, 1, ctypes.byref(gu), ctypes.byref(dn), scratch, nbytes, out, o_dtype, None)
    for fmt, m in ((_lib.W_FP8, 16), (_lib.W_FP8_BLOCK128, 128), (_lib.W_INT8, 16), (_lib.W_NVFP4, 32), (_lib.W_MXFP4, 32), (_lib.W_BF16, 8)):
        gu, dn = weight(fmt, 4 * m, 3 * m), weight(fmt, 40, 2 * m)
        assert need(gu, dn) >= 4 * 4 * (2 * m + 40)
        assert need(weight(fmt, 4 * m, 3 * m + m // 2), dn) == 0                # K not a multiple
        assert need(gu, weight(fmt, 40, m)) == 0                                # H does not match
        assert need(gu, dn, tokens=33) == 0 and need(gu, dn, k=5) == 0 and need(gu, dn, k=0) == 0 and need(gu, dn, x_dtype=3) == 0
        assert call(gu, dn, x=None) == -1 and call(gu, dn, logits=None) == -1 and call(gu, dn, out=None) == -1
        assert call(gu, dn, scratch=None) == -1 and call(weight(fmt, 4 * m, 3 * m, q=None), dn) == -1
        assert call(gu, dn, x=p + 8) == -3 and call(gu, dn, scratch=p + 16) == -3
        assert call(gu, dn, l_dtype=2) == -4 and call(gu, dn, o_dtype=2) == -4
        assert call(gu, dn, nbytes=need(gu, dn) - 1) == -6 and call(gu, dn, tokens=33) == -6
        assert call(gu, dn, tokens=0) == 0
    gu, dn = weight(_lib.W_NVFP4, 128, 64, gs=None), weight(_lib.W_NVFP4, 40, 64)
    assert call(gu, dn) == -1
    assert need(weight(_lib.W_FP8, 64, 64), weight(_lib.W_INT8, 40, 32)) == 0   # two formats
    assert need(weight(6, 64, 64), weight(6, 40, 32)) == 0
    assert need(weight(_lib.W_BF16, 64, 65536), weight(_lib.W_BF16, 40, 32), x_dtype=_lib.F32) == 0      # a row that does not fit
    for K in (36000, 32768):
        assert need(weight(_lib.W_BF16, 64, K), weight(_lib.W_BF16, 40, 32), tokens=1, x_dtype=_lib.F32) > 0
    del keep


@pytest.mark.parametrize("fmt, apart", [(_lib.W_NVFP4, 4), (_lib.W_MXFP4, 8), (_lib.W_FP8_BLOCK128, 2), (_lib.W_INT8, 2)])
def test_moe_decode_refuses_scales_that_it_cannot_load_whole(cdll, fmt, apart):
    """FP4 scale bytes are read 16 at a time, the other formats' scales as fp32 words."""
    keep, p = _buffer()
    for side in range(2):
        gu, dn = _lib.Weight(), _lib.Weight()
        for i, (w, n, k) in enumerate(((gu, 512, 128), (dn, 40, 256))):
            w.format, w.groups, w.n, w.k, w.q, w.scale, w.global_scale = fmt, 4, n, k, p, p + (apart if i == side else 0), p
        assert cdll.dsl_moe_decode(p, _lib.BF16, p, 0, 2, 2, 1, ctypes.byref(gu), ctypes.byref(dn), p, 1 << 30, p, 0, None) == -3
    del keep


def test_quant_int8_of_no_columns_is_refused(cdll):
    """It would leave the scales unwritten."""
    keep, p = _buffer()
    assert cdll.dsl_quant_int8(p, 0, 4, 0, p, p, None) == -2
    assert cdll.dsl_quant_int8(p, 0, 0, 0, p, p, None) == -2
    del keep
