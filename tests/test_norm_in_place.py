"""dsl_rms_norm may write the new residual over x or over the old one: its loads must not take the path for memory that a kernel does
not write, and every element is read before it is written, at every size and alignment."""
import os
import re

import pytest
import torch

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "dsl_tool_b200", "csrc")


def test_rows_are_not_read_as_constants():
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, "norm.cu")).read())
    body = re.search(r"void load\(const T\* p, bool wide\) \{\n(.*?)\n    \}\n", text, re.S).group(1)
    assert "ld.global" in body and ".nc" not in body and "__ldg(" not in body and "ldg256" not in body
    kernel = text[text.index("row_kernel(const RowArgs a)"):text.index("launch_threads(")]
    assert re.findall(r"(\w+)(?:\[p\])?\.load\(", kernel) == ["rx", "rr"]        # x and residual come in through it ...
    assert "load16" not in kernel and "__ldg" not in kernel                      # ... and in no other way


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 16), (9, 256), (700, 528), (2000, 4096), (300, 8192), (5, 16400), (400, 32768)])
@pytest.mark.parametrize("offset", [0, 1])
def test_sum_over_its_inputs(cuda_device, dtype, rows, cols, offset):
    """`offset`: rows that start on 16 but not on 32 bytes."""
    from dsl_tool_b200 import _lib, rms_norm
    g = torch.Generator(device="cuda").manual_seed(rows)
    pad = 16 // torch.empty((), dtype=dtype).element_size() * offset

    def draw():
        return torch.randn(rows * cols + pad, generator=g, device="cuda").to(dtype)[pad:].reshape(rows, cols)
    x, r, w = draw(), draw(), torch.rand(cols, generator=g, device="cuda")
    for fmt, code in ((None, _lib.NORM_NONE), ("int8", _lib.NORM_INT8), ("fp8_block128", _lib.NORM_FP8_GROUP_1X128)):
        want_out, want_s, want_t = rms_norm(x, w, residual=r, format=fmt)
        for over in ("x", "residual"):
            storage = [torch.empty(rows * cols + pad, dtype=dtype, device="cuda")[pad:].reshape(rows, cols).copy_(v) for v in (x, r)]
            xi, ri = storage
            t = xi if over == "x" else ri
            out, s = torch.empty_like(want_out), None if want_s is None else torch.empty_like(want_s)
            rc = _lib.lib().dsl_rms_norm(xi.data_ptr(), _lib.dtype_code(dtype), rows, cols, ri.data_ptr(), w.data_ptr(), _lib.F32, 1e-6, code,
                                         t.data_ptr(), out.data_ptr(), _lib.ptr(s), None, _lib.stream_ptr())
            assert rc == 0 and torch.equal(t, want_t) and torch.equal(out, want_out) and (s is None or torch.equal(s, want_s))
            assert torch.equal(ri if over == "x" else xi, r if over == "x" else x)      # the other input stays
