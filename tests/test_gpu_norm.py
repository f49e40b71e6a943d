"""Root-mean-square norm with residual and 8-bit result: y against 64 bits, the quantised forms bit for bit against the
stand-alone quantisers of the same y, and the chain norm -> linear."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
# relative error of y: a thread's 32 fused products and 10 levels of the tree (42 u), division, addition (2 u) - halved by the root -
# the root (1 u), two products (2 u); u = 2^-24
Y_RTOL = (44 / 2 + 3) * 2.0 ** -24


def _inputs(shape, dtype, gain_dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(shape, generator=g, device="cuda") * 3
    x[torch.rand(shape, generator=g, device="cuda") < 1e-3] = 60.0
    r = torch.randn(shape, generator=g, device="cuda")
    w = torch.rand(shape[-1], generator=g, device="cuda") + 0.5
    w[0] = -w[0]
    return x.to(dtype), r.to(dtype), w.to(gain_dtype)


def _exact(t, w, eps):
    t = t.double()
    return t / torch.sqrt(t.square().mean(-1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("gain_dtype", DTYPES)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 16), (3, 512), (5, 528), (64, 1024), (33, 4096), (2, 8192), (3, 16384), (2, 16400), (2, 32768)])
def test_formats(cuda_device, shape, dtype, gain_dtype):
    from dsl_tool_b200 import quantize_fp8, quantize_int8, rms_norm
    x, r, w = _inputs(shape, dtype, gain_dtype)
    for residual in (None, r):
        t = x if residual is None else (x.float() + r.float()).to(dtype)
        y, none, total = rms_norm(t.float(), w, eps=1e-5)                     # fp32 in, fp32 out: y itself
        assert none is None and total is None and y.dtype == torch.float32
        want = _exact(t, w, 1e-5)
        assert ((y.double() - want).abs() <= want.abs() * Y_RTOL).all()
        out, s, total = rms_norm(x, w, eps=1e-5, residual=residual)
        assert s is None and out.dtype == dtype and torch.equal(out, y.to(dtype))
        assert total is None if residual is None else torch.equal(total, t)
        q, s, total = rms_norm(x, w, eps=1e-5, residual=residual, format="int8")
        assert all(torch.equal(a, b) for a, b in zip((q, s), quantize_int8(y)))
        assert total is None if residual is None else torch.equal(total, t)
        q, s, _ = rms_norm(x, w, eps=1e-5, residual=residual, format="fp8_block128")
        assert all(torch.equal(a, b) for a, b in zip((q, s), quantize_fp8(y, "groupwise")))
        for scale in (0.02, torch.tensor([1e-4], device="cuda")):             # the second saturates
            q, s, _ = rms_norm(x, w, eps=1e-5, residual=residual, format="fp8", scale=scale)
            assert all(torch.equal(a, b) for a, b in zip((q, s), quantize_fp8(y, scale=scale)))


def test_shapes_strides_and_aliases(cuda_device):
    from dsl_tool_b200 import rms_norm
    x, r, w = _inputs((2, 3, 64), torch.bfloat16, torch.bfloat16)
    out, _, total = rms_norm(x, w, residual=r)
    assert out.shape == total.shape == x.shape
    q, s, total8 = rms_norm(x, w, residual=r, format="int8")
    assert q.shape == (6, 64) and s.shape == (6,) and torch.equal(total8, total)
    flat, _, _ = rms_norm(x.reshape(6, 64), w, residual=r.reshape(6, 64))
    assert torch.equal(flat, out.reshape(6, 64))
    one, _, _ = rms_norm((x + r)[0, 0], w)
    assert one.shape == (64,) and torch.equal(one, out[0, 0])
    tall = torch.randn(64, 6, device="cuda").bfloat16()
    assert torch.equal(rms_norm(tall.t(), w)[0], rms_norm(tall.t().contiguous(), w)[0])
    wide = torch.randn(8 + 6 * 64, device="cuda").bfloat16()                  # 16-byte but not 32-byte aligned rows
    assert torch.equal(rms_norm(wide[8:].reshape(6, 64), w)[0], rms_norm(wide[8:].reshape(6, 64).clone(), w)[0])
    gain = torch.randn(128, device="cuda")[::2]
    assert torch.equal(rms_norm(x, gain)[0], rms_norm(x, gain.clone())[0])
    same, _, total = rms_norm(x, w, residual=x)                               # the same tensor twice
    assert torch.equal(total, x + x) and torch.equal(same, rms_norm(x + x, w)[0])
    q, s, total = rms_norm(x[:0], w, residual=r[:0], format="int8")
    assert q.shape == (0, 64) and s.shape == (0,) and total.shape == (0, 3, 64)


def test_sum_may_be_written_in_place(cuda_device):
    """The C entry point lets the new residual replace the old one."""
    from dsl_tool_b200 import _lib, rms_norm
    x, r, w = _inputs((9, 256), torch.bfloat16, torch.float32)
    want_q, want_s, want_t = rms_norm(x, w, residual=r, format="int8")
    q, s = torch.empty_like(want_q), torch.empty_like(want_s)
    rc = _lib.lib().dsl_rms_norm(x.data_ptr(), _lib.BF16, 9, 256, r.data_ptr(), w.data_ptr(), _lib.F32, 1e-6, _lib.NORM_INT8, r.data_ptr(),
                                 q.data_ptr(), s.data_ptr(), None, _lib.stream_ptr())
    assert rc == 0 and torch.equal(q, want_q) and torch.equal(s, want_s) and torch.equal(r, want_t)


def test_special_values(cuda_device):
    from dsl_tool_b200 import rms_norm
    x, _, w = _inputs((7, 256), torch.float32, torch.float32)
    clean = {f: rms_norm(x, w, format=f) for f in (None, "int8", "fp8_block128")}
    x[1, 3], x[2, 9], x[4] = float("nan"), float("inf"), 0.0
    y, _, _ = rms_norm(x, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[2, 9]) and (y[2, :9] == 0).all() and (y[4] == 0).all()
    q, s, _ = rms_norm(x, w, format="int8")
    assert torch.isnan(s[1]) and torch.isnan(s[2]) and s[4].item() == np.float32(1e-12) and not q[4].any()
    q8, s8, _ = rms_norm(x, w, format="fp8_block128")
    assert ((q8[1] & 0x7F) == 0x7F).all() and not (q8[4] & 0x7F).any()      # 0 * -w is -0
    for i in (0, 3, 5, 6):
        assert torch.equal(y[i], clean[None][0][i]) and torch.equal(q[i], clean["int8"][0][i]) and s[i] == clean["int8"][1][i]
        assert torch.equal(q8[i], clean["fp8_block128"][0][i]) and torch.equal(s8[i], clean["fp8_block128"][1][i])


def test_refusals(cuda_device):
    from dsl_tool_b200 import rms_norm
    x, r, w = _inputs((4, 64), torch.bfloat16, torch.bfloat16)
    with pytest.raises(ValueError, match="format must be"):
        rms_norm(x, w, format="nvfp4")
    with pytest.raises(ValueError, match="needs the scale"):
        rms_norm(x, w, format="fp8")
    with pytest.raises(ValueError, match="needs the scale"):
        rms_norm(x, w, format="int8", scale=1.0)
    with pytest.raises(ValueError, match="multiple of 16"):
        rms_norm(x[:, :40], w[:40])
    with pytest.raises(ValueError, match="at most 32768"):
        rms_norm(torch.zeros(1, 32784, device="cuda"), torch.zeros(32784, device="cuda"))
    with pytest.raises(ValueError, match="weight must be"):
        rms_norm(x, w[:32])
    with pytest.raises(ValueError, match="residual must have"):
        rms_norm(x, w, residual=r[:2])
    with pytest.raises(ValueError, match="residual must have"):
        rms_norm(x, w, residual=r.float())
    with pytest.raises(TypeError, match="unsupported input dtype"):
        rms_norm(x.double(), w)
    with pytest.raises(TypeError, match="unsupported input dtype"):
        rms_norm(x, w.double())
    with pytest.raises(ValueError, match="at least one element"):
        rms_norm(x[:, :0], w[:0])
    with pytest.raises(RuntimeError, match="CUDA device"):
        rms_norm(x, w.cpu())


@pytest.mark.parametrize("rows", [1, 40, 300])
@pytest.mark.parametrize("format", ["int8", "fp8_block128", "fp8"])
def test_block_of_projections(cuda_device, rows, format):
    """Residual, norm, gate/up projection with SwiGLU, down projection, next norm - as a block runs them - against the same chain
    of separate calls, bit for bit."""
    from dsl_tool_b200 import linear, pack_weight, quantize_fp8, quantize_int8, rms_norm
    x, r, w = _inputs((rows, 512), torch.bfloat16, torch.bfloat16)
    up = pack_weight(torch.randn(1024, 512, device="cuda") * 0.04, format, gate_up_interleave=True)
    down = pack_weight(torch.randn(512, 512, device="cuda") * 0.04, format)
    scale = 0.05 if format == "fp8" else None
    bf16 = torch.bfloat16
    q, s, t = rms_norm(x, w, residual=r, format=format, scale=scale)
    h = linear(q, up, act_scale=s, activation="swiglu", out_dtype=bf16)
    o = linear(h, down, out_dtype=bf16)
    q2, s2, t2 = rms_norm(o, w, residual=t, format=format, scale=scale)

    def apart(x, r):
        t = (x.float() + r.float()).to(bf16)
        y = rms_norm(t.float(), w)[0]
        if format == "int8":
            return (*quantize_int8(y), t)
        return (*quantize_fp8(y, "groupwise" if format == "fp8_block128" else "per_tensor", scale=scale), t)
    qa, sa, ta = apart(x, r)
    assert torch.equal(qa, q) and torch.equal(sa, s) and torch.equal(ta, t)
    qb, sb, tb = apart(o, t)
    assert torch.equal(qb, q2) and torch.equal(sb, s2) and torch.equal(tb, t2)
    # the product of quantised rows is what the values multiply to: fp32 sums of 512 products, and a bf16 result, of which each
    # element is off by half a step, 2^-8 of its value at most (8 bits: a step is 2^-7 of the power of two below), so their norm too
    values = q.view(torch.int8).double() * s.double()[:, None] if format == "int8" else \
        q.view(torch.float8_e4m3fn).double() * (s.double() if format == "fp8" else s.double().repeat_interleave(128, 1))
    uv = up.q.double() * up.scale.double()[:, None] if format == "int8" else \
        up.q.view(torch.float8_e4m3fn).double() * (up.scale.double() if format == "fp8" else
                                                   up.scale.double()[0].repeat_interleave(128, 0).repeat_interleave(128, 1))
    g = values @ uv.t()
    want = torch.nn.functional.silu(g[:, 0::2]) * g[:, 1::2]
    assert ((h.double() - want).norm() / want.norm()).item() <= 2.0 ** -8 + 2e-5


def test_captured_chain(cuda_device):
    from dsl_tool_b200 import linear, pack_weight, rms_norm
    x, r, w = _inputs((24, 1024), torch.bfloat16, torch.bfloat16)
    p = pack_weight(torch.randn(2048, 1024, device="cuda") * 0.04, "int8")

    def step():
        q, s, t = rms_norm(x, w, residual=r, format="int8")
        return linear(q, p, act_scale=s), t
    step()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for seed in (1, 2):
        a, b, _ = _inputs((24, 1024), torch.bfloat16, torch.bfloat16, seed)
        x.copy_(a)
        r.copy_(b)
        g.replay()
        want = step()
        assert all(torch.equal(i, j) for i, j in zip(out, want))


@pytest.mark.parametrize("format", ["int8", "fp8_block128", "fp8"])
def test_chain_of_no_rows(cuda_device, format):
    """Nothing to do, from the norm to the projection."""
    from dsl_tool_b200 import int8_gemm, linear, pack_weight, rms_norm
    x, r, w = _inputs((0, 512), torch.bfloat16, torch.bfloat16)
    packed = pack_weight(torch.randn(256, 512, device="cuda"), format, gate_up_interleave=True)
    q, s, t = rms_norm(x, w, residual=r, format=format, scale=0.1 if format == "fp8" else None)
    assert q.shape == (0, 512) and t.shape == (0, 512)
    assert linear(q, packed, act_scale=s).shape == (0, 256)
    assert linear(x, packed, activation="swiglu", out_dtype=torch.bfloat16).shape == (0, 128)
    if format == "int8":
        assert int8_gemm(q, packed, s).shape == (0, 256)
        assert int8_gemm(x, torch.randn(512, 256, device="cuda")).shape == (0, 256)
