"""INT8 quantiser and GEMM.  The sums are exact, so results are compared bit for bit: int64 sums rounded to fp32 once, then the
two scale factors in the epilogue's order."""
import numpy as np
import pytest
import torch

from tests.helpers import activations, moe_offsets, weights

pytestmark = pytest.mark.gpu


def _ok():
    from dsl_tool_b200 import _lib
    _lib.check_status()


def quant(x):
    """fp32 rows -> (int8, scales): the definition in IEEE fp32."""
    x = np.asarray(x, np.float32)
    s = np.maximum(np.abs(x).max(1) / np.float32(127), np.float32(1e-12)).astype(np.float32)
    return np.rint(x / s[:, None]).astype(np.int8), s


def product(qa, qb, sa, sb):
    acc = torch.from_numpy(qa).cuda().double() @ torch.from_numpy(qb).cuda().double().t()      # below 2^53: exact
    c = acc.cpu().numpy().astype(np.float32)
    return (c * np.asarray(sa, np.float32).reshape(-1, 1)).astype(np.float32) * np.asarray(sb, np.float32)


def _t(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 16), (3, 512), (7, 528), (129, 4096), (5, 16384), (4, 16400), (2, 32768)])
def test_quantiser(cuda_device, shape, dtype):
    from dsl_tool_b200 import quantize_int8
    x = activations(np.random.default_rng(shape[1]), *shape, outliers=True)
    if shape[0] > 2:
        x[2] = 0.0                                        # an all-zero row: the floor of the scale
        x[1] *= np.float32(1e-5) if dtype != torch.float16 else np.float32(1)
    x[0, :8] = [1.0, 0.5, -0.5, 63.5 / 127, -1.5 / 127, 2.5 / 127, 1e-3, -1.0]
    xt = torch.from_numpy(x).to(dtype)
    q, s = quantize_int8(xt.cuda())
    qo, so = quant(xt.float().numpy())
    assert q.dtype == torch.int8 and (s.cpu().numpy() == so).all() and (q.cpu().numpy() == qo).all()


def test_quantiser_special_values_and_layouts(cuda_device):
    from dsl_tool_b200 import quantize_int8
    x = torch.randn(6, 64, device="cuda")
    x[1, 5], x[2, 7], x[3, 0] = float("nan"), float("inf"), -float("inf")
    x[4] = 1e-30
    q, s = quantize_int8(x)
    assert torch.isnan(s[1]) and torch.isinf(s[2]) and torch.isinf(s[3]) and s[4].item() == np.float32(1e-12)
    assert not q[2].any() and not q[3].any() and not q[4].any()
    q0, s0 = quantize_int8(x[0:1])
    assert torch.equal(q[0:1], q0) and torch.equal(s[0:1], s0) and torch.isfinite(s[5])
    y = torch.randn(64, 40, device="cuda").bfloat16()
    assert all(torch.equal(a, b) for a, b in zip(quantize_int8(y.t()), quantize_int8(y.t().contiguous())))
    wide = torch.randn(8 + 4 * 48, device="cuda").half()
    off = wide[8:].reshape(4, 48)                          # 16-byte but not 32-byte aligned
    assert all(torch.equal(a, b) for a, b in zip(quantize_int8(off), quantize_int8(off.clone())))
    q, s = quantize_int8(x[:0])
    assert q.shape == (0, 64) and s.shape == (0,)


@pytest.mark.parametrize("out", ["float32", "bfloat16"])
@pytest.mark.parametrize("M", [1, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 300, 513])
@pytest.mark.parametrize("N,K", [(256, 128), (520, 1040), (128, 512), (72, 16), (1030, 2064), (33, 4096)])
def test_gemm(cuda_device, M, N, K, out):
    from dsl_tool_b200.gemm_kernels import gemm_int8_quantized
    rng = np.random.default_rng(M * 7 + N)
    qa = rng.integers(-128, 128, (M, K)).astype(np.int8)
    qb = rng.integers(-128, 128, (N, K)).astype(np.int8)
    sa, sb = rng.random(M).astype(np.float32) * 0.05, rng.random(N).astype(np.float32) * 0.01
    got = gemm_int8_quantized(_t(qa), _t(qb), _t(sa), _t(sb), n=N, out_dtype=out)
    _ok()
    want = torch.from_numpy(product(qa, qb, sa, sb))
    assert torch.equal(got.cpu(), want if out == "float32" else want.bfloat16())


@pytest.mark.parametrize("M,N,K", [(1, 8192, 8192), (24, 2048, 28672), (16, 4096, 14336), (60, 1024, 8192), (100, 4096, 4096),
                                   (200, 2048, 14336), (300, 256, 8192), (130, 200, 16384), (4, 20000, 1024), (1000, 5344, 1168)])
def test_gemm_cut_along_k(cuda_device, M, N, K):
    """Weight streaming in clusters and through scratch, and the split tiled kernels: integer sums whatever the cut."""
    from dsl_tool_b200.gemm_kernels import gemm_int8_quantized
    g = torch.Generator(device="cuda").manual_seed(M)
    qa = torch.randint(-127, 128, (M, K), generator=g, device="cuda", dtype=torch.int8)
    qb = torch.randint(-127, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
    qa[0] = 127
    qb[0] = 127                                            # the largest sum: 127 * 127 * K
    ones = torch.ones(1, device="cuda")
    got = gemm_int8_quantized(qa, qb, ones, ones, n=N)
    _ok()
    assert torch.equal(got, (qa.double() @ qb.double().t()).float())


def test_gemm_largest_sum(cuda_device):
    from dsl_tool_b200 import _lib
    from dsl_tool_b200.gemm_kernels import gemm_int8_quantized
    K = _lib.INT8_MAX_K
    for M in (3, 200):
        qa = torch.full((M, K), -128, dtype=torch.int8, device="cuda")
        qb = torch.full((256, K), -128, dtype=torch.int8, device="cuda")
        qb[1] = 127
        got = gemm_int8_quantized(qa, qb, 1.0, 1.0, n=256)
        _ok()
        assert (got[:, 0] == np.float32(16384.0 * K)).all() and (got[:, 1] == np.float32(-128.0 * 127 * K)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,N,K", [(1, 512, 512), (17, 384, 1040), (128, 520, 2048), (257, 768, 1024)])
def test_linear_and_int8_gemm(cuda_device, M, N, K, dtype):
    from dsl_tool_b200 import int8_gemm, linear, pack_weight, quantize_int8
    rng = np.random.default_rng(N)
    a = torch.from_numpy(activations(rng, M, K, outliers=True)).to(dtype).cuda()
    w = torch.from_numpy(weights(rng, N, K)).bfloat16().cuda()
    qa, sa = quant(a.float().cpu().numpy())
    qb, sb = quant(w.float().cpu().numpy())
    want = torch.from_numpy(product(qa, qb, sa, sb)).cuda()
    p = pack_weight(w, "int8")
    assert p.q.dtype == torch.int8 and (p.q.cpu().numpy() == qb).all() and (p.scale.cpu().numpy() == sb).all()
    q, s = quantize_int8(a)
    for got in (linear(a, p), linear(q, p, act_scale=s), int8_gemm(a, w, b_layout="nk"), int8_gemm(a, w.t()), int8_gemm(a, p),
                int8_gemm(q, p, s), int8_gemm(q, p.q, s, p.scale, b_layout="nk"), int8_gemm(q, p.q.t().contiguous(), s, p.scale),
                int8_gemm(a, w, b_layout="nk", cache_weights=True), linear(a.t().contiguous().t(), p)):
        assert torch.equal(got, want)
    assert torch.equal(linear(a, p, out_dtype=torch.bfloat16), want.bfloat16())
    _ok()


@pytest.mark.parametrize("activation", ["swiglu", "geglu"])
@pytest.mark.parametrize("M", [1, 20, 100, 400])
def test_gated(cuda_device, M, activation):
    """silu / gelu of exact pre-activations.  __expf is off by up to 2 + 1.173 |z| ulp (its documented bound), the division by 2,
    the products by half an ulp each, and z itself of geglu (four roundings) by 4 ulp of |z|, i.e. 4 |z| ulp of exp(z)."""
    from dsl_tool_b200 import linear, pack_weight
    H, K = 264, 512
    g = torch.Generator(device="cuda").manual_seed(M)
    a = torch.randn(M, K, generator=g, device="cuda")
    w = torch.randn(2 * H, K, generator=g, device="cuda") * 0.05
    plain = linear(a, pack_weight(w, "int8")).double()
    gate, up = plain[:, :H], plain[:, H:]
    z = gate if activation == "swiglu" else 1.5957691216 * (gate + 0.044715 * gate ** 3)
    want = gate / (1 + torch.exp(-z)) * up
    got = linear(a, pack_weight(w, "int8", gate_up_interleave=True), activation=activation).double()
    _ok()
    ulp = 2.0 ** -23
    assert ((got - want).abs() <= want.abs() * ulp * (8 + 6 * z.abs())).all()


def test_quantised_result(cuda_device):
    from dsl_tool_b200 import linear, pack_weight, quantize_fp4
    a, w = torch.randn(140, 256, device="cuda"), torch.randn(512, 256, device="cuda") * 0.05
    p = pack_weight(w, "int8")
    q, sf, gs = linear(a, p, out_dtype="nvfp4", out_global_scale=0.01)
    want = quantize_fp4(linear(a, p), "nvfp4", global_scale=0.01)
    _ok()
    assert torch.equal(q, want[0]) and torch.equal(sf, want[1])


@pytest.mark.parametrize("tokens,experts,n,k", [(16, 8, 264, 256), (200, 6, 512, 512), (900, 5, 300, 272), (40, 64, 128, 128)])
def test_row_groups(cuda_device, tokens, experts, n, k):
    from dsl_tool_b200 import grouped_gemm, linear, pack_weight
    rng = np.random.default_rng(tokens)
    offs = moe_offsets(rng, tokens, experts, 2)
    M = int(offs[-1])
    a, w = activations(rng, M, k), weights(rng, experts * n, k).reshape(experts, n, k)
    qa, sa = quant(a)
    want = np.zeros((M, n), np.float32)
    for e in range(experts):
        r = slice(int(offs[e]), int(offs[e + 1]))
        if r.stop > r.start:
            qb, sb = quant(w[e])
            want[r] = product(qa[r], qb, sa[r], sb)
    p = pack_weight(_t(w), "int8")
    got = linear(_t(a), p, expert_offsets=_t(offs))
    _ok()
    assert (got.cpu().numpy() == want).all()
    assert torch.equal(grouped_gemm(_t(a), _t(w), expert_offsets=_t(offs), format="int8", b_layout="nk"), got)
    from dsl_tool_b200 import quantize_int8
    q, s = quantize_int8(_t(a))
    assert torch.equal(linear(q, p, act_scale=s, expert_offsets=_t(offs)), got)


def test_moe_forward_with_int8_experts(cuda_device):
    """The layer takes int8 experts through its step-by-step form: every routed row is quantised on its own."""
    from dsl_tool_b200 import MoEWeights, moe_forward
    from dsl_tool_b200.moe import route
    T, E, K, H, D, k = 37, 6, 256, 128, 192, 2
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(T, K, generator=g, device="cuda").bfloat16()
    logits = torch.randn(T, E, generator=g, device="cuda")
    gu, dn = torch.randn(E, 2 * H, K, generator=g, device="cuda") * 0.1, torch.randn(E, D, H, generator=g, device="cuda") * 0.1
    got = moe_forward(x, logits, MoEWeights.pack(gu, dn, "int8"), k)
    _ok()
    ids, wts = route(logits, k)
    want = torch.zeros(T, D, dtype=torch.float64, device="cuda")

    def rounded(v):
        s = (v.abs().amax(-1, keepdim=True).float() / 127).clamp(min=1e-12)
        return torch.round(v.float() / s).double() * s.double()
    for t in range(T):
        for j in range(k):
            e = int(ids[t, j])
            g2 = rounded(x[t:t + 1]) @ rounded(gu[e]).t()
            h = (torch.nn.functional.silu(g2[:, :H]) * g2[:, H:]).bfloat16()
            want[t] += (wts[t, j].double() * (rounded(h) @ rounded(dn[e]).t()).bfloat16().double())[0]
    # both sides round alike; where the last bit of an fp32 sum tips a rounding the other way, a value moves by a step (2^-7 of it in
    # bf16, 1 / 127 of its row's largest in int8): seldom, so far less than half a bf16 step, 2^-8, over all values
    assert ((got.double() - want).norm() / want.norm()).item() < 4e-3


def test_nan_and_infinite_rows_stay_alone(cuda_device):
    from dsl_tool_b200 import linear, pack_weight
    a, w = torch.randn(40, 128, device="cuda"), torch.randn(256, 128, device="cuda")
    p = pack_weight(w, "int8")
    clean = linear(a, p)
    a[3, 4], a[17, 0] = float("nan"), float("inf")
    got = linear(a, p)
    assert torch.isnan(got[3]).all() and torch.isnan(got[17]).all()
    keep = [i for i in range(40) if i not in (3, 17)]
    assert torch.equal(got[keep], clean[keep])


def test_refusals(cuda_device):
    from dsl_tool_b200 import int8_gemm, linear, pack_weight, quantize_int8
    from dsl_tool_b200.gemm_kernels import gemm_int8_quantized
    a, w = torch.randn(4, 64, device="cuda"), torch.randn(32, 64, device="cuda")
    p, f, n = pack_weight(w, "int8"), pack_weight(w, "fp8"), pack_weight(w, "nvfp4")
    q, s = quantize_int8(a)
    one = torch.ones(4, device="cuda")
    with pytest.raises(ValueError, match="multiple of 16"):
        quantize_int8(torch.randn(2, 20, device="cuda"))
    with pytest.raises(ValueError, match="at most 32768"):
        quantize_int8(torch.randn(1, 32784, device="cuda"))
    with pytest.raises(ValueError, match="no global_scale"):
        pack_weight(w, "int8", global_scale=1.0)
    for kw in (dict(row_scale=one), dict(col_scale=torch.ones(32, device="cuda"))):
        for x, more in ((a, {}), (q, dict(act_scale=s)), (a.t().contiguous().t(), {})):
            with pytest.raises(ValueError, match="occupy"):
                linear(x, p, **kw, **more)
    with pytest.raises(TypeError, match="quantised for int8"):
        linear(a, p, act_scale=s)
    with pytest.raises(TypeError, match="quantised for fp8"):
        linear(a, f, act_scale=s[:1])
    with pytest.raises(ValueError, match="FP8 and int8"):
        linear(q, n, act_scale=s)
    with pytest.raises(ValueError, match="4 values"):
        linear(q, p, act_scale=s[:3])
    with pytest.raises(ValueError, match="exclude"):
        linear(q, p, act_scale=s, act_global_scale=1.0)
    with pytest.raises(TypeError):
        gemm_int8_quantized(q.view(torch.uint8), p.q, s, p.scale, n=32)
    with pytest.raises(ValueError, match="scale_a"):
        gemm_int8_quantized(q, p.q, s[:2], p.scale, n=32)
    with pytest.raises(ValueError, match="required"):
        int8_gemm(q, p)
    with pytest.raises(ValueError, match="required"):
        int8_gemm(q, p.q, s, b_layout="nk")
    with pytest.raises(ValueError, match="goes with int8"):
        int8_gemm(a, p, s)
    with pytest.raises(ValueError, match="brings its own"):
        int8_gemm(q, p, s, p.scale)
    with pytest.raises(ValueError, match="need single-group int8"):
        int8_gemm(a, f)
    with pytest.raises(TypeError, match="both be"):
        int8_gemm(q, w.t(), s)
    with pytest.raises(ValueError, match="derived"):
        int8_gemm(a, w.t(), one)
    with pytest.raises(ValueError, match="even number|gate_up"):
        linear(a, p, activation="swiglu")


def test_capture_and_streams(cuda_device):
    """A captured call keeps scratch of its own, and calls on two streams at once do not meet."""
    from dsl_tool_b200 import linear, pack_weight
    p = pack_weight(torch.randn(4096, 4096, device="cuda"), "int8")
    xs = [torch.randn(24, 4096, device="cuda").bfloat16() for _ in range(4)]
    want = [linear(x, p) for x in xs]
    side = torch.cuda.Stream()
    static = xs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = linear(static, p)
    for i in range(4):
        static.copy_(xs[i])
        side.wait_stream(torch.cuda.current_stream())
        g.replay()
        with torch.cuda.stream(side):
            others = [linear(x, p) for x in xs]
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and all(torch.equal(a, b) for a, b in zip(others, want))
    _ok()
