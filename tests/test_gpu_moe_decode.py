"""The few-token MoE layer in three kernels against the layer in 64 bits on the packed weights' own values."""
import numpy as np
import pytest
import torch

from oracle import quant_oracle as O

pytestmark = pytest.mark.gpu

FORMATS = ["fp8", "fp8_block128", "int8", "nvfp4", "mxfp4", "bf16"]


def values(p):
    """What a packed weight stands for: [G, n, k] in 64 bits."""
    G, n, k = p.groups, p.n, p.k
    if p.format == "bf16":
        return p.q.double().reshape(G, n, k)
    if p.format == "int8":
        return p.q.double().reshape(G, n, k) * p.scale.double().reshape(G, n, 1)
    if p.format in ("fp8", "fp8_block128"):
        v = p.q.view(torch.float8_e4m3fn).double().reshape(G, n, k)
        if p.format == "fp8":
            return v * p.scale.double()
        s = p.scale.double().reshape(G, -(-n // 128), -1)
        return v * s.repeat_interleave(128, 1)[:, :n].repeat_interleave(128, 2)[:, :, :k]
    block = 16 if p.format == "nvfp4" else 32
    v = torch.from_numpy(O.e2m1_decode(O.unpack_nibbles(p.q.cpu().numpy()))).double().reshape(G, n, k)
    nblk, tiles = k // block, -(-n // 128)
    per = tiles * (-(-nblk // 4)) * 512
    sf = p.scale.cpu().numpy()
    s = np.stack([O.unswizzle_sf(sf[g * per:(g + 1) * per], n, nblk) for g in range(G)])
    s = O.e4m3_decode(s).astype(np.float64) * float(p.global_scale) if p.format == "nvfp4" else np.exp2(s.astype(np.float64) - 127)
    return (v * torch.from_numpy(s).repeat_interleave(block, 2)).cuda()


def layer(x, logits, w, k, renormalize=True):
    """The layer and, beside it, the sum of the magnitudes that the output adds up (what rounding errors are relative to)."""
    gu, dn = values(w.gate_up), values(w.down)
    T, E = logits.shape
    l = logits.double()
    out = torch.zeros(T, w.down.n, dtype=torch.float64, device="cuda")
    for t in range(T):
        row = l[t].tolist()
        order = sorted((e for e in range(E) if row[e] > -np.inf), key=lambda e: (-row[e], e))[:k]
        if not order:
            continue
        p = torch.softmax(l[t], 0)[order]
        if renormalize:
            p = p / p.sum()
        for j, e in enumerate(order):
            g = gu[e] @ x[t].double()
            h = g[0::2] / (1 + torch.exp(-g[0::2])) * g[1::2]
            out[t] += p[j] * (dn[e] @ h)
    return out


def make(T, E, K, H, D, fmt, dtype=torch.bfloat16, seed=0, logits_dtype=torch.float32):
    from dsl_tool_b200 import MoEWeights
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(T, K, generator=g, device="cuda")
    x[torch.rand(T, K, generator=g, device="cuda") < 1e-3] = 20.0
    logits = torch.randn(T, E, generator=g, device="cuda").to(logits_dtype)
    w = MoEWeights.pack((torch.randn(E, 2 * H, K, generator=g, device="cuda") / K ** 0.5).bfloat16(),
                        (torch.randn(E, D, H, generator=g, device="cuda") / H ** 0.5).bfloat16(), fmt)
    return x.to(dtype), logits, w


def bound(fmt, dtype):
    """Relative error in the 2-norm.  Independent relative errors of the terms of a sum of random signs carry over to it at their own
    size.  The hidden activation is rounded to the 11 bits of f16: half a step is finfo(float16).eps / 2 = 2^-11 of the value (bf16
    weights: to two bf16 terms, the second of the remainder of the first, 2^-8 * 2^-8 = 2^-16), an fp32 x to the same, of which
    gate and up each pass theirs on (silu has a slope of at most 1.1): at most 1 + 2.1 roundings in all.  fp32 sums of up to 1536
    products: 2^-24 times the number of additions a warp makes in a row, below 2^-17."""
    half = 2.0 ** (-16 if fmt == "bf16" else -11)
    return half * (3.1 if dtype == torch.float32 else 1.0) + 2.0 ** -17


def far(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,E,k,K,H,D", [(1, 8, 2, 256, 128, 256), (3, 4, 4, 384, 256, 200), (8, 16, 3, 512, 384, 136), (9, 6, 2, 640, 128, 264),
                                         (16, 8, 8, 256, 256, 128), (17, 40, 5, 256, 128, 72), (32, 8, 2, 1152, 640, 1000), (32, 33, 32, 128, 128, 48),
                                         (5, 1, 1, 1536, 1280, 56), (2, 64, 8, 2048, 768, 2048)])
def test_layer(cuda_device, fmt, T, E, k, K, H, D):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(T, E, K, H, D, fmt)
    want = layer(x, logits, w, k)
    got = moe_decode(x, logits, w, k)
    assert got.shape == (T, D) and got.dtype == torch.float32
    assert far(got, want) <= bound(fmt, x.dtype)
    assert torch.equal(moe_decode(x, logits, w, k), got)                                  # the same bits every time
    assert torch.equal(moe_decode(x, logits, w, k, out_dtype=torch.bfloat16), got.bfloat16())
    one = torch.cat([moe_decode(x[t:t + 1], logits[t:t + 1], w, k) for t in range(min(T, 3))])
    assert far(one, want[:min(T, 3)]) <= bound(fmt, x.dtype)


@pytest.mark.parametrize("fmt,K,H,D", [("nvfp4", 288, 96, 50), ("mxfp4", 32, 32, 2), ("fp8", 272, 144, 17), ("int8", 16, 16, 1), ("bf16", 72, 8, 3),
                                       ("bf16", 1000, 1048, 30), ("nvfp4", 2912, 1440, 96), ("mxfp4", 2912, 1440, 96), ("fp8", 2064, 1040, 40)])
@pytest.mark.parametrize("T", [1, 13])
def test_odd_sizes(cuda_device, fmt, K, H, D, T):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(T, 5, K, H, D, fmt, seed=K)
    assert far(moe_decode(x, logits, w, 2), layer(x, logits, w, 2)) <= bound(fmt, x.dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.bfloat16])
def test_types(cuda_device, fmt, dtype, logits_dtype):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(6, 12, 512, 256, 320, fmt, dtype=dtype, logits_dtype=logits_dtype)
    if logits_dtype == torch.bfloat16:
        logits[2] = logits[2, 0]                                                           # ties: the lower index
    for renormalize in (True, False):
        got = moe_decode(x, logits, w, 3, renormalize=renormalize)
        assert far(got, layer(x, logits, w, 3, renormalize)) <= bound(fmt, dtype)


@pytest.mark.parametrize("fmt,K,H,T", [("bf16", 14336, 128, 7), ("bf16", 256, 14336, 8), ("nvfp4", 14336, 128, 20), ("fp8", 128, 20480, 5),
                                       ("int8", 32768, 32, 3)])
def test_rows_that_do_not_all_fit(cuda_device, fmt, K, H, T):
    """An expert with more rows than its CTA's shared memory holds takes several passes over its weight."""
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(T, 2, K, H, 64, fmt, dtype=torch.float16)
    assert far(moe_decode(x, logits, w, 2), layer(x, logits, w, 2)) <= bound(fmt, x.dtype)


@pytest.mark.parametrize("fmt", FORMATS)
def test_routing_is_the_routers(cuda_device, fmt):
    from dsl_tool_b200 import moe_decode
    from dsl_tool_b200.moe import route
    x, logits, w = make(11, 24, 256, 128, 128, fmt)
    ids, wts = route(logits, 4)
    got = moe_decode(x, logits, w, 4)
    # the same experts with the same weights, asked for one by one: a logit of 0 for the expert, minus infinity for the others
    want = torch.zeros_like(got, dtype=torch.float64)
    for t in range(11):
        for j in range(4):
            alone = torch.full((1, 24), -float("inf"), device="cuda")
            alone[0, int(ids[t, j])] = 0.0
            want[t] += wts[t, j].double() * moe_decode(x[t:t + 1], alone, w, 1)[0].double()
    assert far(got, want) <= 1e-6          # fp32: five roundings of 2^-24 and the sums' other order of K


def test_masked_and_special_logits(cuda_device):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(8, 10, 256, 128, 192, "nvfp4")
    inf = float("inf")
    logits[1] = -inf                                         # nobody
    logits[2, 3:] = -inf                                     # three experts for k = 4
    logits[3, :] = -inf
    logits[3, 7] = -3e38                                     # one, at the type's end
    logits[4] = torch.finfo(torch.float32).min               # all at the lowest value: the first four, a quarter each
    logits[5, 2] = float("nan")
    got = moe_decode(x, logits, w, 4)
    want = layer(x, logits, w, 4)
    assert not got[1].any()
    for t in (0, 2, 3, 4, 6, 7):
        assert far(got[t], want[t]) <= bound("nvfp4", x.dtype)
    assert torch.isnan(got[5]).all()                         # its softmax is
    everything = torch.full_like(logits, -inf)
    assert not moe_decode(x, everything, w, 4).any()
    poison = torch.empty(8, 192, device="cuda").fill_(float("nan"))
    del poison                                               # the next result may land on it: every element is written
    assert not moe_decode(x, everything, w, 4, out_dtype=torch.bfloat16).any()


@pytest.mark.parametrize("fmt", FORMATS)
def test_special_activations_stay_in_their_row(cuda_device, fmt):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(12, 3, 256, 128, 128, fmt)
    clean = moe_decode(x, logits, w, 2)
    x[2, 5], x[9, 0], x[4] = float("nan"), float("inf"), 0.0
    got = moe_decode(x, logits, w, 2)
    assert torch.isnan(got[2]).all() and not torch.isfinite(got[9]).all() and not got[4].any()
    keep = [t for t in range(12) if t not in (2, 4, 9)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("scale", [2.0 ** -60, 2.0 ** 40])
@pytest.mark.parametrize("fmt", ["nvfp4", "bf16", "int8", "mxfp4"])
def test_scale_of_the_rows(cuda_device, fmt, scale):
    """Rows far from 1: f16 products are taken of rows scaled by powers of two."""
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(4, 4, 256, 128, 128, fmt)
    x = x.float()
    x[1] *= scale                                            # the other rows stay
    x = x.bfloat16()
    want, got = layer(x, logits, w, 2), moe_decode(x, logits, w, 2)
    for t in range(4):
        assert torch.isfinite(got[t]).all() and far(got[t], want[t]) <= bound(fmt, x.dtype)


def test_mxfp4_scales_far_apart(cuda_device):
    """Blocks 2^-40 to 2^30 beside one another in a row: each block's sum meets its scale in fp32."""
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(5, 3, 512, 128, 128, "mxfp4")
    g = torch.Generator(device="cuda").manual_seed(5)
    spread = torch.randint(87, 158, w.gate_up.scale.shape, generator=g, device="cuda").to(torch.uint8)
    w.gate_up.scale.copy_(torch.where(w.gate_up.scale > 0, spread - 20, w.gate_up.scale))
    x = (x.float() * 2.0 ** -12).bfloat16()
    want, got = layer(x, logits, w, 2), moe_decode(x, logits, w, 2)
    assert far(got, want) <= bound("mxfp4", x.dtype)
    w.gate_up.scale[0] = 255                                 # NaN block of expert 0, row 0
    assert torch.isnan(moe_decode(x, logits, w, 3)).all()
    w.gate_up.scale.fill_(0)                                 # 2^-127 throughout: everything vanishes, nothing breaks
    assert torch.isfinite(moe_decode(x, logits, w, 2)).all()


def test_against_moe_forward(cuda_device):
    """The layer of quantised GEMMs, whose activations are rounded to the weights' format, lies as far off as that rounding."""
    from dsl_tool_b200 import moe_decode, moe_forward
    x, logits, w = make(16, 16, 1024, 512, 512, "fp8_block128")
    a, b, want = moe_decode(x, logits, w, 4), moe_forward(x, logits, w, 4), layer(x, logits, w, 4)
    assert far(a, want) < far(b, want) < 0.1


def test_strides_threads_capture(cuda_device):
    import threading
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(8, 16, 512, 256, 384, "nvfp4")
    want = moe_decode(x, logits, w, 4)
    assert torch.equal(moe_decode(x.t().contiguous().t(), logits.t().contiguous().t(), w, 4), want)
    static_x, static_l = x.clone(), logits.clone()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = moe_decode(static_x, static_l, w, 4)
        graphs.append((g, out))
    others = [make(8, 16, 512, 256, 384, "nvfp4", seed=s)[:2] for s in (1, 2, 3)]
    results = [moe_decode(a, b, w, 4) for a, b in others]
    side = torch.cuda.Stream()
    for (a, b), r in zip(others, results):
        static_x.copy_(a)
        static_l.copy_(b)
        side.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
            eager = moe_decode(x, logits, w, 4)
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], r) and torch.equal(graphs[1][1], r) and torch.equal(eager, want)
    got = {}

    def work(i):
        got[i] = [moe_decode(a, b, w, 4) for a, b in others]
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(u, v) for r in got.values() for u, v in zip(r, results))


def test_decode_step(cuda_device):
    """Residual and norm, router, experts, residual and norm to the next projection: a decode step's feed-forward half."""
    from dsl_tool_b200 import linear, moe_decode, pack_weight, rms_norm
    x, _, w = make(6, 16, 512, 256, 512, "nvfp4")
    r, gain = torch.randn(6, 512, device="cuda").bfloat16(), torch.rand(512, device="cuda").bfloat16()
    router = pack_weight(torch.randn(16, 512, device="cuda") * 0.1, "bf16")
    proj = pack_weight(torch.randn(256, 512, device="cuda") * 0.05, "int8")
    y, _, t = rms_norm(x, gain, residual=r)
    logits = linear(y, router)
    o = moe_decode(y, logits, w, 4, out_dtype=torch.bfloat16)
    q, s, t2 = rms_norm(o, gain, residual=t, format="int8")
    z = linear(q, proj, act_scale=s)
    want = layer(y, logits, w, 4).bfloat16()
    tw = (want.float() + t.float()).double()
    yw = tw / torch.sqrt(tw.square().mean(1, keepdim=True) + 1e-6) * gain.double()
    # bf16 roundings of o and t (half a step: 2^-8 each) and the int8 rounding of y: at most half a step, amax / 254, in each of
    # a row's 512 elements (rows hold values of 20 sigma, so this is the largest part)
    steps = (yw.abs().amax(1) / 254).norm() * 512 ** 0.5 / yw.norm()
    assert far(z, yw @ values(proj)[0].t()) <= 2 * 2.0 ** -8 + steps.item()


def test_refusals(cuda_device):
    from dsl_tool_b200 import MoEWeights, moe_decode
    x, logits, w = make(4, 6, 256, 128, 128, "nvfp4")
    with pytest.raises(ValueError, match="at most 32 tokens"):
        moe_decode(torch.zeros(33, 256, device="cuda"), torch.zeros(33, 6, device="cuda"), w, 2)
    with pytest.raises(ValueError, match="k must lie"):
        moe_decode(x, logits, w, 7)
    with pytest.raises(ValueError, match="k must lie"):
        moe_decode(x, logits, w, 0)
    with pytest.raises(ValueError, match="logits must be"):
        moe_decode(x, logits[:3], w, 2)
    with pytest.raises(TypeError, match="logits must be"):
        moe_decode(x, logits.half(), w, 2)
    with pytest.raises(TypeError, match="x must be"):
        moe_decode(x.double(), logits, w, 2)
    with pytest.raises(ValueError, match="x must be"):
        moe_decode(x[:, :128], logits, w, 2)
    with pytest.raises(ValueError, match="out_dtype"):
        moe_decode(x, logits, w, 2, out_dtype=torch.float16)
    with pytest.raises(ValueError, match="all 6 experts"):
        moe_decode(x, logits, MoEWeights(w.gate_up, w.down, 0, 3, 6), 2)
    plain = make(4, 6, 256, 128, 128, "nvfp4")[2]
    plain.gate_up.gate_up_interleaved = False
    with pytest.raises(ValueError, match="gate_up_interleave"):
        moe_decode(x, logits, plain, 2)
    bad = make(4, 6, 256, 128, 128, "nvfp4")[2]
    bad.down.scale = bad.down.scale[:-512]
    with pytest.raises(ValueError, match="lays them out"):
        moe_decode(x, logits, bad, 2)
    with pytest.raises(ValueError, match="fit a CTA"):
        x2, l2, w2 = make(1, 2, 65536, 32, 16, "bf16", dtype=torch.float32)
        moe_decode(x2, l2, w2, 1)
    assert moe_decode(x[:0], logits[:0], w, 2).shape == (0, 128)


@pytest.mark.parametrize("fmt", ["bf16", "int8", "nvfp4", "mxfp4"])
def test_most_tokens_experts_and_slots(cuda_device, fmt):
    """32 tokens that choose 32 of 1024 experts each: 1024 entries, hundreds of experts with one or a few rows."""
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(32, 1024, 128, 32, 24, fmt)
    got = moe_decode(x, logits, w, 32)
    assert far(got, layer(x, logits, w, 32)) <= bound(fmt, x.dtype)
    assert torch.equal(moe_decode(x, logits, w, 32), got)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("T,k", [(32, 1), (31, 2)])
def test_all_tokens_choose_the_same_experts(cuda_device, fmt, T, k):
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(T, 300, 384, 128, 200, fmt)
    logits[:, [7, 299]] += 100.0
    assert far(moe_decode(x, logits, w, k), layer(x, logits, w, k)) <= bound(fmt, x.dtype)


@pytest.mark.parametrize("K", [8, 72, 136])
def test_infinite_weight_at_the_end_of_a_row(cuda_device, K):
    """What stands behind a row's end in a step of 64 bytes adds nothing to it, not the NaN that an infinity against a zero makes."""
    from dsl_tool_b200 import moe_decode
    x, logits, w = make(3, 2, K, 16, 24, "bf16")
    x[:, K - 1] = x[:, K - 1].abs() + 0.5
    w.gate_up.q[10, K - 1] = float("inf")                   # gate 5 of expert 0
    got, want = moe_decode(x, logits, w, 2), layer(x, logits, w, 2)
    assert torch.isinf(want).all()
    assert torch.equal(got.double(), want)
