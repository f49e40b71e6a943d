"""Operators of a quantised language model next to the framework's GEMMs, as measurable cases: inputs, the plain form in elementary
torch operations, the call that a user of the framework makes, and the result in 64 bits.

* ``int8_linear``  activations [M, K] times a weight of 8-bit integers with one scale per output channel; the activations are
                   quantised within the call with one scale per token.
* ``norm``         root-mean-square norm of x (+ residual), the result in 8 bits with its scales, the sum as new residual.
* ``norm_linear``  the norm with an 8-bit result and the int8 product that reads it, as a layer's projections use them.
* ``moe_decode``   a whole mixture-of-experts feed-forward layer for a few tokens: routing, gate/up, SwiGLU, down, combine, the
                   activations unquantised, the experts' weights in any packed format.
"""
from __future__ import annotations

import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
# bytes of a packed weight per element, scales included
_PACKED = {"fp8": 1.0, "fp8_block128": 1.0 + 4.0 / (128 * 128), "int8": 1.0, "nvfp4": 0.5 + 1.0 / 16, "mxfp4": 0.5 + 1.0 / 32, "bf16": 2.0}
_EPS = 1e-6


def _int8_linear(name, m, k, n, activation="none", out="bf16", dtype="bf16"):
    case = dict(op="int8_linear", m=m, k=k, n=n, activation=activation, out=out, dtype=dtype)
    return dict(case, name=name) if name else case


def _norm(name, m, k, format, residual, dtype="bf16"):
    case = dict(op="norm", m=m, k=k, format=format, residual=residual, dtype=dtype)
    return dict(case, name=name) if name else case


def _norm_linear(name, m, k, n, residual, dtype="bf16"):
    case = dict(op="norm_linear", m=m, k=k, n=n, residual=residual, dtype=dtype)
    return dict(case, name=name) if name else case


def _moe(name, format, tokens, experts, topk, k, h, d, dtype="bf16"):
    case = dict(op="moe_decode", format=format, tokens=tokens, experts=experts, topk=topk, k=k, h=h, d=d, dtype=dtype)
    return dict(case, name=name) if name else case


def listed():
    return [
        # one sequence generating text: one token through a square projection with an int8 weight
        _int8_linear("int8_m1", 1, 8192, 8192),
        # a small odd batch of sequences through the 70B MLP's down projection: the long K
        _int8_linear("int8_m24", 24, 28672, 8192),
        # a ragged chunk of prefill through the 8B MLP's gate/up projection, gate folded into the product
        _int8_linear("int8_swiglu_m1000", 1000, 4096, 28672, activation="swiglu"),
        # prefill through the 8B MLP's up projection, result in fp32: the largest product
        _int8_linear("int8_m4096_fp32", 4096, 4096, 14336, out="fp32"),
        # one token's norm before block-scaled FP8 projections: latency is all there is
        _norm("norm_fp8_m1", 1, 4096, "fp8_block128", True),
        # the norm of a long prefill before block-scaled FP8 projections: the largest one
        _norm("norm_fp8_m8192", 8192, 8192, "fp8_block128", True),
        # a decode batch: residual, norm, int8 projection
        _norm_linear("norm_int8_m16", 16, 4096, 14336, True),
        # a ragged prefill in fp16: the first norm of a model (no residual yet) and its int8 projection
        _norm_linear("norm_int8_m2047", 2047, 4096, 4096, False, dtype="fp16"),
        # one sequence generating text: one token through a layer of 64 experts in NVFP4
        _moe("moe_nvfp4_t1", "nvfp4", 1, 64, 8, 4096, 1536, 4096),
        # eight sequences through the layer with block-scaled FP8 experts
        _moe("moe_fp8_block_t8", "fp8_block128", 8, 64, 8, 4096, 1536, 4096),
        # three sequences through a layer of few large unquantised experts
        _moe("moe_bf16_t3", "bf16", 3, 8, 2, 4096, 14336, 4096),
        # sixteen sequences through a layer of many experts in MXFP4, odd sizes: the most rows
        _moe("moe_mxfp4_t16", "mxfp4", 16, 128, 8, 2912, 1440, 2880),
    ]


def _log(rng, low, high, multiple=1):
    """A whole number between low and high, spread over the logarithm, a multiple of `multiple`."""
    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(-(-low // multiple), min(high // multiple, round(v / multiple))) * multiple


def draw(rng):
    op = rng.choices(("int8_linear", "norm", "norm_linear", "moe_decode"), weights=(3, 2, 2, 4))[0]
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "int8_linear":
        k, n = _log(rng, 1024, 28672, 16), _log(rng, 1024, 28672, 2)
        m = _log(rng, 1, 128) if rng.random() < 0.5 else _log(rng, 129, 8192)
        m = max(1, min(m, int(4096.0 * 4096 * 14336 / (k * n))))
        return _int8_linear(None, m, k, n, rng.choice(("none", "none", "swiglu")), rng.choice(("bf16", "fp32")), dtype)
    if op == "norm":
        k = _log(rng, 512, 16384, 16)
        return _norm(None, max(1, min(_log(rng, 1, 16384), 8192 * 4096 // k)), k, rng.choice(("fp8_block128", "fp8_block128", "fp8")),
                     rng.random() < 0.7, dtype)
    if op == "norm_linear":
        k, n = _log(rng, 1024, 8192, 16), _log(rng, 1024, 14336, 2)
        m = _log(rng, 1, 128) if rng.random() < 0.5 else _log(rng, 129, 8192)
        return _norm_linear(None, max(1, min(m, int(2048.0 * 8192 * 8192 / (k * n)))), k, n, rng.random() < 0.7, dtype)
    format = rng.choice(("nvfp4", "mxfp4", "fp8_block128", "fp8", "int8", "bf16"))
    multiple = 128 if format == "fp8_block128" else 32
    experts = rng.choice((8, 16, 32, 64, 128))
    topk = rng.choice((1, 2, 4, 6, 8))
    k, h, d = _log(rng, 1024, 4096, multiple), _log(rng, 512, 1536, multiple), _log(rng, 1024, 4096, 2)
    return _moe(None, format, _log(rng, 1, 16), experts, topk, k, h, d, rng.choice(("bf16", "bf16", "fp16")))


# ---- inputs ------------------------------------------------------------------------------------------------------------------

def _activations(gen, shape, dtype):
    """Activations as they come: N(0, 1) with one value in a thousand at 20."""
    a = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    big = torch.rand(shape, generator=gen, device="cuda") < 1e-3
    a = torch.where(big, torch.copysign(torch.full_like(a, 20.0), a), a)
    return a.to(_DTYPES[dtype])


def _tiles(scale_bytes, groups, n):
    """Scale bytes [groups * n, blocks] -> the framework's tile layout: per group and 128 rows x 4 blocks 512 bytes, byte (r, c) at
    (r % 32) * 16 + (r / 32) * 4 + c, zeros where there is no row or block."""
    blocks = scale_bytes.shape[1]
    s = scale_bytes.reshape(groups, n, blocks)
    s = torch.nn.functional.pad(s, (0, -blocks % 4, 0, -n % 128))
    s = s.reshape(groups, s.shape[1] // 128, 4, 32, s.shape[2] // 4, 4)
    return s.permute(0, 1, 4, 3, 2, 5).contiguous().reshape(-1)


def _untile(tiles, groups, n, blocks):
    s = tiles.reshape(groups, -(-n // 128), -(-blocks // 4), 32, 4, 4).permute(0, 1, 4, 3, 2, 5)
    return s.reshape(groups, -(-n // 128) * 128, -(-blocks // 4) * 4)[:, :n, :blocks]


def _packed_weight(gen, groups, n, k, format):
    """A weight N(0, 0.02) in a packed format: {"q", "scale", "global_scale"} laid out as the framework keeps it."""
    w = torch.randn((groups * n, k), generator=gen, device="cuda", dtype=torch.bfloat16).mul_(0.02)
    if format == "bf16":
        return dict(q=w, scale=None, global_scale=None)
    if format == "fp8":
        s = (w.abs().amax().float() / 448.0).reshape(1)
        return dict(q=(w.float() / s).to(torch.float8_e4m3fn).view(torch.uint8), scale=s, global_scale=None)
    if format == "int8":
        s = w.abs().amax(dim=1).float().div_(127.0).clamp_(min=1e-12)
        return dict(q=w.float().div_(s[:, None]).round_().to(torch.int8), scale=s, global_scale=None)
    if format == "fp8_block128":
        p = torch.nn.functional.pad(w.reshape(groups, n, k), (0, 0, 0, -n % 128)).reshape(groups, -(-n // 128), 128, k // 128, 128)
        s = p.abs().amax(dim=(2, 4)).float().div_(448.0).clamp_(min=1e-12)
        q = (p.float() / s[:, :, None, :, None]).reshape(groups, -1, k)[:, :n].reshape(groups * n, k)
        return dict(q=q.to(torch.float8_e4m3fn).view(torch.uint8), scale=s, global_scale=None)
    block = 16 if format == "nvfp4" else 32
    b = w.reshape(groups * n, k // block, block)
    amax = b.abs().amax(dim=2).float()
    if format == "nvfp4":
        gs = (amax.amax() / 2688.0).reshape(1)
        code = (amax / 6.0 / gs).to(torch.float8_e4m3fn)
        step = code.float() * gs
        code = code.view(torch.uint8)
    else:
        gs = None
        e = torch.floor(torch.log2(amax.clamp(min=1e-30))) - 2
        code, step = (e + 127).to(torch.uint8), torch.exp2(e)
    a = b.float() / step.clamp(min=1e-30)[:, :, None]
    m = a.abs()
    nibble = sum((m > t).to(torch.uint8) for t in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)) + (a < 0).to(torch.uint8) * 8
    nibble = nibble.reshape(groups * n, k // 2, 2)
    return dict(q=nibble[:, :, 0] | (nibble[:, :, 1] << 4), scale=_tiles(code, groups, n), global_scale=gs)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op = case["op"]
    state = dict(case=case)
    if op == "moe_decode":
        e, k, h, d = case["experts"], case["k"], case["h"], case["d"]
        state["x"] = _activations(gen, (case["tokens"], k), case["dtype"])
        state["logits"] = torch.randn((case["tokens"], e), generator=gen, device="cuda", dtype=torch.float32)
        state["gate_up"] = _packed_weight(gen, e, 2 * h, k, case["format"])
        state["down"] = _packed_weight(gen, e, d, h, case["format"])
        if own:
            from dsl_tool_b200 import MoEWeights, PackedWeight
            state["w"] = MoEWeights(PackedWeight(case["format"], **state["gate_up"], groups=e, n=2 * h, k=k, gate_up_interleaved=True),
                                    PackedWeight(case["format"], **state["down"], groups=e, n=d, k=h), 0, e, e)
        return state
    m, k = case["m"], case["k"]
    state["x"] = _activations(gen, (m, k), case["dtype"])
    if op != "int8_linear":
        state["gain"] = torch.rand((k,), generator=gen, device="cuda").add_(0.5).to(_DTYPES[case["dtype"]])
        state["residual"] = torch.randn((m, k), generator=gen, device="cuda").mul_(2.0).to(_DTYPES[case["dtype"]]) if case["residual"] else None
        # a calibrated scale of the norm's result for the per-tensor format
        state["scale"] = torch.full((1,), 20.0 / 448.0, device="cuda") if case.get("format") == "fp8" else None
    if op != "norm":
        state["weight"] = _packed_weight(gen, 1, case["n"], k, "int8")
        if own:
            from dsl_tool_b200 import PackedWeight
            state["w"] = PackedWeight("int8", **state["weight"], groups=1, n=case["n"], k=k, gate_up_interleaved=case.get("activation") == "swiglu")
    return state


# ---- plain forms -------------------------------------------------------------------------------------------------------------

def _int8_rows(y):
    """One scale per row, amax / 127, and the row's whole numbers: nearest, ties to even."""
    s = (y.abs().amax(dim=1, keepdim=True) / torch.full((), 127.0, device=y.device)).clamp_(min=1e-12)
    return torch.round(y / s), s


def _int8_product(y, weight):
    q, s = _int8_rows(y)
    return (q @ weight["q"].float().t()) * s * weight["scale"]


def _rms(state):
    x, r = state["x"], state["residual"]
    total = x if r is None else (x.float() + r.float()).to(x.dtype)        # the residual as the next layer reads it
    z = total.float()
    y = z * torch.rsqrt((z * z).mean(dim=1, keepdim=True) + _EPS) * state["gain"].float()
    return y, (None if r is None else total)


def _values(packed, groups, n, k, format, ids):
    """The values of the weights of experts `ids` in fp32: [len(ids), n, k]."""
    q = packed["q"].reshape(groups, n, -1)[ids]
    if format == "bf16":
        return q.float()
    if format == "fp8":
        return q.view(torch.float8_e4m3fn).float() * packed["scale"]
    if format == "int8":
        return q.float() * packed["scale"].reshape(groups, n, 1)[ids]
    if format == "fp8_block128":
        s = packed["scale"][ids].repeat_interleave(128, dim=1)[:, :n].repeat_interleave(128, dim=2)
        return q.view(torch.float8_e4m3fn).float() * s
    e2m1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=q.device)
    pairs = torch.stack((e2m1.repeat(16), e2m1.repeat_interleave(16)), dim=1)      # byte -> (low, high) nibble's value
    block = 16 if format == "nvfp4" else 32
    tiles = packed["scale"][:groups * (-(-n // 128)) * (-(-(k // block) // 4)) * 512]
    s = _untile(tiles, groups, n, k // block)[ids]
    s = s.contiguous().view(torch.float8_e4m3fn).float() * packed["global_scale"] if format == "nvfp4" else torch.exp2(s.float() - 127.0)
    return (pairs[q.int()].reshape(len(ids), n, k // block, block) * s[:, :, :, None]).reshape(len(ids), n, k)


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "int8_linear":
        y = _int8_product(state["x"].float(), state["weight"])
        if case["activation"] == "swiglu":
            y = y[:, 0::2] * torch.sigmoid(y[:, 0::2]) * y[:, 1::2]
        return y.to(_DTYPES[case["out"]])
    if op == "norm":
        y, total = _rms(state)
        m, k = y.shape
        if case["format"] == "fp8":
            q, s = (y / state["scale"]).clamp(-448.0, 448.0), None
        else:
            groups = torch.nn.functional.pad(y, (0, -k % 128)).reshape(m, -1, 128)
            s = (groups.abs().amax(dim=2) / torch.full((), 448.0, device=y.device)).clamp_(min=1e-12)
            q = (groups / s[:, :, None]).reshape(m, -1)[:, :k]
        return dict(q=q.contiguous().to(torch.float8_e4m3fn), s=s, total=total)
    if op == "norm_linear":
        y, total = _rms(state)
        return dict(y=_int8_product(y, state["weight"]).to(torch.bfloat16), total=total)
    t, e, k, h, d, topk = (case[v] for v in ("tokens", "experts", "k", "h", "d", "topk"))
    order = torch.sort(state["logits"], dim=1, descending=True, stable=True)[1][:, :topk]
    p = torch.exp(state["logits"] - state["logits"].amax(dim=1, keepdim=True))
    p = torch.gather(p / p.sum(dim=1, keepdim=True), 1, order)
    p = p / p.sum(dim=1, keepdim=True)
    ids = order.reshape(-1)
    rows = state["x"].float().repeat_interleave(topk, dim=0)
    g = torch.bmm(_values(state["gate_up"], e, 2 * h, k, case["format"], ids), rows[:, :, None])[:, :, 0]
    g = g[:, 0::2] * torch.sigmoid(g[:, 0::2]) * g[:, 1::2]
    y = torch.bmm(_values(state["down"], e, d, h, case["format"], ids), g[:, :, None])[:, :, 0]
    return (y.reshape(t, topk, d) * p[:, :, None]).sum(dim=1).to(torch.bfloat16)


def run(state):
    if not own:
        return _plain(state)
    import dsl_tool_b200 as dsl
    case = state["case"]
    op = case["op"]
    if op == "int8_linear":
        return dsl.linear(state["x"], state["w"], out_dtype=_DTYPES[case["out"]], activation=case["activation"])
    if op == "norm":
        q, s, total = dsl.rms_norm(state["x"], state["gain"], eps=_EPS, residual=state["residual"], format=case["format"], scale=state["scale"])
        return dict(q=q.view(torch.float8_e4m3fn), s=None if case["format"] == "fp8" else s, total=total)
    if op == "norm_linear":
        q, s, total = dsl.rms_norm(state["x"], state["gain"], eps=_EPS, residual=state["residual"], format="int8")
        return dict(y=dsl.linear(q, state["w"], act_scale=s, out_dtype=torch.bfloat16), total=total)
    return dsl.moe_decode(state["x"], state["logits"], state["w"], case["topk"], out_dtype=torch.bfloat16)


def work(case):
    op = case["op"]
    if op == "moe_decode":
        t, e, k, h, d = (case[v] for v in ("tokens", "experts", "k", "h", "d"))
        used = e * (1.0 - (1.0 - case["topk"] / e) ** t)        # experts that some token is routed to, on average
        return {"bytes": used * h * (2 * k + d) * _PACKED[case["format"]] + t * k * _BYTES[case["dtype"]] + t * e * 4 + t * d * 2,
                "flops": 2.0 * t * case["topk"] * h * (2 * k + d)}
    m, k = case["m"], case["k"]
    size = _BYTES[case["dtype"]]
    bytes_ = m * k * size
    if op != "int8_linear":
        bytes_ += k * size + (2 * m * k * size if case["residual"] else 0)      # gain, residual in and out
    if op == "norm":
        return {"bytes": bytes_ + m * k + (4 * m * (-(-k // 128)) if case["format"] == "fp8_block128" else 0), "flops": 6.0 * m * k}
    n = case["n"]
    columns = n // 2 if case.get("activation") == "swiglu" else n
    return {"bytes": bytes_ + n * k + 4 * n + m * columns * _BYTES[case.get("out", "bf16")], "flops": 2.0 * m * n * k}


# ---- in 64 bits --------------------------------------------------------------------------------------------------------------

def _exact_int8(y, weight):
    """The int8 product of the rows y: scales and quotients are fp32 by definition, everything else is exact."""
    amax = y.abs().max(dim=1).values
    s = (amax / 127.0).float().clamp(min=1e-12).double()
    q = (y / s[:, None]).float().double().round()
    return torch.mm(q, weight["q"].double().t()) * torch.outer(s, weight["scale"].double())


def _exact_rms(state):
    x = state["x"].double()
    total = None
    if state["residual"] is not None:
        total = (x + state["residual"].double()).to(state["x"].dtype)
        x = total.double()
    return x / torch.sqrt(x.square().sum(dim=1, keepdim=True) / x.shape[1] + _EPS) * state["gain"].double(), total


def _exact_expert(packed, e, n, k, format):
    """One expert's weight from its bits."""
    q = packed["q"][e * n:(e + 1) * n]
    if format in ("bf16", "int8"):
        w = q.double()
        return w if format == "bf16" else w * packed["scale"][e * n:(e + 1) * n].double()[:, None]
    if format in ("fp8", "fp8_block128"):
        w = q.view(torch.float8_e4m3fn).double()
        if format == "fp8":
            return w * packed["scale"].double()
        rows, cols = torch.arange(n, device=q.device) // 128, torch.arange(k, device=q.device) // 128
        return w * packed["scale"][e].double()[rows][:, cols]
    bits = torch.empty((n, k), dtype=torch.int64, device=q.device)
    bits[:, 0::2], bits[:, 1::2] = q.long() & 15, q.long() >> 4
    exponent, fraction = (bits >> 1) & 3, (bits & 1).double()
    w = torch.where(exponent == 0, 0.5 * fraction, (1.0 + 0.5 * fraction) * torch.exp2(exponent.double() - 1.0))
    w = torch.where(bits >= 8, -w, w)
    block = 16 if format == "nvfp4" else 32
    kt = -(-(k // block) // 4)
    r, c = torch.arange(n, device=q.device)[:, None], torch.arange(k, device=q.device)[None, :] // block
    at = ((e * (-(-n // 128)) + r // 128) * kt + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4
    code = packed["scale"][at]
    return w * (code.view(torch.float8_e4m3fn).double() * packed["global_scale"].double() if format == "nvfp4" else torch.exp2(code.double() - 127.0))


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "int8_linear":
        y = _exact_int8(state["x"].double(), state["weight"])
        if case["activation"] == "swiglu":
            gate, up = y[:, 0::2], y[:, 1::2]
            y = gate / (1.0 + torch.exp(-gate)) * up
        return y
    if op == "norm_linear":
        y, total = _exact_rms(state)
        return dict(y=_exact_int8(y, state["weight"]), total=total)
    if op == "norm":
        y, total = _exact_rms(state)
        if case["format"] == "fp8":
            return dict(q=(y / state["scale"].double()).clamp(-448, 448).float().to(torch.float8_e4m3fn).double(), s=None, total=total)
        k = y.shape[1]
        starts = range(0, k, 128)
        s = torch.stack([y[:, i:i + 128].abs().max(dim=1).values / 448.0 for i in starts], dim=1).clamp(min=1e-12)
        q = torch.cat([y[:, i:i + 128] / s[:, i // 128, None] for i in starts], dim=1)
        return dict(q=q.float().to(torch.float8_e4m3fn).double(), s=s, total=total)
    t, e, k, h, d, topk = (case[v] for v in ("tokens", "experts", "k", "h", "d", "topk"))
    logits = state["logits"].double()
    out = torch.zeros((t, d), dtype=torch.float64, device="cuda")
    chosen = [sorted(range(e), key=lambda j, row=row: (-row[j], j))[:topk] for row in logits.tolist()]
    for j in sorted({j for row in chosen for j in row}):
        tokens = [i for i in range(t) if j in chosen[i]]
        share = torch.stack([torch.exp(logits[i, j]) / torch.exp(logits[i, chosen[i]]).sum() for i in tokens])
        g = state["x"][tokens].double() @ _exact_expert(state["gate_up"], j, 2 * h, k, case["format"]).t()
        hidden = g[:, 0::2] / (1.0 + torch.exp(-g[:, 0::2])) * g[:, 1::2]
        out[tokens] += share[:, None] * (hidden @ _exact_expert(state["down"], j, d, h, case["format"]).t())
    return out
