"""What the 8-bit floating point operators are measured on: the cases, their inputs, the work they cannot do without, their
plain form in elementary torch operations, and their values in 64 bits.

    quant    activations [T, H] -> e4m3 values and one scale per token and group of 128 features
    silu     gate/up rows [T, 2 I] -> silu(g) * u as e4m3 values and group scales (in front of down_proj)
    norm     RMSNorm, with or without the residual add, -> e4m3 values and group scales (in front of qkv_proj / gate_up_proj)
    gemm     the matrix product of e4m3 activations and weights, one scale per token group and per 128 x 128 weight block
    linear   fp16 / bf16 activations times such a weight, as a linear layer's forward runs it

Scales: amax of the group / 448, amax at least 2^-96.  A last group or block may be shorter than 128.
"""
import math

import torch

own = False

DEV = "cuda"
GROUP = 128
QMAX = 448.0            # the largest finite e4m3 value
AMAX_MIN = 2.0 ** -96
E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---- cases -----------------------------------------------------------------------------------------
def listed():
    return [
        # o_proj / qkv_proj input of a decode batch (hidden 4096): launch latency
        {"name": "quant 16x4096", "op": "quant", "T": 16, "H": 4096, "dtype": "bf16"},
        # down_proj input of a 4096-token prefill, quantised by itself: bandwidth
        {"name": "quant 4096x14336", "op": "quant", "T": 4096, "H": 14336, "dtype": "bf16"},
        # one user's token through the MLP activation: launch latency
        {"name": "silu 1x14336", "op": "silu", "T": 1, "H": 14336, "dtype": "bf16"},
        # the MLP activation of a 4096-token prefill: bandwidth
        {"name": "silu 4096x14336", "op": "silu", "T": 4096, "H": 14336, "dtype": "bf16"},
        # the norm in front of gate_up_proj in a decode batch: launch latency
        {"name": "norm 16x4096", "op": "norm", "T": 16, "H": 4096, "dtype": "bf16", "residual": True},
        # the norm of a larger model's prefill, fp16: bandwidth
        {"name": "norm 4096x8192", "op": "norm", "T": 4096, "H": 8192, "dtype": "fp16", "residual": True},
        # gate_up_proj of a decode batch: the weights' bytes
        {"name": "gemm 16x28672x4096", "op": "gemm", "T": 16, "N": 28672, "K": 4096, "dtype": "bf16", "bias": False},
        # a small ragged layer: no size a multiple of the tile or the group
        {"name": "gemm 333x1000x1080", "op": "gemm", "T": 333, "N": 1000, "K": 1080, "dtype": "fp16", "bias": True},
        # o_proj of a short prefill: between bandwidth and matrix rate
        {"name": "gemm 512x4096x4096", "op": "gemm", "T": 512, "N": 4096, "K": 4096, "dtype": "bf16", "bias": False},
        # gate_up_proj of a 4096-token prefill: matrix rate
        {"name": "gemm 4096x28672x4096", "op": "gemm", "T": 4096, "N": 28672, "K": 4096, "dtype": "bf16", "bias": False},
        # qkv_proj of one user's token: weights' bytes and latency
        {"name": "linear 1x6144x4096", "op": "linear", "T": 1, "N": 6144, "K": 4096, "dtype": "bf16", "bias": True},
        # down_proj of a large decode batch: a long K
        {"name": "linear 128x4096x14336", "op": "linear", "T": 128, "N": 4096, "K": 14336, "dtype": "bf16", "bias": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quant", "silu", "norm", "gemm", "gemm", "linear"])
    case = {"op": op, "T": _log(rng, 1, 4096), "dtype": rng.choice(["bf16", "fp16"])}
    if op in ("quant", "silu", "norm"):
        h = _log(rng, 256, 14336)
        case["H"] = h if rng.random() < 0.25 else max(8, h // 8 * 8)
        if op == "norm":
            case["residual"] = rng.random() < 0.7
    else:
        n, k = _log(rng, 128, 28672), _log(rng, 128, 14336)
        while n * k > 28672 * 4096:
            n = max(1, n // 2)
        case["N"] = n if rng.random() < 0.25 else max(16, n // 16 * 16)
        case["K"] = k if rng.random() < 0.15 else max(16, k // 16 * 16)
        case["bias"] = rng.random() < 0.3
    return case


def work(case):
    T = case["T"]
    if case["op"] in ("quant", "silu", "norm"):
        H = case["H"]
        out = T * H + 4 * T * _blocks(H)
        if case["op"] == "quant":
            return {"bytes": 2 * T * H + out, "flops": 3 * T * H}
        if case["op"] == "silu":
            return {"bytes": 4 * T * H + out, "flops": 8 * T * H}
        res = 4 * T * H if case["residual"] else 0
        return {"bytes": 2 * T * H + res + 2 * H + out, "flops": 8 * T * H}
    N, K = case["N"], case["K"]
    weight = N * K + 4 * _blocks(N) * _blocks(K) + (2 * N if case["bias"] else 0)
    x = 2 * T * K if case["op"] == "linear" else T * K + 4 * T * _blocks(K)
    return {"bytes": x + weight + 2 * T * N, "flops": 2 * T * N * K}


def _blocks(n):
    return (n + GROUP - 1) // GROUP


# ---- inputs ----------------------------------------------------------------------------------------
def _activations(T, H, dt, gen):
    """Token rows as a decoder's residual stream has them: tokens of different size, a few channels far above the others."""
    x = torch.randn(T, H, generator=gen, device=DEV)
    x *= torch.exp(0.5 * torch.randn(T, 1, generator=gen, device=DEV))
    big = torch.rand(H, generator=gen, device=DEV) < 0.01
    return (x * torch.where(big, 12.0, 1.0)).to(dt)


def _pad(x, rows=1):
    return torch.nn.functional.pad(x, (0, -x.shape[1] % GROUP, 0, -x.shape[0] % rows))


def _weight(N, K, gen):
    """A dense weight in 128 x 128 blocks: e4m3 values and fp32 scales, as a checkpoint holds them."""
    w = torch.randn(N, K, generator=gen, device=DEV) / K ** 0.5
    w *= torch.exp(0.3 * torch.randn(N, 1, generator=gen, device=DEV))
    NB, KB = _blocks(N), _blocks(K)
    b = _pad(w, GROUP).view(NB, GROUP, KB, GROUP)
    s = b.abs().amax((1, 3)).clamp_min(AMAX_MIN) / QMAX
    q = (b / s.view(NB, 1, KB, 1)).to(E4M3).view(NB * GROUP, KB * GROUP)
    return q.view(torch.uint8)[:N, :K].contiguous().view(E4M3), s


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    dt, T, op = DTYPES[case["dtype"]], case["T"], case["op"]
    s = {"op": op, "dt": dt}
    if op == "quant":
        s["x"] = _activations(T, case["H"], dt, gen)
    elif op == "silu":
        s["x"] = (2 * torch.randn(T, 2 * case["H"], generator=gen, device=DEV)).to(dt)
    elif op == "norm":
        H = case["H"]
        s["x"] = torch.randn(T, H, generator=gen, device=DEV).to(dt)
        s["residual"] = _activations(T, H, dt, gen) if case["residual"] else None
        s["w"] = (1 + 0.2 * torch.randn(H, generator=gen, device=DEV)).to(dt)
        s["eps"] = 1e-5
    else:
        N, K = case["N"], case["K"]
        x = _activations(T, K, dt, gen)
        s["w"], s["ws"] = _weight(N, K, gen)
        s["bias"] = torch.randn(N, generator=gen, device=DEV).to(dt) if case["bias"] else None
        if op == "linear":
            s["x"] = x
        else:
            q, xs = _quant(x.float())
            s["q"], s["xs"] = q, xs.t().contiguous().t()      # [T, K / 128], tokens adjacent in memory, as the quantising operators return it
    return s


# ---- the plain form, in 32 bits --------------------------------------------------------------------
def _quant(v):
    """fp32 rows -> (e4m3 values, fp32 group scales)."""
    T, H = v.shape
    b = _pad(v).view(T, -1, GROUP)
    s = b.abs().amax(2).clamp_min(AMAX_MIN) / QMAX
    q = (b / s.unsqueeze(2)).to(E4M3).view(T, -1)
    return (q if q.shape[1] == H else q.view(torch.uint8)[:, :H].contiguous().view(E4M3)), s


def _matmul(q, xs, w, ws, bias, dt):
    K, N = q.shape[1], w.shape[0]
    x = q.float() * xs.repeat_interleave(GROUP, 1)[:, :K]
    wd = w.float() * ws.repeat_interleave(GROUP, 0)[:N].repeat_interleave(GROUP, 1)[:, :K]
    y = x @ wd.t()
    return (y if bias is None else y + bias.float()).to(dt)


def _silu_mul(x):
    g, u = x.float().chunk(2, 1)
    return g / (1 + torch.exp(-g)) * u


def _plain(s):
    if s["op"] == "quant":
        return _quant(s["x"].float())
    if s["op"] == "silu":
        return _quant(_silu_mul(s["x"]))
    if s["op"] == "norm":
        z = s["x"].float()
        if s["residual"] is not None:
            z = z + s["residual"].float()
            s["residual"].copy_(z)
        v = z * torch.rsqrt((z * z).mean(1, keepdim=True) + s["eps"]) * s["w"].float()
        return (*_quant(v), s["residual"])
    if s["op"] == "gemm":
        return _matmul(s["q"], s["xs"], s["w"], s["ws"], s["bias"], s["dt"])
    return _matmul(*_quant(s["x"].float()), s["w"], s["ws"], s["bias"], s["dt"])


# ---- one pass --------------------------------------------------------------------------------------
def run(s):
    if not own:
        return _plain(s)
    from vllm_pq_amd import ops
    if s["op"] == "quant":
        return ops.fp8_group_quant(s["x"])
    if s["op"] == "silu":
        return ops.silu_and_mul_fp8(s["x"])
    if s["op"] == "norm":
        if s["residual"] is None:
            return (*ops.rms_norm_fp8(s["x"], s["w"], s["eps"]), None)
        return (*ops.fused_add_rms_norm_fp8(s["x"], s["residual"], s["w"], s["eps"]), s["residual"])
    if s["op"] == "gemm":
        return ops.fp8_block_gemm(s["q"], s["xs"], s["w"], s["ws"], s["bias"], s["dt"])
    return ops.fp8_block_linear(s["x"], s["w"], s["ws"], s["bias"])


# ---- the values in 64 bits -------------------------------------------------------------------------
def _round_e4m3(v):
    """Nearest e4m3 value (ties to even) of float64 values up to 448 in magnitude: 3 bits behind the leading one, at least 2^-9 a step."""
    step = torch.ldexp(torch.ones_like(v), (torch.frexp(v).exponent - 4).clamp_min(-9))
    return torch.round(v / step) * step


def _exact_quant(v):
    """Row by row of groups, padded groups apart; the scale is held in 32 bits and the values are divided by what is held."""
    qs, ss = [], []
    for k in range(0, v.shape[1], GROUP):
        g = v[:, k:k + GROUP]
        s = (g.abs().amax(1, keepdim=True).clamp_min(AMAX_MIN) / QMAX).float().double()
        qs.append(_round_e4m3(g / s))
        ss.append(s)
    return torch.cat(qs, 1), torch.cat(ss, 1)


def _exact_product(q, s, w, ws, bias):
    wd = w.double()
    for j in range(ws.shape[0]):
        for k in range(ws.shape[1]):
            wd[j * GROUP:(j + 1) * GROUP, k * GROUP:(k + 1) * GROUP] *= ws[j, k].double()
    xd = q.double()
    for k in range(ws.shape[1]):
        xd[:, k * GROUP:(k + 1) * GROUP] *= s[:, k:k + 1].double()
    y = torch.mm(xd, wd.t())
    return y if bias is None else y + bias.double()


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quant":
        return _exact_quant(s["x"].double())
    if s["op"] == "silu":
        half = s["x"].shape[1] // 2
        g, u = s["x"][:, :half].double(), s["x"][:, half:].double()
        return _exact_quant(g * torch.sigmoid(g) * u)
    if s["op"] == "norm":
        z = s["x"].double()
        if s["residual"] is not None:
            z = z + s["residual"].double()
        rms = torch.sqrt(z.square().sum(1, keepdim=True) / z.shape[1] + s["eps"])
        return (*_exact_quant(z / rms * s["w"].double()), z if s["residual"] is not None else None)
    if s["op"] == "gemm":
        return _exact_product(s["q"], s["xs"], s["w"], s["ws"], s["bias"])
    q, xs = _exact_quant(s["x"].double())
    return _exact_product(q, xs, s["w"], s["ws"], s["bias"])
