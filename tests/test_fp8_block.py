"""Linears in 8-bit floating point with scale blocks of 128 (pq_fp8_*): refusals on the CPU, and on the GPU every operator
through the public entry points against the definition in 64 bits.

Tolerances, from the arithmetic:
  fp8_group_quant   the scale is one correctly rounded fp32 division and the value one correctly rounded quotient followed
                    by one rounding to e4m3: bit for bit.  (A quotient rounded to 53 bits and then to 24 is the quotient
                    rounded to 24: 53 >= 2 * 24 + 2.)
  silu / norm       v in fp32: silu(g) takes exp(-g) with an error of |g| 2^-23 from the rounded exponent and a few units of
                    2^-24 (|g| < 16 here); the mean of squares sums at most 100 terms in a row (100 * 2^-24, halved by the root).
                    Both stay below V = 2^-17 relative.  The scale then carries V too, and q * scale is off v by half an
                    e4m3 step (2^-4 of |v|, or 2^-10 scale below the smallest normal) plus V.
  products          The matrix instruction (v_mfma_f32_16x16x128_f8f6f4) takes 8 products at a time, cuts each toward zero to
                    a multiple of 2^-13 of the power of two that the largest one's operand exponents give, and adds the groups
                    with fp32 precision (test_gpu_matrix_instruction shows all three).  The largest product of a group is exact
                    (8 significant bits), so a group is off by less than 7 * 2^-13 of its largest product, and a block by less than
                    7 * 2^-13 of its sum of magnitudes.  Then 16 groups, KB blocks and up to 16 waves, each addition off by at
                    most 2^-22 of the sum of magnitudes S:  (7 * 2^-13 + (16 + KB + 16) 2^-22) S, and half a step of the act dtype.
"""
import math

import pytest
import torch

from vllm_pq_amd import _lib, ops

DEV = "cuda:0"
F8 = torch.float8_e4m3fn
V = 2.0 ** -17
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}     # half the smallest step
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
gpu = pytest.mark.gpu


def blocks(n):
    return (n + 127) // 128


# ---- definitions in 64 bits ------------------------------------------------------------------------
def groups_of(v):
    return torch.nn.functional.pad(v, (0, -v.shape[-1] % 128)).unflatten(-1, (-1, 128))


def quant64(v):
    """(q as float64 values, scale) of float64 rows, by the definition."""
    g = groups_of(v)
    s = (g.abs().amax(-1).clamp_min(2.0 ** -96).float() / torch.tensor(448.0)).double()
    q = (g / s.unsqueeze(-1)).float().to(F8)
    return q.flatten(-2)[..., :v.shape[-1]].double(), s


def check_quant(q, s, v, loose):
    """loose: v is known to a relative error of V, else exactly."""
    q64, s64 = quant64(v)
    q, s = q.cpu(), s.cpu()
    assert q.dtype == F8 and s.dtype == torch.float32 and q.shape == v.shape and s.shape == s64.shape
    if not loose:
        assert torch.equal(s.double(), s64)
        assert torch.equal(q.double(), q64), int((q.double() != q64).sum())
        return
    assert ((s.double() - s64).abs() <= V * s64).all()
    sd = s.double().repeat_interleave(128, -1)[..., :v.shape[-1]]
    err = (q.double() * sd - v).abs()
    tol = torch.maximum(2.0 ** -4 * v.abs(), 2.0 ** -10 * sd) * (1 + 2.0 ** -10) + 2 * V * v.abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


def expand(w, ws):
    N, K = w.shape
    return w.double() * ws.double().repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]


def check_gemm(y, q, s, w, ws, bias, dev="cpu"):
    K = w.shape[1]
    x64 = q.to(dev).double().reshape(-1, K) * s.to(dev).double().reshape(-1, s.shape[-1]).repeat_interleave(128, 1)[:, :K]
    w64 = expand(w.to(dev), ws.to(dev))
    want, mag = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    if bias is not None:
        want, mag = want + bias.to(dev).double(), mag + bias.to(dev).double().abs()
    got = y.to(dev).double().reshape(want.shape)
    sums = 7 * 2.0 ** -13 + (32 + blocks(K)) * 2.0 ** -22
    tol = HALF[y.dtype] * want.abs() + sums * mag * (1 + HALF[y.dtype]) + SMALLEST[y.dtype]
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())


def activations(gen, T, H, dt, scale=1.0):
    x = torch.randn(T, H, generator=gen) * torch.exp(0.5 * torch.randn(T, 1, generator=gen))
    return (scale * x * torch.where(torch.rand(H, generator=gen) < 0.02, 12.0, 1.0)).to(dt)


def weight(gen, N, K):
    w = torch.randn(N, K, generator=gen) / max(K, 1) ** 0.5
    NB, KB = blocks(N), blocks(K)
    ws = torch.exp(0.5 * torch.randn(NB, KB, generator=gen)) * 2.0 ** -9
    return (w / ws.repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)[:, :K]).clamp(-448, 448).to(F8), ws


# ---- CPU: refusals ---------------------------------------------------------------------------------
def test_capability_bit():
    assert _lib.load().pq_caps() & (1 << 10)


def _quant_rc(fn="pq_fp8_group_quant", **kw):
    a = dict(x=256, xs=256, T=4, H=128, dtype=1, q=256, qs=128, s=256, ss=4)
    a.update(kw)
    return getattr(_lib.load(), fn)(a["x"], a["xs"], a["T"], a["H"], a["dtype"], a["q"], a["qs"], a["s"], a["ss"], None)


def test_quant_refusals_need_no_gpu():
    for fn in ("pq_fp8_group_quant", "pq_silu_and_mul_fp8"):
        assert _quant_rc(fn, dtype=2) == 1 and "dtype" in _lib.last_error()
        assert _quant_rc(fn, T=-1) == 1 and _quant_rc(fn, H=-5) == 1
        assert _quant_rc(fn, xs=127) == 1 and "strides" in _lib.last_error()
        assert _quant_rc(fn, qs=127) == 1
        assert _quant_rc(fn, ss=3) == 1 and "scale_group_stride" in _lib.last_error()
        for p in ("x", "q", "s"):
            assert _quant_rc(fn, **{p: None}) == 1 and "NULL" in _lib.last_error()
        assert _quant_rc(fn, T=0) == 0 and _quant_rc(fn, H=0) == 0      # nothing to do, nothing launched
    assert _quant_rc("pq_silu_and_mul_fp8", xs=255) == 1                # the input row is twice as long


def test_rows_that_do_not_fit_the_index_are_refused():
    big = 2 ** 31 - 1
    assert _quant_rc("pq_fp8_group_quant", H=big, xs=big, qs=big) == 2 and "elements" in _lib.last_error()
    assert _norm_rc(H=big, xs=big, rs=big, qs=big) == 2
    assert _gemm_rc(N=big, ys=big) == 1 and _gemm_rc(K=big, qs=big, wst=big, wss=big) == 1


def _norm_rc(**kw):
    a = dict(x=256, xs=128, r=256, rs=128, w=256, T=4, H=128, dtype=1, q=256, qs=128, s=256, ss=4)
    a.update(kw)
    return _lib.load().pq_fused_add_rms_norm_fp8(a["x"], a["xs"], a["r"], a["rs"], a["w"], 1e-5, a["T"], a["H"], a["dtype"],
                                                 a["q"], a["qs"], a["s"], a["ss"], None)


def test_norm_refusals_need_no_gpu():
    assert _norm_rc(r=None) == 1 and "residual" in _lib.last_error()
    assert _norm_rc(w=None) == 1 and _norm_rc(rs=100) == 1 and _norm_rc(xs=100) == 1
    assert _norm_rc(H=16392, xs=16392, rs=16392, qs=16392) == 2         # longer than a block holds
    assert _norm_rc(T=0) == 0


def _gemm_rc(linear=False, **kw):
    a = dict(q=256, T=4, qs=256, s=256, st=1, sg=4, w=256, wst=256, ws=256, wss=2, b=None, N=64, K=256, dtype=1, y=256, ys=64,
             tmp=256, tb=1 << 20)
    a.update(kw)
    L = _lib.load()
    tail = (a["w"], a["wst"], a["ws"], a["wss"], a["b"], a["N"], a["K"], a["dtype"], a["y"], a["ys"])
    if linear:
        return L.pq_fp8_block_linear(a["q"], a["T"], a["qs"], *tail, a["tmp"], a["tb"], None)
    return L.pq_fp8_block_gemm(a["q"], a["T"], a["qs"], a["s"], a["st"], a["sg"], *tail, a["tmp"], a["tb"], None)


@pytest.mark.parametrize("linear", [False, True])
def test_gemm_refusals_need_no_gpu(linear):
    for kw in (dict(dtype=3), dict(T=-1), dict(N=-1), dict(K=-1), dict(qs=255), dict(wst=255), dict(wss=1), dict(ys=63),
               dict(q=None), dict(w=None), dict(ws=None), dict(y=None)):
        assert _gemm_rc(linear, **kw) == 1, kw
    assert _gemm_rc(linear, T=0) == 0 and _gemm_rc(linear, N=0, ys=0) == 0
    if linear:
        need = _lib.load().pq_fp8_block_linear_tmp_bytes(64, 64, 256)
        assert _lib.load().pq_fp8_block_linear_tmp_bytes(1, 64, 256) == 0      # quantised inside
        assert need > 0
        assert _gemm_rc(True, T=64, tb=need - 1) == 3 and "tmp" in _lib.last_error()
        assert _gemm_rc(True, T=64, tmp=None) == 3 and _gemm_rc(True, T=64, tmp=264) == 1
        assert _lib.load().pq_fp8_block_linear_tmp_bytes(0, 64, 256) == 0
    else:
        assert _gemm_rc(st=-1) == 1 and _gemm_rc(s=None) == 1 and _gemm_rc(tmp=264) == 1


def test_linear_refuses_rows_too_far_apart():
    assert _gemm_rc(True, T=1, wst=2 ** 26) == 2 and "weight_row_stride" in _lib.last_error()     # where it quantises inside


def test_ops_raise_on_cpu_tensors():
    x, w = torch.zeros(2, 256, dtype=torch.bfloat16), torch.zeros(128, 256).to(F8)
    ws, one = torch.ones(1, 2), torch.ones(256, dtype=torch.bfloat16)
    for call in (lambda: ops.fp8_group_quant(x), lambda: ops.silu_and_mul_fp8(x), lambda: ops.rms_norm_fp8(x, one, 1e-5),
                 lambda: ops.fused_add_rms_norm_fp8(x, x, one, 1e-5), lambda: ops.fp8_block_linear(x, w, ws),
                 lambda: ops.fp8_block_gemm(x.to(F8), torch.ones(2, 2), w, ws)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


# ---- GPU: quantising operators ---------------------------------------------------------------------
SHAPES = [(1, 128), (3, 8), (5, 1), (2, 129), (7, 136), (16, 4096), (33, 2040), (4, 5000), (130, 257), (2100, 2056), (1, 16384)]


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,H", SHAPES)
def test_gpu_group_quant(T, H, dt):
    x = activations(torch.Generator().manual_seed(T * 7 + H), T, H, DT[dt])
    check_quant(*ops.fp8_group_quant(x.to(DEV)), x.double(), False)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,I", SHAPES)
def test_gpu_silu_and_mul_fp8(T, I, dt):
    x = (2 * torch.randn(T, 2 * I, generator=torch.Generator().manual_seed(T + I))).to(DT[dt])
    g, u = x.double().chunk(2, -1)
    check_quant(*ops.silu_and_mul_fp8(x.to(DEV)), g / (1 + torch.exp(-g)) * u, True)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("T,H", SHAPES + [(3, 8192), (2, 12288), (2, 16383)])
def test_gpu_norm_fp8(T, H, add, dt):
    gen = torch.Generator().manual_seed(3 * T + H)
    x, w = activations(gen, T, H, DT[dt]), (1 + 0.2 * torch.randn(H, generator=gen)).to(DT[dt])
    res = activations(gen, T, H, DT[dt]) if add else None
    xd = x.to(DEV)
    z = x.float()
    if add:
        z = z + res.float()
        rd = res.to(DEV)
        q, s = ops.fused_add_rms_norm_fp8(xd, rd, w.to(DEV), 1e-5)
        assert torch.equal(rd.cpu(), z.to(DT[dt]))
    else:
        q, s = ops.rms_norm_fp8(xd, w.to(DEV), 1e-5)
    assert torch.equal(xd.cpu(), x)
    z = z.double()
    check_quant(q, s, z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-5) * w.double(), True)


@gpu
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("eps", [1e-5, 1e-30])
def test_gpu_norm_fp8_small_values(eps, add):
    """Rows and groups far below 1: the floor 2^-96 is one of the normed values, which 1 / rms makes up to 316 (1e15) times as
    large.  The values are known to V there too: z is exact, z^2 and its sum count only where they are beside eps, and a
    subnormal step (2^-149) is below V of the smallest numbers that matter (2^-10 of 2^-96 / 448, over rms)."""
    gen = torch.Generator().manual_seed(5)
    H, dt = 640, torch.bfloat16
    size = torch.zeros(9, H)
    for row, exponent in enumerate((-90, -97, -100, -104, -110), 1):
        size[row] = 2.0 ** exponent
    size[6], size[6, 128:256] = 2.0 ** -5, 2.0 ** -99          # small groups beside ordinary ones
    size[7], size[7, :128] = 2.0 ** -40, 2.0 ** -110
    size[8], size[8, 256:384] = 1.0, 2.0 ** -96
    x, res = ((torch.randn(9, H, generator=gen) * size).to(dt) for _ in range(2))
    w = (1 + 0.2 * torch.randn(H, generator=gen)).to(dt)
    z = x.float() + res.float() if add else x.float()
    if add:
        rd = res.to(DEV)
        q, s = ops.fused_add_rms_norm_fp8(x.to(DEV), rd, w.to(DEV), eps)
        assert torch.equal(rd.cpu(), z.to(dt))
    else:
        q, s = ops.rms_norm_fp8(x.to(DEV), w.to(DEV), eps)
    z = z.double()
    check_quant(q, s, z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps) * w.double(), True)
    assert not q[0].float().any() and (s[0].cpu() == torch.tensor(2.0 ** -96) / 448).all()


@gpu
def test_gpu_quant_extremes():
    """Zeros, a single value, the largest and smallest values, ties between two e4m3 numbers, infinities and NaN."""
    x = torch.zeros(10, 256, dtype=torch.bfloat16)
    x[1, 3] = -2.5
    x[2, :] = torch.finfo(torch.bfloat16).max
    x[3, :] = 2.0 ** -120
    x[4, :128] = torch.arange(-64, 64) * 7.0           # amax 448: scale exactly 1, every value on or between e4m3 numbers
    x[5, 0], x[5, 1] = 1e-30, 1e30
    x[6, 130] = float("inf")
    x[7, 5] = float("nan")
    x[8, 128:] = torch.linspace(-1, 1, 128).to(torch.bfloat16)
    x[9, 255] = -float("inf")
    q, s = (t.cpu() for t in ops.fp8_group_quant(x.to(DEV)))
    fine = [0, 1, 2, 3, 4, 5, 8]
    check_quant(q[fine], s[fine], x[fine].double(), False)
    assert s[0, 0] == torch.tensor(2.0 ** -96) / 448 and not q[0].double().any()
    assert s[4, 0] == 1.0
    for t, b, j in ((6, 1, 130), (9, 1, 255)):         # only the group with the infinity, and in it only the infinity
        assert math.isinf(s[t, b]) and math.isfinite(s[t, 1 - b])
        assert math.isnan(q[t, j].float()) and int(torch.isnan(q[t].float()).sum()) == 1
    assert math.isnan(s[7, 0]) and math.isfinite(s[7, 1]) and torch.isnan(q[7, :128].float()).all()
    # and a product that reads them: NaN for these tokens, nothing else touched
    gen = torch.Generator().manual_seed(1)
    w, ws = weight(gen, 48, 256)
    y = ops.fp8_block_gemm(q.to(DEV), s.to(DEV), w.to(DEV), ws.to(DEV)).cpu()
    assert torch.isnan(y[[6, 7, 9]]).all()
    # token 2 apart: 256 terms of 3.4e38 times weights of about 1/16 are sums of magnitude 4e39, above the largest fp32
    # number (3.4e38), so its sums overflow on the way even where the result would not
    assert float((s[2].double().repeat_interleave(128) * 448) @ expand(w, ws)[0].abs()) > torch.finfo(torch.float32).max
    fine.remove(2)
    check_gemm(y[fine], q[fine], s[fine], w, ws, None)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_gpu_silu_extremes(dt):
    """The type's lowest and largest values in either half (masked or unset rows), gates far below zero, products near the end
    of fp32, infinities and NaN.  Where silu is not 0 the gates are within 16 of 0, so V holds as it does above."""
    dt = DT[dt]
    low, high = torch.finfo(dt).min, torch.finfo(dt).max
    rows = [(low, low), (low, 1.0), (low, high), (-1000.0, high), (-1.0, low), (-5.0, low), (-0.0, low), (1.0, high / 2), (low, 0.0), (0.0, high),
            (high / 4, 1.0), (-300.0, -2.0)]
    g = torch.stack([torch.full((128,), a) for a, _ in rows]).to(dt)
    u = torch.stack([torch.full((128,), b) for _, b in rows]).to(dt)
    u[:, 64:] *= 0.5
    q, s = (t.cpu() for t in ops.silu_and_mul_fp8(torch.cat((g, u), 1).to(DEV)))
    v = g.double() * torch.sigmoid(g.double()) * u.double()
    assert torch.isfinite(s).all()
    check_quant(q, s, v, True)
    for a, b in ((math.inf, 1.0), (-math.inf, 1.0), (math.nan, 1.0), (1.0, math.inf), (1.0, math.nan)):
        g[0], u[0] = 1.0, 1.0
        g[0, 5], u[0, 5] = a, b
        s = ops.silu_and_mul_fp8(torch.cat((g, u), 1).to(DEV))[1].cpu()
        assert not math.isfinite(s[0, 0]) and torch.isfinite(s[1:]).all()


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_gpu_silu_largest_gates(dt):
    """Gates up to the type's largest value, each product finite in fp32.  Above 88 silu(g) is g to the last place."""
    dt = DT[dt]
    high = torch.finfo(dt).max
    gates = [88.5, 127.0, 128.0, 129.0, 200.0, 1000.0, high / 4, high / 2, 0.7 * high, 0.75 * high, high]
    g = torch.tensor([[a] * 128 for a in gates for _ in range(4)]).to(dt)
    u = torch.tensor([[0.5, 1.0, -0.25, 0.0]] * len(gates)).view(-1, 1).repeat(1, 128).to(dt)
    u[:, 64:] *= 0.5
    g[:, 1::2] = torch.linspace(-15.0, 88.0, 64).to(dt)       # beside ordinary ones
    q, s = (t.cpu() for t in ops.silu_and_mul_fp8(torch.cat((g, u), 1).to(DEV)))
    assert torch.isfinite(s).all() and torch.isfinite(q.float()).all()
    check_quant(q, s, g.double() * torch.sigmoid(g.double()) * u.double(), True)


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_gpu_silu_gates_far_below_zero(dt):
    """silu(-90) is 1e-37, which a large u makes an ordinary number again.  The exponential's error grows with the rounded
    exponent put back to first order only, (|t| 2^-24)^2: below V by far."""
    dt = DT[dt]
    high = torch.finfo(dt).max
    gates = [-80.0, -87.0, -87.5, -88.0, -88.5, -90.0, -100.0, -104.0, -125.0, -150.0, -170.0, -174.0, -175.0, -176.0, -200.0]
    g = torch.tensor([[a] * 128 for a in gates for _ in range(4)]).to(dt)
    u = torch.tensor([[high, -high / 2, 1.0, -high / 64]] * len(gates)).view(-1, 1).repeat(1, 128).to(dt)
    u[:, 1::2] *= 0.625
    g[:, 64:] += 1.0 / 2
    near = (2 * torch.randn(len(g), 256, generator=torch.Generator().manual_seed(1))).to(dt)
    gg, uu = torch.cat((g, near), 1), torch.cat((u, near.flip(1)), 1)         # two ordinary groups beside each
    q, s = (t.cpu() for t in ops.silu_and_mul_fp8(torch.cat((gg, uu), 1).to(DEV)))
    assert torch.isfinite(s).all()
    check_quant(q, s, gg.double() * torch.sigmoid(gg.double()) * uu.double(), True)
    # and those keep their bits where the gates beside them are ordinary too
    gg[:, :128] = 1.0
    q1, s1 = (t.cpu() for t in ops.silu_and_mul_fp8(torch.cat((gg, uu), 1).to(DEV)))
    assert torch.equal(q1[:, 128:].float(), q[:, 128:].float()) and torch.equal(s1[:, 1:], s[:, 1:])


@gpu
def test_gpu_quant_strides_shapes_and_empty():
    gen = torch.Generator().manual_seed(2)
    base = activations(gen, 12, 700, torch.bfloat16)
    bd = base.to(DEV)
    for view in (lambda b: b[:, 8:8 + 512], lambda b: b[:, 3:3 + 300], lambda b: b[::2, :256], lambda b: b.t()[:256],
                 lambda b: b[:1].expand(5, 700), lambda b: b.view(3, 4, 700), lambda b: b.view(3, 4, 700)[:, 1:3, 16:144],
                 lambda b: b[4]):
        v = view(base)
        q, s = ops.fp8_group_quant(view(bd))
        check_quant(q, s, v.double(), False)
    for shape in ((0, 128), (4, 0), (0, 3, 40)):
        q, s = ops.fp8_group_quant(torch.empty(shape, dtype=torch.bfloat16, device=DEV))
        assert q.shape == shape and s.shape == shape[:-1] + (blocks(shape[-1]),)


@gpu
def test_gpu_quant_leaves_what_is_outside_its_rows():
    """Rows inside wider buffers: bytes behind a row, rows behind the last token, scales of other tokens stay as they were."""
    T, H = 5, 200
    x = torch.randn(T, H, device=DEV).to(torch.float16)
    for H_used in (200, 131):
        q = torch.full((T + 2, H + 24), 0x55, dtype=torch.uint8, device=DEV)
        s = torch.full((3, T + 3), -7.0, device=DEV)
        rc = _lib.load().pq_fp8_group_quant(x.data_ptr(), H, T, H_used, 0, q.data_ptr(), H + 24, s.data_ptr(), T + 3,
                                            torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert (q[T:] == 0x55).all() and (q[:, H_used:] == 0x55).all()
        assert (s[:, T:] == -7).all() and (s[2] == -7).all()
        check_quant(q[:T, :H_used].contiguous().view(F8), s[:2, :T].t(), x[:, :H_used].cpu().double(), False)


# ---- GPU: products ---------------------------------------------------------------------------------
GEMMS = [(1, 16, 128), (1, 1, 1), (3, 7, 5), (16, 128, 256), (17, 130, 384), (5, 1000, 1080), (33, 96, 2048), (64, 257, 640),
         (100, 48, 127), (129, 300, 129), (2, 4096, 4096), (333, 1000, 1080), (70, 40, 3000), (257, 513, 528), (300, 640, 131), (90, 70, 20), (40, 100, 16), (33, 65, 12), (50, 60, 148), (2, 100, 20), (16, 40, 4100), (4, 8200, 144), (9, 64, 8200),
         (16, 96, 14336), (3, 50, 16384), (4, 33, 16400), (1, 9000, 1024), (7, 33, 131), (16, 20, 257), (1, 40, 1003), (2, 300, 4098), (8, 48, 1024),
         (512, 1024, 512), (700, 700, 1600)]


@gpu
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("T,N,K", GEMMS)
def test_gpu_block_gemm_and_linear(T, N, K, dt):
    gen = torch.Generator().manual_seed(T + 3 * N + 7 * K)
    x = activations(gen, T, K, DT[dt])
    w, ws = weight(gen, N, K)
    bias = torch.randn(N, generator=gen).to(DT[dt]) if (T + N) % 2 else None
    bd = None if bias is None else bias.to(DEV)
    q, s = ops.fp8_group_quant(x.to(DEV))
    y = ops.fp8_block_gemm(q, s, w.to(DEV), ws.to(DEV), bd, DT[dt])
    assert y.shape == (T, N) and y.dtype == DT[dt]
    check_gemm(y, q, s, w, ws, bias)
    assert torch.equal(y, ops.fp8_block_gemm(q, s, w.to(DEV), ws.to(DEV), bd, DT[dt]))       # the same bits every time
    z = ops.fp8_block_linear(x.to(DEV), w.to(DEV), ws.to(DEV), bd)
    assert z.dtype == DT[dt]
    check_gemm(z, q, s, w, ws, bias)
    if K % 4 == 0:      # the quantised rows have the same layout to both: the same kernel, the same bits
        assert torch.equal(y, z)


@gpu
@pytest.mark.parametrize("T,N,K", [(3, 70, 2064), (4, 20, 1168), (2, 40, 2576), (1, 9000, 2048), (1, 33, 3600), (16, 600, 2176), (7, 8300, 2400),
                                   (13, 24, 1151)])
def test_gpu_few_tokens_any_number_of_blocks(T, N, K):
    """9 to 29 scale blocks over 8 waves: two, three and four of a wave, whole and short, quantised inside and before."""
    test_gpu_block_gemm_and_linear(T, N, K, "bf16")


@gpu
@pytest.mark.parametrize("T,N,K", [(2500, 6100, 1000), (2560, 6144, 1040), (1000, 4000, 1084), (1024, 4096, 512), (520, 4096, 2000),
                                   (250, 4096, 1152), (64, 512, 8192), (40, 1000, 14300), (300, 4096, 14336), (17, 257, 4100),
                                   (4096, 300, 260)])
def test_gpu_block_gemm_tiles(T, N, K):
    """Sizes that take each tile shape, whole and ragged, with K in one range and in several (the scratch is the caller's: without
    it the same call runs in one range)."""
    gen = torch.Generator().manual_seed(T + N + K)
    q, s = ops.fp8_group_quant(activations(gen, T, K, torch.bfloat16).to(DEV))
    w, ws = (t.to(DEV) for t in weight(gen, N, K))
    bias = torch.randn(N, generator=gen).to(torch.bfloat16).to(DEV)
    y = ops.fp8_block_gemm(q, s, w, ws, bias)
    check_gemm(y, q, s, w, ws, bias, DEV)
    if (T, N, K) in ((64, 512, 8192), (40, 1000, 14300)):
        assert ops._fp8_tmp_bytes("pq_fp8_block_gemm_tmp_bytes", T, N, K) > 0
    z = torch.empty_like(y)
    assert _lib.load().pq_fp8_block_gemm(q.data_ptr(), T, K, s.data_ptr(), 1, T, w.data_ptr(), K, ws.data_ptr(), blocks(K),
                                         bias.data_ptr(), N, K, 1, z.data_ptr(), N, None, 0,
                                         torch.cuda.current_stream().cuda_stream) == 0
    check_gemm(z, q, s, w, ws, bias, DEV)


@gpu
@pytest.mark.parametrize("T,N,K", [(17, 130, 18), (40, 257, 1001), (300, 700, 4099), (1000, 520, 2001), (64, 512, 8195), (200, 30, 15), (33, 5, 127)])
def test_gpu_block_gemm_any_length(T, N, K):
    """A K that is no multiple of 4: with the scratch (operands laid out there), without it, and with rows inside wider ones."""
    gen = torch.Generator().manual_seed(T + N + K)
    q, s = ops.fp8_group_quant(activations(gen, T, K, torch.float16).to(DEV))
    w, ws = (t.to(DEV) for t in weight(gen, N, K))
    bias = torch.randn(N, generator=gen).to(torch.float16).to(DEV)
    y = ops.fp8_block_gemm(q, s, w, ws, bias, torch.float16)
    check_gemm(y, q, s, w, ws, bias, DEV)
    # around each row of both operands: bytes that are NaN as e4m3
    qw, ww = (torch.full((t.shape[0] + 2, K + 21), 0x7f, dtype=torch.uint8, device=DEV) for t in (q, w))
    qw[1:-1, 9:K + 9], ww[1:-1, 9:K + 9] = q.view(torch.uint8), w.view(torch.uint8)
    args = (qw[1:-1, 9:K + 9].view(F8), s, ww[1:-1, 9:K + 9].view(F8), ws, bias, torch.float16)
    assert torch.equal(y, ops.fp8_block_gemm(*args))
    z = torch.empty_like(y)
    tmp = torch.full((ops._fp8_tmp_bytes("pq_fp8_block_gemm_tmp_bytes", T, N, K) + 64,), 0x7f, dtype=torch.uint8, device=DEV)
    for scratch in (0, 16, tmp.numel() - 64):       # none, too little, what is asked for
        z.zero_()
        assert _lib.load().pq_fp8_block_gemm(args[0].data_ptr(), T, K + 21, s.data_ptr(), 1, T, args[2].data_ptr(), K + 21, ws.data_ptr(),
                                             blocks(K), bias.data_ptr(), N, K, 0, z.data_ptr(), N, tmp.data_ptr() if scratch else None,
                                             scratch, torch.cuda.current_stream().cuda_stream) == 0
        check_gemm(z, q, s, w, ws, bias, DEV)
        assert (tmp[-64:] == 0x7f).all()
    assert torch.equal(y, z)


@gpu
@pytest.mark.parametrize("T,N,K", [(4, 40, 300), (4, 40, 4096 + 300), (40, 64, 384), (40, 64, 131), (300, 200, 640), (300, 4096, 1152)])
def test_gpu_gemm_infinite_scales(T, N, K):
    """An infinite scale of a token's (row block's) last group and finite values: the sums are infinite, with the values' sign,
    also where a wave has no group of its own behind it."""
    q = torch.ones(T, K, device=DEV).to(F8)
    w = torch.ones(N, K, device=DEV).to(F8)
    w[1::2] = torch.full((), -1.0).to(F8)
    s, ws = torch.ones(T, blocks(K), device=DEV), torch.ones(blocks(N), blocks(K), device=DEV)
    sign = torch.ones(N, device=DEV)
    sign[1::2] = -1
    s[1::2, -1] = math.inf
    y = ops.fp8_block_gemm(q, s, w, ws).float()
    assert torch.equal(y[1::2], (sign * math.inf).expand(T // 2, N))
    assert torch.isfinite(y[::2]).all()
    ws[0, -1] = math.inf
    y = ops.fp8_block_gemm(q, s, w, ws).float()
    assert torch.equal(y[:, :128], (sign[:128] * math.inf).expand(T, min(N, 128)))
    assert torch.isfinite(y[::2, 128:]).all()


@gpu
def test_gpu_matrix_instruction():
    """What the tolerance of the products rests on, seen through the operator: 448 * 448 and its negative cancel, and what is
    left of a small product tells how it was held.  A lane holds 32 of the block's features, in groups of 8."""
    def left(small, at, big=448.0):
        x, w = torch.zeros(1, 128), torch.zeros(1, 128)
        x[0, 0], w[0, 0], x[0, 32], w[0, 32] = big, big, big, -big
        x[0, at], w[0, at] = small
        one = torch.ones(1, 1, device=DEV)
        return float(ops.fp8_block_gemm(x.to(F8).to(DEV), one, w.to(F8).to(DEV), one, None, torch.float16))
    for at in range(1, 8):           # beside the large one: multiples of 2^(8 + 8 - 13) = 8, toward zero
        assert [left((v, 1), at) for v in (7, 8, 15, 16, 30)] == [0, 8, 8, 16, 24]
        assert [left((v, -1), at) for v in (7, 8, 15, 16, 30)] == [0, -8, -8, -16, -24]
    assert [left((v, 1), 3, 240.0) for v in (1, 2, 3)] == [0, 2, 2]      # 2^(7 + 7 - 13) = 2
    for at in (8, 15, 17, 64, 127):  # in another group: fp32
        assert [left((v, 1), at) for v in (0.0625, 0.5, 7, 15)] == [0.0625, 0.5, 7, 15]


@gpu
@pytest.mark.parametrize("T", [4, 40, 300])
def test_gpu_gemm_layouts(T):
    """Strided operands, scales in either order and broadcast, leading dimensions, weights inside wider rows, no features."""
    gen = torch.Generator().manual_seed(T)
    N, K = 272, 400
    x = activations(gen, T, K, torch.bfloat16)
    w, ws = weight(gen, N, K)
    q, s = ops.fp8_group_quant(x.to(DEV))
    wd, wsd = w.to(DEV), ws.to(DEV)
    y = ops.fp8_block_gemm(q, s, wd, wsd)
    check_gemm(y, q, s, w, ws, None)
    assert torch.equal(y, ops.fp8_block_gemm(q, s.contiguous(), wd, wsd))
    assert torch.equal(y, ops.fp8_block_gemm(q.view(2, T // 2, K), s.reshape(2, T // 2, -1), wd, wsd).view(T, N))
    for pad in (16, 3):          # rows inside wider buffers, 16-byte aligned and not
        wide = torch.zeros(N, K + pad, dtype=torch.uint8, device=DEV)
        wide[:, :K] = wd.view(torch.uint8)
        qw = torch.zeros(T, K + pad, dtype=torch.uint8, device=DEV)
        qw[:, :K] = q.view(torch.uint8)
        for a, b in ((q, wide[:, :K].view(F8)), (qw[:, :K].view(F8), wd), (qw[:, :K].view(F8), wide[:, :K].view(F8))):
            check_gemm(ops.fp8_block_gemm(a, s, b, wsd), q, s, w, ws, None)
    one = torch.full((1, 1), 0.25, device=DEV).expand(T, blocks(K))
    check_gemm(ops.fp8_block_gemm(q, one, wd, wsd), q, one, w, ws, None)
    bias = torch.randn(N, device=DEV).to(torch.bfloat16)
    none = ops.fp8_block_gemm(q[:, :0], s[:, :0], wd[:, :0], wsd[:, :0], bias)
    assert torch.equal(none, bias.expand(T, N))
    assert ops.fp8_block_gemm(q[:0], s[:0], wd, wsd).shape == (0, N)
    assert ops.fp8_block_linear(x.to(DEV)[:, :0], wd[:, :0], wsd[:, :0], bias).shape == (T, N)
    assert ops.fp8_block_gemm(q, s, wd[:0], wsd[:0]).shape == (T, 0)


@gpu
@pytest.mark.parametrize("T", [5, 40, 300])
def test_gpu_gemm_leaves_what_is_outside_its_rows(T):
    N, K = 200, 384
    gen = torch.Generator().manual_seed(9)
    q, s = ops.fp8_group_quant(activations(gen, T, K, torch.float16).to(DEV))
    w, ws = weight(gen, N, K)
    wd, wsd = w.to(DEV), ws.to(DEV)
    for cols in (N, N - 3):
        y = torch.full((T + 3, N + 8), 31.0, dtype=torch.float16, device=DEV)
        rc = _lib.load().pq_fp8_block_gemm(q.data_ptr(), T, K, s.data_ptr(), s.stride(0), s.stride(1), wd.data_ptr(), K,
                                           wsd.data_ptr(), 3, None, cols, K, 0, y.data_ptr(), N + 8, None, 0,
                                           torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        assert (y[T:] == 31).all() and (y[:, cols:] == 31).all()
        check_gemm(y[:T, :cols], q, s, w[:cols], ws[:blocks(cols)], None)


@gpu
@pytest.mark.parametrize("T,N,stride", [(600, 520, 2 ** 23 - 128), (600, 520, 2 ** 23 + 128), (16, 600, 2 ** 23), (5, 72, 2 ** 26 - 64),
                                        (3, 33, 2 ** 27)])
def test_gpu_offsets_past_32_bits(T, N, stride):
    """Rows so far apart that the last ones lie more than 2^32 elements behind the first: weights, outputs and, for many tokens,
    activations."""
    K = 272
    gen = torch.Generator().manual_seed(N)
    x = activations(gen, T, K, torch.bfloat16).to(DEV)
    q, s = ops.fp8_group_quant(x)
    w, ws = (t.to(DEV) for t in weight(gen, N, K))

    def spread(t):
        rows = torch.empty(t.shape[0] * stride, dtype=t.dtype, device=DEV).view(t.shape[0], stride)[:, :t.shape[1]]
        return rows.copy_(t) if t.dtype != F8 else rows.view(torch.uint8).copy_(t.view(torch.uint8)).view(F8)
    far = spread(w)
    check_gemm(ops.fp8_block_gemm(q, s, far, ws), q, s, w, ws, None, DEV)
    del far
    if T > 16:
        far = spread(q)
        check_gemm(ops.fp8_block_gemm(far, s, w, ws), q, s, w, ws, None, DEV)
        del far
        far = spread(x)
        q2, s2 = ops.fp8_group_quant(far)
        assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
        check_gemm(ops.fp8_block_linear(far, w, ws), q, s, w, ws, None, DEV)
        one = torch.ones(K, dtype=x.dtype, device=DEV)
        for a, b in zip(ops.rms_norm_fp8(far, one, 1e-5), ops.rms_norm_fp8(x, one, 1e-5)):
            assert torch.equal(a.float(), b.float())
        del far
    y = torch.empty(T * stride, dtype=torch.bfloat16, device=DEV).view(T, stride)[:, :N]
    assert _lib.load().pq_fp8_block_gemm(q.data_ptr(), T, K, s.data_ptr(), 1, T, w.data_ptr(), K, ws.data_ptr(), 3, None, N, K, 1,
                                         y.data_ptr(), stride, None, 0, torch.cuda.current_stream().cuda_stream) == 0
    check_gemm(y.contiguous(), q, s, w, ws, None, DEV)


@gpu
@pytest.mark.parametrize("T,N,stride", [(1, 72, 2 ** 26 - 16), (1, 72, 2 ** 26), (5, 40, 2 ** 27)])
def test_gpu_linear_of_few_tokens_and_rows_far_apart(T, N, stride):
    """Tokens that are quantised inside the product's launch, and before it where the weight's rows are too far apart for that."""
    K = 272
    gen = torch.Generator().manual_seed(T + N)
    x = activations(gen, T, K, torch.bfloat16).to(DEV)
    w, ws = (t.to(DEV) for t in weight(gen, N, K))
    bias = torch.randn(N, generator=gen).to(torch.bfloat16).to(DEV)
    far = torch.empty(N * stride, dtype=torch.uint8, device=DEV).view(N, stride)[:, :K].copy_(w.view(torch.uint8)).view(F8)
    q, s = ops.fp8_group_quant(x)
    y = ops.fp8_block_linear(x, far, ws, bias)
    check_gemm(y, q, s, w, ws, bias, DEV)
    assert torch.equal(y, ops.fp8_block_linear(x, w, ws, bias))
    assert torch.equal(y, ops.fp8_block_linear(x.view(1, T, K), far, ws, bias)[0])


@gpu
@pytest.mark.parametrize("T", [3, 16, 40, 300])
@pytest.mark.parametrize("K", [256, 384, 1027, 4500])
def test_gpu_a_token_stands_for_itself(T, K):
    """A padding row of infinities or NaN leaves the other tokens' outputs as they were, bit for bit."""
    gen = torch.Generator().manual_seed(T + K)
    N = 200
    x = activations(gen, T, K, torch.bfloat16).to(DEV)
    w, ws = (t.to(DEV) for t in weight(gen, N, K))
    y, z = ops.fp8_block_linear(x, w, ws), ops.fp8_block_gemm(*ops.fp8_group_quant(x), w, ws)
    for bad in (math.nan, math.inf):
        x[1] = bad
        rest = [t for t in range(T) if t != 1]
        for got, want in ((ops.fp8_block_linear(x, w, ws), y), (ops.fp8_block_gemm(*ops.fp8_group_quant(x), w, ws), z)):
            assert torch.equal(got[rest], want[rest]) and got[1].isnan().all()


@gpu
def test_gpu_refusals():
    x = torch.zeros(4, 256, dtype=torch.bfloat16, device=DEV)
    w, ws = torch.zeros(130, 256, device=DEV).to(F8), torch.ones(2, 2, device=DEV)
    q, s = ops.fp8_group_quant(x)
    good = (q, s, w, ws)
    assert ops.fp8_block_gemm(*good).shape == (4, 130)
    bad = [(q.float(), s, w, ws), (q, s.double(), w, ws), (q, s[:, :1], w, ws), (q, s[:3], w, ws), (q, s, w[:, :128], ws),
           (q, s, w.float(), ws), (q, s, w, ws[:1]), (q, s, w, ws.half()), (q, s, w, ws.view(4)),
           (q, s, w, ws, torch.zeros(129, dtype=torch.bfloat16, device=DEV)),
           (q, s, w, ws, torch.zeros(130, device=DEV)), (q, s, w, ws, None, torch.float32)]
    for args in bad:
        with pytest.raises(ValueError):
            ops.fp8_block_gemm(*args)
    with pytest.raises(RuntimeError):
        ops.fp8_block_gemm(q, s.cpu(), w, ws)
    one = torch.ones(256, dtype=torch.bfloat16, device=DEV)
    for call in (lambda: ops.fp8_group_quant(x.float()), lambda: ops.fp8_group_quant(x[0, 0]), lambda: ops.silu_and_mul_fp8(x[:, :255]),
                 lambda: ops.rms_norm_fp8(x, one[:255], 1e-5), lambda: ops.rms_norm_fp8(x, one.half(), 1e-5),
                 lambda: ops.fused_add_rms_norm_fp8(x, x[:3], one, 1e-5), lambda: ops.fused_add_rms_norm_fp8(x, x.half(), one, 1e-5),
                 lambda: ops.fused_add_rms_norm_fp8(x, torch.zeros(256, 4, dtype=x.dtype, device=DEV).t(), one, 1e-5),
                 lambda: ops.fused_add_rms_norm_fp8(x, None, one, 1e-5),
                 lambda: ops.fp8_block_linear(x.float(), w, ws), lambda: ops.fp8_block_linear(x[:, :128], w, ws),
                 lambda: ops.rms_norm_fp8(torch.zeros(1, 16392, dtype=x.dtype, device=DEV),
                                          torch.zeros(16392, dtype=x.dtype, device=DEV), 1e-5)):
        with pytest.raises(ValueError):
            call()


# ---- GPU: together ---------------------------------------------------------------------------------
def _mlp(x, res, nw, wgu, wsgu, wd, wsd):
    """The 8-bit half of a decoder layer: norm with the residual add, gate_up_proj, activation, down_proj."""
    q, s = ops.fused_add_rms_norm_fp8(x, res, nw, 1e-5)
    gu = ops.fp8_block_gemm(q, s, wgu, wsgu, None, x.dtype)
    a, sa = ops.silu_and_mul_fp8(gu)
    return ops.fp8_block_gemm(a, sa, wd, wsd, None, x.dtype), gu, res


@gpu
@pytest.mark.parametrize("T", [1, 16, 70, 300])
def test_gpu_mlp_composes(T):
    gen = torch.Generator().manual_seed(T)
    H, I = 512, 1040
    x, res = (torch.randn(T, H, generator=gen).to(torch.bfloat16) for _ in range(2))
    nw = (1 + 0.1 * torch.randn(H, generator=gen)).to(torch.bfloat16)
    (wgu, wsgu), (wd, wsd) = weight(gen, 2 * I, H), weight(gen, H, I)
    y, gu, r = _mlp(x.to(DEV), res.to(DEV), nw.to(DEV), wgu.to(DEV), wsgu.to(DEV), wd.to(DEV), wsd.to(DEV))
    # the chain in 64 bits with its 8-bit roundings: a value that lies on the other side of a rounding there moves a product by
    # one step of one of its terms, far below the act dtype's half step summed over the chain's two products
    z = (x.float() + res.float()).double()
    q, s = quant64(z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-5) * nw.double())
    deq = lambda q, s: q * s.repeat_interleave(128, -1)[..., :q.shape[-1]]  # noqa: E731
    g64 = deq(q, s) @ expand(wgu, wsgu).t()
    g, u = gu.cpu().double().chunk(2, -1)
    q, s = quant64(g / (1 + torch.exp(-g)) * u)
    y64 = deq(q, s) @ expand(wd, wsd).t()
    for got, want in ((gu, g64), (y, y64)):
        assert (got.cpu().double() - want).norm() / want.norm() < 2.0 ** -8
    assert torch.equal(r.cpu(), z.to(torch.bfloat16))


@gpu
@pytest.mark.parametrize("T", [1, 16, 200])
def test_gpu_graph_streams_and_compiled_route(T):
    """Captured into a graph and replayed with eager work between; issued on another stream; through the registered ops."""
    gen = torch.Generator().manual_seed(T)
    H, I = 256, 512
    dt = torch.bfloat16
    nw = torch.ones(H, dtype=dt, device=DEV)
    (wgu, wsgu), (wd, wsd) = ((t.to(DEV) for t in weight(gen, n, k)) for n, k in ((2 * I, H), (H, I)))
    x, res = torch.zeros(T, H, dtype=dt, device=DEV), torch.zeros(T, H, dtype=dt, device=DEV)

    def step():
        y = _mlp(x, res, nw, wgu, wsgu, wd, wsd)
        return y[0], y[1], ops.fp8_block_linear(x, wgu, wsgu), *ops.fp8_group_quant(x)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    side = torch.cuda.Stream()
    for i in range(4):
        xi, ri = (torch.randn(T, H, generator=gen).to(dt).to(DEV) for _ in range(2))
        x.copy_(xi), res.copy_(ri)
        graph.replay()
        torch.cuda.synchronize()
        got, got_res = [o.clone() for o in outs], res.clone()
        res.copy_(ri)
        want = step()
        assert torch.equal(got_res, res)
        for a, b in zip(got, want):
            assert torch.equal(a.float(), b.float())
        res.copy_(ri)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = step()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(other, want):
            assert torch.equal(a.float(), b.float())
    o = torch.ops.pq_amd
    res.copy_(ri)
    q, s = o.fused_add_rms_norm_fp8(x, res, nw, 1e-5)
    a, sa = o.silu_and_mul_fp8(o.fp8_block_gemm(q, s, wgu, wsgu, None, dt))
    assert torch.equal(o.fp8_block_gemm(a, sa, wd, wsd, None, dt), want[0])
    assert torch.equal(o.fp8_block_linear(x, wgu, wsgu, None), want[2])
    q2, s2 = o.rms_norm_fp8(x, nw, 1e-5)
    q3, s3 = ops.rms_norm_fp8(x, nw, 1e-5)
    assert torch.equal(q2.float(), q3.float()) and torch.equal(s2, s3)
    assert torch.equal(o.fp8_group_quant(x)[1], want[4])


def test_fake_implementations_match_the_real_layouts():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 5, 600, dtype=torch.bfloat16, device="cuda")
        q, s = torch.ops.pq_amd.fp8_group_quant(x)
        assert q.shape == (3, 5, 600) and q.dtype == F8 and s.shape == (3, 5, 5) and s.stride() == (5, 1, 15)
        q, s = torch.ops.pq_amd.silu_and_mul_fp8(x)
        assert q.shape == (3, 5, 300) and s.shape == (3, 5, 3)
        w = torch.empty(70, 300, dtype=F8, device="cuda")
        y = torch.ops.pq_amd.fp8_block_gemm(q, s, w, torch.empty(1, 3, device="cuda"), None, torch.float16)
        assert y.shape == (3, 5, 70) and y.dtype == torch.float16


@gpu
@pytest.mark.parametrize("T,N,K", [(40, 512, 8192), (300, 200, 1001), (4, 300, 8200), (1, 512, 1024), (128, 256, 4096)])
def test_gpu_scratch_in_graphs_and_on_two_streams(T, N, K):
    """Calls that use scratch (ranges of K, laid-out operands): two graphs of them replayed in turn while weights and scales change,
    and two streams at once."""
    gen = torch.Generator().manual_seed(T * K)
    dt = torch.bfloat16
    sets = []
    for _ in range(2):
        x = activations(gen, T, K, dt).to(DEV)
        w, ws = (t.to(DEV) for t in weight(gen, N, K))
        sets.append((x, w, ws))

    def call(x, w, ws):
        return ops.fp8_block_gemm(*ops.fp8_group_quant(x), w, ws), ops.fp8_block_linear(x, w, ws)
    for a in sets:
        call(*a)
    torch.cuda.synchronize()
    graphs = []
    for a in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call(*a)
        graphs.append((g, out))
    for i in range(3):
        for x, w, ws in sets:
            x.copy_(activations(gen, T, K, dt))
            fresh, scales = weight(gen, N, K)
            w.view(torch.uint8).copy_(fresh.view(torch.uint8))
            ws.copy_(scales)
        for g, _ in graphs:
            g.replay()
        want = [call(*a) for a in sets]
        for (_, got), w in zip(graphs, want):
            assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        results = []
        for s, a in zip(streams, sets):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                results.append([call(*a) for _ in range(4)])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for many, w in zip(results, want):
            for got in many:
                assert torch.equal(got[0], w[0]) and torch.equal(got[1], w[1])
