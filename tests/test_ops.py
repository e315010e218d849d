"""The model-free operators (evodiff_amd.ops) against plain implementations in 64 bits: block-scaled 8-bit quantisation, the
product on it, log probabilities of given tokens with entropy and top alternatives, and their gradient.

Tolerances are counted in roundings (``torch.finfo(t).eps / 2`` each, relative):

* quantised values, scales and tokens are compared exactly;
* a product of Kb blocks: every product of two e4m3 values is exact in fp32, and at most 128 * Kb + 1 additions round, each by
  at most 2^-24 of the sum of magnitudes so far; then one rounding to the output type;
* a log probability: sum and reference value of one row.  A sum of n positive terms in chains of at most c additions
  (c = ceil(n / 64) + 64 bounds every form) is off by c * 2^-24, its terms by (4 + 2 log n) * 2^-24 together (exponential,
  difference, and the sums of d exp(d) weighted by the distribution), the logarithm and three differences by 2^-22 of
  the values they join.
"""
import ctypes
import math

import numpy as np
import pytest
import torch

from evodiff_amd import _lib, ops

TOP = 448.0
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ---- plain implementations -------------------------------------------------------------------------------------------

def e4m3(y):
    """Round fp64 values within +-448 to e4m3, to nearest even, from the format's definition."""
    exponent = torch.frexp(y.abs())[1]
    step = torch.ldexp(torch.ones_like(y), (exponent - 4).clamp(min=-9))
    return torch.round(y / step) * step


def plain_quantize(x, square):
    """(values fp64 (m, kb * 128) with NaN where x has no finite value, exponents int (blocks, kb)) on the CPU."""
    x = x.detach().cpu().double()
    m, k = x.shape
    kb = -(-k // 128)
    rows = -(-m // 128) * 128 if square else m
    full = torch.zeros((rows, kb * 128), dtype=torch.float64)
    full[:m, :k] = x
    tile = full.view(-1, 128 if square else 1, kb, 128)
    amax = torch.where(torch.isfinite(tile), tile.abs(), torch.zeros_like(tile)).amax((1, 3))
    mant, exp = torch.frexp(amax / TOP)
    s = torch.where(mant == 0.5, exp - 1, exp)
    s = torch.where(amax > 0, s, torch.full_like(s, -126)).clamp(-126, 127)
    scale = torch.ldexp(torch.ones_like(amax), s)[:, None, :, None]
    y = tile / scale
    q = torch.where(torch.isfinite(y), e4m3(torch.where(torch.isfinite(y), y, torch.zeros_like(y))), torch.full_like(y, math.nan))
    return q.view(full.shape)[:m], s


def dequantized(q, s, square):
    scale = torch.ldexp(torch.ones(s.shape, dtype=torch.float64), s)
    if square:
        scale = scale.repeat_interleave(128, 0)[:q.shape[0]]
    return q * scale.repeat_interleave(128, 1)


def exponents(scale):
    return scale.view(torch.uint8).cpu().int() - 127


def plain_logprobs(x, targets, top_k, select=None, n_classes=None):
    """fp64 (logprob, entropy, top_logprob, top_token) with the conventions of ``ops.token_logprobs``; x (rows, v)."""
    x = x.detach().cpu().double()[:, :n_classes]
    rows, n = x.shape
    logprob, entropy = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    top, token = torch.zeros((rows, top_k), dtype=torch.float64), torch.full((rows, top_k), -1)
    for r in range(rows):
        if select is not None and not select[r]:
            continue
        row = x[r]
        empty, bad = bool((row == -math.inf).all()), bool((torch.isnan(row) | (row == math.inf)).any())
        lp = torch.full_like(row, math.nan) if bad else row.clone() if empty else row - torch.logsumexp(row, 0)
        t = int(targets[r])
        logprob[r] = lp[t] if 0 <= t < n else math.nan
        p = torch.exp(lp)
        entropy[r] = math.nan if bad else 0.0 if empty else -(torch.where(p > 0, p * lp, torch.zeros_like(p))).sum()
        order = torch.sort(row, descending=True, stable=True).indices[:top_k]
        token[r], top[r] = order, lp[order]
    return logprob, entropy, top, token


def logprob_tolerance(x, n):
    span = float(x[torch.isfinite(x)].abs().max()) if torch.isfinite(x).any() else 0.0
    return (-(-n // 64) + 64 + 4 + 2 * math.log(max(n, 2))) * 2.0 ** -24 + 2.0 ** -22 * max(span if span < 1e4 else 0.0, 1.0)


def rel_ok(got, want, tol_abs, tol_rel=2.0 ** -22):
    got, want = got.detach().cpu().double(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf])
    ok = torch.isfinite(want)
    off = (got[ok] - want[ok]).abs() - (tol_abs + tol_rel * want[ok].abs())
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


# ---- on the CPU: what the entry points refuse before anything is launched ---------------------------------------------

def test_refusals_of_the_c_entry_points():
    lib = _lib.load()
    p = ctypes.c_void_p(1 << 20)         # never read: every call below is refused on the host
    odd = ctypes.c_void_p((1 << 20) + 1)

    def refused(rc, text):
        assert rc == -1 and text in lib.ed_last_error().decode(), lib.ed_last_error()

    for fn in (lib.ed_fp8_quantize_rows, lib.ed_fp8_quantize_weight):
        refused(fn(p, 3, 128, 4, 128, p, p, None), "dtype")
        refused(fn(p, 0, 128, -1, 128, p, p, None), "range")
        refused(fn(p, 0, 128, 4, 0, p, p, None), "range")
        refused(fn(p, 0, 128, 1 << 29, 1 << 20, p, p, None), "range")
        refused(fn(p, 0, -1, 4, 128, p, p, None), "stride")
        refused(fn(None, 0, 128, 4, 128, p, p, None), "null")
        refused(fn(p, 0, 128, 4, 128, None, p, None), "null")
        refused(fn(odd, 1, 128, 4, 128, p, p, None), "aligned")
        refused(fn(p, 0, 128, 4, 128, odd, p, None), "16 bytes")
        assert fn(None, 0, 128, 0, 128, None, None, None) == 0      # no rows: nothing to do

    def linear(x=p, xd=1, rs=256, xs=None, w=p, ws=p, b=None, o=p, od=1, m=4, n=8, k=256, wk=p, wb=1 << 20):
        return lib.ed_fp8_linear(x, xd, rs, xs, w, ws, b, o, od, m, n, k, wk, wb, None)

    refused(linear(xd=7), "dtype")
    refused(linear(od=3), "dtype")
    refused(linear(xd=3, rs=200, xs=p), "bytes apart")
    refused(linear(xd=3, rs=256, xs=None), "null")
    refused(linear(xd=3, x=ctypes.c_void_p((1 << 20) + 8), xs=p), "16 bytes")
    refused(linear(w=None), "null")
    refused(linear(w=odd), "16 bytes")
    refused(linear(o=odd), "aligned")
    refused(linear(b=odd), "aligned")
    refused(linear(n=0), "range")
    refused(linear(k=0), "range")
    refused(linear(m=1 << 29, n=1 << 20, k=1), "range")
    need = lib.ed_fp8_linear_workspace(65536, 8, 256, 1, 1)  # (rows enough to be brought to 8 bits by a launch of their own)
    assert need >= 65536 * 2 * 129
    refused(linear(m=65536, wb=need - 1), "workspace")
    refused(linear(m=65536, wk=None, wb=need), "workspace")
    refused(linear(m=65536, wk=odd, wb=need), "workspace")
    assert linear(m=0, x=None) == 0

    def logprobs(x=p, dt=0, rs=31, inner=4, outer=0, rows=4, n=31, t=p, sel=None, k=2, lp=p, h=p, st=None, tl=p, tt=p,
                 wk=p, wb=1 << 30):
        return lib.ed_token_logprobs(x, dt, rs, inner, outer, rows, n, t, sel, k, lp, h, st, tl, tt, wk, wb, None)

    refused(logprobs(dt=3), "dtype")
    refused(logprobs(n=0), "range")
    refused(logprobs(n=1 << 30), "range")
    refused(logprobs(rows=-1), "range")
    refused(logprobs(rs=-1), "strides")
    refused(logprobs(inner=0), "inner_rows")
    refused(logprobs(k=32), "top_k")
    refused(logprobs(n=64, k=33), "top_k")
    refused(logprobs(k=-1), "top_k")
    refused(logprobs(x=None), "null")
    refused(logprobs(x=odd), "aligned")
    refused(logprobs(h=None), "null")
    refused(logprobs(lp=None), "null")
    refused(logprobs(tt=None), "null")
    assert logprobs(rows=0, x=None) == 0
    need = lib.ed_token_logprobs_workspace(1, 131072, 20)
    if need > 0:
        refused(logprobs(rows=1, n=131072, k=20, wb=need - 1), "workspace")

    def backward(cols=31, st=p, h=p, t=p, tt=p, gl=p, gh=p, gt=p, d=p, k=2):
        return lib.ed_token_logprobs_backward(p, 0, 31, 4, 0, 4, 31, cols, t, None, k, st, h, tt, gl, gh, gt, d, None)

    refused(backward(cols=30), "columns")
    refused(backward(st=None), "null")
    refused(backward(d=None), "null")
    refused(backward(t=None), "targets")
    refused(backward(tt=None), "top_token")
    refused(backward(d=odd), "aligned")
    assert lib.ed_score_tokens(None, p, None, p, None, 1, 1, 31, 0, p, p, None, None, 1, None) == -1


def test_there_is_no_cpu_path():
    x, w = torch.zeros((2, 128)), ops.Fp8Weight(torch.zeros((4, 128), dtype=torch.float8_e4m3fn), torch.zeros((1, 1), dtype=torch.float8_e8m0fnu))
    for call in (lambda: ops.quantize_fp8(x), lambda: ops.quantize_fp8_weight(x), lambda: ops.linear_fp8(x, w),
                 lambda: ops.token_logprobs(x, torch.zeros(2, dtype=torch.long))):
        with pytest.raises(_lib.EvoDiffHipError, match="no CPU path"):
            call()


# ---- on the GPU ------------------------------------------------------------------------------------------------------

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = torch.device("cuda", 0)
    torch.cuda.set_device(d)
    return d


def rand(dev, shape, seed, dtype=torch.float32, spread=0.0):
    g = torch.Generator(device="cpu")
    g.manual_seed(seed)
    x = torch.randn(shape, generator=g)
    if spread:
        x = x * torch.exp(spread * torch.randn(shape[-1:], generator=g))
    return x.to(dtype).to(dev)


@gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 1000), (130, 384), (128, 8), (200, 1111), (64, 1280)])
@pytest.mark.parametrize("square", [False, True])
def test_quantize(dev, m, k, dtype, square):
    x = rand(dev, (m, k), m * 10007 + k, dtype, 1.0)
    q, scale = (ops.quantize_fp8_weight if square else ops.quantize_fp8)(x)
    want, s = plain_quantize(x, square)
    assert torch.equal(exponents(scale), s.int())
    assert torch.equal(q.cpu().double(), want)


@gpu
def test_quantize_every_bfloat16_value_and_every_border(dev):
    """All bf16 bit patterns, one to a block with a larger neighbour that fixes the scale, and as a block's own largest."""
    bits = (torch.arange(65536, dtype=torch.int32) << 16).view(torch.float32)
    x = torch.zeros((65536, 128))
    x[:, 3] = bits
    x[:, 77] = 448.0
    for col in (448.0, 0.0):                     # the neighbour fixes the scale at 1, or there is none
        x[:, 77] = col
        q, scale = ops.quantize_fp8(x.to(dev))
        want, s = plain_quantize(x, False)
        assert torch.equal(exponents(scale), s.int())
        got = q.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())


@gpu
def test_quantize_not_finite_and_strided(dev):
    x = rand(dev, (9, 300), 5, torch.float32)
    x[0, 5], x[1, 200], x[2, 299] = math.inf, math.nan, -math.inf
    x[3] = math.nan
    x[4] = 0.0
    x[5] = 1e-45                                 # below every scale
    x[6] = 3.4e38
    for v in (x, x[:, 1:], x[:, ::2], x.t(), x[::3], x[:1].expand(6, 300)):
        q, scale = ops.quantize_fp8(v)
        want, s = plain_quantize(v, False)
        assert torch.equal(exponents(scale), s.int())
        got = q.cpu().double()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(), want.nan_to_num())
    q, scale = ops.quantize_fp8(x.view(3, 3, 300))
    assert q.shape == (9, 384) and scale.shape == (9, 3)
    q, scale = ops.quantize_fp8(x[:0])
    assert q.shape == (0, 384) and scale.shape == (0, 3)


def check_product(dev, x, w, bias, out_dtype, got):
    xq, xs = plain_quantize(x.reshape(-1, x.shape[-1]), False)
    wq, ws = plain_quantize(w, True)
    xd, wd = dequantized(xq, xs, False), dequantized(wq, ws, True)
    want = xd @ wd.t()
    size = xd.abs() @ wd.abs().t()
    if bias is not None:
        want, size = want + bias.cpu().double(), size + bias.cpu().double().abs()
    sums = ((xd.shape[1] + 2) * 2.0 ** -24 + (0 if out_dtype == torch.float32 else 7 * 2.0 ** -13)) * size
    tol = sums + (want.abs() + sums) * HALF[out_dtype] + 2.0 ** -25
    off = (got.cpu().double().view(want.shape) - want).abs() - tol
    assert got.dtype == out_dtype and float(off.max()) <= 0, float(off.max())


SHAPES = [(1, 16, 16), (1, 1280, 1280), (1, 1, 1), (2, 31, 1280), (4, 100, 129), (8, 640, 1111), (15, 257, 512), (16, 256, 2048),
          (17, 64, 128), (31, 1000, 384), (64, 31, 1024), (65, 129, 127), (127, 320, 640), (128, 128, 128), (129, 255, 1000),
          (200, 1280, 1280), (256, 512, 896), (300, 1000, 1111), (511, 513, 2049), (777, 31, 40), (1024, 768, 256)]


@gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear(dev, m, n, k, dtype):
    x, w = rand(dev, (m, k), m + n, dtype, 1.0), rand(dev, (n, k), m + k, torch.float32) / k ** 0.5
    bias = rand(dev, (n,), 3) if (m + n) % 2 else None
    weight = ops.quantize_fp8_weight(w)
    got = ops.linear_fp8(x, weight, bias)
    check_product(dev, x, w, bias, dtype, got)
    again = ops.linear_fp8(ops.quantize_fp8(x), weight, bias, out_dtype=dtype)
    assert torch.equal(got, again)               # quantised inside or before: the same, bit for bit
    assert torch.equal(got, ops.linear_fp8(x, weight, bias))


# every height of tile, with the K loop whole and cut into 2 to 16 pieces, for both forms of the product
TILES = [(2464, 700, 131), (3141, 69, 5865), (261, 435, 3519), (437, 197, 4522), (17, 32, 8836), (1313, 2530, 33), (8321, 205, 4465),
         (130, 3588, 11846), (67, 3371, 7154), (1548, 81, 15631), (2953, 2751, 139), (4813, 3500, 34), (9831, 279, 13156),
         (605, 391, 1714), (394, 340, 2966), (212, 307, 5999), (24, 33, 8385), (1601, 1231, 1701), (9189, 66, 3400), (4546, 65, 4542),
         (73, 2086, 8165), (1636, 1048, 129), (2572, 1302, 32), (512, 1280, 1280), (40, 1296, 1000)]


@gpu
@pytest.mark.parametrize("m,n,k", TILES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_linear_tiles(dev, m, n, k, dtype):
    x, w = rand(dev, (m, k), m + n, dtype, 1.0), rand(dev, (n, k), m + k, torch.float32) / k ** 0.5
    bias = rand(dev, (n,), 3) if (m + n) % 2 else None
    weight = ops.quantize_fp8_weight(w)
    got = ops.linear_fp8(x, weight, bias)
    rows = sorted({r for at in range(0, m + 64, 64) for r in (at - 1, at) if 0 <= r < m} | {m - 1})
    rows = torch.tensor(rows if len(rows) <= 96 else rows[:32] + rows[len(rows) // 2 - 16:len(rows) // 2 + 16] + rows[-32:], device=dev)
    check_product(dev, x[rows], w, bias, dtype, got[rows])
    # every row against the product of what was rounded to 8 bits (2.6 % of a value each on average, 3.7 % together), so that none
    # is left out: 6 % over all of them, 25 % in the worst row of few channels; a wrong row is off by its whole length
    near = x.float() @ w.t() + (bias if bias is not None else 0)
    assert float((got.float() - near).norm() / near.norm()) < 0.06
    assert float((got.float() - near).norm(dim=1).max() / near.norm(dim=1).mean()) < 0.25
    again = ops.linear_fp8(ops.quantize_fp8(x), weight, bias, out_dtype=dtype)
    assert torch.equal(got, again) and torch.equal(got, ops.linear_fp8(x, weight, bias))


@gpu
@pytest.mark.parametrize("m", [1, 7, 40, 300])
@pytest.mark.parametrize("out_dtype", DTYPES)
def test_linear_types_layouts_and_edges(dev, m, out_dtype):
    """Batched, strided and unaligned inputs, every output type, and memory around the output left as it was."""
    k, n = 200, 45
    weight_values = rand(dev, (n, k), 2) / k ** 0.5
    weight = ops.quantize_fp8_weight(weight_values)
    base = rand(dev, (m, 2, k + 3), 9, torch.float16, 0.5)
    for x in (base[:, 0, 1:k + 1], base[:, 1, :k], base[..., 2:k + 2], base[:, 0, :k].t().contiguous().t()):
        got = ops.linear_fp8(x, weight, None, out_dtype=out_dtype)
        assert got.shape == x.shape[:-1] + (n,)
        check_product(dev, x, weight_values, None, out_dtype, got)
    lib, x = _lib.load(), base[:, 0, :k].contiguous()
    guard = torch.full((m * n + 64,), 7.0, dtype=out_dtype, device=dev)
    out = guard[32:32 + m * n]
    code = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[out_dtype]
    need = lib.ed_fp8_linear_workspace(m, n, k, _lib.DT_FP16, code)
    ws = torch.empty(need + 16, dtype=torch.uint8, device=dev)
    _lib.check(lib.ed_fp8_linear(x.data_ptr(), _lib.DT_FP16, k, None, weight.q.data_ptr(), weight.scale.data_ptr(), None,
                                 out.data_ptr(), code, m, n, k, ws.data_ptr() if need else None, need,
                                 torch.cuda.current_stream().cuda_stream))
    assert torch.equal(out.view(m, n), ops.linear_fp8(x, weight, out_dtype=out_dtype))
    assert bool((guard[:32] == 7).all()) and bool((guard[32 + m * n:] == 7).all())


@gpu
@pytest.mark.parametrize("m", [1, 20, 200])
def test_linear_carries_what_is_not_finite_to_its_row_alone(dev, m):
    x, w = rand(dev, (m, 384), 1), rand(dev, (70, 384), 2)
    clean = ops.linear_fp8(x, ops.quantize_fp8_weight(w))
    x[0, 130] = math.inf
    got = ops.linear_fp8(x, ops.quantize_fp8_weight(w))
    assert bool(torch.isnan(got[0]).all()) and torch.equal(got[1:], clean[1:])
    assert bool((ops.linear_fp8(torch.zeros_like(x), ops.quantize_fp8_weight(w)) == 0).all())


@gpu
def test_linear_refusals(dev):
    w = ops.quantize_fp8_weight(rand(dev, (64, 256), 0))
    x = rand(dev, (4, 256), 1)
    with pytest.raises(RuntimeError, match="channels"):
        ops.linear_fp8(x[:, :128], w)
    with pytest.raises(RuntimeError, match="x must be float32"):
        ops.linear_fp8(x.double(), w)
    with pytest.raises(RuntimeError, match="out_dtype"):
        ops.linear_fp8(x, w, out_dtype=torch.float64)
    with pytest.raises(RuntimeError, match="bias"):
        ops.linear_fp8(x, w, torch.zeros(63, device=dev))
    with pytest.raises(RuntimeError, match="bias"):
        ops.linear_fp8(x, w, torch.zeros(64, device=dev, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError, match="weight.scale"):
        ops.linear_fp8(x, ops.Fp8Weight(w.q, w.scale[:, :1].contiguous()))
    with pytest.raises(RuntimeError, match="weight.q"):
        ops.linear_fp8(x, ops.Fp8Weight(w.q.view(torch.uint8), w.scale))
    with pytest.raises(RuntimeError, match="x.scale"):
        r = ops.quantize_fp8(x)
        ops.linear_fp8(ops.Fp8Rows(r.q, r.scale[:2].contiguous()), w)
    with pytest.raises(_lib.EvoDiffHipError, match="no gradient"):
        ops.linear_fp8(x.clone().requires_grad_(), w)
    with torch.no_grad():
        ops.linear_fp8(x.clone().requires_grad_(), w)
    with pytest.raises(RuntimeError, match="weight must be"):
        ops.quantize_fp8_weight(x.view(2, 2, 256))
    assert ops.linear_fp8(x[:0], w).shape == (0, 64)


def make_logits(dev, rows, v, dtype, seed, masked):
    x = rand(dev, (rows, v), seed) * 2.5
    if masked:
        x[:, torch.arange(v) % 3 == 1] = -math.inf
        x[0, :] = -math.inf                                    # a row without a class
        if rows > 1:
            x[1, 1:] = -math.inf                               # a row with one
            x[1, 0] = -3.0
        if rows > 2:
            x[2, ::2] = torch.finfo(dtype).min                 # masks of the type's lowest value
    return x.to(dtype)


ROWS = [(1, 1, 1), (1, 2, 2), (64, 31, 5), (5, 32, 32), (7, 33, 0), (3, 64, 8), (9, 65, 20), (70, 255, 5), (2, 256, 1), (5, 257, 20),
        (33, 1000, 8), (3, 1024, 32), (4, 1025, 20), (3, 4099, 5), (5, 8192, 20), (2, 32000, 20), (1, 50257, 20), (3, 131072, 20), (1, 131071, 0)]


@gpu
@pytest.mark.parametrize("rows,v,k", ROWS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_token_logprobs(dev, rows, v, k, dtype, masked):
    x = make_logits(dev, rows, v, dtype, rows + v, masked)
    targets = torch.randint(0, v, (rows,), generator=torch.Generator().manual_seed(v))
    select = torch.arange(rows) % 4 != 3 if rows > 4 else None
    got = ops.token_logprobs(x, targets.to(dev), k, None if select is None else select.to(dev))
    want = plain_logprobs(x, targets, k, select)
    tol = logprob_tolerance(x.float().cpu(), v)
    assert torch.equal(got.top_token.cpu(), want[3])
    rel_ok(got.logprob, want[0], tol)
    rel_ok(got.entropy, want[1], 2 * tol)
    rel_ok(got.top_logprob, want[2], tol)


@gpu
@pytest.mark.parametrize("v", [5, 40, 700, 5000, 40000])
def test_token_logprobs_ties_and_orders(dev, v):
    """Constant rows, rows in rising and falling order, few distinct values, -0 beside 0, a late and an early spike."""
    k = min(v, 20)
    x = torch.zeros((8, v))
    x[1] = torch.arange(v) * (20.0 / v)
    x[2] = -x[1]
    x[3] = (torch.arange(v) * 7919 % 5).float()
    x[4, ::2] = -0.0
    x[5, -1] = 9.0
    x[6, 0] = 9.0
    x[7] = (torch.arange(v) * 104729 % 97).float()
    targets = torch.arange(8) % v
    for dtype in DTYPES:
        xd = x.to(dtype).to(dev)
        got, want = ops.token_logprobs(xd, targets.to(dev), k), plain_logprobs(xd, targets, k)
        assert torch.equal(got.top_token.cpu(), want[3])
        tol = logprob_tolerance(xd.float().cpu(), v)
        rel_ok(got.logprob, want[0], tol)
        rel_ok(got.entropy, want[1], 2 * tol)
        rel_ok(got.top_logprob, want[2], tol)


@gpu
@pytest.mark.parametrize("v", [31, 300, 3000, 70000])
def test_token_logprobs_not_finite_and_out_of_range(dev, v):
    x = rand(dev, (7, v), v)
    x[1, v // 2], x[2, 3], x[3, 0] = math.nan, math.inf, -math.inf
    x[4] = math.nan
    targets = torch.tensor([v, 1, 2, 0, 0, -1, v - 1])
    got = ops.token_logprobs(x, targets.to(dev), 5)
    assert torch.isnan(got.logprob.cpu()).tolist() == [True, True, True, False, True, True, False]
    assert float(got.logprob[3]) == -math.inf
    assert torch.isnan(got.entropy.cpu()).tolist() == [False, True, True, False, True, False, False]
    assert torch.isnan(got.top_logprob.cpu()).all(1).tolist() == [False, True, True, False, True, False, False]
    assert int(got.top_token.min()) >= 0 and int(got.top_token.max()) < v
    want = plain_logprobs(x, targets, 5)
    for r in (0, 3, 5, 6):
        assert torch.equal(got.top_token[r].cpu(), want[3][r])
    xg = x.clone().requires_grad_()
    out = ops.token_logprobs(xg, targets.to(dev), 5)
    grad, = torch.autograd.grad(out.logprob.sum(), xg)
    assert torch.isnan(grad).all(1).tolist() == [True, True, True, False, True, True, False]


@gpu
@pytest.mark.parametrize("v", [31, 500, 20000])
def test_token_logprobs_views_classes_and_shapes(dev, v):
    x = rand(dev, (4, 6, v + 5), 3, torch.bfloat16)
    targets = torch.randint(0, v - 3, (4, 5), device=dev)
    for view in (x[:, :-1, :v], x[:, 1:, 5:], x[:, :5, 1:v + 1], x.transpose(0, 1)[:5].transpose(0, 1)[..., :v],
                 x[:, :1, :v].expand(4, 5, v), x[:, :5, :v].transpose(1, 2).contiguous().transpose(1, 2)):
        got = ops.token_logprobs(view, targets, 3, n_classes=v - 3)
        want = ops.token_logprobs(view.reshape(20, -1)[:, :v - 3].contiguous(), targets.reshape(20), 3)
        # tokens are equal; a row's sums are taken in an order that goes by its alignment, so that two layouts of it differ by
        # up to twice what either may be off the exact value (the entropy, a sum and a quotient more, twice that)
        tol = logprob_tolerance(view.float().cpu(), v - 3)
        assert torch.equal(got.top_token.reshape(20, 3), want.top_token)
        rel_ok(got.logprob.reshape(20), want.logprob.cpu(), 2 * tol, 2.0 ** -21)
        rel_ok(got.entropy.reshape(20), want.entropy.cpu(), 4 * tol, 2.0 ** -21)
        rel_ok(got.top_logprob.reshape(20, 3), want.top_logprob.cpu(), 2 * tol, 2.0 ** -21)
        assert got.logprob.shape == (4, 5) and got.top_token.shape == (4, 5, 3)
    one = ops.token_logprobs(x[0, 0, :v], torch.tensor(3, device=dev), 2)
    assert one.logprob.shape == () and one.top_token.shape == (2,)
    none = ops.token_logprobs(x[:, :5, :v], None, 3, n_classes=v - 3)
    assert none.logprob is None and torch.equal(none.top_token, ops.token_logprobs(x[:, :5, :v], targets, 3, n_classes=v - 3).top_token)
    empty = ops.token_logprobs(x[:, :0, :v], targets[:, :0], 3)
    assert empty.logprob.shape == (4, 0) and empty.top_logprob.shape == (4, 0, 3)
    assert torch.equal(ops.token_logprobs(x[:, :5, :v], targets.int()).logprob, ops.token_logprobs(x[:, :5, :v], targets).logprob)


@gpu
def test_token_logprobs_refusals(dev):
    x, t = rand(dev, (4, 31), 0), torch.zeros(4, dtype=torch.long, device=dev)
    for bad in (dict(top_k=32), dict(top_k=-1), dict(n_classes=32), dict(n_classes=0), dict(n_classes=3, top_k=4)):
        with pytest.raises(RuntimeError, match="top_k|n_classes"):
            ops.token_logprobs(x, t, **bad)
    with pytest.raises(RuntimeError, match="targets"):
        ops.token_logprobs(x, t[:3])
    with pytest.raises(RuntimeError, match="targets"):
        ops.token_logprobs(x, t.float())
    with pytest.raises(RuntimeError, match="select"):
        ops.token_logprobs(x, t, select=t)
    with pytest.raises(RuntimeError, match="logits"):
        ops.token_logprobs(x.double(), t)


def plain_grad(x, targets, token, select, g_lp, g_h, g_top, n_classes=None):
    """The formula in 64 bits, row by row on the CPU."""
    x = x.detach().cpu().double()
    grad = torch.zeros_like(x)
    n = x.shape[1] if n_classes is None else n_classes
    for r in range(len(x)):
        row = x[r, :n]
        if (select is not None and not select[r]) or bool((row == -math.inf).all()):
            continue
        lp = row - torch.logsumexp(row, 0)
        p = torch.exp(lp)
        plp = torch.where(p > 0, p * lp, torch.zeros_like(p))
        h = -plp.sum()
        d = -p * (g_lp[r] + g_top[r].sum()) - g_h[r] * (plp + p * h)
        if targets is not None:
            d[targets[r]] += g_lp[r]
        d.scatter_add_(0, token[r], g_top[r])
        grad[r, :n] = d
    return grad


@gpu
@pytest.mark.parametrize("rows,v,k", [(1, 1, 1), (64, 31, 5), (5, 33, 0), (6, 64, 20), (5, 300, 8), (5, 1025, 5), (6, 4099, 20), (5, 32000, 8), (3, 50257, 0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", [False, True])
def test_gradient(dev, rows, v, k, dtype, masked):
    x = make_logits(dev, rows, v, dtype, rows + v, masked).requires_grad_()
    g = torch.Generator().manual_seed(v)
    targets = torch.randint(0, v, (rows,), generator=g)
    select = torch.arange(rows) % 5 != 4 if rows > 4 else None
    g_lp, g_h, g_top = torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn((rows, k), generator=g)
    out = ops.token_logprobs(x, targets.to(dev), k, None if select is None else select.to(dev))
    grad, = torch.autograd.grad(out[:3], x, (g_lp.to(dev), g_h.to(dev), g_top.to(dev)))
    want = plain_grad(x, targets, out.top_token.cpu().clamp(min=0), select, g_lp.double(), g_h.double(), g_top.double())
    # p is off by the tolerance of a log probability (relative), and multiplies terms of these sizes; then one rounding
    size = g_lp.abs() + g_top.abs().sum(1) + g_h.abs() * 64
    tol = 4 * logprob_tolerance(x.detach().float().cpu(), v) * size[:, None].double()
    off = (grad.cpu().double() - want).abs() - (tol + (want.abs() + tol) * HALF[dtype] + torch.finfo(dtype).smallest_normal * HALF[dtype] * 2)
    assert grad.dtype == dtype and float(off.max()) <= 0, float(off.max())
    assert torch.equal(torch.autograd.grad(ops.token_logprobs(x, targets.to(dev), k, None if select is None else select.to(dev))[:3], x,
                                           (g_lp.to(dev), g_h.to(dev), g_top.to(dev)))[0], grad)


@gpu
@pytest.mark.parametrize("v", [17, 700])
def test_gradient_against_differences(dev, v):
    """Central differences of the 64-bit definition along random directions, and partial sets of incoming gradients."""
    x = rand(dev, (3, v), v).requires_grad_()
    targets = torch.tensor([0, v - 1, v // 2])
    out = ops.token_logprobs(x, targets.to(dev), 4)
    weights = [torch.tensor([0.7, -1.3, 2.0]), torch.tensor([1.1, 0.4, -0.6]), torch.linspace(-1, 1, 12).view(3, 4)]

    def value(z, parts):
        f = plain_logprobs(z, targets, 4)
        return sum(float((f[i] * weights[i].double()).sum()) for i in parts)

    for parts in ((0,), (1,), (2,), (0, 1, 2)):
        grad, = torch.autograd.grad([out[i] for i in parts], x, [weights[i].to(dev) for i in parts], retain_graph=True)
        for seed in range(3):
            step = torch.randn((3, v), generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
            eps = 1e-5
            base = x.detach().cpu().double()
            slope = (value(base + eps * step, parts) - value(base - eps * step, parts)) / (2 * eps)
            assert abs(float((grad.cpu().double() * step).sum()) - slope) < 2e-5 * max(1.0, float(step.abs().max())) * v ** 0.5


@gpu
def test_gradient_is_taken_once_and_in_any_grad_mode(dev):
    x = rand(dev, (4, 31), 0).requires_grad_()
    t = torch.zeros(4, dtype=torch.long, device=dev)
    grad, = torch.autograd.grad(ops.token_logprobs(x, t).logprob.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(grad.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        grad.sum().backward()
    want, = torch.autograd.grad(ops.token_logprobs(x, t).logprob.sum(), x)
    assert torch.equal(grad, want)
    with torch.no_grad():
        assert not ops.token_logprobs(x, t).logprob.requires_grad
    assert not ops.token_logprobs(x.detach(), t).logprob.requires_grad
    out = ops.token_logprobs(x, t, 3)
    assert out.entropy.requires_grad and out.top_logprob.requires_grad and not out.top_token.requires_grad
    out.entropy.mean().backward()
    assert x.grad is not None and x.grad.shape == x.shape


@gpu
def test_gradient_of_views_classes_broadcast_and_missing_targets(dev):
    v = 40
    base = rand(dev, (3, 5, v), 1).requires_grad_()
    targets = torch.randint(0, 30, (3, 4), device=dev)
    out = ops.token_logprobs(base[:, :-1], targets, 2, n_classes=30)
    grad, = torch.autograd.grad(out.logprob.sum() + out.entropy.sum(), base)
    ref = torch.log_softmax(base.detach().double()[:, :-1, :30], -1).requires_grad_()
    logits = base.detach().double()[:, :-1, :30].requires_grad_()
    lp = torch.log_softmax(logits, -1)
    want, = torch.autograd.grad(lp.gather(2, targets[..., None]).sum() - (lp.exp() * lp).sum(), logits)
    assert bool((grad[:, -1] == 0).all()) and bool((grad[:, :, 30:] == 0).all())
    assert float((grad[:, :-1, :30].double() - want).abs().max()) < 1e-5
    one = rand(dev, (1, v), 2).requires_grad_()                       # one row under many: its gradient is their sum
    many = ops.token_logprobs(one.expand(6, v), torch.arange(6, device=dev))
    grad, = torch.autograd.grad(many.logprob.sum(), one)
    lp = one.detach().double().requires_grad_()
    want, = torch.autograd.grad(torch.log_softmax(lp, -1)[0, :6].sum(), lp)
    assert float((grad.double() - want).abs().max()) < 1e-5
    out = ops.token_logprobs(one, None, 3)
    grad, = torch.autograd.grad(out.entropy.sum() + out.top_logprob.sum(), one)
    lp = torch.log_softmax(one.detach().double(), -1)
    want = plain_grad(one, None, out.top_token.cpu(), None, torch.zeros(1).double(), torch.ones(1).double(), torch.ones((1, 3)).double())
    assert float((grad.cpu().double() - want).abs().max()) < 1e-5


@gpu
def test_rows_that_share_nothing_with_their_batch(dev):
    """A row's results do not depend on the rows beside it, however many there are."""
    for v in (31, 3000, 50000):
        x = rand(dev, (300, v), 7, torch.bfloat16)
        t = torch.randint(0, v, (300,), device=dev)
        whole = ops.token_logprobs(x, t, 5)
        for r in (0, 150, 299):
            part = ops.token_logprobs(x[r:r + 1], t[r:r + 1], 5)
            assert torch.equal(part.top_token[0], whole.top_token[r])
            assert abs(float(part.logprob[0]) - float(whole.logprob[r])) <= 2 * logprob_tolerance(x.float().cpu(), v)


@gpu
def test_long_offsets(dev):
    """Rows that start past 2^31 elements, in logits and in a product's activations."""
    rows, v = 70000, 32000
    big = torch.empty(rows * v, dtype=torch.bfloat16, device=dev)
    x = big.view(rows, v)
    x[-2:] = rand(dev, (2, v), 1, torch.bfloat16)
    x[:2] = 0
    tail = torch.tensor([5, 6], device=dev)
    strided = torch.as_strided(x, (2, v), (v * (rows - 1), 1))
    got = ops.token_logprobs(strided, tail, 4)
    want = ops.token_logprobs(torch.stack([x[0], x[-1]]), tail, 4)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    w = ops.quantize_fp8_weight(rand(dev, (64, v), 2))
    assert torch.equal(ops.linear_fp8(strided, w), ops.linear_fp8(torch.stack([x[0], x[-1]]), w))


@gpu
def test_linear_long_offsets(dev):
    """Operands and outputs past 2^32 bytes and elements.  Small whole numbers: exact in 8 bits, every sum exact in fp32."""
    k, m = 131072, 40008
    base = torch.randint(-2, 3, (8, k), device=dev).bfloat16()
    x = torch.empty((m // 8, 8, k), dtype=torch.bfloat16, device=dev)
    x.copy_(base.expand_as(x))
    x = x.view(m, k)
    last = torch.randint(-2, 3, (24, k), device=dev).bfloat16()
    x[-24:] = last
    w = torch.randint(-2, 3, (48, k), device=dev).bfloat16()
    weight = ops.quantize_fp8_weight(w)
    want, want_last = base.double().cpu() @ w.double().cpu().T, last.double().cpu() @ w.double().cpu().T
    for rows in (x, ops.quantize_fp8(x)):
        out = ops.linear_fp8(rows, weight, out_dtype=torch.float32).cpu().double()
        assert torch.equal(out[-24:], want_last)
        assert torch.equal(out[:-24].view(-1, 8, 48), want.expand(m // 8 - 3, 8, 48))
    del x, rows
    a, b = torch.randint(-3, 4, (66001, 8), device=dev).bfloat16(), torch.randint(-3, 4, (66003, 8), device=dev).bfloat16()
    out = ops.linear_fp8(a, ops.quantize_fp8_weight(b))  # 4.4e9 values, under 2^8: exact in bf16
    for rows in (slice(0, 300), slice(65020, 65200), slice(65900, 66001)):
        assert torch.equal(out[rows].cpu().double(), a[rows].cpu().double() @ b.cpu().double().T)


@gpu
@pytest.mark.parametrize("rows,v", [(70001, 31001), (70000007, 31)])
def test_log_probabilities_and_gradient_past_32_bits(dev, rows, v):
    """More than 2^31 logits: the first, middle and last rows as they are alone (fp32 sums in another order: 1e-5 is 80 roundings;
    gradients rounded to bf16 on both sides: 2^-7)."""
    some = rand(dev, (1024, v), 1, torch.bfloat16)
    x = torch.empty((rows, v), dtype=torch.bfloat16, device=dev)
    for at in range(0, rows, 1024):
        if v > 100 or at == 0 or at + 1024 >= rows or at % (1 << 20) == 0:
            x[at:at + 1024] = some[:min(1024, rows - at)]
    pick = torch.tensor([0, 5, 1 << 16, (1 << 16) + 1, (rows - 1) // 1024 * 1024, rows - 1], device=dev)
    if v <= 100:
        pick = torch.tensor([0, 5, 64 << 20, (64 << 20) + 1, (rows - 1) // 1024 * 1024, rows - 1], device=dev)
    targets = torch.arange(rows, device=dev) % v
    x.requires_grad_()
    out = ops.token_logprobs(x, targets, 2)
    few = x.detach()[pick].requires_grad_()
    want = ops.token_logprobs(few, targets[pick], 2)
    for a, b in zip(out, want):
        assert torch.equal(a[pick], b) if a.dtype == torch.long else torch.allclose(a[pick], b, rtol=1e-5, atol=1e-5)
    grad, = torch.autograd.grad(out.logprob, x, torch.ones_like(out.logprob))
    want_grad, = torch.autograd.grad(want.logprob, few, torch.ones_like(want.logprob))
    assert torch.allclose(grad[pick].float(), want_grad.float(), rtol=2 ** -7, atol=1e-6)


@gpu
def test_together_captured_and_on_other_streams(dev):
    """A scoring step as a program runs it - hidden rows, an 8-bit head, log probabilities, the gradient to the logits - eager,
    in two captured graphs that replay in turn, and on another stream."""
    hidden, head = rand(dev, (50, 320), 1, torch.bfloat16), ops.quantize_fp8_weight(rand(dev, (1000, 320), 2) / 18)
    one = hidden[:1].clone()
    targets = torch.randint(0, 1000, (50,), device=dev)
    ones = torch.ones(50, device=dev)

    def step(h, t):
        logits = ops.linear_fp8(h, head, out_dtype=torch.float32).requires_grad_()
        out = ops.token_logprobs(logits, t, 5)
        grad, = torch.autograd.grad((out.logprob, out.entropy), logits, (ones[:len(t)], ones[:len(t)]))
        return [t.detach() for t in out] + [grad]

    eager, eager_one = step(hidden, targets), step(one, targets[:1])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            on_side = step(hidden, targets)
            step(one, targets[:1])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(eager, on_side))
    graphs = []
    for h, t in ((hidden, targets), (one, targets[:1])):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            captured = step(h, t)
        graphs.append((g, captured))
    for i in range(4):
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (_, captured), want in zip(graphs, (eager, eager_one)):
            assert all(torch.equal(a, b) for a, b in zip(captured, want))
        hidden.copy_(rand(dev, (50, 320), 10 + i, torch.bfloat16))
        one.copy_(hidden[:1])
        eager, eager_one = step(hidden, targets), step(one, targets[:1])
    logits = ops.linear_fp8(hidden, head, out_dtype=torch.float32)
    want = plain_logprobs(logits, targets.cpu(), 5)
    assert torch.equal(eager[3].cpu(), want[3])


@gpu
def test_capture_with_an_eager_graph_of_the_leaf(dev):
    """Refused while that graph is alive (only the forward is tried); captured, replayed and right once it is gone."""
    logits, targets = rand(dev, (40, 700), 3).requires_grad_(), torch.randint(0, 700, (40,), device=dev)
    ones = torch.ones(40, device=dev)

    def step():
        out = ops.token_logprobs(logits, targets, 3)
        return torch.autograd.grad((out.logprob, out.entropy), logits, (ones, ones))[0]

    want = step()
    alive = ops.token_logprobs(logits, targets, 3)
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.token_logprobs(logits, targets, 3)
    assert torch.equal(torch.autograd.grad((alive.logprob, alive.entropy), logits, (ones, ones))[0], want)
    del alive
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = step()
    for _ in range(3):
        captured.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, want)
        assert torch.equal(step(), want)


@gpu
def test_model_score_tokens(dev):
    """The model's own path: score_tokens agrees with the model's logits in 64 bits and with score_nll, for both precisions."""
    from evodiff_amd.model import ByteNetLMTime
    torch.manual_seed(0)
    m = ByteNetLMTime(31, 8, 256, 3, 5, 128, padding_idx=28, final_ln=True, slim=False, activation="gelu").eval()
    x = torch.randint(0, 26, (3, 50), device=dev)
    y = torch.zeros(3, dtype=torch.long, device=dev)
    targets = torch.randint(0, 26, (3, 50), device=dev)
    select = torch.rand((3, 50), device=dev) < 0.5
    for precision in ("fp32", "bf16"):
        m.precision = precision
        logits = m(x, y)
        got = m.score_tokens(x, y, targets, select=select, n_classes=26, top_k=5)
        want = plain_logprobs(logits.reshape(150, 31), targets.reshape(-1).cpu(), 5, select.reshape(-1).cpu(), 26)
        tol = logprob_tolerance(logits.cpu(), 26)
        assert torch.equal(got.top_token.reshape(150, 5).cpu(), want[3])
        rel_ok(got.logprob.reshape(-1), want[0], tol)
        rel_ok(got.entropy.reshape(-1), want[1], 2 * tol)
        rel_ok(got.top_logprob.reshape(150, 5), want[2], tol)
        nll = m.score_nll(x, y, targets, select=select, n_classes=26)
        assert float((got.logprob + nll).abs().max()) < 1e-4
        again = m.score_tokens(x, y, targets, select=select, n_classes=26, top_k=5)
        assert all(torch.equal(a, b) for a, b in zip(got, again))
    with pytest.raises(ValueError):
        m.score_tokens(x, y, targets, n_classes=32)
    with pytest.raises(ValueError):
        m.score_tokens(x, y, targets, n_classes=4, top_k=5)
    with pytest.raises(ValueError):
        m.score_tokens(x, y, targets[:, :-1])
    with pytest.raises(_lib.EvoDiffHipError):
        m.score_tokens(x, y, torch.full_like(targets, 30), n_classes=26)


# ---- the model in 8 bits --------------------------------------------------------------------------------------------

def bytenet(d_model, n_layers, r, slim=True, activation="gelu", causal=False, timesteps=None, kernel_size=5):
    from evodiff_amd.model import ByteNetLMTime
    torch.manual_seed(3)
    m = ByteNetLMTime(31, 8, d_model, n_layers, kernel_size, r, padding_idx=28, final_ln=True, slim=slim, activation=activation,
                      causal=causal, timesteps=timesteps).eval()
    with torch.no_grad():
        for name, p in m.named_parameters():  # (norms and biases that are not their initial ones and zeros)
            if p.dim() == 1:
                p.add_(0.2 * torch.randn_like(p))
    m.precision = "fp8"
    return m


def plain_block(block, dilation, x, causal, activation):
    """What a block adds to the residual stream x (B, L, D), fp64 on the CPU: LayerNorms and activations in 64 bits, the operands
    of each product rounded to 8 bits with the scales of the definition, products' outputs rounded to bf16 but the last."""
    act = torch.nn.functional.gelu if activation == "gelu" else torch.relu

    def rows(v, norm):
        v = act(torch.nn.functional.layer_norm(v, v.shape[-1:], norm.weight.double().cpu(), norm.bias.double().cpu(), norm.eps))
        flat = v.reshape(-1, v.shape[-1])
        return dequantized(*plain_quantize(flat, False), False)[:, :v.shape[-1]].reshape(v.shape)

    def weight(w):
        return dequantized(*plain_quantize(w, True), True)[:, :w.shape[1]]

    def bf16(v):
        return v.bfloat16().double()

    pff1, pff2, conv = block.sequence1[2].conv, block.sequence2[2].conv, block.conv
    y = bf16(rows(x, block.sequence1[0]) @ weight(pff1.weight[:, :, 0]).T + pff1.bias.double())
    z = rows(y, block.sequence1[3])
    taps, length = conv.weight.shape[2], x.shape[1]
    center = taps - 1 if causal else taps // 2
    y = conv.bias.double().repeat(z.shape[0], length, 1)
    for t in range(taps):
        shift = (t - center) * dilation
        lo, hi = max(0, -shift), min(length, length - shift)
        if lo < hi:
            y[:, lo:hi] += z[:, lo + shift:hi + shift] @ weight(conv.weight[:, :, t]).T
    return rows(bf16(y), block.sequence2[0]) @ weight(pff2.weight[:, :, 0]).T + pff2.bias.double()


@gpu
@pytest.mark.parametrize("batch,length,kw", [
    (3, 50, dict(d_model=256, n_layers=8, r=128)),                                       # taps that reach no row
    (1, 1, dict(d_model=64, n_layers=2, r=2)),
    (2, 300, dict(d_model=96, n_layers=3, r=4, slim=False, activation="relu")),          # channels that end inside a block
    (5, 33, dict(d_model=320, n_layers=4, r=8, causal=True)),
    (1, 129, dict(d_model=640, n_layers=2, r=2, timesteps=20, slim=False)),
    (40, 64, dict(d_model=1024, n_layers=2, r=64)),
    (7, 500, dict(d_model=384, n_layers=2, r=128, slim=False)),
    (2, 70, dict(d_model=2048, n_layers=1, r=1, slim=False, kernel_size=3)),
    (4, 100, dict(d_model=128, n_layers=2, r=2, kernel_size=1)),
])
def test_model_in_8_bits(dev, batch, length, kw):
    """Every block against its plain form from the same residual stream, position by position, in 2-norms.

    The first product's operands differ from the plain form's where a relative difference of 1e-6 in the LayerNorm (3e-5 with
    the fitted GELU) turns a rounding: an expected square of difference * step, the steps 2^-4 to 2^-3 of a value, so 0.2 %; the
    products keep that share, the second quantiser turns 2e-3 into sqrt(2e-3 * 0.09) = 1.3 %, the third that into 3.4 %.  The
    bound is 10 %, three times that; a tap left out of five is 45 %, one of three blocks at twice its scale 58 %."""
    m = bytenet(**kw)
    x = torch.randint(0, 26, (batch, length), device=dev)
    y = torch.randint(0, kw.get("timesteps") or 1, (batch,), device=dev)
    logits, acts = m(x, y, return_blocks=True)
    again = m(x, y)
    assert torch.equal(logits, again)
    acts = acts.double().cpu()
    for i, (block, dilation) in enumerate(zip(m.embedder.layers, m.embedder.dilations)):
        want = plain_block(block, dilation, acts[i], kw.get("causal", False), kw.get("activation", "gelu"))
        got = acts[i + 1] - acts[i]
        worst = float(((got - want).norm(dim=2) / want.norm(dim=2)).detach().max())
        print("block", i, "dilation", dilation, "worst position", worst)
        assert worst < 0.1
    tail = torch.nn.functional.layer_norm(acts[-1], acts.shape[-1:], m.last_norm.weight.double(), m.last_norm.bias.double(), m.last_norm.eps)
    tail = tail @ m.decoder.conv.weight[:, :, 0].double().T + m.decoder.conv.bias.double()
    assert float((logits.cpu() - tail).detach().abs().max()) < 1e-4 * float(tail.detach().abs().max())


@gpu
def test_model_in_8_bits_scores_lengths_in_turn_and_new_weights(dev):
    m = bytenet(256, 4, 8)
    y = torch.zeros(6, dtype=torch.long, device=dev)
    calls = [torch.randint(0, 26, s, device=dev) for s in ((6, 90), (2, 17), (5, 200), (6, 91), (1, 1))]
    first = [m(x, y[:len(x)]) for x in calls]
    for x, want in zip(reversed(calls), reversed(first)):  # the zero rows of one length are another's values
        assert torch.equal(m(x, y[:len(x)]), want)
    x, logits = calls[0], first[0]
    targets = torch.randint(0, 26, x.shape, device=dev)
    select = torch.rand(x.shape, device=dev) < 0.5
    got = m.score_tokens(x, y, targets, select=select, n_classes=26, top_k=4)
    want = plain_logprobs(logits.reshape(-1, 31), targets.reshape(-1).cpu(), 4, select.reshape(-1).cpu(), 26)
    tol = logprob_tolerance(logits.cpu(), 26)
    assert torch.equal(got.top_token.reshape(-1, 4).cpu(), want[3])
    rel_ok(got.logprob.reshape(-1), want[0], tol)
    rel_ok(got.entropy.reshape(-1), want[1], 2 * tol)
    assert float((got.logprob + m.score_nll(x, y, targets, select=select, n_classes=26)).abs().max()) < 1e-4
    with torch.no_grad():
        m.embedder.layers[1].conv.weight.mul_(-1)
    changed, acts = m(x, y, return_blocks=True)
    assert not torch.equal(changed, logits)
    acts = acts.double().cpu()
    want = plain_block(m.embedder.layers[1], m.embedder.dilations[1], acts[1], False, "gelu")
    assert float(((acts[2] - acts[1] - want).norm(dim=2) / want.norm(dim=2)).detach().max()) < 0.1
    other = bytenet(256, 4, 8)
    other.precision = "bf16"
    other(x, y)
    m.precision = "bf16"  # a handle that has run in 8 bits runs in the others as before
    with torch.no_grad():
        m.embedder.layers[1].conv.weight.mul_(-1)
    m.precision = "fp8"
    assert torch.equal(m(x, y), logits)
    m.precision = "bf16"
    assert torch.equal(m(x, y), other(x, y))


@gpu
def test_model_in_8_bits_refuses_the_sampling_loops(dev):
    m = bytenet(64, 2, 2)
    order = torch.arange(10, dtype=torch.int32, device=dev)
    with pytest.raises(_lib.EvoDiffHipError, match="sampling loops"):
        m.oadm_sample(torch.full((2, 10), 28, device=dev), order, torch.rand((10, 2), device=dev), 26)
    m.precision = "fp4"
    with pytest.raises(ValueError, match="fp8"):
        m(torch.zeros((1, 4), dtype=torch.long, device=dev), torch.zeros(1, dtype=torch.long, device=dev))
