"""The operators that carry a scoring run beside the model itself, each as a measured case and in its plain form.

Three operators: quantisation to 8-bit floating point with a scale for each block of 128, the matrix product on operands of
that form, and the log probabilities of given tokens with entropy and top alternatives (forward, and with the gradient to the
logits).  ``run`` computes a case in elementary torch operations (``own`` false) or calls ``evodiff_amd.ops`` (``own`` true).
"""
import math

import torch

own = False

BLOCK = 128           # values that share a scale: 128 channels of a row, or 128 x 128 weights
TOP = 448.0           # the largest finite value of float8_e4m3fn
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the activations of one block of the 640M model at 64 sequences of 256, on their way into an 8-bit product
        {"name": "quantize_rows_16384x1280", "op": "quantize_rows", "m": 16384, "k": 1280, "dtype": "bf16"},
        # the weights of a five-tap convolution of that model, taps stacked, as a checkpoint is loaded
        {"name": "quantize_weight_6400x1280", "op": "quantize_weight", "m": 6400, "k": 1280, "dtype": "fp32"},
        # one token of one sequence through a 1280 x 1280 projection: the smallest product, latency alone
        {"name": "linear_1x1280x1280", "op": "linear", "m": 1, "n": 1280, "k": 1280, "dtype": "bf16", "out": "bf16", "bias": True},
        # eight sequences, one token each, through a wide layer: the weights are streamed once
        {"name": "linear_8x8192x8192", "op": "linear", "m": 8, "n": 8192, "k": 8192, "dtype": "bf16", "out": "bf16", "bias": False},
        # a ragged batch through an odd head, kept in 32 bits: every edge of a tile is cut
        {"name": "linear_300x1000x1111", "op": "linear", "m": 300, "n": 1000, "k": 1111, "dtype": "fp32", "out": "fp32", "bias": True},
        # the 1x1 projection of the 640M model at 64 sequences of 256
        {"name": "linear_16384x1280x1280", "op": "linear", "m": 16384, "n": 1280, "k": 1280, "dtype": "bf16", "out": "bf16", "bias": True},
        # the largest product: compute-bound
        {"name": "linear_8192x8192x8192", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "dtype": "bf16", "out": "bf16", "bias": False},
        # one autoregressive step of 64 sequences over the protein alphabet
        {"name": "logprobs_64x31", "op": "logprobs", "rows": 64, "v": 31, "dtype": "fp32", "top": 5, "masked": False, "skip": False},
        # one step of eight sequences over a large vocabulary: few rows, a long axis
        {"name": "logprobs_8x131072", "op": "logprobs", "rows": 8, "v": 131072, "dtype": "bf16", "top": 20, "masked": False, "skip": False},
        # scoring whole prompts over an odd vocabulary, some classes forbidden, padded positions left out
        {"name": "logprobs_4096x50257", "op": "logprobs", "rows": 4096, "v": 50257, "dtype": "bf16", "top": 20, "masked": True, "skip": True},
        # a loss on the protein alphabet at 64 sequences of 256, with an entropy term: forward and gradient
        {"name": "train_16384x31", "op": "train", "rows": 16384, "v": 31, "dtype": "fp32", "top": 0, "masked": False, "skip": True},
        # a loss on a text vocabulary with a term on the eight top alternatives: forward and gradient
        {"name": "train_4096x32000", "op": "train", "rows": 4096, "v": 32000, "dtype": "bf16", "top": 8, "masked": True, "skip": False},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["quantize_rows", "quantize_weight", "linear", "linear", "logprobs", "logprobs", "train"])
    if op in ("quantize_rows", "quantize_weight"):
        m, k = _log(rng, 1, 16384), _log(rng, 16, 8192)
        return {"op": op, "m": m, "k": k, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
    if op == "linear":
        m, n, k = _log(rng, 1, 16384), _log(rng, 16, 8192), _log(rng, 16, 8192)
        dtype = rng.choice(["bf16", "bf16", "fp32", "fp16"])
        return {"op": op, "m": min(m, 8192 ** 3 // (n * k)), "n": n, "k": k, "dtype": dtype, "out": rng.choice([dtype, "fp32"]),
                "bias": rng.random() < 0.5}
    v = _log(rng, 2, 131072)
    rows = min(_log(rng, 1, 16384), 4096 * 32000 // v)
    return {"op": op, "rows": rows, "v": v, "dtype": rng.choice(["fp32", "bf16", "bf16", "fp16"]),
            "top": min(v, rng.choice([0, 1, 5, 8, 20])), "masked": rng.random() < 0.5, "skip": rng.random() < 0.5}


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    s = dict(case)
    if case["op"] in ("quantize_rows", "quantize_weight", "linear"):
        # activations behind a LayerNorm and a GELU: mostly near zero, a few channels far larger
        x = torch.randn((case["m"], case["k"]), generator=g, device=dev)
        x *= torch.exp(torch.randn(case["k"], generator=g, device=dev))
        s["x"] = (x if case["op"] != "quantize_weight" else x / case["k"] ** 0.5).to(dtype)
    if case["op"] == "linear":
        w = torch.randn((case["n"], case["k"]), generator=g, device=dev) / case["k"] ** 0.5
        s["wq"], s["ws"] = _quantize(w, True)      # laid out once, as a program keeps its weights
        s["b"] = torch.randn(case["n"], generator=g, device=dev) if case["bias"] else None
    if case["op"] in ("logprobs", "train"):
        rows, v, top = case["rows"], case["v"], case["top"]
        x = torch.randn((rows, v), generator=g, device=dev).mul_(2.5)
        if case["masked"]:                          # forbidden classes, never all of a row
            ban = torch.rand((1, v), generator=g, device=dev) < 0.3
            ban[0, 0] = False
            x.masked_fill_(ban, -math.inf)
        s["targets"] = torch.randint(0, v, (rows,), generator=g, device=dev)
        # the token that a model is scored on is a likely one more often than not
        likely = torch.rand(rows, generator=g, device=dev) < 0.6
        at = torch.arange(rows, device=dev)
        x[at[likely], s["targets"][likely]] = 6.0
        s["logits"] = x.to(dtype)
        if case["masked"]:                          # a given token is never a forbidden one
            s["targets"] = torch.where(torch.isinf(x[at, s["targets"]]), torch.zeros_like(s["targets"]), s["targets"])
        s["select"] = torch.rand(rows, generator=g, device=dev) < 0.85 if case["skip"] else None
        if case["op"] == "train":
            s["g_logprob"] = torch.randn(rows, generator=g, device=dev)
            s["g_entropy"] = torch.randn(rows, generator=g, device=dev) * 0.1
            s["g_top"] = torch.randn((rows, top), generator=g, device=dev) * 0.2
    return s


# ---- plain forms -----------------------------------------------------------------------------------------------------

def _blocks(x):
    """(m, k) -> fp32 (m, blocks, 128), zeros behind k."""
    m, k = x.shape
    kb = -(-k // BLOCK)
    return torch.nn.functional.pad(x.float(), (0, kb * BLOCK - k)).view(m, kb, BLOCK)


def _quantize(x, square):
    """float8_e4m3fn values (m, blocks * 128) and float8_e8m0fnu scales: a power of two for 128 channels of a row, or for
    128 x 128 weights (``square``), the smallest with which the block's largest value stays within 448."""
    m = x.shape[0]
    b = _blocks(x)
    kb = b.shape[1]
    amax = b.abs().amax(-1)                                                     # (m, kb)
    if square:
        mb = -(-m // BLOCK)
        amax = torch.nn.functional.pad(amax, (0, 0, 0, mb * BLOCK - m)).view(mb, BLOCK, kb).amax(1)
    bits = amax.view(torch.int32)                                               # amax = 2^(e - 127) * (1 + f / 2^23)
    e, f = bits >> 23, bits & 0x7FFFFF
    byte = (e - 8 + (f > 0x600000).int()).clamp(1, 254)                         # 448 = 2^8 * (1 + 0x600000 / 2^23)
    inverse = ((254 - byte) << 23).view(torch.float32)                          # 2^(127 - byte), exact
    if square:
        inverse = inverse.repeat_interleave(BLOCK, 0)[:m]
    q = (b * inverse.unsqueeze(-1)).to(torch.float8_e4m3fn).view(m, kb * BLOCK)
    return q, byte.to(torch.uint8).view(torch.float8_e8m0fnu)


def _dequantize(q, scale, square):
    factor = (scale.view(torch.uint8).int() << 23).view(torch.float32)          # 2^(byte - 127); bytes are 1 .. 254
    if square:
        factor = factor.repeat_interleave(BLOCK, 0)[:q.shape[0]]
    return (q.float().view(q.shape[0], -1, BLOCK) * factor.unsqueeze(-1)).view(q.shape)


def _plain_linear(s):
    x = _dequantize(*_quantize(s["x"], False), False)
    y = x @ _dequantize(s["wq"], s["ws"], True).t()
    if s["b"] is not None:
        y = y + s["b"]
    return y.to(DTYPES[s["out"]])


def _top(x, k):
    """The k largest values of each row, ties to the lowest index: one ordered whole number for value and index."""
    v = x.shape[1]
    bits = (x + 0.0).view(torch.int32)                                          # (-0 and 0 are one value)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    key = (order << 32) + (v - 1 - torch.arange(v, device=x.device))
    return v - 1 - (torch.topk(key, k, dim=1).values & 0xFFFFFFFF)


def _plain_logprobs(s):
    x = s["logits"].float()
    m = x.amax(1, keepdim=True)
    d = x - m
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    log_s = torch.log(total)
    logprob = d.gather(1, s["targets"].unsqueeze(1)).squeeze(1) - log_s.squeeze(1)
    entropy = (log_s - torch.where(e > 0, d * e, torch.zeros_like(d)).sum(1, keepdim=True) / total).squeeze(1)
    token = _top(x, s["top"])
    top = d.gather(1, token) - log_s
    if s["select"] is not None:
        keep = s["select"]
        logprob, entropy = logprob * keep, entropy * keep
        top = torch.where(keep.unsqueeze(1), top, torch.zeros_like(top))
        token = torch.where(keep.unsqueeze(1), token, torch.full_like(token, -1))
    return logprob, entropy, top, token, d - log_s


def _plain_train(s):
    logprob, entropy, top, token, logp = _plain_logprobs(s)
    p = torch.exp(logp)
    weight = s["g_logprob"] + s["g_top"].sum(1)
    grad = -p * weight.unsqueeze(1)
    grad -= torch.where(p > 0, p * (logp + entropy.unsqueeze(1)), torch.zeros_like(p)) * s["g_entropy"].unsqueeze(1)
    grad.scatter_add_(1, s["targets"].unsqueeze(1), s["g_logprob"].unsqueeze(1))
    grad.scatter_add_(1, token.clamp(min=0), s["g_top"])
    if s["select"] is not None:
        grad = torch.where(s["select"].unsqueeze(1), grad, torch.zeros_like(grad))
    return logprob, entropy, top, token, grad.to(s["logits"].dtype)


def run(s):
    op = s["op"]
    if own:
        from evodiff_amd import ops
        if op == "quantize_rows":
            return tuple(ops.quantize_fp8(s["x"]))
        if op == "quantize_weight":
            return tuple(ops.quantize_fp8_weight(s["x"]))
        if op == "linear":
            return ops.linear_fp8(s["x"], ops.Fp8Weight(s["wq"], s["ws"]), s["b"], out_dtype=DTYPES[s["out"]])
        if op == "logprobs":
            return tuple(ops.token_logprobs(s["logits"], s["targets"], top_k=s["top"], select=s["select"]))
        logits = s["logits"].detach().requires_grad_()
        out = ops.token_logprobs(logits, s["targets"], top_k=s["top"], select=s["select"])
        grad, = torch.autograd.grad(out[:3], logits, (s["g_logprob"], s["g_entropy"], s["g_top"]))
        return tuple(t.detach() for t in out) + (grad,)
    if op in ("quantize_rows", "quantize_weight"):
        return _quantize(s["x"], op == "quantize_weight")
    if op == "linear":
        return _plain_linear(s)
    return _plain_logprobs(s)[:4] if op == "logprobs" else _plain_train(s)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    op, es = case["op"], SIZE[case["dtype"]]
    if op in ("quantize_rows", "quantize_weight"):
        m, k = case["m"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": m * k * es + m * kb * BLOCK + kb * (m if op == "quantize_rows" else -(-m // BLOCK)), "flops": 2.0 * m * k}
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        kb = -(-k // BLOCK)
        return {"bytes": m * k * es + n * kb * BLOCK + -(-n // BLOCK) * kb + m * n * SIZE[case["out"]] + 4 * n * case["bias"],
                "flops": 2.0 * m * n * k}
    rows, v, top = case["rows"], case["v"], case["top"]
    small = rows * (8 + 8 + 12 * top + case["skip"])
    if op == "logprobs":
        return {"bytes": rows * v * es + small, "flops": 6.0 * rows * v}
    return {"bytes": 2 * rows * v * es + small + rows * (8 + 4 * top), "flops": 14.0 * rows * v}


# ---- 64 bits, from the definitions -----------------------------------------------------------------------------------

def _power(s):
    """2^s in 64 bits, exactly (a power function on the GPU is not)."""
    return ((s.long() + 1023) << 52).view(torch.float64)


def _exact_scale(amax):
    """2^s, s the smallest whole number with amax <= 448 * 2^s, within [-126, 127]; -126 for an empty block."""
    mantissa, exponent = torch.frexp(amax / TOP)                                # amax / 448 = mantissa * 2^exponent, [1/2, 1)
    s = torch.where(mantissa == 0.5, exponent - 1, exponent)
    s = torch.where(amax > 0, s, torch.full_like(s, -126)).clamp(-126, 127)
    return _power(s)


def _exact_quantize(x, square):
    m, k = x.shape
    kb = -(-k // BLOCK)
    full = torch.zeros((-(-m // BLOCK) * BLOCK if square else m, kb * BLOCK), dtype=torch.float64, device=x.device)
    full[:m, :k] = x.double()
    tile = full.view(-1, BLOCK if square else 1, kb, BLOCK)
    scale = _exact_scale(tile.abs().amax((1, 3)))                               # (row blocks, kb)
    y = tile / scale[:, None, :, None]
    step = _power((torch.frexp(y.abs())[1] - 4).clamp(min=-9))   # 3 bits behind the leading one
    q = (torch.round(y / step) * step).view(full.shape)[:m]
    return q, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op in ("quantize_rows", "quantize_weight"):
        return _exact_quantize(s["x"], op == "quantize_weight")
    if op == "linear":
        q, scale = _exact_quantize(s["x"], False)
        x = q * scale.repeat_interleave(BLOCK, 1)
        scale = _power(s["ws"].view(torch.uint8).int() - 127)
        w = s["wq"].double() * scale.repeat_interleave(BLOCK, 0)[:case["n"]].repeat_interleave(BLOCK, 1)
        y = torch.mm(x, w.t().contiguous())
        return y if s["b"] is None else y + s["b"].double()
    x = s["logits"].double()
    logp = x - torch.logsumexp(x, 1, keepdim=True)
    p = torch.exp(logp)
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    entropy = -plogp.sum(1)
    logprob = logp[torch.arange(len(x), device=x.device), s["targets"]]
    top = torch.topk(logp, case["top"], dim=1).values
    token = _top(s["logits"].float(), case["top"]) if op == "train" else None
    keep = s["select"] if s["select"] is not None else torch.ones(len(x), dtype=torch.bool, device=x.device)
    zero = torch.zeros((), dtype=torch.float64, device=x.device)
    shown = (torch.where(keep, logprob, zero), torch.where(keep, entropy, zero), torch.where(keep[:, None], top, zero), None)
    if op == "logprobs":
        return shown
    pull = torch.zeros_like(p)                                                  # d loss / d log p, then through log softmax
    pull.scatter_add_(1, s["targets"][:, None], s["g_logprob"].double()[:, None])
    pull.scatter_add_(1, token, s["g_top"].double())
    grad = pull - p * pull.sum(1, keepdim=True) - s["g_entropy"].double()[:, None] * (plogp + p * entropy[:, None])
    return shown + (torch.where(keep[:, None], grad, zero),)
