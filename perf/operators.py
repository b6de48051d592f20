"""The operators of projections in 8 bits and of the probabilities that a model gives to tokens, at the sizes at which the engine runs
them: the dense decoder's layers at the benchmark's 3B and 7B sizes, from one token to a whole prompt.

``norm``      the residual sum takes a branch's output, and its RMS norm leaves in 8 bits with a scale to each 128 features
``quantize``  rows (attention's output) into the same form
``product``   rows in 8 bits times a matrix in 8 bits, both with a scale to each 128 of k
``gated``     the gate's and the up product with their activation, into 8 bits for the product that follows
``logprobs``  of each row of logits: the log probability of a given token, the distribution's entropy, the most probable tokens

A number in 8 bits is a float8_e4m3fn; a scale is a power of two (float8_e8m0fnu): the smallest with which the block's largest magnitude
stays within 448.  Tensors of 8-bit rows: ``q`` [R, K] with rows of whole 16 bytes, ``s`` [R, ceil(K / 128)] with rows of whole 4 bytes.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
BLOCK = 128
EPS = 1e-6


def case(name, op, rows, k, n=0, parts=0, dtype="bfloat16", bias=False, act="silu", top=0, masked=False):
    """``k``: features of a row (the vocabulary for logprobs); ``n``: features of the result; ``parts``: a branch's output as so many
    float32 partial sums, 0: whole in bfloat16; ``dtype``: of the input of quantize and logprobs, of the result of product."""
    return {"name": name, "op": op, "rows": rows, "k": k, "n": n, "parts": parts, "dtype": dtype, "bias": bias, "act": act, "top": top,
            "masked": masked}


def listed():
    return [
        # one person's next token: the norm before a layer's products, on the attention product's partial sums
        case("norm_3b_1", "norm", 1, 2048, parts=4),
        # a document in one step
        case("norm_7b_2048", "norm", 2048, 3584),
        # attention's output of a server's decode step, and of a prompt
        case("quantize_7b_23", "quantize", 23, 3584),
        case("quantize_3b_2048", "quantize", 2048, 2048),
        # one token's down projection: all latency and bandwidth
        case("down_3b_1", "product", 1, 11008, 2048),
        # queries, keys and values of 23 requests decoding together
        case("qkv_7b_23", "product", 23, 3584, 4608, bias=True),
        # a full server's logits
        case("vocabulary_7b_64", "product", 64, 3584, 152064, dtype="float32"),
        # a prompt's down projection
        case("down_7b_2048", "product", 2048, 18944, 3584),
        # the feed-forward's first half of 8 requests, and of a prompt: the largest product of a layer
        case("gated_3b_8", "gated", 8, 2048, 11008),
        case("gated_7b_2048", "gated", 2048, 3584, 18944),
        # what a few users' tokens are shown with; a prompt scored token by token
        case("logprobs_3b_8", "logprobs", 8, 151936, dtype="float32", top=5),
        case("logprobs_7b_509", "logprobs", 509, 152064, dtype="float32", top=20),
    ]


def _log(rng, lo, hi):
    n = max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))
    return n + 1 if n == 3072 else n


def draw(rng):
    """Another case of these ranges: widths of the two models or any others, odd ones too."""
    op = rng.choice(["norm", "quantize", "product", "product", "product", "gated", "gated", "logprobs"])
    width = rng.choice([2048, 3584, _log(rng, 64, 4096), 8 * _log(rng, 16, 500) + 8])
    if op == "norm":
        c = case("", op, _log(rng, 1, 2048), width, parts=rng.choice([0, 0, 1, 2, 3, 5, 8]))
        if c["parts"]:
            c["rows"] = min(c["rows"], 256)
    elif op == "quantize":
        c = case("", op, _log(rng, 1, 2048), rng.choice([width, _log(rng, 64, 8192)]), dtype=rng.choice(["bfloat16", "bfloat16", "float32"]))
    elif op == "product":
        k, n = rng.choice([(2048, 2560), (2048, 2048), (11008, 2048), (3584, 4608), (3584, 3584), (18944, 3584), (width, _log(rng, 64, 20000)),
                           (_log(rng, 64, 12000), width)])
        c = case("", op, _log(rng, 1, 2048), k, n, dtype=rng.choice(["bfloat16", "bfloat16", "float32"]), bias=rng.random() < 0.3)
    elif op == "gated":
        k, n = rng.choice([(2048, 11008), (3584, 18944), (width, _log(rng, 64, 9000))])
        c = case("", op, _log(rng, 1, 1800), k, n, act=rng.choice(["silu", "silu", "gelu_tanh"]), bias=rng.random() < 0.2)
    else:
        c = case("", op, _log(rng, 1, 400), rng.choice([151936, 152064, 32000, _log(rng, 1000, 150000)]),
                 dtype=rng.choice(["float32", "float32", "bfloat16"]), top=rng.choice([0, 1, 5, 20]), masked=rng.random() < 0.3)
    del c["name"]
    return c


# ---- what a user's program holds ----------------------------------------------------------------------------------

def _numbers(gen, shape, std):
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=gen)


def _rows8(x):
    """Rows in 8 bits as a program keeps them: (q, s), rows of whole 16 and of whole 4 bytes."""
    R, K = x.shape
    q, s = _to8(x)
    q8 = torch.zeros((R, -(-K // 16) * 16), dtype=torch.float8_e4m3fn, device=DEVICE)[:, :K]
    s8 = torch.zeros((R, -(-s.shape[1] // 4) * 4), dtype=torch.uint8, device=DEVICE)[:, :s.shape[1]]
    q8.copy_(q)
    s8.copy_(s.view(torch.uint8))
    return q8, s8.view(torch.float8_e8m0fnu)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    R, K, N, op = case["rows"], case["k"], case["n"], case["op"]
    st = {"case": case}
    if op == "norm":
        # a residual sum as it is some layers deep: a few features are much larger than the others
        big = 1.0 + 20.0 * (torch.rand(K, generator=gen, device=DEVICE) < 0.01)
        st["x"] = _numbers(gen, (R, K), 1.0) * big
        st["delta"] = _numbers(gen, (case["parts"], R, K), 0.1) if case["parts"] else _numbers(gen, (R, K), 0.1).bfloat16()
        st["weight"] = 1.0 + _numbers(gen, (K,), 0.1)
    elif op == "quantize":
        st["x"] = _numbers(gen, (R, K), 0.5).to(getattr(torch, case["dtype"]))
    elif op in ("product", "gated"):
        rows = 2 * N if op == "gated" else N
        st["x"] = _rows8(_numbers(gen, (R, K), 1.0))
        st["w"] = tuple(torch.empty_strided((rows, t.shape[1]), t.stride(), dtype=t.dtype, device=DEVICE) for t in _rows8(_numbers(gen, (1, K), 1.0)))
        step = max(1, (1 << 27) // K)
        for i in range(0, rows, step):                   # a piece at a time: the vocabulary's matrix is two gigabytes in 32 bits
            q, s = _rows8(_numbers(gen, (min(step, rows - i), K), K ** -0.5))
            st["w"][0][i:i + step].copy_(q)
            st["w"][1].view(torch.uint8)[i:i + step].copy_(s.view(torch.uint8))
        st["bias"] = _numbers(gen, (rows,), 0.1) if case["bias"] else None
    else:
        z = _numbers(gen, (R, K), 2.5)
        if case["masked"]:                               # a grammar that leaves a tenth of the vocabulary
            z = torch.where(torch.rand(K, generator=gen, device=DEVICE) < 0.9, torch.full_like(z, -math.inf), z)
        z[:, 0] = 0.0
        st["logits"] = z.to(getattr(torch, case["dtype"]))
        # tokens as a sampler finds them: more likely ones more often
        u = torch.rand((R, 8), generator=gen, device=DEVICE)
        near = (u * K).long().clamp_(max=K - 1)
        best = near.gather(1, st["logits"].float().gather(1, near).argmax(1, keepdim=True))
        st["tokens"] = best[:, 0].to(torch.int32)
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _blocks(y):
    """[R, K] -> [R, ceil(K / 128), 128], zeros behind the end."""
    R, K = y.shape
    n = -(-K // BLOCK)
    return torch.nn.functional.pad(y, (0, n * BLOCK - K)).view(R, n, BLOCK)


def _exponent(y):
    """The exponents of the scales of [R, n, 128]: 448 = 1.75 * 2^8."""
    m, e = torch.frexp(y.abs().amax(2))
    return torch.where(m == 0, torch.zeros_like(e), (e - 9 + (m > 0.875)).clamp(-126, 127))


def _to8(y):
    b = _blocks(y)
    e = _exponent(b)
    q = torch.ldexp(b, -e.unsqueeze(2)).view(y.shape[0], -1)[:, :y.shape[1]].to(torch.float8_e4m3fn)
    return q, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _from8(rows, dtype):
    q, s = rows
    factor = torch.ldexp(torch.ones((), dtype=dtype, device=q.device), s.view(torch.uint8).int() - 127)
    return (_blocks(q.to(dtype)) * factor.unsqueeze(2)).view(q.shape[0], -1)[:, :q.shape[1]]


def _act(g, u, act):
    if act == "gelu_tanh":
        return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g))) * u
    return g / (1.0 + torch.exp(-g)) * u


def _log_probabilities(z, tokens, top):
    m = z.amax(1, keepdim=True)
    w = torch.exp(z - m)
    total = w.sum(1, keepdim=True)
    log_total = torch.log(total)
    shifted = torch.where(w > 0, z - m, torch.zeros_like(z))
    entropy = log_total[:, 0] - (w * shifted).sum(1) / total[:, 0]
    of_token = (z.gather(1, tokens.long().unsqueeze(1)) - m - log_total)[:, 0]
    # the largest first, of equal ones the lowest index: both in one 64-bit key
    V = z.shape[1]
    bits = (z.float() + 0.0).contiguous().view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    keys = order * (1 << 20) + (V - 1 - torch.arange(V, device=z.device))
    ids = V - 1 - (torch.topk(keys, top, dim=1).values & ((1 << 20) - 1))
    return of_token, entropy, ids.to(torch.int32), z.gather(1, ids) - m - log_total


def _plain(st):
    c = st["case"]
    if c["op"] == "norm":
        d = st["delta"].float()
        st["x"] = st["x"] + (d.sum(0) if c["parts"] else d)
        x = st["x"]
        y = x * (1.0 / torch.sqrt((x * x).mean(1, keepdim=True) + EPS)) * st["weight"]
        return (x,) + _to8(y)
    if c["op"] == "quantize":
        return _to8(st["x"].float())
    if c["op"] == "logprobs":
        return _log_probabilities(st["logits"].float(), st["tokens"], c["top"])
    y = torch.matmul(_from8(st["x"], torch.float32), _from8(st["w"], torch.float32).t())
    if st["bias"] is not None:
        y = y + st["bias"]
    if c["op"] == "product":
        return y.to(getattr(torch, c["dtype"]))
    return _to8(_act(y[:, :c["n"]], y[:, c["n"]:], c["act"]))


# ---- the framework's operators -------------------------------------------------------------------------------------

def _own(st):
    from qwen_decoder_b200 import kernels
    c = st["case"]
    R, K, N, op = c["rows"], c["k"], c["n"], c["op"]
    if op == "norm":
        out = kernels.fp8_rows(R, K, DEVICE)
        kernels.add_rmsnorm_fp8(st["x"], st["delta"], st["weight"], out, EPS)
        return st["x"], out.q, out.s
    if op == "quantize":
        out = kernels.fp8_rows(R, K, DEVICE)
        kernels.quantize_fp8(st["x"], out)
        return out.q, out.s
    if op == "product":
        out = torch.empty((R, N), dtype=getattr(torch, c["dtype"]), device=DEVICE)
        kernels.gemm_fp8(kernels.Fp8Rows(*st["x"]), kernels.Fp8Rows(*st["w"]), st["bias"], out)
        return out
    if op == "gated":
        out = kernels.fp8_rows(R, N, DEVICE)
        kernels.gemm_fp8_gated(kernels.Fp8Rows(*st["x"]), kernels.Fp8Rows(*st["w"]), st["bias"], out,
                               kernels.ACT_GATED_GELU if c["act"] == "gelu_tanh" else kernels.ACT_SILU)
        return out.q, out.s
    return tuple(kernels.token_logprobs(st["logits"], st["tokens"], c["top"]))


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without, and its results in 64 bits -----------------------------------------------------

def work(case):
    R, K, N, op = case["rows"], case["k"], case["n"], case["op"]
    size = 4 if case["dtype"] == "float32" else 2
    rows8 = lambda r, k: r * (k + -(-k // BLOCK))        # noqa: E731
    if op == "norm":
        return {"bytes": R * K * (8 + (4 * case["parts"] or 2)) + 4 * K + rows8(R, K), "flops": R * K * (8 + case["parts"])}
    if op == "quantize":
        return {"bytes": R * K * size + rows8(R, K), "flops": 3 * R * K}
    if op == "logprobs":
        return {"bytes": R * (K * size + 4 + 8 + 8 * case["top"]), "flops": 6 * R * K}
    if op == "product":
        return {"bytes": rows8(R, K) + rows8(N, K) + R * N * size + (4 * N if case["bias"] else 0), "flops": 2 * R * N * K}
    return {"bytes": rows8(R, K) + rows8(2 * N, K) + rows8(R, N) + (8 * N if case["bias"] else 0), "flops": 4 * R * N * K}


def _exact8(y):
    """What rows in 8 bits stand for, before the rounding to 8 bits: y over its block's scale, and the scales."""
    R, K = y.shape
    b = torch.zeros((R, -(-K // BLOCK) * BLOCK), dtype=torch.float64, device=y.device)
    b[:, :K] = y
    b = b.view(R, -1, BLOCK)
    peak = b.abs().max(2).values
    scale = torch.exp2(torch.ceil(torch.log2(peak / 448.0)))
    scale = torch.where(peak > 448.0 * scale, 2.0 * scale, torch.where(peak <= 224.0 * scale, 0.5 * scale, scale))   # a logarithm rounded across
    scale = torch.where(peak == 0, torch.ones_like(scale), scale)
    return (b / scale.unsqueeze(2)).view(R, -1)[:, :K], scale


def exact(case, seed):
    st = prepare(case, seed)
    R, K, N, op = case["rows"], case["k"], case["n"], case["op"]
    if op == "norm":
        d = st["delta"].double()
        x = st["x"].double() + (d.sum(0) if case["parts"] else d)
        return (x,) + _exact8(x * torch.rsqrt(x.square().mean(1, keepdim=True) + EPS) * st["weight"].double())
    if op == "quantize":
        return _exact8(st["x"].double())
    if op == "logprobs":
        z = st["logits"].double()
        lp = z - torch.logsumexp(z, 1, keepdim=True)
        p = torch.exp(lp)
        entropy = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1)
        top = torch.sort(lp, dim=1, descending=True, stable=True).values[:, :case["top"]]
        return lp.gather(1, st["tokens"].long().unsqueeze(1))[:, 0], entropy, None, top
    scales = [t.view(torch.uint8).double().sub(127).exp2().repeat_interleave(BLOCK, 1)[:, :K] for t in (st["x"][1], st["w"][1])]
    x, rows = st["x"][0].double() * scales[0], st["w"][0].shape[0]
    y = torch.empty((R, rows), dtype=torch.float64, device=DEVICE)
    for i in range(0, rows, 16384):
        y[:, i:i + 16384] = x @ (st["w"][0][i:i + 16384].double() * scales[1][i:i + 16384]).t()
    if st["bias"] is not None:
        y += st["bias"].double()
    if op == "product":
        return y
    g, u = y[:, :N], y[:, N:]
    if case["act"] == "gelu_tanh":
        h = g * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (g + 0.044715 * g ** 3)) * u
    else:
        h = g * torch.sigmoid(g) * u
    return _exact8(h)
