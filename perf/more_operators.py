"""The operators of a cache in 8 bits, and the choice of a token from the nucleus of its distribution, at the sizes at which the engine runs
them: the dense decoder's layers at the benchmark's sizes, from one token to long contexts.

``write``   q, k and v of tokens take their bias and their position's rotation; q leaves in bfloat16, k and v go to their slots of the cache
            in 8 bits with a scale to each row
``decode``  attention of single tokens over the keys and values of such a cache
``chunk``   attention of portions of several requests' tokens over such a cache, causal
``sample``  a token by temperature, top-k, top-p and min-p from a given number in [0, 1)

A number in 8 bits is a float8_e4m3fn; a scale is a power of two (float8_e8m0fnu): the smallest with which the row's largest magnitude stays
within 448.  A page of ``page_size`` tokens is a row of bytes: the keys [kv heads, page_size, d], the values likewise, then the scales
[kv heads, page_size, 2] of key and value.
"""
import math

import torch

own = False
DEVICE = "cuda:0"
MODELS = {"05b": (14, 2, 64), "3b": (16, 2, 128), "7b": (28, 4, 128), "32b": (40, 8, 128)}      # query heads, kv heads, head size


def attention(name, op, heads, tokens, before, page=16, window=0):
    """``tokens``: new tokens of each request, ``before``: tokens cached ahead of them; texts of numbers with commas."""
    return {"name": name, "op": op, "H": heads[0], "G": heads[1], "d": heads[2], "tokens": ",".join(map(str, tokens)),
            "before": ",".join(map(str, before)), "page": page, "window": window}


def write(name, heads, tokens, parts=0, bias=True, pairing="half", rotary=0, page=16):
    """``parts``: q, k and v as so many float32 partial sums, 0: whole in bfloat16; ``rotary``: features of a head that turn, 0: all."""
    return {"name": name, "op": "write", "H": heads[0], "G": heads[1], "d": heads[2], "tokens": str(tokens), "parts": parts, "bias": bias,
            "pairing": pairing, "rotary": rotary or heads[2], "page": page}


def sample(name, rows, vocabulary, top_k=0, top_p=1.0, min_p=0.0, temperature=0.8, mixed=False):
    """``mixed``: every row has settings of its own around these."""
    return {"name": name, "op": "sample", "rows": rows, "V": vocabulary, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "temperature": temperature, "mixed": mixed}


def listed():
    ragged = [500 + (i * 1531) % 3500 for i in range(23)]
    return [
        # one person's next token
        write("write_3b_1", MODELS["3b"], 1, parts=4),
        # a server's decode step
        write("write_7b_64", MODELS["7b"], 64, bias=False),
        # a document in one step
        write("write_7b_2048", MODELS["7b"], 2048),
        # one person's next token behind a page of text, and behind a book
        attention("decode_3b_1", "decode", MODELS["3b"], [1], [2047]),
        attention("decode_7b_1_long", "decode", MODELS["7b"], [1], [100000]),
        # requests of many lengths, and a full server of long ones
        attention("decode_7b_23_ragged", "decode", MODELS["7b"], [1] * 23, ragged),
        attention("decode_7b_64", "decode", MODELS["7b"], [1] * 64, [8191] * 64),
        # three prompts that share a step
        attention("chunk_3b_512_of_3", "chunk", MODELS["3b"], [201, 140, 171], [0, 655, 333]),
        # a short question about a long document
        attention("chunk_7b_37_long", "chunk", MODELS["7b"], [37], [32000]),
        # a portion of a long document
        attention("chunk_7b_2048", "chunk", MODELS["7b"], [2048], [6144]),
        # one person's token, a server's
        sample("sample_3b_1", 1, 151936, top_p=0.9),
        sample("sample_7b_64", 64, 152064, top_k=50, top_p=0.95, min_p=0.02, mixed=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    """Another case of these ranges: heads of the models or any others, ragged requests, rows with settings of their own."""
    op = rng.choice(["write", "decode", "decode", "chunk", "chunk", "sample"])
    if rng.random() < 0.6:
        heads = MODELS[rng.choice(sorted(MODELS))]
    else:
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = (kv * rng.randint(1, 16), kv, rng.choice([64, 128]))
    page = rng.choice([16, 16, 16, 32, 64])
    if op == "write":
        c = write("", heads, _log(rng, 1, 2000), rng.choice([0, 0, 1, 2, 4]), rng.random() < 0.7, rng.choice(["half", "adjacent"]),
                  rng.choice([0, 0, heads[2] // 2]), page)
        if c["parts"] > 1:
            c["tokens"] = str(min(int(c["tokens"]), 128))
    elif op == "decode":
        n, most = _log(rng, 1, 128), _log(rng, 40, 8000)
        if n <= 4:
            most = _log(rng, 40, 60000)
        even = rng.random() < 0.3
        c = attention("", op, heads, [1] * n, [most if even else _log(rng, 1, most) for _ in range(n)], page,
                      rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    elif op == "chunk":
        n = rng.choice([1, 1, 2, 3, 5, 8])
        tokens = [_log(rng, 1, 2000 // n) for _ in range(n)]
        most = max(1, min(30000, int(1.5e8 / (n * max(tokens) * heads[0]))))
        c = attention("", op, heads, tokens, [rng.choice([0, _log(rng, 1, most)]) for _ in range(n)], page, rng.choice([0, 0, 0, _log(rng, 16, 4096)]))
    else:
        c = sample("", _log(rng, 1, 64), rng.choice([151936, 152064, 32000, _log(rng, 1000, 150000)]), rng.choice([0, 0, 1, 20, 50, 1500]),
                   rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]), rng.choice([0.0, 0.0, 0.02, 0.1]), rng.choice([0.3, 0.7, 1.0, 1.5]), rng.random() < 0.5)
        if c["top_p"] == 1.0 and c["min_p"] == 0.0:
            c["min_p"] = 0.05
    del c["name"]
    return c


# ---- what a user's program holds ----------------------------------------------------------------------------------

def _numbers(gen, shape, std):
    return torch.empty(shape, dtype=torch.float32, device=DEVICE).normal_(0.0, std, generator=gen)


def _int(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _lists(case):
    tokens = [int(t) for t in case["tokens"].split(",")]
    return tokens, [int(t) for t in case["before"].split(",")]


def _split(pages, G, ps, d):
    """The numbers [pages, 2, G, ps, d] and the scales [pages, G, ps, 2] of rows of bytes."""
    n = 2 * G * ps * d
    return (pages[:, :n].view(torch.float8_e4m3fn).view(-1, 2, G, ps, d), pages[:, n:].view(torch.float8_e8m0fnu).view(-1, G, ps, 2))


def _pool(gen, n, G, ps, d):
    """Pages as a model's earlier steps left them: keys with some large features, values of changing size."""
    pages = torch.zeros((n, G * ps * (2 * d + 2)), dtype=torch.uint8, device=DEVICE)
    q, s = _split(pages, G, ps, d)
    offset = _numbers(gen, (G, 1, d), 1.0) * (1.0 + 4.0 * (torch.rand((G, 1, d), generator=gen, device=DEVICE) < 0.03))
    step = max(1, (1 << 26) // (G * ps * d))
    for i in range(0, n, step):
        m = min(step, n - i)
        rows = torch.stack([_numbers(gen, (m, G, ps, d), 1.0) + offset,
                            _numbers(gen, (m, G, ps, d), 0.5) * torch.exp2(_numbers(gen, (m, G, ps, 1), 0.7))], 1)
        q8, e = _to8(rows)
        q[i:i + m] = q8
        s[i:i + m] = e.permute(0, 2, 3, 1).view(torch.float8_e8m0fnu)
    return pages


def _tables(rotary, positions):
    """cos and sin as the engine makes them: angles in 64 bits, tables in 32."""
    inv = 1000000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=DEVICE) / rotary)
    angle = torch.arange(positions, dtype=torch.float64, device=DEVICE).unsqueeze(1) * inv
    return torch.cos(angle).float(), torch.sin(angle).float()


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    st = {"case": case}
    if case["op"] == "sample":
        R, V = case["rows"], case["V"]
        z = _numbers(gen, (R, V), 2.5)
        z[:, 0] = 0.0
        around = (torch.rand((4, R), generator=gen, device=DEVICE) if case["mixed"] else torch.full((4, R), 0.5, device=DEVICE))
        st["logits"] = z
        st["temperature"] = case["temperature"] * (0.5 + around[0])
        st["top_k"] = (case["top_k"] * 2 * around[1]).ceil().to(torch.int32)
        st["top_p"] = (case["top_p"] + (1.0 - case["top_p"]) * (around[2] - 0.5)).clamp(max=1.0)
        st["min_p"] = case["min_p"] * 2 * around[3]
        st["draws"] = torch.rand(R, generator=gen, device=DEVICE)
        return st
    H, G, d, ps = case["H"], case["G"], case["d"], case["page"]
    if case["op"] == "write":
        T, W = int(case["tokens"]), (H + 2 * G) * d
        st["qkv"] = _numbers(gen, (case["parts"], T, W), case["parts"] ** -0.5) if case["parts"] else _numbers(gen, (T, W), 1.0).bfloat16()
        st["bias"] = _numbers(gen, (W,), 1.0) * (1.0 + 10.0 * (torch.rand(W, generator=gen, device=DEVICE) < 0.02)) if case["bias"] else None
        st["cos"], st["sin"] = _tables(case["rotary"], 32768)
        st["positions"] = torch.randint(0, 32768, (T,), generator=gen, device=DEVICE, dtype=torch.int32)
        n = -(-T // ps) + 2
        st["pages"] = _pool(gen, n, G, ps, d)
        st["slots"] = torch.randperm(n * ps, generator=gen, device=DEVICE)[:T].to(torch.int32)
        return st
    tokens, before = _lists(case)
    blocks = [-(-(b + t) // ps) for t, b in zip(tokens, before)]
    order = torch.randperm(sum(blocks) + 3, generator=gen, device=DEVICE).to(torch.int32)
    table, at = torch.full((len(tokens), max(blocks)), -1, dtype=torch.int32, device=DEVICE), 0
    for r, b in enumerate(blocks):
        table[r, :b] = order[at:at + b]
        at += b
    st["pages"], st["table"] = _pool(gen, sum(blocks) + 3, G, ps, d), table
    st["q"] = _numbers(gen, (sum(tokens), H * d), 1.0).bfloat16()
    st["start"] = _int(before)
    st["cu"] = _int([0] + tokens).cumsum(0).to(torch.int32)
    st["request"] = torch.repeat_interleave(torch.arange(len(tokens), device=DEVICE, dtype=torch.int32), _int(tokens).long())
    st["positions"] = st["start"][st["request"].long()] + torch.arange(sum(tokens), device=DEVICE, dtype=torch.int32) - st["cu"][st["request"].long()]
    st["longest"] = max(b + t for t, b in zip(tokens, before))
    return st


# ---- the plain forms ----------------------------------------------------------------------------------------------

def _to8(y):
    """Rows (the last dimension) in 8 bits, and the bytes of their scales: 448 = 1.75 * 2^8."""
    m, e = torch.frexp(y.abs().amax(-1))
    e = torch.where(m == 0, torch.zeros_like(e), (e - 9 + (m > 0.875)).clamp(-126, 127))
    return torch.ldexp(y, -e.unsqueeze(-1)).float().to(torch.float8_e4m3fn), (e + 127).to(torch.uint8)


def _turn(x, cos, sin, rotary, half):
    """Rows [T, heads, d], their first ``rotary`` features turned by angles [T, rotary / 2]: pairs (p, p + rotary / 2), or neighbours."""
    cos, sin = cos.unsqueeze(1), sin.unsqueeze(1)
    r = x[..., :rotary]
    a, b = (r[..., :rotary // 2], r[..., rotary // 2:]) if half else (r[..., ::2], r[..., 1::2])
    pair = a * cos - b * sin, a * sin + b * cos
    r = torch.cat(pair, -1) if half else torch.stack(pair, -1).flatten(-2)
    return torch.cat([r, x[..., rotary:]], -1)


def _plain_write(st):
    c = st["case"]
    H, G, d, ps = c["H"], c["G"], c["d"], c["page"]
    x = st["qkv"].double()                               # (64 bits: a scale changes where the largest magnitude is next to a border)
    x = x.sum(0) if c["parts"] else x
    if st["bias"] is not None:
        x = x + st["bias"]
    x = x.view(-1, H + 2 * G, d)
    at = st["positions"].long()
    turned = _turn(x[:, :H + G], st["cos"][at].double(), st["sin"][at].double(), c["rotary"], c["pairing"] == "half")
    q8, e = _to8(torch.stack([turned[:, H:], x[:, H + G:]], 1))
    numbers, scales = _split(st["pages"], G, ps, d)
    page, offset = st["slots"].long() // ps, st["slots"].long() % ps
    numbers.view(torch.uint8).permute(0, 3, 1, 2, 4)[page, offset] = q8.view(torch.uint8)
    scales.view(torch.uint8).transpose(1, 2)[page, offset] = e.transpose(1, 2)
    return turned[:, :H].flatten(1).bfloat16(), numbers, scales


def _keys_values(st):
    """float32 [requests, tokens, kv heads, d] each, through the block table."""
    c = st["case"]
    G, d, ps = c["G"], c["d"], c["page"]
    numbers, scales = _split(st["pages"][st["table"].clamp(min=0).long().flatten()], G, ps, d)
    byte = scales.view(torch.uint8).int()
    factor = torch.ldexp(torch.ones_like(byte, dtype=torch.float32), byte - 127)
    rows = numbers.float() * factor.permute(0, 3, 1, 2).unsqueeze(-1)
    rows = rows.view(len(st["table"]), -1, 2, G, ps, d).permute(2, 0, 1, 4, 3, 5)
    return rows.reshape(2, len(st["table"]), -1, G, d).unbind(0)


def _plain_attention(st):
    c = st["case"]
    H, G, d = c["H"], c["G"], c["d"]
    k, v = _keys_values(st)
    # every request's tokens in a row of their own, padded to the longest
    n = (st["cu"][1:] - st["cu"][:-1]).long()
    place = torch.arange(int(n.max()), device=DEVICE)
    flat = (st["cu"][:-1, None].long() + place).clamp(max=len(st["q"]) - 1)
    q = st["q"].float()[flat].view(len(n), -1, G, H // G, d)
    z = torch.einsum("rtghd,rlgd->rghtl", q, k) * d ** -0.5
    at = (st["start"][:, None] + place)[:, :, None]
    key = torch.arange(k.shape[1], device=DEVICE)
    seen = (key <= at) & (key > at - (c["window"] or k.shape[1] + 1))
    w = torch.exp(z - z.masked_fill(~seen[:, None, None], -math.inf).amax(-1, keepdim=True)) * seen[:, None, None]
    y = torch.einsum("rghtl,rlgd->rtghd", w / w.sum(-1, keepdim=True), v)
    return y.flatten(2)[(place < n[:, None])].bfloat16()


def _plain_sample(st):
    """In 64 bits: which token a number falls to changes where it is next to a border."""
    z, V = st["logits"].double(), st["logits"].shape[1]
    order = torch.sort(z, dim=1, descending=True).values
    w = torch.exp((z - order[:, :1]) / st["temperature"].double().unsqueeze(1))
    ranked = torch.exp((order - order[:, :1]) / st["temperature"].double().unsqueeze(1))
    k = st["top_k"].long()
    kth = order.gather(1, (torch.where((k > 0) & (k < V), k, torch.full_like(k, V)) - 1).unsqueeze(1))
    ranked = torch.where(order >= kth, ranked, torch.zeros_like(ranked))
    sums = torch.cumsum(ranked, 1)
    reached = sums >= st["top_p"].double().unsqueeze(1) * sums[:, -1:]
    last = order.gather(1, reached.int().argmax(1, keepdim=True))
    last = torch.where(st["top_p"].unsqueeze(1) < 1.0, torch.maximum(last, kth), kth)
    kept = torch.where((z >= last) & (w >= st["min_p"].double().unsqueeze(1)), w, torch.zeros_like(w))
    sums = torch.cumsum(kept, 1)
    hit = (sums >= st["draws"].double().unsqueeze(1) * sums[:, -1:]) & (kept > 0)
    return hit.int().argmax(1).to(torch.int32)


def _plain(st):
    return {"write": _plain_write, "decode": _plain_attention, "chunk": _plain_attention, "sample": _plain_sample}[st["case"]["op"]](st)


# ---- the framework's operators -------------------------------------------------------------------------------------

def _own(st):
    from qwen_decoder_b200 import kernels
    c = st["case"]
    if c["op"] == "sample":
        out = torch.empty(c["rows"], dtype=torch.int32, device=DEVICE)
        kernels.sample_nucleus(st["logits"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], st["draws"], out)
        return out
    H, G, d, ps = c["H"], c["G"], c["d"], c["page"]
    if c["op"] == "write":
        q = torch.empty((int(c["tokens"]), H * d), dtype=torch.bfloat16, device=DEVICE)
        kernels.rope_kv_write_fp8(st["qkv"], st["bias"], q, H, G, d, c["rotary"], 1 if c["pairing"] == "half" else 0, st["cos"], st["sin"],
                                  st["positions"], st["pages"], st["slots"], ps)
        return (q,) + tuple(kernels.fp8_page_views(st["pages"], G, ps, d))
    out = torch.empty_like(st["q"])
    if c["op"] == "decode":
        kernels.decode_attention_fp8(st["q"], out, st["pages"], st["table"], st["request"], st["positions"], H, G, d, ps, d ** -0.5,
                                     c["window"], st["longest"])
    else:
        kernels.prefill_attention_fp8(st["q"], out, st["pages"], st["table"], st["cu"], st["start"], H, G, d, ps, d ** -0.5, c["window"],
                                      st["longest"])
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---- what a pass cannot do without, and its results in 64 bits -----------------------------------------------------

def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (4 * case["V"] + 24), "flops": 4 * case["rows"] * case["V"]}
    H, G, d = case["H"], case["G"], case["d"]
    if case["op"] == "write":
        T, W = int(case["tokens"]), (H + 2 * G) * d
        return {"bytes": T * (W * (4 * case["parts"] or 2) + 2 * H * d + 2 * G * (d + 1) + 4 * case["rotary"] + 8) + (4 * W if case["bias"] else 0),
                "flops": T * (W * (case["parts"] + 1) + 3 * (H + G) * case["rotary"])}
    keys, pairs = 0, 0
    for t, b in zip(*_lists(case)):
        window = case["window"] or b + t
        keys += min(b + t, window + t - 1)
        pairs += sum(min(b + i + 1, window) for i in range(t))
    T = sum(_lists(case)[0])
    return {"bytes": keys * G * 2 * (d + 1) + 4 * T * H * d, "flops": 4 * pairs * H * d}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(st)
    H, G, d, ps = case["H"], case["G"], case["d"], case["page"]
    numbers, scales = _split(st["pages"], G, ps, d)
    numbers, scales = numbers.double(), torch.exp2(scales.view(torch.uint8).double() - 127)
    if case["op"] == "write":
        x = st["qkv"].double()
        x = x.sum(0) if case["parts"] else x
        x = (x + st["bias"] if st["bias"] is not None else x).view(-1, H + 2 * G, d)
        rot = case["rotary"]
        z = x[..., :rot]
        z = torch.complex(*((z[..., :rot // 2], z[..., rot // 2:]) if case["pairing"] == "half" else (z[..., 0::2], z[..., 1::2])))
        at = st["positions"].long()
        z = z * torch.complex(st["cos"][at].double(), st["sin"][at].double()).unsqueeze(1)
        y = x.clone()
        if case["pairing"] == "half":
            y[..., :rot // 2], y[..., rot // 2:rot] = z.real, z.imag
        else:
            y[..., 0:rot:2], y[..., 1:rot:2] = z.real, z.imag
        y[:, H + G:] = x[:, H + G:]
        peak = y[:, H:].abs().max(-1).values
        scale = torch.exp2(torch.ceil(torch.log2(peak / 448.0)))
        scale = torch.where(peak > 448.0 * scale, 2.0 * scale, torch.where(peak <= 224.0 * scale, 0.5 * scale, scale))      # a logarithm rounded across
        for t, slot in enumerate(st["slots"].tolist()):
            numbers[slot // ps, :, :, slot % ps] = (y[t, H:] / scale[t, :, None]).view(2, G, d)
            scales[slot // ps, :, slot % ps] = scale[t].view(2, G).t()
        return y[:, :H].flatten(1), numbers, scales
    numbers *= scales.permute(0, 3, 1, 2).unsqueeze(-1)
    out = torch.empty((len(st["q"]), H, d), dtype=torch.float64, device=DEVICE)
    at = 0
    for r, (t, b) in enumerate(zip(*_lists(case))):
        rows = numbers[st["table"][r].clamp(min=0).long()].permute(1, 2, 0, 3, 4).reshape(2, G, -1, d)[:, :, :b + t]
        for i in range(0, t, 128):
            n = min(128, t - i)
            q = st["q"][at + i:at + i + n].double().view(n, G, H // G, d).permute(1, 2, 0, 3).reshape(G, -1, d)
            z = (q @ rows[0].transpose(1, 2) / math.sqrt(d)).view(G, H // G, n, b + t)
            pos = torch.arange(b + i, b + i + n, device=DEVICE).unsqueeze(1)
            key = torch.arange(b + t, device=DEVICE)
            hidden = key > pos
            if case["window"]:
                hidden |= key <= pos - case["window"]
            p = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
            out[at + i:at + i + n] = (p.view(G, -1, b + t) @ rows[1]).view(G, H // G, n, d).permute(2, 0, 1, 3).reshape(n, H, d)
        at += t
    return out.flatten(1)


def _exact_sample(st):
    """Row by row, candidates in their order."""
    found = []
    for r in range(len(st["logits"])):
        z = st["logits"][r].double()
        p = torch.softmax((z - z.max()) / st["temperature"][r].double(), 0)
        k, V = int(st["top_k"][r]), len(z)
        rank = torch.argsort(z, descending=True, stable=True)
        n = k if 0 < k < V else V
        n = int((z >= z[rank[n - 1]]).sum())
        if float(st["top_p"][r]) < 1.0:
            mass = torch.cumsum(p[rank[:n]], 0)
            n = int((mass < st["top_p"][r].double() * mass[-1]).sum()) + 1
        keep = (z >= z[rank[n - 1]]) & (p >= st["min_p"][r].double() * p.max())
        ids = torch.nonzero(keep)[:, 0]
        mass = torch.cumsum(p[ids], 0)
        found.append(int(ids[min(int((mass < st["draws"][r].double() * mass[-1]).sum()), len(ids) - 1)]))
    return _int(found)
