"""A cache in 8 bits, the attention over it and the choice of a token, in float64 from their formulas, with bounds on what the kernels' roundings
may be off by."""
import math

import torch

E4M3_HALF_STEP, BF16_HALF_STEP, FP16_HALF_STEP, FP32_HALF_STEP = 2.0 ** -4, 2.0 ** -8, 2.0 ** -11, 2.0 ** -24


def powers(scales):
    """float8_e8m0fnu -> float64; the byte 255 is no number."""
    b = scales.view(torch.uint8).to(torch.float64)
    return torch.where(b == 255, torch.full_like(b, math.nan), torch.exp2(b - 127))


def scale_of(rows):
    """The smallest power of two with which the largest magnitude of each row stays within 448; 1 for zeros."""
    peak = rows.abs().amax(-1)
    m, e = torch.frexp(peak)
    e = torch.where(m > 0.875, e - 8, e - 9).clamp(-126, 127)
    return torch.where(peak == 0, torch.ones_like(peak), torch.exp2(e.to(torch.float64)))


def filled_pages(gen, n, G, ps, d, spread=1.0):
    """A pool of pages with random rows whose sizes differ by powers of two."""
    from qwen_decoder_b200 import kernels
    pages = torch.zeros((n, kernels.fp8_page_bytes(G, ps, d)), dtype=torch.uint8)
    numbers, scales = kernels.fp8_page_views(pages, G, ps, d)
    rows = torch.randn((n, 2, G, ps, d), generator=gen, dtype=torch.float64) * torch.exp2(spread * torch.randn((n, 2, G, ps, 1), generator=gen, dtype=torch.float64))
    s = scale_of(rows)
    numbers.copy_((rows / s.unsqueeze(-1)).float().to(torch.float8_e4m3fn))
    scales.view(torch.uint8).copy_((torch.log2(s) + 127).to(torch.uint8).permute(0, 2, 3, 1))
    return pages


def page_rows(pages, G, ps, d):
    """float64 [n, 2, G, ps, d]."""
    from qwen_decoder_b200 import kernels
    numbers, scales = kernels.fp8_page_views(pages, G, ps, d)
    return numbers.to(torch.float32).to(torch.float64) * powers(scales).permute(0, 3, 1, 2).unsqueeze(-1)


def attention(q, pages, table, reqs, positions, H, G, d, ps, scale, window, weight_half_step):
    """(out float64 [T, H d], bound): rows of tokens that see nothing are zeros.  ``weight_half_step``: of the number a weight is rounded to."""
    rows = page_rows(pages, G, ps, d)
    out, bound = torch.zeros((len(q), H, d), dtype=torch.float64), torch.zeros((len(q), H, d), dtype=torch.float64)
    for t, (r, pos) in enumerate(zip(reqs, positions)):
        if pos < 0:
            continue
        lo = max(0, pos - window + 1) if window else 0
        blocks = table[r, lo // ps:pos // ps + 1].long()
        kv = rows[blocks].permute(1, 2, 0, 3, 4).reshape(2, G, -1, d)[:, :, lo % ps:lo % ps + pos - lo + 1]
        k, v = kv.repeat_interleave(H // G, 1)
        x = q[t].to(torch.float64).view(H, 1, d)
        z = (x * k).sum(-1) * scale
        # a score in float32: the sum's terms, and a few products behind it
        off = (d + 8) * FP32_HALF_STEP * ((x * k).abs().sum(-1) * abs(scale)).amax(-1, keepdim=True)
        p = torch.softmax(z, -1)
        out[t] = (p.unsqueeze(-1) * v).sum(1)
        around = (p.unsqueeze(-1) * v.abs()).sum(1)
        # weights (of value's scale and softmax) far below the largest: a float16's smallest steps
        size = v.abs().amax(-1)
        least = z.shape[-1] * 2.0 ** -25 * (p * size).amax(-1, keepdim=True) if weight_half_step == FP16_HALF_STEP else 0.0
        # every weight's rounding, its power of two (2 units) and its share of the scores' error, in numerator and denominator
        bound[t] = BF16_HALF_STEP * out[t].abs() + around * (weight_half_step + 2 * off.expm1() + 16 * FP32_HALF_STEP + z.shape[-1] * FP32_HALF_STEP) + least
    return out.reshape(len(q), -1), bound.reshape(len(q), -1) * (1 + 2.0 ** -6) + 1e-30


def sample(z, temperature, top_k, top_p, min_p, draw):
    """(token, margin): the margin is how near the draw or the nucleus' edge comes to a border, relative to all of the weight."""
    z = z.to(torch.float64)
    V = len(z)
    if temperature == 0:
        return int(torch.argmax(z)), 1.0
    w = torch.exp((z - z.max()) / temperature)
    w = torch.where(torch.isnan(w), torch.zeros_like(w), w)
    order = torch.sort(z, descending=True, stable=True)
    last = order.values[(top_k if 0 < top_k < V else V) - 1]
    margin = 1.0
    if top_p < 1.0:
        ranked = torch.where(order.values >= last, w[order.indices], torch.zeros_like(w))
        mass = torch.cumsum(ranked, 0)
        at = int((mass < top_p * mass[-1]).sum())
        near = (mass / mass[-1] - top_p).abs()
        margin = float(near.min())
        last = torch.maximum(last, order.values[at])
    keep = (z >= last) & (w >= min(min_p, 1.0))            # (the largest logit stays)
    ids = torch.nonzero(keep)[:, 0]
    mass = torch.cumsum(w[ids], 0)
    share = mass / mass[-1]
    at = min(int((mass < draw * mass[-1]).sum()), len(ids) - 1)
    if min_p > 0 and bool((w < 1).any()):
        margin = min(margin, float((w[w < 1] / min_p - 1).abs().min()))
    return int(ids[at]), min(margin, float((share - draw).abs()[:-1].min()) if len(ids) > 1 else 1.0)
