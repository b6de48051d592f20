"""The cache in 8 bits and attention over it, against float64."""
import math

import pytest
import torch

import plain_fp8_cache as plain
from qwen_decoder_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def tables(rot, n):
    inv = 1e4 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(n, dtype=torch.float64)[:, None] * inv
    return torch.cos(angle).float(), torch.sin(angle).float()


def turned(x, cos, sin, rot, half):
    y = x.clone()
    if rot:
        a, b = (x[..., :rot // 2], x[..., rot // 2:rot]) if half else (x[..., 0:rot:2], x[..., 1:rot:2])
        c, s = cos.double()[:, None], sin.double()[:, None]
        if half:
            y[..., :rot // 2], y[..., rot // 2:rot] = a * c - b * s, a * s + b * c
        else:
            y[..., 0:rot:2], y[..., 1:rot:2] = a * c - b * s, a * s + b * c
    return y


def check_write(x, bias, H, G, d, rot, half, ps, slots, n_pages, seed=0, positions=None):
    """x: float64-exact rows as given to the kernel ([T, W] or [n, T, W]), on the CPU."""
    gen = torch.Generator().manual_seed(seed)
    T = x.shape[-2]
    cos, sin = tables(rot, 500) if rot else (None, None)
    positions = torch.randint(0, 500, (T,), generator=gen, dtype=torch.int32) if positions is None else positions
    before = plain.filled_pages(gen, n_pages, G, ps, d)
    pages, q = before.to(DEV), torch.empty((T, H * d), dtype=torch.bfloat16, device=DEV)
    to = lambda t: None if t is None else t.to(DEV)
    kernels.rope_kv_write_fp8(to(x), to(bias), q, H, G, d, rot, int(half), to(cos), to(sin), to(positions), pages, to(slots), ps)
    terms = x.double() if x.dim() == 3 else x.double()[None]
    whole, size = terms.sum(0), terms.abs().sum(0)
    if bias is not None:
        whole, size = whole + bias.double(), size + bias.double().abs()
    whole, size = whole.view(T, H + 2 * G, d), size.view(T, H + 2 * G, d)
    at = positions.long()
    y = whole.clone()
    if rot:
        y[:, :H + G] = turned(whole[:, :H + G], cos[at], sin[at], rot, half)
    # q: one rounding to bfloat16 of sums and two products in float32, of the pair's terms
    pair = size[:, :H].amax(-1, keepdim=True) * 2
    off = (q.cpu().double().view(T, H, d) - y[:, :H]).abs()
    assert bool((off <= plain.BF16_HALF_STEP * y[:, :H].abs() + (terms.shape[0] + 6) * plain.FP32_HALF_STEP * pair).all())
    # k and v: the scale exactly, numbers by half a step (two roundings: to float32, to 8 bits)
    want, got = before.clone(), pages.cpu()
    numbers, scales = kernels.fp8_page_views(got, G, ps, d)
    w_numbers, w_scales = kernels.fp8_page_views(want, G, ps, d)
    for t, slot in enumerate(slots.tolist()):
        if slot < 0 or slot >= n_pages * ps:
            continue
        rows = y[t, H:].view(2, G, d)
        s = plain.scale_of(rows)
        assert torch.equal(plain.powers(scales[slot // ps, :, slot % ps]), s.t())
        n = numbers[slot // ps, :, :, slot % ps].float().double()
        exact = rows / s.unsqueeze(-1)
        assert bool(((n - exact).abs() <= (plain.E4M3_HALF_STEP * exact.abs()).clamp(min=2.0 ** -10) * (1 + 2.0 ** -20)).all())
        w_numbers.view(torch.uint8)[slot // ps, :, :, slot % ps] = numbers.view(torch.uint8)[slot // ps, :, :, slot % ps]
        w_scales.view(torch.uint8)[slot // ps, :, slot % ps] = scales.view(torch.uint8)[slot // ps, :, slot % ps]
    assert torch.equal(want, got)                       # every other byte of the pool as it was


@pytest.mark.parametrize("T,H,G,d,rot,half,parts,bias,ps", [
    (1, 16, 2, 128, 128, True, 4, True, 16), (1, 16, 2, 128, 128, False, 0, False, 16), (5, 7, 7, 64, 64, True, 1, True, 16), (3, 16, 1, 64, 32, True, 0, True, 32),
    (70, 28, 4, 128, 128, True, 0, True, 16), (70, 6, 3, 128, 64, False, 2, True, 48), (9, 5, 1, 128, 0, True, 3, False, 16), (2, 1, 1, 64, 8, False, 0, True, 16),
    (300, 28, 4, 128, 128, True, 0, False, 16), (301, 9, 3, 64, 64, True, 2, True, 64), (300, 10, 5, 128, 112, True, 0, True, 16)])
def test_write(guard_regions, T, H, G, d, rot, half, parts, bias, ps):
    gen = torch.Generator().manual_seed(T + H)
    W = (H + 2 * G) * d
    x = torch.randn((parts, T, W), generator=gen) if parts else torch.randn((T, W), generator=gen).bfloat16()
    b = torch.randn(W, generator=gen) * 3 if bias else None
    n_pages = T // ps + 3
    check_write(x, b, H, G, d, rot, half, ps, torch.randperm(n_pages * ps, generator=gen)[:T].to(torch.int32), n_pages)


def test_write_float32_rows_zeros_and_sizes(guard_regions):
    """Whole rows in float32; a row of zeros, of the smallest and of large numbers; largest magnitudes at 448 and just above."""
    H, G, d, ps = 2, 2, 64, 16
    x = torch.randn((6, (H + 2 * G) * d), generator=torch.Generator().manual_seed(1))
    x[1] = 0
    x[2] *= 1e-30
    x[3] *= 1e30
    x[4, H * d + 5], x[5, H * d + 5] = 448.0, 448.00006
    x[4, (H + G) * d + 5], x[5, (H + G) * d + 5] = 448.0 * 2 ** 9, 448.00006 * 2 ** 9
    check_write(x, None, H, G, d, 0, True, ps, torch.tensor([0, 17, 5, 31, 16, 2], dtype=torch.int32), 2)


def test_write_rows_behind_the_last(guard_regions):
    gen = torch.Generator().manual_seed(3)
    x = torch.randn((7, 6 * 64), generator=gen).bfloat16()
    slots = torch.tensor([4, -1, 19, -1, 40, 32, 1 << 30], dtype=torch.int32)
    check_write(x, None, 2, 2, 64, 64, True, 16, slots, 2, positions=torch.tensor([3, 1, 499, 0, 7, 8, 9], dtype=torch.int32))


def test_write_no_numbers():
    H, G, d, ps = 2, 2, 64, 16
    x = torch.ones((4, (H + 2 * G) * d))
    x[0, H * d + 3] = math.inf
    x[1, (H + G) * d + 3] = math.nan
    pages, q = kernels.fp8_pages(1, G, ps, d, DEV), torch.empty((4, H * d), dtype=torch.bfloat16, device=DEV)
    kernels.rope_kv_write_fp8(x.to(DEV), None, q, H, G, d, 0, 1, None, None, torch.zeros(4, dtype=torch.int32, device=DEV), pages,
                              torch.arange(4, dtype=torch.int32, device=DEV), ps)
    s = kernels.fp8_page_views(pages, G, ps, d)[1].view(torch.uint8).cpu()
    none = (s[0, :, :4] == 255).nonzero().tolist()
    assert none == [[0, 0, 0], [0, 1, 1]] and bool((s[0, :, 4:] == 0).all())


# ---- attention of single tokens --------------------------------------------------------------------------------

def a_cache(gen, lengths, G, ps, d, spread=1.0, extra=2):
    """(pages, table) on the CPU: requests of so many cached tokens, pages in a shuffled order, no page behind the last."""
    blocks = [max(1, -(-n // ps)) for n in lengths]
    order = torch.randperm(sum(blocks) + extra, generator=gen)
    table, at = torch.full((len(lengths), max(blocks)), -1, dtype=torch.int32), 0
    for r, b in enumerate(blocks):
        table[r, :b] = order[at:at + b].int()
        at += b
    return plain.filled_pages(gen, sum(blocks) + extra, G, ps, d, spread), table


def check_decode(lengths, H, G, d, ps=16, window=0, reqs=None, positions=None, spread=1.0, seed=0, q_scale=1.0, max_keys=None, pages=None):
    gen = torch.Generator().manual_seed(seed)
    made, table = a_cache(gen, lengths, G, ps, d, spread)
    pages = made if pages is None else pages(made, table)
    reqs = list(range(len(lengths))) if reqs is None else reqs
    positions = [lengths[r] - 1 for r in reqs] if positions is None else positions
    q = (torch.randn((len(reqs), H * d), generator=gen) * q_scale).bfloat16()
    want, bound = plain.attention(q, made, table, reqs, positions, H, G, d, ps, d ** -0.5, window, plain.FP16_HALF_STEP)
    out = torch.empty((len(reqs), H * d), dtype=torch.bfloat16, device=DEV)
    kernels.decode_attention_fp8(q.to(DEV), out, pages.to(DEV), table.to(DEV), torch.tensor(reqs, dtype=torch.int32, device=DEV),
                                 torch.tensor(positions, dtype=torch.int32, device=DEV), H, G, d, ps, d ** -0.5, window, max_keys)
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), (off / bound).argmax())
    return out


@pytest.mark.parametrize("H,G,d", [(16, 2, 128), (28, 4, 128), (14, 2, 64), (40, 8, 128), (3, 3, 64), (16, 1, 128), (9, 1, 64), (11, 1, 128)])
@pytest.mark.parametrize("lengths", [[1], [16], [17], [2, 15, 129, 128, 127], [700, 3, 2100]])
def test_decode(guard_regions, H, G, d, lengths):
    check_decode(lengths, H, G, d)


@pytest.mark.parametrize("ps", [32, 48, 64])
def test_decode_page_sizes(guard_regions, ps):
    check_decode([1, 100, 333, ps, ps + 1], 14, 2, 64, ps=ps)


@pytest.mark.parametrize("window", [1, 15, 16, 17, 100, 128, 5000])
def test_decode_window(guard_regions, window):
    check_decode([1, 14, 16, 100, 129, 1000], 12, 2, 128, window=window)


def test_decode_many_tokens(guard_regions):
    """More tokens than a launch takes, several of one request, some that see nothing."""
    gen = torch.Generator().manual_seed(5)
    reqs = torch.randint(0, 3, (1500,), generator=gen).tolist()
    lengths = [40, 300, 7]
    positions = [int(torch.randint(-1, lengths[r], (1,), generator=gen)) for r in reqs]
    check_decode(lengths, 2, 1, 64, reqs=reqs, positions=positions)


def test_decode_long(guard_regions):
    check_decode([20000, 5], 7, 1, 128)
    check_decode([9000] * 3, 8, 4, 64)


@pytest.mark.parametrize("T", [5, 31, 33, 64, 130, 400, 1100])
@pytest.mark.parametrize("H,G,d", [(8, 2, 128), (3, 3, 64), (9, 1, 64)])
def test_decode_ragged(guard_regions, T, H, G, d):
    """Tokens of lengths from nothing on beside a few long ones, whose keys several CTAs have."""
    gen = torch.Generator().manual_seed(T)
    lengths = [5000, 700, 129, 1]
    reqs = [0, 3] + torch.randint(0, 4, (T - 2,), generator=gen).tolist()
    short = torch.rand((T,), generator=gen) < 0.7
    positions = [4999, 0] + [int(torch.randint(-1, min(lengths[r], 300) if short[t + 2] else lengths[r], (1,), generator=gen)) for t, r in enumerate(reqs[2:])]
    check_decode(lengths, H, G, d, reqs=reqs, positions=positions)
    if T in (33, 130):
        check_decode(lengths, H, G, d, reqs=reqs, positions=positions, window=1500)
        check_decode(lengths, H, G, d, reqs=reqs[:-1] + [0], positions=[-1] * (T - 1) + [4999])
        check_decode(lengths, H, G, d, reqs=[0] * T, positions=[4999 - t % 7 for t in range(T)])


def test_decode_scales_far_apart(guard_regions):
    """Values whose scales lie 2^20 and more apart, scores that leave one key nearly alone."""
    check_decode([300, 40, 1000], 8, 2, 128, spread=8.0, q_scale=0.01)
    check_decode([300, 40, 1000], 8, 2, 128, spread=2.0, q_scale=8.0)
    check_decode([300, 40, 1000], 8, 2, 64, spread=1.0, q_scale=1e-20)


def test_decode_max_keys(guard_regions):
    check_decode([1, 500, 130], 8, 2, 128, max_keys=500)


def test_decode_what_nobody_sees(guard_regions):
    """Rows behind a token's position and pages of nobody that are no numbers, and window's lost keys."""
    def spoiled(pages, table):
        G, ps, d = 2, 16, 128
        bad = pages.clone()
        used = set()
        numbers, scales = kernels.fp8_page_views(bad, G, ps, d)
        for r, n in enumerate([1, 18, 500]):
            for key in range(table.shape[1] * ps):
                page = int(table[r, key // ps])
                if page >= 0 and (key >= n or key <= n - 1 - 40):
                    numbers.view(torch.uint8)[page, :, :, key % ps] = 0x7f
                    scales.view(torch.uint8)[page, :, key % ps] = 255
            used |= {int(p) for p in table[r] if p >= 0}
        for page in range(len(bad)):
            if page not in used:
                bad[page] = 255
        return bad
    check_decode([1, 18, 500], 8, 2, 128, window=40, pages=spoiled)


@pytest.mark.parametrize("which", [0, 1])
def test_decode_no_number_that_is_seen(which):
    gen = torch.Generator().manual_seed(2)
    H, G, d, ps = 4, 2, 64, 16
    pages, table = a_cache(gen, [300, 300], G, ps, d)
    numbers, scales = kernels.fp8_page_views(pages, G, ps, d)
    scales.view(torch.uint8)[int(table[0, 3]), 1, 5, which] = 255        # request 0, kv head 1
    out = torch.empty((2, H * d), dtype=torch.bfloat16, device=DEV)
    q = torch.randn((2, H * d), generator=gen).bfloat16().to(DEV)
    kernels.decode_attention_fp8(q, out, pages.to(DEV), table.to(DEV), torch.arange(2, dtype=torch.int32, device=DEV),
                                 torch.full((2,), 299, dtype=torch.int32, device=DEV), H, G, d, ps, 0.1)
    none = out.isnan().view(2, H, d).cpu()
    assert bool(none[0, 2:].all()) and not bool(none[0, :2].any()) and not bool(none[1].any())


def test_decode_repeats_and_rows_apart():
    """The same bits again, from rows that lie apart, for a token alone and among others whose shares differ; rows between untouched."""
    gen = torch.Generator().manual_seed(8)
    H, G, d, ps = 8, 2, 128, 16
    pages, table = a_cache(gen, [2500, 90, 1], G, ps, d)
    q = torch.randn((3, H * d), generator=gen).bfloat16().to(DEV)
    args = (pages.to(DEV), table.to(DEV), torch.arange(3, dtype=torch.int32, device=DEV), torch.tensor([2499, 89, 0], dtype=torch.int32, device=DEV), H, G, d, ps, 0.1)
    a, b = (torch.empty_like(q) for _ in range(2))
    kernels.decode_attention_fp8(q, a, *args)
    kernels.decode_attention_fp8(q, b, *args)
    assert torch.equal(a, b)
    wide, out = torch.zeros((3, H * d + 64), dtype=torch.bfloat16, device=DEV), torch.full((3, H * d + 8), 7.0, dtype=torch.bfloat16, device=DEV)
    wide[:, :H * d] = q
    kernels.decode_attention_fp8(wide[:, :H * d], out[:, :H * d], *args)
    assert torch.equal(out[:, :H * d], a) and bool((out[:, H * d:] == 7).all())


def test_decode_in_graphs_on_other_streams():
    """Two captured graphs and a call replayed side by side on streams of their own give what they give alone, lengths changed in between."""
    gen = torch.Generator().manual_seed(9)
    H, G, d, ps = 28, 4, 128, 16
    pages, table = a_cache(gen, [3000, 3000], G, ps, d)
    pages, table = pages.to(DEV), table.to(DEV)
    reqs = torch.arange(2, dtype=torch.int32, device=DEV)
    sets = []
    for i in range(2):
        q = torch.randn((2, H * d), generator=gen).bfloat16().to(DEV)
        pos, out = torch.tensor([2999, 17], dtype=torch.int32, device=DEV), torch.empty_like(q)
        call = lambda q=q, out=out, pos=pos: kernels.decode_attention_fp8(q, out, pages, table, reqs, pos, H, G, d, ps, 0.1, 0, 3000)
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        sets.append((q, pos, out, call, graph, torch.cuda.Stream()))
    for lengths in ([2999, 17], [5, 2998], [1500, 1501]):
        alone = []
        for q, pos, out, call, graph, stream in sets:
            pos.copy_(torch.tensor(lengths, dtype=torch.int32))
            call()
            alone.append(out.clone())
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for *_, graph, stream in sets:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for (q, pos, out, *_), want in zip(sets, alone):
            assert torch.equal(out, want)


def test_write_then_decode_behind_other_work():
    """Positions, slots and tables written by the work just before, on the same stream."""
    gen = torch.Generator().manual_seed(4)
    H, G, d, ps, T = 14, 2, 64, 16, 40
    x = torch.randn((T, (H + 2 * G) * d), generator=gen).bfloat16().to(DEV)
    cos, sin = (t.to(DEV) for t in tables(d, 64))
    outs = []
    for lazy in (False, True):
        pages, q, out = kernels.fp8_pages(4, G, ps, d, DEV), torch.empty((T, H * d), dtype=torch.bfloat16, device=DEV), torch.empty((T, H * d), dtype=torch.bfloat16, device=DEV)
        pos, slots, table, reqs = (torch.zeros(n, dtype=torch.int32, device=DEV) for n in (T, T, 3, T))
        torch.cuda.synchronize()
        if lazy:
            torch.cuda._sleep(2_000_000)
        pos.copy_(torch.arange(T, dtype=torch.int32, device=DEV))
        table.copy_(torch.tensor([2, 0, 3], dtype=torch.int32, device=DEV))
        slots.copy_(table[(pos // ps).long()] * ps + pos % ps)
        kernels.rope_kv_write_fp8(x, None, q, H, G, d, d, 1, cos, sin, pos, pages, slots, ps)
        kernels.decode_attention_fp8(q, out, pages, table.view(1, 3), reqs, pos, H, G, d, ps, d ** -0.5)
        torch.cuda.synchronize()
        outs.append(out.clone())
    assert torch.equal(*outs)


# ---- attention of portions ---------------------------------------------------------------------------------------

def check_prefill(tokens, before, H, G, d, ps=16, window=0, spread=1.0, seed=0, q_scale=1.0, spoil=None, extra_rows=(0, 0), **kw):
    """Portions of so many tokens behind so many cached ones; ``extra_rows`` of q and out before and behind them stay as they are."""
    gen = torch.Generator().manual_seed(seed)
    lengths = [b + t for b, t in zip(before, tokens)]
    pages, table = a_cache(gen, lengths, G, ps, d, spread)
    T, (ahead, behind) = sum(tokens), extra_rows
    q = (torch.randn((T, H * d), generator=gen) * q_scale).bfloat16()
    reqs = [r for r, t in enumerate(tokens) for _ in range(t)]
    positions = [b + i for b, t in zip(before, tokens) for i in range(t)]
    want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, window, plain.BF16_HALF_STEP)
    if spoil is not None:
        spoil(pages, table, lengths)
    wide = torch.zeros((ahead + T + behind, H * d), dtype=torch.bfloat16)
    wide[ahead:ahead + T] = q
    out = torch.full(wide.shape, 7.0, dtype=torch.bfloat16, device=DEV)
    cu = [ahead]
    for t in tokens:
        cu.append(cu[-1] + t)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    args = (wide.to(DEV), out, pages.to(DEV), table.to(DEV), i32(cu), i32(before), H, G, d, ps, d ** -0.5, window)
    kernels.prefill_attention_fp8(*args, **kw)
    kernels.check_status()
    got = out.cpu()
    assert bool((got[:ahead] == 7).all()) and bool((got[ahead + T:] == 7).all())
    off = (got[ahead:ahead + T].double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), divmod(int((off / bound).argmax()), H * d))
    return args


@pytest.mark.parametrize("H,G,d", [(16, 2, 128), (28, 4, 128), (14, 2, 64), (5, 1, 128), (3, 3, 64), (16, 1, 128), (11, 1, 64)])
@pytest.mark.parametrize("tokens,before", [([1], [0]), ([5], [0]), ([130], [0]), ([20, 1, 37], [0, 200, 3]), ([129], [127]), ([300, 2], [100, 511])])
def test_prefill(guard_regions, H, G, d, tokens, before):
    check_prefill(tokens, before, H, G, d)


@pytest.mark.parametrize("ps", [32, 48, 64])
def test_prefill_page_sizes(guard_regions, ps):
    check_prefill([ps, ps + 1, 3], [0, 77, 2 * ps - 1], 14, 2, 64, ps=ps)
    check_prefill([ps, ps + 1, 3], [0, 77, 2 * ps - 1], 4, 2, 128, ps=ps)


@pytest.mark.parametrize("window", [1, 16, 100, 128, 129, 5000])
def test_prefill_window(guard_regions, window):
    check_prefill([140, 1, 33], [0, 300, 250], 12, 2, 128, window=window)
    check_prefill([20], [3000], 8, 1, 64, window=window)


@pytest.mark.parametrize("tokens,before", [([1], [5000]), ([37], [4000]), ([3, 40], [9000, 10]), ([17], [1100])])
@pytest.mark.parametrize("H,G,d", [(7, 1, 128), (4, 2, 64)])
def test_prefill_shares_of_keys(guard_regions, tokens, before, H, G, d):
    """Few rows behind many keys: several CTAs have a share of them, some of which a request's rows do not reach."""
    check_prefill(tokens, before, H, G, d, extra_rows=(2, 3), n_tokens=sum(tokens))


def test_prefill_rows_around(guard_regions):
    check_prefill([33, 150], [70, 0], 8, 2, 128, extra_rows=(9, 4))
    check_prefill([0, 33, 0, 5], [0, 70, 0, 2], 8, 2, 128, extra_rows=(0, 1))


def test_prefill_many_requests(guard_regions):
    gen = torch.Generator().manual_seed(11)
    tokens = torch.randint(1, 4, (300,), generator=gen).tolist()
    before = torch.randint(0, 40, (300,), generator=gen).tolist()
    check_prefill(tokens, before, 4, 2, 64)


def test_prefill_scales_far_apart(guard_regions):
    check_prefill([60, 9], [200, 40], 8, 2, 128, spread=8.0, q_scale=0.01)
    check_prefill([60, 9], [200, 40], 8, 2, 128, spread=2.0, q_scale=8.0)
    check_prefill([60, 9], [200, 40], 8, 2, 64, q_scale=1e-20)


def test_prefill_what_nobody_sees(guard_regions):
    """Rows behind a request's last token, pages of nobody and keys before every row's window that are no numbers."""
    def spoil(pages, table, lengths):
        numbers, scales = kernels.fp8_page_views(pages, 2, 16, 128)
        used = set()
        for r, n in enumerate(lengths):
            used |= {int(p) for p in table[r] if p >= 0}
            for key in list(range(n, table.shape[1] * 16)) + list(range(0, max(0, n - 41 - 100))):
                page = int(table[r, key // 16])
                if page >= 0:
                    numbers.view(torch.uint8)[page, :, :, key % 16] = 0x7f
                    scales.view(torch.uint8)[page, :, key % 16] = 255
        for page in range(len(pages)):
            if page not in used:
                pages[page] = 255
    check_prefill([41, 7, 100], [300, 0, 13], 8, 2, 128, window=100, spoil=spoil)


@pytest.mark.parametrize("which", [0, 1])
def test_prefill_no_number_that_some_see(which):
    """A key or value that is no number: the rows from its own on are none, in its head alone; a window past it is not."""
    gen = torch.Generator().manual_seed(2)
    H, G, d, ps = 4, 2, 64, 16
    pages, table = a_cache(gen, [300], G, ps, d)
    kernels.fp8_page_views(pages, G, ps, d)[1].view(torch.uint8)[int(table[0, 3]), 1, 5, which] = 255        # key 53 of kv head 1
    q = torch.randn((300, H * d), generator=gen).bfloat16().to(DEV)
    for window, last in ((0, 300), (20, 73)):
        out = torch.empty_like(q)
        kernels.prefill_attention_fp8(q, out, pages.to(DEV), table.to(DEV), torch.tensor([0, 300], dtype=torch.int32, device=DEV),
                                      torch.zeros(1, dtype=torch.int32, device=DEV), H, G, d, ps, 0.1, window)
        none = out.isnan().view(300, H, d).cpu()
        want = torch.zeros((300, H, d), dtype=torch.bool)
        want[53:last, 2:] = True
        assert torch.equal(none, want)


def test_prefill_is_decode(guard_regions):
    """Single tokens through both kernels, within both bounds; the same bits again, in a graph on another stream."""
    args = check_prefill([1, 1, 1], [0, 400, 77], 8, 2, 128)
    q, out, pages, table, cu, start, H, G, d, ps, scale, window = args
    first, other = out.clone(), torch.empty_like(out)
    kernels.decode_attention_fp8(q, other, pages, table, torch.arange(3, dtype=torch.int32, device=DEV), start, H, G, d, ps, scale)
    assert float((other.double() - first.double()).abs().max()) < 2.0 ** -5 * float(first.double().abs().max())
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with torch.cuda.graph(graph):
        kernels.prefill_attention_fp8(*args)
    out.zero_()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)


def test_prefill_wait_that_runs_out():
    kernels.check_status()
    check_prefill([5], [0], 2, 1, 64)
    kernels.wait_probe("attention_fp8_chunk")
    with pytest.raises(kernels.KernelError, match="attention_fp8_chunk"):
        kernels.check_status()
    check_prefill([5], [0], 2, 1, 64)


# ---- scales of values anywhere -----------------------------------------------------------------------------------

def moved(pages, table, lengths, G, d, ps, by):
    """The values' scales of keys [128 i, 128 (i + 1)) times 2^by[i], the last entry for all behind."""
    pages = pages.clone()
    scales = kernels.fp8_page_views(pages, G, ps, d)[1].view(torch.uint8)
    for r, n in enumerate(lengths):
        for key in range(n):
            at = scales[int(table[r, key // ps]), :, key % ps, 1]
            new = at.int() + by[min(key // 128, len(by) - 1)]
            assert 1 <= int(new.min()) and int(new.max()) <= 254
            at.copy_(new.to(torch.uint8))
    return pages


def both_kernels(q, pages, table, tokens, before, H, G, d, ps):
    """Rows of the portions' kernel, and of the single tokens' one."""
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    reqs = [r for r, t in enumerate(tokens) for _ in range(t)]
    positions = [b + i for b, t in zip(before, tokens) for i in range(t)]
    q, pages, table = q.to(DEV), pages.to(DEV), table.to(DEV)
    a, b = torch.empty_like(q), torch.empty_like(q)
    kernels.prefill_attention_fp8(q, a, pages, table, i32([0] + tokens).cumsum(0).to(torch.int32), i32(before), H, G, d, ps, d ** -0.5)
    kernels.decode_attention_fp8(q, b, pages, table, i32(reqs), i32(positions), H, G, d, ps, d ** -0.5)
    kernels.check_status()
    return reqs, positions, a.cpu().double(), b.cpu().double()


@pytest.mark.parametrize("tokens,before", [([20, 3], [300, 0]), ([3], [4000])])
@pytest.mark.parametrize("by", [-110, 60, 120])
@pytest.mark.parametrize("H,G,d", [(8, 2, 128), (4, 2, 64)])
def test_values_times_a_power_of_two(guard_regions, H, G, d, by, tokens, before):
    gen, ps = torch.Generator().manual_seed(21), 16
    lengths = [b + t for b, t in zip(before, tokens)]
    pages, table = a_cache(gen, lengths, G, ps, d)
    q = torch.randn((sum(tokens), H * d), generator=gen).bfloat16()
    reqs, positions, *got = both_kernels(q, moved(pages, table, lengths, G, d, ps, [by]), table, tokens, before, H, G, d, ps)
    for out, step in zip(got, (plain.BF16_HALF_STEP, plain.FP16_HALF_STEP)):
        want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, 0, step)
        # a score and its value's scale add up to numbers below 256, three roundings of 2^-17 each: 3% of a weight's own 2^-11; bfloat16's least step
        assert bool(((out - want * 2.0 ** by).abs() <= bound * 2.0 ** by * (1 + 2.0 ** -4) + 2.0 ** -133).all())


@pytest.mark.parametrize("by", [[0, -110, 0], [-110, 0], [0, 0, -110], [-110, 100, -60], [100, -110], [20, -20, 0, 20]])
@pytest.mark.parametrize("tokens,before", [([20, 3], [500, 90]), ([3], [4000])])
def test_values_of_keys_far_apart(guard_regions, tokens, before, by):
    """Values that are next to nothing beside others take their share of the softmax all the same."""
    gen, H, G, d, ps = torch.Generator().manual_seed(22), 8, 2, 128, 16
    lengths = [b + t for b, t in zip(before, tokens)]
    pages, table = a_cache(gen, lengths, G, ps, d)
    pages = moved(pages, table, lengths, G, d, ps, by)
    q = torch.randn((sum(tokens), H * d), generator=gen).bfloat16()
    reqs, positions, *got = both_kernels(q, pages, table, tokens, before, H, G, d, ps)
    for out, step in zip(got, (plain.BF16_HALF_STEP, plain.FP16_HALF_STEP)):
        want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, 0, step)
        assert bool(((out - want).abs() <= bound * (1 + 2.0 ** -4)).all()), float(((out - want).abs() / bound).max())


def test_prefill_rows_before_the_first_position(guard_regions):
    """Rows at positions below zero see nothing: zeros; a list of rows that ends behind q's is cut."""
    gen, H, G, d, ps = torch.Generator().manual_seed(23), 4, 2, 64, 16
    pages, table = a_cache(gen, [40, 30], G, ps, d)
    q = torch.randn((60, H * d), generator=gen).bfloat16()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
    for cu, start, tokens in (([0, 40, 60], [-7, 5], (40, 20)), ([0, 45, 60], [-200, 0], (45, 15)), ([0, 40, 90], [0, 5], (40, 20))):
        out = torch.full_like(q, 7.0).to(DEV)
        kernels.prefill_attention_fp8(q.to(DEV), out, pages.to(DEV), table.to(DEV), i32(cu), i32(start), H, G, d, ps, d ** -0.5)
        kernels.check_status()
        reqs, positions = [0] * tokens[0] + [1] * tokens[1], [start[r] + i for r, t in enumerate(tokens) for i in range(t)]
        want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, 0, plain.BF16_HALF_STEP)
        assert bool(((out.cpu().double() - want).abs() <= bound).all())


# ---- large sizes -------------------------------------------------------------------------------------------------

def test_pages_past_32_bits():
    """Written, and attended to by both kernels, at the end of a pool of more than 2^32 bytes as at its beginning."""
    gen, H, G, d, ps = torch.Generator().manual_seed(31), 8, 4, 128, 16
    n = (1 << 32) // kernels.fp8_page_bytes(G, ps, d) + 1000
    pool = torch.empty((n, kernels.fp8_page_bytes(G, ps, d)), dtype=torch.uint8, device=DEV)
    T, before, lengths = 40, [260, 0], [290, 10]
    pages, table = a_cache(gen, lengths, G, ps, d, extra=0)
    blocks = len(pages)
    x = torch.randn((T, (H + 2 * G) * d), generator=gen).bfloat16().to(DEV)
    reqs = torch.tensor([0] * 30 + [1] * 10, dtype=torch.int32, device=DEV)
    positions = torch.tensor([260 + i for i in range(30)] + list(range(10)), dtype=torch.int32, device=DEV)
    cu, start = torch.tensor([0, 30, 40], dtype=torch.int32, device=DEV), torch.tensor(before, dtype=torch.int32, device=DEV)
    got = []
    for first in (0, n - blocks):
        pool[first:first + blocks] = pages.to(DEV)
        at = torch.where(table >= 0, table + first, table).to(DEV)
        slots = (at[reqs.long(), positions.long() // ps] * ps + positions % ps).to(torch.int32)
        q, a, b = (torch.empty((T, H * d), dtype=torch.bfloat16, device=DEV) for _ in range(3))
        kernels.rope_kv_write_fp8(x, None, q, H, G, d, 0, 1, None, None, positions, pool, slots, ps)
        kernels.prefill_attention_fp8(q, a, pool, at, cu, start, H, G, d, ps, d ** -0.5)
        kernels.decode_attention_fp8(q, b, pool, at, reqs, positions, H, G, d, ps, d ** -0.5)
        kernels.check_status()
        got.append((q, a, b, pool[first:first + blocks].clone()))
        pool[first:first + blocks] = 255
    assert all(torch.equal(x, y) for x, y in zip(*got)) and not bool(got[0][1].isnan().any())
    want, bound = plain.attention(got[0][0].cpu(), got[0][3].cpu(), table, reqs.tolist(), positions.tolist(), H, G, d, ps, d ** -0.5, 0, plain.BF16_HALF_STEP)
    assert bool(((got[0][1].cpu().double() - want).abs() <= bound).all())


def test_prefill_many_rows(guard_regions):
    """More rows than one round of multiprocessors has room for, in one request and in several."""
    check_prefill([1500, 700], [100, 0], 2, 2, 64)
    check_prefill([1200], [0], 16, 2, 64, window=300)
