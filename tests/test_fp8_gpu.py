"""Rows and products in 8 bits (``csrc/rows_fp8.cu``, ``csrc/gemm_fp8.cu``) against float64: odd sizes, strides, parts, blocks of zeros and
of no numbers, the edges of tiles and of blocks, shares of K."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("guard_regions")]
DEV = "cuda:0"


def generator(*sizes):
    return torch.Generator(device=DEV).manual_seed(sum(s * 31 ** i for i, s in enumerate(sizes)) % (1 << 31))


def numbers(shape, g, spread=0):
    """Normal numbers, blocks of 128 up to 2^spread apart."""
    x = torch.empty(shape, device=DEV, dtype=torch.float32).normal_(generator=g)
    if spread:
        n = -(-shape[-1] // 128)
        e = torch.randint(-spread, 1, (*shape[:-1], n), generator=g, device=DEV)
        x = torch.ldexp(x, e.repeat_interleave(128, -1)[..., :shape[-1]])
    return x


def room(R, K):
    """``kernels.fp8_rows`` between margins that are looked at when a test ends (its own room does not go through torch.empty)."""
    from qwen_decoder_b200 import kernels
    kb = -(-K // 128)
    return kernels.Fp8Rows(torch.empty((R, -(-K // 16) * 16), dtype=torch.float8_e4m3fn, device=DEV)[:, :K],
                           torch.empty((R, -(-kb // 4) * 4), dtype=torch.float8_e8m0fnu, device=DEV)[:, :kb])


def scales_of(peak):
    """The scale of a block by its definition: the smallest power of two with peak <= 448 * scale, 1 of zeros, 2^-126 at least."""
    e = torch.ceil(torch.log2(peak / 448.0))
    for step in (-1, 1):                                   # a logarithm may be rounded across a whole number
        e = torch.where((peak <= 448.0 * torch.exp2(e - 1)) if step < 0 else (peak > 448.0 * torch.exp2(e)), e + step, e)
    s = torch.exp2(e.clamp(min=-126))
    return torch.where(peak == 0, torch.ones_like(s), s)


def blocks(y):
    n = -(-y.shape[1] // 128)
    return torch.nn.functional.pad(y, (0, n * 128 - y.shape[1])).view(y.shape[0], n, 128)


def spread_out(s, K):
    return s.repeat_interleave(128, 1)[:, :K]


def check_rows(rows, y, off):
    """rows holds y in 8 bits, of numbers that may be ``off`` from y (float64, elementwise): scales by their definition, of a peak that may
    be so far off; numbers rounded to nearest: half of e4m3's step is 2^-4 of a number at most, 2^-10 among the smallest."""
    s = rows.s.float().double()
    peak, wide = blocks(y.abs()).amax(2), blocks(off).amax(2)
    assert ((s >= scales_of((peak - wide).clamp(min=0))) | (s >= scales_of(peak))).all() and (s <= scales_of(peak + wide)).all()
    s = spread_out(s, y.shape[1])
    got, want = rows.q.double(), y / s
    assert ((got - want).abs() <= torch.clamp((want.abs() + off / s) * 2.0 ** -4, min=2.0 ** -10) + off / s).all()


def rows_of(x):
    from qwen_decoder_b200 import kernels
    out = room(*x.shape)
    kernels.quantize_fp8(x, out)
    return out


def value(rows):
    return rows.q.double() * spread_out(rows.s.float().double(), rows.shape[1])


# ---- rows -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,K,pad", [(1, 1, 0), (3, 127, 0), (2, 128, 4), (5, 129, 3), (1, 2048, 0), (23, 1000, 24), (300, 3584, 0), (4, 517, 1)])
def test_rows_as_they_are(T, K, pad, dtype):
    x = numbers((T, K + pad), generator(T, K), spread=20).to(dtype)[:, :K]
    got = rows_of(x)
    b = blocks(x.double())
    s = scales_of(b.abs().amax(2))
    assert torch.equal(got.s.float().double(), s)
    # a quotient by a power of two is exact: the same rounding to 8 bits as of the quotient in 32 bits
    want = (x.double() / spread_out(s, K)).float().to(torch.float8_e4m3fn)
    assert torch.equal(got.q.view(torch.uint8), want.view(torch.uint8))


def test_edges_of_the_scale():
    x = torch.zeros(8, 256, device=DEV)
    x[0, 3] = 448.0                                        # the largest number of the scale 1 ...
    x[1, 3] = math.nextafter(448.0, 1e9) * (1 + 2.0 ** -20)  # ... and one above it
    x[2, 200] = -2.0 ** -140                               # a subnormal: the smallest scale
    x[3, 5] = 3.4028234663852886e38
    x[4, 7], x[5, 7], x[6, 130] = float("inf"), float("nan"), -float("inf")
    got = rows_of(x)
    s = got.s.float()
    assert s[0].tolist() == [1.0, 1.0] and s[1].tolist() == [2.0, 1.0] and s[2].tolist() == [1.0, 2.0 ** -126] and s[3, 0] == 2.0 ** 120
    assert s[4, 0].isnan() and s[5, 0].isnan() and s[6, 1].isnan() and s[4, 1] == 1 and s[6, 0] == 1
    q = got.q.float()
    assert q[0, 3] == 448 and q[1, 3] == 224 and q[7].abs().max() == 0 and q[2, 200] == 0 and 224 < q[3, 5] <= 448
    assert q[4, :128].isnan().all() and q[5, :128].isnan().all() and q[6, 128:].isnan().all() and not q[4, 128:].isnan().any()


@pytest.mark.parametrize("n", [1, 2, 7])
@pytest.mark.parametrize("K", [130, 512])
def test_parts_are_added_first(n, K):
    parts = numbers((n, 9, K), generator(n, K))
    total = parts[0]
    for p in parts[1:]:
        total = total + p
    got, want = rows_of_parts(parts), rows_of(total)
    assert torch.equal(got.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(got.s.view(torch.uint8), want.s.view(torch.uint8))


def rows_of_parts(parts):
    from qwen_decoder_b200 import kernels
    out = room(*parts.shape[1:])
    kernels.quantize_fp8(parts, out)
    return out


def gated(g, u, act):
    if act:
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("T,F,n,bias", [(1, 1, 1, True), (7, 200, 3, True), (3, 1001, 1, False), (64, 512, 2, False)])
def test_gate(T, F, n, bias, act):
    from qwen_decoder_b200 import kernels
    g = generator(T, F, n)
    parts, b = numbers((n, T, 2 * F), g), numbers((2 * F,), g) if bias else None
    out = room(T, F)
    kernels.gate_fp8(parts, out, b, act)
    z = parts.double().sum(0) + (b.double() if bias else 0)
    # n + 1 roundings of 2^-24 of what is added; the activation's slope is below 1.2, its exponential and quotient within 2^-20
    size = parts.double().abs().sum(0) + (b.double().abs() if bias else 0)
    off = (n + 1) * 2.0 ** -24 * size
    h = gated(z[:, :F], z[:, F:], act)
    check_rows(out, h, 1.2 * off[:, :F] * z[:, F:].abs() + (z[:, :F].abs() + off[:, :F]) * off[:, F:] + 2.0 ** -20 * (z[:, :F] * z[:, F:]).abs())


def test_gate_of_infinities():
    from qwen_decoder_b200 import kernels
    z = torch.ones(3, 256, device=DEV)
    z[0, 0], z[1, 0], z[2, 0] = -float("inf"), float("inf"), float("nan")
    out = room(3, 128)
    kernels.gate_fp8(z, out)
    assert out.q[0, 0].float() == 0 and not out.s[0].float().isnan().any() and out.s[1:].float().isnan().all()


@pytest.mark.parametrize("T,D,parts,scaled", [(1, 1, 0, False), (1, 2048, 4, False), (5, 1001, 3, True), (64, 3584, 0, True), (3, 20001, 2, False),
                                              (2, 40000, 1, False), (130, 130, 0, False)])
def test_norm(T, D, parts, scaled):
    from qwen_decoder_b200 import kernels
    g = generator(T, D, parts)
    x, w, f = numbers((T, D), g), 1 + 0.1 * numbers((D,), g), numbers((D,), g) if scaled else None
    delta = numbers((parts, T, D), g) if parts else numbers((T, D), g).bfloat16()
    d = delta.double().sum(0) if parts else delta.double()
    size = delta.double().abs().sum(0) if parts else d.abs()
    if scaled:
        d, size = d * f.double(), size * f.double().abs()
    sums, off = x.double() + d, (parts + 3) * 2.0 ** -24 * (x.double().abs() + size)
    y = sums * torch.rsqrt(sums.square().mean(1, keepdim=True) + 1e-6) * w.double()
    out, kept = room(T, D), x.clone()
    kernels.add_rmsnorm_fp8(x, delta, w, out, 1e-6, delta_scale=f)
    assert ((x.double() - sums).abs() <= off).all()
    # a thread's up to 64 squares and a tree of 10 levels, a quotient, a root and three products: below 2^-17; the sums' own error apart
    inv = torch.rsqrt(sums.square().mean(1, keepdim=True) + 1e-6)
    mean_off = (off.square().mean(1, keepdim=True)).sqrt() * inv
    own = 2.0 ** -17 * y.abs() + (off * inv + sums.abs() * inv * mean_off) * w.double().abs()
    check_rows(out, y, own)
    # chosen rows, the sum left as it was
    rows = torch.tensor([T - 1, 0], dtype=torch.int32, device=DEV)
    again, few = kept.clone(), room(2, D)
    kernels.add_rmsnorm_fp8(again, delta, w, few, 1e-6, rows=rows, write_back=False, delta_scale=f)
    assert torch.equal(again, kept) and torch.equal(few.q.view(torch.uint8), out.q[rows.long()].view(torch.uint8))
    assert torch.equal(few.s.view(torch.uint8), out.s.view(torch.uint8)[rows.long()])


def test_norm_of_zeros_and_without_delta():
    from qwen_decoder_b200 import kernels
    x = torch.zeros(2, 300, device=DEV)
    x[1, 7] = 3.0
    out = room(2, 300)
    kernels.add_rmsnorm_fp8(x, None, torch.ones(300, device=DEV), out, 1e-6)
    assert out.q[0].float().abs().max() == 0 and (out.s[0].float() == 1).all()
    assert float(value(out)[1, 7]) == pytest.approx(300 ** 0.5, rel=2.0 ** -4) and (out.q[1].float() != 0).sum() == 1


# ---- products ---------------------------------------------------------------------------------------------------------
def sums_off(x, w):
    """Of a float32 sum in the tensor cores: an addition to every 32 of k, cut off at 2^-23 of what is added up at most, and the pieces' own."""
    K = x.shape[1]
    return (K / 32 + K / 1024 + 10) * 2.0 ** -23 * (value(x).abs() @ value(w).abs().T)


def operands(T, N, K):
    g = generator(T, N, K)
    return rows_of(numbers((T, K), g, spread=6)), rows_of(numbers((N, K), g, spread=6) * K ** -0.5), numbers((N,), g)


PRODUCTS = [(1, 1, 1), (1, 64, 128), (5, 200, 1000), (8, 97, 5000), (9, 530, 1601), (16, 40, 4500), (17, 33, 129), (127, 130, 512), (128, 2049, 640), (129, 96, 2056), (257, 264, 1024),
            (300, 1000, 1500), (700, 514, 300)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T,N,K", PRODUCTS)
def test_product(T, N, K, dtype):
    from qwen_decoder_b200 import kernels
    x, w, bias = operands(T, N, K)
    want, off = value(x) @ value(w).T, sums_off(x, w)
    plans = {None} | ({kernels.FP8_FEW} if T <= kernels.FP8_FEW_TOKENS else set())
    for cg in (1, 2):
        for bn in (32, 48, 64, 96, 128, 192, 208, 224, 240, 256):
            for splits in (1, 2, 3, 8):
                if (cg == 1 or splits == 1) and (bn % 32 == 0 or cg * splits == 1) and splits <= -(-K // 128) and not (dtype == torch.float32 and bn > 128):
                    plans.add((cg, bn, splits))
    for plan in sorted(plans, key=str):
        for b in (None, bias):
            out = torch.full((T, N + 5), -7.0, dtype=dtype, device=DEV)[:, :N] if plan is None else torch.full((T, N), -7.0, dtype=dtype, device=DEV)
            try:
                kernels.gemm_fp8(x, w, b, out, plan)
            except kernels.KernelError:
                # sums of a share that have no room in shared memory are refused
                assert plan is not None and plan[2] > 1
                continue
            full = want if b is None else want + b.double()
            close = (2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -23) * full.abs() + off
            assert ((out.double() - full).abs() <= close).all(), plan
    kernels.check_status()


@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("T,F,K,bias", [(1, 1, 1, True), (8, 1000, 300, False), (5, 200, 1000, True), (128, 128, 512, False), (129, 384, 640, True),
                                        (300, 1001, 1500, False), (1000, 136, 200, True)])
def test_gated_product(T, F, K, bias, act):
    from qwen_decoder_b200 import kernels
    x, w, b = operands(T, 2 * F, K)
    z = value(x) @ value(w).T + (b.double() if bias else 0)
    off = sums_off(x, w) + 2.0 ** -23 * z.abs()
    h = gated(z[:, :F], z[:, F:], act)
    wide = 1.2 * off[:, :F] * z[:, F:].abs() + (z[:, :F].abs() + off[:, :F]) * off[:, F:] + 2.0 ** -20 * (z[:, :F] * z[:, F:]).abs()
    for plan in (None, (1, 256, 1), (2, 256, 1)):
        out = room(T, F)
        kernels.gemm_fp8_gated(x, w, b if bias else None, out, act, plan)
        check_rows(out, h, wide)
    kernels.check_status()


@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("T,plan", [(1, None), (9, None), (30, (1, 256, 1)), (90, (1, 256, 1)), (200, (1, 256, 1)), (200, (2, 256, 1))])
def test_gated_scales_are_of_the_sums_as_they_are(T, plan, act):
    """Largest magnitudes a few millionths off where the scale doubles, of sums that the tensor cores cut off by as much.  The activation of a
    large gate is the gate; roundings of the gate, of up, of their product and of the quotient are 5 times 2^-24 at most."""
    from qwen_decoder_b200 import kernels
    K, blocks = 8192, 40
    F = 128 * blocks
    g = generator(T, K, act)
    x = rows_of(numbers((1, K), g, spread=5).abs().expand(T, K).contiguous())
    w = torch.zeros((2 * F, K), device=DEV)
    at = torch.randint(0, 128, (blocks,), generator=g, device=DEV) + 128 * torch.arange(blocks, device=DEV)      # the feature that counts
    w[at] = numbers((blocks, K), g, spread=5).abs() * 64 / K
    w[at + F] = numbers((blocks, K), g, spread=5).abs() * 64 / K
    w = rows_of(w)
    z = (value(x)[:1] @ value(w).T)[0]
    gate, up = z[at], z[at + F]
    # biases that bring up to where the product is so many millionths beyond 1.75 times a power of two
    off = torch.linspace(-4e-6, 4e-6, blocks, device=DEV, dtype=torch.float64)
    bias = torch.zeros(2 * F, device=DEV)
    bias[at] = torch.clamp(30 - gate, min=0).float()
    gate = gate + bias[at].double()
    edge = 1.75 * torch.exp2(torch.floor(torch.log2(gate * up / 1.75)))
    bias[at + F] = (edge * (1 + off) / gate - up).float()
    h = gate * (up + bias[at + F].double())
    far = (h / edge - 1).abs() > 5 * 2.0 ** -24
    assert far.sum() > 30
    out = room(T, F)
    kernels.gemm_fp8_gated(x, w, bias, out, act, plan)
    s = out.s.float().double()
    assert (s == torch.where(h > edge, 2 * edge / 448, edge / 448))[:, far].all()
    kernels.check_status()


def test_few_tokens_and_several_tiles_to_a_cta():
    from qwen_decoder_b200 import kernels
    for T in (1, 8, 13):
        x, w, bias = operands(T, 12345, 700)
        out = torch.empty(T, 12345, device=DEV)
        kernels.gemm_fp8(x, w, bias, out, kernels.FP8_FEW)
        want = value(x) @ value(w).T + bias.double()
        assert ((out.double() - want).abs() <= 2.0 ** -23 * want.abs() + sums_off(x, w)).all()


@pytest.mark.parametrize("T,plan", [(5, (1, 256, 1)), (40, (1, 256, 1)), (140, (2, 256, 1)), (140, (1, 256, 1))])
def test_no_numbers_and_infinities_in_a_gated_product(T, plan):
    """A block that holds one makes its rows' sums none and the result's whole blocks with them; sums that are infinite do the same, but for
    gates of minus infinity, which close."""
    from qwen_decoder_b200 import kernels
    F = 300
    x, w, _ = operands(T, 2 * F, 384)
    clean = room(T, F)
    kernels.gemm_fp8_gated(x, w, None, clean, 0, plan)
    x.s.view(torch.uint8)[2, 1] = 255
    w.s.view(torch.uint8)[130, 0] = 255                    # a row of the gate, of the second block of features
    bias = torch.zeros(2 * F, device=DEV)
    bias[299] = -float("inf")                              # a closed gate, of the third
    out = room(T, F)
    kernels.gemm_fp8_gated(x, w, bias, out, 0, plan)
    none = torch.zeros(T, 3, dtype=torch.bool, device=DEV)
    none[2], none[:, 1] = True, True
    assert torch.equal(out.s.float().isnan(), none)
    rows = [r for r in range(T) if r != 2]
    assert torch.equal(out.q[rows, :128].view(torch.uint8), clean.q[rows, :128].view(torch.uint8))
    assert (out.q[rows, 299].float() == 0).all() and out.q[2].float().isnan().all()
    kernels.check_status()


def test_rows_behind_the_end_are_not_taken():
    """Numbers that end within 16 bytes, and rows of a larger matrix: what lies behind them, here no numbers, is in no sum."""
    from qwen_decoder_b200 import kernels
    x, w, _ = operands(7, 40, 389)
    wide = lambda r: kernels.Fp8Rows(torch.nn.functional.pad(r.q.view(torch.uint8), (0, 400 - 389), value=0x7f)[:, :389].view(torch.float8_e4m3fn), r.s)  # noqa: E731
    want = value(x) @ value(w).T
    for plan in (kernels.FP8_FEW, (1, 64, 1), (1, 32, 2)):
        out = torch.empty(7, 40, device=DEV)
        kernels.gemm_fp8(wide(x), wide(w), None, out, plan)
        assert ((out.double() - want).abs() <= 2.0 ** -23 * want.abs() + sums_off(x, w)).all(), plan


def test_products_of_several_tiles_to_a_worker():
    """More tiles than multiprocessors: accumulators in turn, with whole and with overlapping columns, in both forms."""
    from qwen_decoder_b200 import kernels
    x, w, _ = operands(520, 19000, 256)
    want, off = value(x) @ value(w).T, sums_off(x, w)
    for plan in ((1, 256, 1), (2, 256, 1), (1, 32, 1), (2, 224, 1), (1, 240, 1)):
        out = torch.empty(520, 19000, dtype=torch.bfloat16, device=DEV)
        kernels.gemm_fp8(x, w, None, out, plan)
        assert ((out.double() - want).abs() <= 2.0 ** -8 * want.abs() + off).all(), plan
    out = torch.empty(520, 19000, device=DEV)
    kernels.gemm_fp8(x, w, None, out, (2, 128, 1))
    assert ((out.double() - want).abs() <= off).all()
    h = gated(want[:, :9500], want[:, 9500:], 0)
    wide = 1.2 * off[:, :9500] * want[:, 9500:].abs() + (want[:, :9500].abs() + off[:, :9500]) * off[:, 9500:] + 2.0 ** -20 * (want[:, :9500] * want[:, 9500:]).abs()
    for plan in ((1, 256, 1), (2, 256, 1)):
        rows = room(520, 9500)
        kernels.gemm_fp8_gated(x, w, None, rows, 0, plan)
        check_rows(rows, h, wide)
    kernels.check_status()


@pytest.mark.parametrize("plan", [None, (0, 0, 0), (1, 64, 1), (1, 96, 3)])
def test_a_block_of_no_numbers_reaches_its_rows_sums_alone(plan):
    from qwen_decoder_b200 import kernels
    x, w, _ = operands(5, 70, 384)
    x.s.view(torch.uint8)[2, 1] = 255
    w.s.view(torch.uint8)[64, 0] = 255
    out = torch.empty(5, 70, device=DEV)
    kernels.gemm_fp8(x, w, None, out, plan)
    none = torch.zeros(5, 70, dtype=torch.bool, device=DEV)
    none[2], none[:, 64] = True, True
    assert torch.equal(out.isnan(), none)


@pytest.mark.parametrize("T, plan, gated_one", [(4, None, False), (64, None, False), (300, None, False), (4, (1, 128, 4), False),
                                                (12, (0, 0, 0), False), (4, None, True), (64, None, True), (300, None, True)])
def test_weights_that_the_launches_before_write(T, plan, gated_one):
    """Both operands rounded right before the product, which must not read either earlier: results as of the same operands at rest."""
    from qwen_decoder_b200 import kernels
    N, K = 4096, 4096
    g = generator(T, 7)
    x, w = numbers((T, K), g).bfloat16(), numbers((N, K), g).bfloat16()
    xr, wr = room(T, K), room(N, K)

    def product():
        if gated_one:
            out = room(T, N // 2)
            kernels.gemm_fp8_gated(xr, wr, None, out)
            return out.q.view(torch.uint8), out.s.view(torch.uint8)
        out = torch.empty((T, N), device="cuda")
        kernels.gemm_fp8(xr, wr, None, out, plan)
        return (out,)

    kernels.quantize_fp8(x, xr)
    kernels.quantize_fp8(w, wr)
    torch.cuda.synchronize()
    want = product()
    zeros = torch.zeros_like(w)
    for order in range(8):
        kernels.quantize_fp8(zeros, wr)
        torch.cuda.synchronize()
        for rows, source in ((wr, w), (xr, x))[::-1 if order % 2 else 1]:
            kernels.quantize_fp8(source, rows)
        for got, wanted in zip(product(), want):
            assert torch.equal(got, wanted)


@pytest.mark.parametrize("plan", [(0, 0, 0), (1, 64, 1), (1, 96, 3)])
def test_rows_apart_and_scales_apart(plan):
    from qwen_decoder_b200 import kernels
    x, w, _ = operands(9, 100, 384)
    apart = lambda t, n: torch.cat([t.view(torch.uint8), torch.full((t.shape[0], n), 0x7f, dtype=torch.uint8, device=DEV)], 1)[:, :t.shape[1]].view(t.dtype)  # noqa: E731
    a, b = torch.empty(9, 100, device=DEV), torch.empty(9, 100, device=DEV)
    kernels.gemm_fp8(x, w, None, a, plan)
    kernels.gemm_fp8(kernels.Fp8Rows(apart(x.q, 16), apart(x.s, 5)), kernels.Fp8Rows(apart(w.q, 48), apart(w.s, 1)), None, b, plan)
    assert torch.equal(a, b)


def test_on_another_stream_and_in_a_graph():
    from qwen_decoder_b200 import kernels
    g = generator(3)
    x, w, gu = numbers((40, 512), g), operands(40, 256, 512)[1], operands(40, 600, 512)[1]
    first, second, out = room(40, 512), room(40, 300), torch.empty(40, 256, device=DEV)

    def chain():
        kernels.add_rmsnorm_fp8(x, None, torch.ones(512, device=DEV), first, 1e-6)
        kernels.gemm_fp8(first, w, None, out)
        kernels.gemm_fp8_gated(first, gu, None, second)

    chain()
    torch.cuda.synchronize()
    want, rows = out.clone(), second.q.view(torch.uint8).clone()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out.zero_()
        chain()
    side.synchronize()
    assert torch.equal(out, want) and torch.equal(second.q.view(torch.uint8), rows)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        chain()
    out.zero_()
    second.q.view(torch.uint8).zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(second.q.view(torch.uint8), rows)


def test_nothing_to_do():
    from qwen_decoder_b200 import kernels
    w = operands(1, 64, 256)[1]
    none = room(0, 256)
    kernels.quantize_fp8(torch.empty(0, 256, device=DEV), none)
    kernels.gemm_fp8(none, w, None, torch.empty(0, 64, device=DEV))
    kernels.gemm_fp8_gated(none, w, None, room(0, 32))
    kernels.add_rmsnorm_fp8(torch.empty(0, 256, device=DEV), None, torch.ones(256, device=DEV), none, 1e-6)
    torch.cuda.synchronize()
