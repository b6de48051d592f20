"""Operators in 8 bits where their calls are unusual: pairs of which one CTA has no rows, operands that the launch before writes, a row alone
and among others, scales and numbers of blocks whose largest magnitude lies where the scale doubles, deep gates."""
import pytest
import torch

from test_fp8_gpu import DEV, check_rows, gated, operands, room, rows_of, sums_off, value

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("guard_regions")]


@pytest.mark.parametrize("T", [1, 8, 13])
def test_gated_products_of_few_tokens_in_pairs_with_several_tiles(T):
    """Pairs of which the second CTA has no rows (up to 8 tokens) or few, and more tiles than pairs: a tile's sums stay until they have been
    read, whichever CTA has them."""
    from qwen_decoder_b200 import kernels
    F, K = 40000, 384
    x, w, b = operands(T, 2 * F, K)
    z = value(x) @ value(w).T + b.double()
    off = sums_off(x, w) + 2.0 ** -23 * z.abs()
    wide = 1.2 * off[:, :F] * z[:, F:].abs() + (z[:, :F].abs() + off[:, :F]) * off[:, F:] + 2.0 ** -20 * (z[:, :F] * z[:, F:]).abs()
    h = gated(z[:, :F], z[:, F:], 0)
    for _ in range(3):
        for plan in ((2, 256, 1), (1, 256, 1)):
            out = room(T, F)
            kernels.gemm_fp8_gated(x, w, b, out, 0, plan)
            check_rows(out, h, wide)
    kernels.check_status()


@pytest.mark.parametrize("rows,D", [(1, 2048), (3, 8192), (400, 4096), (2, 20000)])
def test_norm_weights_that_the_launch_before_writes(rows, D):
    """A norm whose weights are the sums of the product right before it: as with the same weights at rest."""
    from qwen_decoder_b200 import kernels
    x, gains, _ = operands(1, D, 8192)
    weight = torch.zeros(1, D, device=DEV)
    stream = torch.empty(rows, D, device=DEV).normal_()
    want, out = room(rows, D), room(rows, D)
    kernels.gemm_fp8(x, gains, None, weight)
    torch.cuda.synchronize()
    kernels.add_rmsnorm_fp8(stream, None, weight[0], want, 1e-6)
    for _ in range(8):
        weight.zero_()
        torch.cuda.synchronize()
        kernels.gemm_fp8(x, gains, None, weight)
        kernels.add_rmsnorm_fp8(stream, None, weight[0], out, 1e-6)
        assert torch.equal(out.q.view(torch.uint8), want.q.view(torch.uint8)) and torch.equal(out.s.view(torch.uint8), want.s.view(torch.uint8))


@pytest.mark.parametrize("D,parts,scaled", [(1, 0, False), (517, 3, False), (2048, 0, False), (2048, 4, True), (3584, 0, True), (5000, 0, False),
                                            (8192, 2, False), (20000, 0, True)])
def test_a_row_of_the_norm_alone_and_among_others(D, parts, scaled):
    """Whatever number of rows is normed with it, a row's sum and its 8 bits are the same."""
    from qwen_decoder_b200 import kernels
    T = 700
    x, w = torch.empty(T, D, device=DEV).normal_() * 3, 1 + 0.1 * torch.empty(D, device=DEV).normal_()
    delta = torch.empty(parts, T, D, device=DEV).normal_() if parts else torch.empty(T, D, device=DEV).normal_().bfloat16()
    scale = torch.empty(D, device=DEV).normal_() if scaled else None
    kept, whole = x.clone(), room(T, D)
    kernels.add_rmsnorm_fp8(x, delta, w, whole, 1e-6, delta_scale=scale)
    for at, n in ((0, 1), (5, 1), (699, 1), (100, 148), (100, 300), (200, 500)):
        some, out = kept[at:at + n].clone(), room(n, D)
        kernels.add_rmsnorm_fp8(some, delta[..., at:at + n, :].contiguous(), w, out, 1e-6, delta_scale=scale)
        assert torch.equal(some, x[at:at + n])
        assert torch.equal(out.q.view(torch.uint8), whole.q[at:at + n].view(torch.uint8))
        assert torch.equal(out.s.view(torch.uint8), whole.s[at:at + n].view(torch.uint8))


@pytest.mark.parametrize("T,plan", [(9, (1, 256, 1)), (200, (1, 256, 1)), (200, (2, 256, 1)), (200, None)])
def test_gated_scales_where_all_blocks_are_near_the_edge(T, plan):
    """More blocks to a CTA whose largest magnitude lies where the scale doubles than it keeps: equal rows, hundreds of such blocks in each.
    The activation of a large gate is the gate; roundings of the gate, of up, of their product and of the quotient are 5 times 2^-24 at most."""
    from qwen_decoder_b200 import kernels
    K, blocks = 8192, 3000 if T == 9 else 400
    F = 128 * blocks
    x = rows_of(torch.empty(1, K, device=DEV).normal_().abs().expand(T, K).contiguous())
    some = rows_of(torch.empty(2 * blocks, K, device=DEV).normal_().abs() * 64 / K)       # the features that count: gates, then ups
    at = 128 * torch.arange(blocks, device=DEV) + torch.arange(blocks, device=DEV) * 37 % 128
    w = room(2 * F, K)
    w.q.view(torch.uint8).zero_()
    w.s.view(torch.uint8).fill_(127)
    for part, to in ((slice(0, blocks), at), (slice(blocks, None), at + F)):
        w.q.view(torch.uint8)[to] = some.q.view(torch.uint8)[part]
        w.s.view(torch.uint8)[to] = some.s.view(torch.uint8)[part]
    z = (value(x)[:1] @ value(some).T)[0]
    gate, up = z[:blocks], z[blocks:]
    off = torch.linspace(-3e-6, 3e-6, blocks, device=DEV, dtype=torch.float64)[torch.randperm(blocks, device=DEV)]
    bias = torch.zeros(2 * F, device=DEV)
    bias[at] = torch.clamp(30 - gate, min=0).float()
    gate = gate + bias[at].double()
    edge = 1.75 * torch.exp2(torch.floor(torch.log2(gate * up / 1.75)))
    bias[at + F] = (edge * (1 + off) / gate - up).float()
    h = gate * (up + bias[at + F].double())
    far = (h / edge - 1).abs() > 5 * 2.0 ** -24
    assert far.sum() > 0.8 * blocks
    out = room(T, F)
    kernels.gemm_fp8_gated(x, w, bias, out, 0, plan)
    s = out.s.float().double()
    assert (s == torch.where(h > edge, 2 * edge / 448, edge / 448))[:, far].all()
    assert (out.q[:, at].float() == torch.where(s > (edge / 448)[None], 224.0, 448.0)).all()
    kernels.check_status()


def deep(g, u, act):
    """``gated`` without the cancellation of 1 + tanh."""
    return g * torch.sigmoid(1.5957691216057308 * (g + 0.044715 * g ** 3) if act else g) * u


@pytest.mark.parametrize("act", [0, 2])
def test_deep_gates(act):
    """Gates far below zero, relative to the activation itself, which is tiny beside gate and up: within 6 units of 2^-23 of itself."""
    from qwen_decoder_b200 import kernels
    T, F = 40, 1000
    z = torch.empty(T, 2 * F, device=DEV).normal_()
    low = torch.tensor([10, 20, 40, 60] if act == 0 else [3, 5, 7, 8.5], device=DEV).repeat(T // 4)[:, None]
    z[:, :F] = -low * (1 + 0.2 * torch.rand(T, F, device=DEV))
    out = room(T, F)
    kernels.gate_fp8(z, out, None, act)
    g, u = z[:, :F].double(), z[:, F:].double()
    h = deep(g, u, act)
    check_rows(out, h, 6 * 2.0 ** -23 * h.abs())


@pytest.mark.parametrize("act", [0, 2])
@pytest.mark.parametrize("T,plan", [(3, None), (60, (1, 256, 1)), (200, (2, 256, 1))])
def test_gated_scales_of_deep_gates(T, plan, act):
    """Largest magnitudes of deep gates some ten millionths off where the scale doubles: the activation's own error does not decide."""
    from qwen_decoder_b200 import kernels
    K, blocks = 128, 400
    F = 128 * blocks
    x, w, _ = operands(T, 2 * F, K)
    w.q.zero_()                                            # gate and up are their biases
    at = 128 * torch.arange(blocks, device=DEV) + torch.arange(blocks, device=DEV) % 128
    bias = torch.zeros(2 * F, device=DEV)
    bias[at] = -torch.linspace(10, 80, blocks, device=DEV) if act == 0 else -torch.linspace(2.5, 9, blocks, device=DEV)
    gate = bias[at].double()
    off = torch.linspace(-1e-6, 1e-6, blocks, device=DEV, dtype=torch.float64)[torch.randperm(blocks, device=DEV)]
    bias[at + F] = (1.75 * (1 + off) / deep(gate, 1.0, act)).float()
    h = deep(gate, bias[at + F].double(), act).abs()
    far = (h / 1.75 - 1).abs() > 1e-12
    assert far.sum() > blocks - 10
    out = room(T, F)
    kernels.gemm_fp8_gated(x, w, bias, out, act, plan)
    s = out.s.float().double()
    assert (s == torch.where(h > 1.75, 2.0 ** -7, 2.0 ** -8))[:, far].all()
    kernels.check_status()


@pytest.mark.parametrize("T,plan", [(3, None), (30, (1, 256, 1)), (90, (1, 256, 1)), (200, (2, 256, 1))])
@pytest.mark.parametrize("lower", [False, True])
def test_numbers_of_blocks_whose_scale_is_looked_at_again(lower, T, plan):
    """Beside the largest magnitude near the edge lie some among e4m3's smallest numbers: whichever scale it comes to be, they are rounded once,
    to it.  The tensor cores cut sums off towards zero: a product of sums seems smaller, and ``lower`` one of a gate about -3 larger."""
    from qwen_decoder_b200 import kernels
    K, blocks = 8192, 64
    F = 128 * blocks
    x = rows_of(torch.empty(1, K, device=DEV).normal_().abs().expand(T, K).contiguous())
    some = torch.empty(2 * blocks, K, device=DEV).normal_().abs() * 64 / K       # the features that count: gates, then ups
    if lower:
        some[:blocks] *= -3 / 26
        some[blocks:] = 0
    some = rows_of(some)
    at = 128 * torch.arange(blocks, device=DEV) + torch.arange(blocks, device=DEV) * 37 % 128
    w = room(2 * F, K)
    w.q.view(torch.uint8).zero_()
    w.s.view(torch.uint8).fill_(127)
    for part, to in ((slice(0, blocks), at), (slice(blocks, None), at + F)):
        w.q.view(torch.uint8)[to] = some.q.view(torch.uint8)[part]
        w.s.view(torch.uint8)[to] = some.s.view(torch.uint8)[part]
    z = (value(x)[:1] @ value(some).T)[0]
    gate, up = z[:blocks], z[blocks:]
    # the others: gates of 30, the activation of which is 30, and ups that bring them to 2^-11 to 2^-4 of the scale
    bias = torch.zeros(2 * F, device=DEV)
    bias[:F] = 30
    bias[at] = 0 if lower else torch.clamp(30 - gate, min=0).float()
    closed = gated(gate + bias[at].double(), 1.0, 0)
    edge = 1.75 * torch.exp2(torch.floor(torch.log2(closed.abs() * (1 if lower else up) / 1.75)))
    small = torch.exp2(-11 + 7 * torch.rand(F, device=DEV)) * (1 - 2 * torch.randint(0, 2, (F,), device=DEV))
    bias[F:] = small * (edge / 448).float().repeat_interleave(128) / 30
    off = torch.linspace(-3e-6, 3e-6, blocks, device=DEV, dtype=torch.float64)[torch.randperm(blocks, device=DEV)]
    bias[at + F] = (edge * (1 + off) / closed - up).float()
    g = torch.zeros(2 * F, dtype=torch.float64, device=DEV)
    g[at], g[at + F] = gate, up
    h = gated((g + bias.double())[:F], (g + bias.double())[F:], 0)
    peak = h[at].abs()
    far = (peak / edge - 1).abs() > 1e-10
    assert far.sum() > blocks - 4
    out = room(T, F)
    kernels.gemm_fp8_gated(x, w, bias, out, 0, plan)
    assert (out.s.float().double() == torch.where(peak > edge, 2 * edge / 448, edge / 448))[:, far].all()
    # of the largest the sums' error, of the others the activation's
    check_rows(out, h.expand(T, F), (6 * 2.0 ** -23 * h.abs()).scatter(0, at, 1e-5 * peak).expand(T, F))
    kernels.check_status()


@pytest.mark.parametrize("plan", [[1, 64, 1], (1, 64), (1, 64, 1, 1), (1, "64", 1), (1, 64, 2 ** 40), 64, "plan"])
def test_plans_that_are_none(plan):
    from qwen_decoder_b200 import kernels
    x, w, _ = operands(3, 64, 256)
    with pytest.raises(kernels.KernelError, match="plan"):
        kernels.gemm_fp8(x, w, None, torch.empty(3, 64, device=DEV), plan)
    with pytest.raises(kernels.KernelError, match="plan"):
        kernels.gemm_fp8_gated(x, w, None, room(3, 32), 0, plan)


def test_plans_of_the_current_device():
    from qwen_decoder_b200 import kernels
    for sizes in ((4, 2048, 2048), (40, 4608, 3584), (500, 3584, 18944)):
        assert kernels.gemm_fp8_plan(*sizes) == kernels.gemm_fp8_plan(*sizes, device="cuda") == kernels.gemm_fp8_plan(*sizes, device=torch.device(DEV))


@pytest.mark.parametrize("T,plan", [(3, None), (16, (1, 256, 1)), (30, (1, 256, 1)), (90, (1, 256, 1)), (200, (2, 256, 1))])
def test_blocks_that_several_threads_tell_of(T, plan):
    """Four equal largest magnitudes near the edge in every block, in all quarters of its features: it is looked at again and again, and stays."""
    from qwen_decoder_b200 import kernels
    K, blocks, four = 8192, 90, 4
    F = 128 * blocks
    x = rows_of(torch.empty(1, K, device=DEV).normal_().abs().expand(T, K).contiguous())
    some = rows_of(torch.empty(2 * blocks, K, device=DEV).normal_().abs() * 64 / K)
    at = 128 * torch.arange(blocks, device=DEV)[:, None] + torch.tensor([3, 40, 77, 126], device=DEV)
    w = room(2 * F, K)
    w.q.view(torch.uint8).zero_()
    w.s.view(torch.uint8).fill_(127)
    for part, to in ((slice(0, blocks), at), (slice(blocks, None), at + F)):
        w.q.view(torch.uint8)[to.flatten()] = some.q.view(torch.uint8)[part].repeat_interleave(four, 0)
        w.s.view(torch.uint8)[to.flatten()] = some.s.view(torch.uint8)[part].repeat_interleave(four, 0)
    z = (value(x)[:1] @ value(some).T)[0]
    gate, up = z[:blocks], z[blocks:]
    bias = torch.zeros(2 * F, device=DEV)
    bias[at] = torch.clamp(30 - gate, min=0).float()[:, None]
    gate = gate + bias[at[:, 0]].double()
    edge = 1.75 * torch.exp2(torch.floor(torch.log2(gate * up / 1.75)))
    off = torch.linspace(-2e-6, 2e-6, blocks, device=DEV, dtype=torch.float64)[torch.randperm(blocks, device=DEV)]
    bias[at + F] = (edge * (1 + off) / gate - up).float()[:, None]
    h = gated(gate, up + bias[at[:, 0] + F].double(), 0)
    far = (h / edge - 1).abs() > 1e-10
    assert far.sum() > blocks - 4
    for _ in range(3):
        out = room(T, F)
        kernels.gemm_fp8_gated(x, w, bias, out, 0, plan)
        s = out.s.float().double()
        assert (s == torch.where(h > edge, 2 * edge / 448, edge / 448))[:, far].all()
        assert (out.q[:, at.flatten()].float() == torch.where(s > (edge / 448)[None], 224.0, 448.0).repeat_interleave(four, 1)).all()
        assert (out.q.float() != 0).sum() == T * blocks * four
    kernels.check_status()


@pytest.mark.parametrize("T", [1, 7, 16, 40, 300])
def test_weights_that_rest(T):
    """``resident`` says when weights are read, not what is made of them."""
    from qwen_decoder_b200 import kernels
    x, w, bias = operands(T, 1200, 1000)
    torch.cuda.synchronize()
    for dtype in (torch.bfloat16, torch.float32):
        a, b = torch.empty(T, 1200, dtype=dtype, device=DEV), torch.empty(T, 1200, dtype=dtype, device=DEV)
        kernels.gemm_fp8(x, w, bias, a)
        kernels.gemm_fp8(x, w, bias, b, resident=True)
        assert torch.equal(a, b)
    a, b = room(T, 600), room(T, 600)
    kernels.gemm_fp8_gated(x, w, bias, a)
    kernels.gemm_fp8_gated(x, w, bias, b, resident=True)
    assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.s.view(torch.uint8), b.s.view(torch.uint8))
