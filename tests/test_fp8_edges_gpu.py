"""Operators in 8 bits where their calls are unusual: pairs of which one CTA has no rows, operands that the launch before writes, a row alone
and among others, scales and numbers of blocks whose largest magnitude lies where the scale doubles, deep gates."""
import pytest
import torch

from test_fp8_gpu import DEV, check_rows, gated, operands, room, sums_off, value

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
