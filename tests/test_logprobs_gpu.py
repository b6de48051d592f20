"""Log probabilities of tokens (``csrc/logprobs.cu``) against float64: ties, masks, rows in order, rows of nothing, odd sizes and strides."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("guard_regions")]
DEV = "cuda:0"
INF = math.inf


def check(z, tokens, top):
    from qwen_decoder_b200 import kernels
    lp, entropy, ids, tops = (t.cpu() for t in kernels.token_logprobs(z, tokens, top))
    z, tokens = z.double().cpu(), tokens.long().cpu()
    V = z.shape[1]
    m = z.amax(1, keepdim=True)
    shift = torch.where(z == -INF, z, z - torch.where(m == -INF, torch.zeros_like(m), m))
    e = torch.exp(shift)
    S = e.sum(1, keepdim=True)
    log_p = torch.where(S > 0, shift - torch.log(S), torch.full_like(z, -INF))
    terms = torch.where(e > 0, e * shift, torch.zeros_like(e))
    H = torch.where(S[:, 0] > 0, torch.log(S[:, 0]) - terms.sum(1) / S[:, 0], torch.zeros(z.shape[0], dtype=torch.float64))
    # a thread adds up to V / 256 + 16 terms, then 8 levels and 8 CTAs; a term's exponential 2^-20; the sum's relative error is the logarithm's
    eps = (V / 256 + 64) * 2.0 ** -24 + 2.0 ** -20
    off = lambda p: eps + 2.0 ** -22 * (p.abs() + torch.log(S.clamp(min=1)))     # noqa: E731
    want = log_p.gather(1, tokens[:, None])
    assert torch.equal(want[:, 0] == -INF, lp == -INF)
    assert ((lp[:, None].double() - want).abs() <= off(want)).masked_fill(want == -INF, True).all()
    assert ((entropy.double() - H).abs() <= 3 * eps * (1 - terms.sum(1) / S[:, 0].clamp(min=1)) + 2.0 ** -21 * (1 + torch.log(S[:, 0].clamp(min=1)))).all()
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top]        # of equal ones the lowest index first
    assert torch.equal(ids.long(), order)
    want = log_p.gather(1, order)
    assert torch.equal(want == -INF, tops == -INF)
    assert ((tops.double() - want).abs() <= off(want)).masked_fill(want == -INF, True).all()


def some(R, V, seed=0):
    return torch.randint(0, V, (R,), generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=torch.int32)


def normal(R, V, std=2.5):
    return torch.empty(R, V, device=DEV).normal_(0, std, generator=torch.Generator(device=DEV).manual_seed(R * 7 + V))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("R,V,top", [(1, 1, 0), (1, 1, 1), (2, 31, 31), (3, 257, 32), (1, 4096, 5), (5, 4097, 1), (2, 8192, 20), (1, 151936, 20),
                                     (9, 50001, 7), (70, 32000, 0), (160, 20000, 3), (700, 5000, 32)])
def test_random_rows(R, V, top, dtype):
    check(normal(R, V).to(dtype), some(R, V), top)


@pytest.mark.parametrize("top", [1, 8, 9, 32])
@pytest.mark.parametrize("kind", ["equal", "rising", "falling", "steps", "peak", "two values", "zeros of both signs", "lowest"])
def test_rows_in_order(kind, top):
    V = 33000
    i = torch.arange(V, device=DEV, dtype=torch.float32)
    row = {"equal": 0 * i + 3, "rising": i / 1024, "falling": -i / 1024, "steps": torch.floor(i / 4096), "peak": -(i - 20000).abs() / 64,
           "two values": (i % 3 == 0).float(), "zeros of both signs": torch.where(i % 2 == 0, -0.0 * i, 0 * i),
           "lowest": torch.full_like(i, torch.finfo(torch.float32).min)}[kind]
    for R in (1, 3, 400):
        check(row.repeat(R, 1), some(R, V), top)


def test_masks():
    V = 20000
    z = torch.full((5, V), -INF, device=DEV)
    z[0, 17], z[0, 19999] = 1.0, 2.0                       # two tokens left
    z[1, 5] = -300.0                                       # one
    z[2] = torch.where(torch.arange(V, device=DEV) % 10 == 3, normal(1, V)[0], z[2])
    z[3, :4] = torch.finfo(torch.float32).min              # the type's lowest value among infinities
    # (row 4: none)
    check(z, torch.tensor([17, 5, 0, 2, 9], dtype=torch.int32, device=DEV), 6)


def test_large_logits_and_small_differences():
    z = normal(4, 10000, 1e-4) + 1000.0
    z[1] *= 1e30
    z[2] = normal(1, 10000)[0] * 1e4
    check(z, some(4, 10000), 4)


def test_no_numbers_and_infinities():
    from qwen_decoder_b200 import kernels
    z = normal(4, 9000)
    clean = z.clone()
    z[1, 8000], z[2, 3] = float("nan"), INF
    got = kernels.token_logprobs(z, some(4, 9000), 5)
    want = kernels.token_logprobs(clean, some(4, 9000), 5)
    for g, w in zip(got[:2] + got[3:], want[:2] + want[3:]):
        assert g[[1, 2]].isnan().all() and torch.equal(g[[0, 3]], w[[0, 3]])
    assert got[2][2, 0] == 3 and torch.equal(got[2][[0, 1, 3]], want[2][[0, 1, 3]])
    only = torch.full((1, 300), float("nan"), device=DEV)
    only[0, 7] = 1.0
    ids = kernels.token_logprobs(only, some(1, 300), 3)[2]
    assert ids.tolist() == [[7, -1, -1]]


def test_tokens_outside_of_the_row():
    from qwen_decoder_b200 import kernels
    z = normal(3, 500)
    lp = kernels.token_logprobs(z, torch.tensor([-1, 500, 499], dtype=torch.int32, device=DEV))[0]
    assert lp.isnan().tolist() == [True, True, False]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("first,pad", [(0, 8), (1, 0), (3, 5)])
def test_rows_apart(first, pad, dtype):
    z = normal(6, 12000 + first + pad).to(dtype)[:, first:12000 + first]
    check(z, some(6, 12000), 9)


def test_a_row_alone_and_among_others():
    """How many rows there are decides how many CTAs share one; the ids are the same, the sums within their rounding."""
    from qwen_decoder_b200 import kernels
    z, t = normal(600, 9000), some(600, 9000)
    many, one = kernels.token_logprobs(z, t, 8), kernels.token_logprobs(z[5:6], t[5:6], 8)
    assert torch.equal(many[2][5:6], one[2]) and float((many[0][5:6] - one[0]).abs().max()) <= 1e-5
    again = kernels.token_logprobs(z, t, 8)
    assert all(torch.equal(a, b) for a, b in zip(many, again))


def test_nothing_to_do():
    from qwen_decoder_b200 import kernels
    out = kernels.token_logprobs(torch.empty(0, 100, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV), 4)
    assert [tuple(t.shape) for t in out] == [(0,), (0,), (0, 4), (0, 4)]
