"""Tokens by temperature, top-k, top-p and min-p against float64."""
import math

import pytest
import torch

import plain_fp8_cache as plain
from qwen_decoder_b200 import kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# weights are off by 3 2^-44 of the largest each: sums of V, and the whole that they are compared with a share of, which is at least the largest, by V 3 2^-44
NEAR = lambda V: 2 * V * 3 * 2.0 ** -44 + 2.0 ** -43


def run(z, temperature, top_k, top_p, min_p, draws, **kw):
    out = torch.full((len(z),), -7, dtype=torch.int32, device=DEV)
    f = lambda v: torch.tensor(v, dtype=torch.float32, device=DEV)
    kernels.sample_nucleus(z, f(temperature), torch.tensor(top_k, dtype=torch.int32, device=DEV), f(top_p), f(min_p), f(draws), out, **kw)
    return out.tolist()


def check(z, temperature, top_k, top_p, min_p, draws, least=0.75):
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    got = run(z.to(DEV), temperature, top_k, top_p, min_p, draws)
    checked = 0
    for r in range(len(z)):
        want, margin = plain.sample(z[r], f32(temperature[r]), top_k[r], f32(top_p[r]), f32(min_p[r]), f32(draws[r]))
        if margin > NEAR(z.shape[1]):
            checked += 1
            assert got[r] == want, (r, got[r], want, margin)
    assert checked >= len(z) * least
    return got


SETTINGS = [(0.8, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.7, 50, 0.95, 0.0), (1.5, 1500, 0.99, 0.01), (0.3, 1, 0.5, 0.0), (1.0, 0, 0.999, 0.0), (2.0, 20, 1.0, 0.3),
            (0.0, 40, 0.9, 0.1), (1.0, 7, 1.0, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.0), (1.0, 0, 1.0, 5.0), (1e-3, 0, 0.9, 0.0), (50.0, 0, 0.9, 0.0)]


@pytest.mark.parametrize("R,V", [(R, V) for R in (1, 5, 70) for V in (1, 2, 31, 1000, 4097, 32000, 151936) if R < 70 or V < 40000])      # (40 long rows: below)
def test_rows(guard_regions, R, V):
    gen = torch.Generator().manual_seed(V + R)
    z = torch.randn((R, V), generator=gen) * 2.5
    rows = [SETTINGS[(r * 5 + V) % len(SETTINGS)] for r in range(R)]
    check(z, *(list(c) for c in zip(*rows)), torch.rand(R, generator=gen).tolist())


@pytest.mark.parametrize("setting", SETTINGS)
def test_settings(guard_regions, setting):
    gen = torch.Generator().manual_seed(3)
    z = torch.randn((8, 9001), generator=gen) * 2.5
    check(z, *([v] * 8 for v in setting), torch.rand(8, generator=gen).tolist())


def test_many_long_rows(guard_regions):
    """More rows than clusters run at a time, too long for shared memory."""
    gen = torch.Generator().manual_seed(6)
    z = torch.randn((40, 152064), generator=gen) * 2.5
    rows = [SETTINGS[r % len(SETTINGS)] for r in range(40)]
    check(z, *(list(c) for c in zip(*rows)), torch.rand(40, generator=gen).tolist())
    big = torch.randn((150, 60000), generator=gen) * 2.5
    rows = [SETTINGS[r % len(SETTINGS)] for r in range(150)]
    check(big, *(list(c) for c in zip(*rows)), torch.rand(150, generator=gen).tolist())


def test_equal_logits(guard_regions):
    """Rows of one value, of two, of steps: logits that are equal are in or out together."""
    V = 5000
    z = torch.zeros((6, V))
    z[1, 2500:] = 1.0
    z[2] = torch.arange(V).float() // 100 * 0.01
    z[3] = torch.randint(0, 4, (V,), generator=torch.Generator().manual_seed(0)).float()
    z[4, 7] = 1e-30
    z[5] = -0.0
    z[5, 100:] = 0.0
    for k, p, m, u in ((0, 0.5, 0.0, 0.7501), (100, 1.0, 0.0, 0.3), (100, 0.3, 0.0, 0.99999), (0, 1.0, 0.9, 0.123), (1, 0.9, 0.0, 0.5), (0, 0.9, 0.0, 0.0001)):
        check(z, [1.0] * 6, [k] * 6, [p] * 6, [m] * 6, [u] * 6, 0.3)       # (a draw of a half is a border of most)


def test_masked_rows(guard_regions):
    """Masks of minus infinity and of the lowest number, rows that leave one token or nothing, no numbers, infinities."""
    gen = torch.Generator().manual_seed(1)
    V, low = 20000, torch.finfo(torch.float32).min
    z = torch.randn((4, V), generator=gen)
    z[0, 100:] = -math.inf
    z[1, 50:] = low
    z[2] = -math.inf
    z[2, 1234] = -3.0
    z[3, :19990] = low
    check(z, [1.0] * 4, [0, 70, 5, 0], [0.95] * 4, [0.0, 0.01, 0.0, 0.0], [0.3, 0.9, 0.5, 0.99])
    odd = torch.randn((6, V), generator=gen)
    odd[0] = -math.inf
    odd[1, 777] = math.inf
    odd[2, 5:] = math.nan
    odd[3] = math.nan
    odd[4] = low
    odd[5, 3:] = -math.inf
    got = run(odd.to(DEV), [1.0] * 6, [0] * 6, [0.9] * 6, [0.01] * 6, [0.4] * 6)
    assert got[0] == 0 and got[1] == 777 and got[2] in range(5) and got[3] == 0 and got[5] in range(3) and 0 <= got[4] < V
    assert run(odd.to(DEV), [0.0] * 6, [0] * 6, [0.9] * 6, [0.01] * 6, [0.4] * 6)[1] == 777


def test_draws_at_the_ends(guard_regions):
    gen = torch.Generator().manual_seed(2)
    z = torch.randn((4, 3000), generator=gen)
    z[:, 0] = -math.inf
    got = run(z.to(DEV), [1.0] * 4, [0] * 4, [0.9] * 4, [0.0] * 4, [0.0, 1.0 - 2.0 ** -24, 1.0, 2.0])
    kept = []
    for r in range(4):
        p = torch.softmax(z[r].double(), 0)
        order = torch.argsort(p, descending=True)
        n = int((torch.cumsum(p[order], 0) < float(torch.tensor(0.9))).sum()) + 1
        kept.append(sorted(order[:n].tolist()))
    assert got[0] == kept[0][0] and got[1] == kept[1][-1] and got[2] == kept[2][-1] and got[3] == int(z[3].argmax())


def test_rows_apart_misaligned_only_and_graph():
    """Rows that lie apart and off 16 bytes; rows without top-p and min-p left alone; a captured call follows its inputs."""
    gen = torch.Generator().manual_seed(5)
    R, V = 6, 4099
    z = torch.randn((R, V), generator=gen) * 2
    wide = torch.zeros((R, V + 4), device=DEV)
    wide[:, 1:V + 1] = z.to(DEV)
    args = ([0.9] * R, [0, 30] * 3, [0.9, 1.0] * 3, [0.0] * R, torch.rand(R, generator=gen).tolist())
    want = run(z.to(DEV), *args)
    assert run(wide[:, 1:V + 1], *args) == want
    assert run(z.to(DEV), *args, only=True) == [w if i % 2 == 0 else -7 for i, w in enumerate(want)]
    dev = [torch.tensor(a, dtype=t, device=DEV) for a, t in zip(args, (torch.float32, torch.int32, torch.float32, torch.float32, torch.float32))]
    zd, out = z.to(DEV), torch.empty(R, dtype=torch.int32, device=DEV)
    kernels.sample_nucleus(zd, *dev, out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.sample_nucleus(zd, *dev, out)
    zd.copy_(z.flip(1))
    dev[4].copy_(1 - dev[4])
    graph.replay()
    again = torch.empty_like(out)
    kernels.sample_nucleus(zd, *dev, again)
    assert torch.equal(out, again)


def test_a_token_does_not_depend_on_the_rows_beside_it():
    gen = torch.Generator().manual_seed(7)
    z = (torch.randn((1, 151936), generator=gen) * 2.5).expand(90, -1).contiguous().to(DEV)
    u = torch.rand(1, generator=gen).item()
    alone = run(z[:1], [0.8], [0], [0.9], [0.0], [u])[0]
    assert set(run(z, [0.8] * 90, [0] * 90, [0.9] * 90, [0.0] * 90, [u] * 90)) == {alone}
    assert set(run(z[:7], [0.8] * 7, [0] * 7, [0.9] * 7, [0.0] * 7, [u] * 7)) == {alone}
