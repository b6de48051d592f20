"""Single tokens over a cache in 8 bits, however a call of them is cut: rounds, lengths far below what the call allows for, scratch memory that holds no
numbers before."""
import ctypes
import math

import pytest
import torch

import plain_fp8_cache as plain
from qwen_decoder_b200 import kernels
from test_fp8_cache_gpu import a_cache, both_kernels

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def launch(q, pages, table, reqs, positions, H, G, d, ps, window, max_keys):
    """The launcher on scratch of exactly the size that it asks for, no numbers before."""
    lib, T, LL = kernels.library("attention_fp8_decode"), len(reqs), ctypes.c_longlong
    lib.qd_decode_attention_fp8_scratch.restype = LL
    floats = lib.qd_decode_attention_fp8_scratch(T, H, G, d, window, max_keys, kernels.sm_count())
    scratch = torch.full((max(floats, 4),), math.nan, device=DEV)
    out = torch.full((T, H * d), 7.0, dtype=torch.bfloat16, device=DEV)
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    code = lib.qd_decode_attention_fp8(at(q), LL(q.stride(0)), at(out), LL(out.stride(0)), at(pages), LL(len(pages)), at(table), table.shape[1], table.shape[0], at(reqs),
                                       at(positions), T, H, G, d, ps, ctypes.c_float(d ** -0.5), window, max_keys, at(scratch) if floats else None,
                                       kernels.sm_count(), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert code == 0
    return out, floats


def check(lengths, H, G, d, ps=16, window=0, reqs=None, positions=None, max_keys=None, columns=0, seed=0, dealt=None):
    """Through the entry point and through the launcher; ``columns``: of the table, at least (no pages behind the requests' own)."""
    gen = torch.Generator().manual_seed(seed)
    pages, table = a_cache(gen, lengths, G, ps, d)
    if columns > table.shape[1]:
        table = torch.cat([table, torch.full((len(lengths), columns - table.shape[1]), -1, dtype=torch.int32)], 1)
    reqs = list(range(len(lengths))) if reqs is None else reqs
    positions = [lengths[r] - 1 for r in reqs] if positions is None else positions
    q = torch.randn((len(reqs), H * d), generator=gen).bfloat16()
    want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, window, plain.FP16_HALF_STEP)
    args = q.to(DEV), pages.to(DEV), table.to(DEV), int32(reqs), int32(positions)
    out = torch.empty((len(reqs), H * d), dtype=torch.bfloat16, device=DEV)
    kernels.decode_attention_fp8(args[0], out, *args[1:], H, G, d, ps, d ** -0.5, window, max_keys)
    other, floats = launch(*args, H, G, d, ps, window, table.shape[1] * ps if max_keys is None else max_keys)
    kernels.check_status()
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), divmod(int((off / bound).argmax()), H * d))
    assert torch.equal(out, other)
    assert dealt is None or (floats > 0) == dealt


@pytest.mark.parametrize("H,G,d,T,window", [(28, 4, 128, 1050, 0), (14, 2, 64, 1080, 0), (7, 1, 128, 1130, 0), (40, 8, 128, 1036, 0), (28, 4, 128, 1050, 1700), (14, 2, 64, 2100, 0)])
def test_rounds_with_plans_of_their_own(guard_regions, H, G, d, T, window):
    """1,024 tokens go in clusters, what is left over is dealt out."""
    gen = torch.Generator().manual_seed(T)
    left = T % 1024
    positions = torch.randint(-1, 40, (T - left,), generator=gen).tolist() + torch.randint(1200, 2048, (left,), generator=gen).tolist()
    check([40, 2048], H, G, d, reqs=[0] * (T - left) + [1] * left, positions=positions, max_keys=2048, window=window, dealt=True)


def test_scratch_that_is_missing():
    """A call that takes scratch memory is refused without."""
    lib, LL = kernels.library("attention_fp8_decode"), ctypes.c_longlong
    q, out = (torch.zeros((1, 7 * 128), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    pages, table, zero = kernels.fp8_pages(2, 1, 16, 128, DEV), torch.zeros((1, 4000), dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    code = lib.qd_decode_attention_fp8(at(q), LL(896), at(out), LL(896), at(pages), LL(2), at(table), 4000, 1, at(zero), at(zero), 1, 7, 1, 128, 16, ctypes.c_float(0.1), 0,
                                       64000, None, kernels.sm_count(), None)
    assert code == kernels.ERR_UNSUPPORTED
    lib = kernels.library("attention_fp8_chunk")
    cu = int32([0, 1])
    code = lib.qd_prefill_attention_fp8(at(q), LL(896), at(out), LL(896), at(pages), LL(2), at(table), 4000, at(cu), at(zero), 1, 1, 1, 7, 1, 128, 16, ctypes.c_float(0.1), 0,
                                        64000, None, kernels.sm_count(), None)
    assert code == kernels.ERR_UNSUPPORTED
    torch.cuda.synchronize()


@pytest.mark.parametrize("lengths,H,G,d,keys", [([1001], 28, 4, 128, 100001), ([8001], 28, 4, 128, 32768), ([5001, 5001], 14, 2, 64, 65536), ([16385], 16, 2, 128, 17408),
                                                ([200] * 3, 7, 1, 128, 40000), ([1], 28, 4, 128, 100001), ([300] * 40, 8, 2, 64, 30000)])
def test_tokens_alike_far_below_the_most(guard_regions, lengths, H, G, d, keys):
    """More CTAs than the keys have units, since the call allows for more keys than there are."""
    check(lengths, H, G, d, columns=-(-keys // 16), dealt=True)
    check(lengths, H, G, d, columns=-(-keys // 16), max_keys=keys - 5, window=700 if keys > 50000 else 0, dealt=None)


def test_replays_of_other_lengths(guard_regions):
    """One captured call that is dealt out, replayed with lengths short, long, alike and not."""
    gen, H, G, d, ps = torch.Generator().manual_seed(12), 14, 2, 64, 16
    pages, table = a_cache(gen, [9000, 9000, 9000], G, ps, d)
    q = torch.randn((3, H * d), generator=gen).bfloat16()
    args = pages.to(DEV), table.to(DEV), torch.arange(3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    qd, out = q.to(DEV), torch.empty((3, H * d), dtype=torch.bfloat16, device=DEV)
    call = lambda: kernels.decode_attention_fp8(qd, out, *args, H, G, d, ps, d ** -0.5, 0, 9000)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for positions in ([8999, 8999, 8999], [3, 3, 3], [0, 8000, 17], [500, 500, 500], [-1, -1, -1], [2500, 2500, -1], [100, 100, 100], [8999, 1, 1]):
        args[3].copy_(torch.tensor(positions, dtype=torch.int32))
        out.fill_(7.0)
        graph.replay()
        want, bound = plain.attention(q, pages, table, [0, 1, 2], positions, H, G, d, ps, d ** -0.5, 0, plain.FP16_HALF_STEP)
        off = (out.cpu().double() - want).abs()
        assert bool((off <= bound).all()), (positions, float((off / bound).max()))


@pytest.mark.parametrize("keys,dealt", [(16, False), (3000, False), (9000, True)])
def test_positions_far_below_zero(guard_regions, keys, dealt):
    """Any position below zero is a token that sees nothing."""
    positions = [-1, -2 ** 31, keys - 1, -2 ** 31 + 100, -200, 3, -2 ** 31 + 15]
    check([keys], 14, 2, 64, reqs=[0] * 7, positions=positions, dealt=dealt)
    check([keys], 14, 2, 64, reqs=[0] * 7, positions=positions, window=5)


@pytest.mark.parametrize("by", [110, -60])
@pytest.mark.parametrize("H,G,d", [(8, 2, 128), (4, 2, 64), (12, 1, 64)])
def test_keys_times_a_power_of_two_and_queries_over_it(guard_regions, H, G, d, by):
    """Scores are what they are however large or small keys alone are."""
    gen, ps, lengths = torch.Generator().manual_seed(24), 16, [300, 23]
    pages, table = a_cache(gen, lengths, G, ps, d)
    scales = kernels.fp8_page_views(pages, G, ps, d)[1].view(torch.uint8)
    scales[..., 0] = (scales[..., 0].int() + by).to(torch.uint8)
    q = (torch.randn((23, H * d), generator=gen) * 2.0 ** -by).bfloat16()
    reqs, positions, *got = both_kernels(q, pages, table, [20, 3], [280, 20], H, G, d, ps)
    want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, 0, plain.FP16_HALF_STEP)
    for out in got:
        assert bool(((out - want).abs() <= bound).all())
