"""The cache in 8 bits at the ends of its ranges: numbers of every size, scratch memory of exactly the size asked for, launches counted."""
import ctypes
import math
import os
import subprocess
import sys

import pytest
import torch

import plain_fp8_cache as plain
from qwen_decoder_b200 import kernels
from test_fp8_cache_engine_gpu import folder, runner_of
from test_fp8_cache_gpu import a_cache, check_prefill, check_write

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def int32(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def test_write_of_the_largest_and_the_smallest_numbers(guard_regions):
    """Every scale that there is, from 2^-126 to that of the largest float32 number; q is zeros."""
    H, G, d, ps = 1, 1, 64, 16
    gen = torch.Generator().manual_seed(41)
    x = torch.zeros((255, 3 * d))
    sizes = torch.exp2(torch.arange(-126, 129, dtype=torch.float64)).clamp(max=torch.finfo(torch.float32).max)
    x[:, d:] = (sizes[:, None] * (torch.rand((255, 2 * d), generator=gen, dtype=torch.float64) * 2 - 1)).float()
    x[:, d + 7] = x[:, 2 * d + 9] = sizes.float()
    x[-1, 2 * d + 9] = -torch.finfo(torch.float32).max
    check_write(x, None, H, G, d, 0, True, ps, torch.randperm(255, generator=gen).to(torch.int32), 16)


def test_launches_are_counted():
    """As the kernels are: in clusters one, dealt out with the one that joins, a round of 1,024 tokens after the other."""
    gen, H, G, d, ps = torch.Generator().manual_seed(42), 7, 1, 128, 16
    pages, table = (t.to(DEV) for t in a_cache(gen, [2048, 40], G, ps, d))
    wide = torch.cat([table, torch.full((2, 2000), -1, dtype=torch.int32, device=DEV)], 1)
    q, out = (torch.zeros((1200, H * d), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    zeros = torch.zeros(1200, dtype=torch.int32, device=DEV)

    def launched(call):
        count = kernels.launches()
        call()
        return kernels.launches() - count

    decode = lambda T, table, keys: launched(lambda: kernels.decode_attention_fp8(q[:T], out[:T], pages, table, zeros[:T], zeros[:T], H, G, d, ps, 0.1, 0, keys))
    assert [decode(1, table, 2048), decode(1, wide, None), decode(1150, table, 2048), decode(1024, table, 2048)] == [1, 2, 3, 1]
    prefill = lambda T, table: launched(lambda: kernels.prefill_attention_fp8(q[:T], out[:T], pages, table[:1], int32([0, T]), zeros[:1], H, G, d, ps, 0.1))
    assert [prefill(300, table[:, :20]), prefill(3, wide)] == [1, 2]
    assert launched(lambda: kernels.rope_kv_write_fp8(torch.zeros((4, 9 * d), device=DEV), None, q[:4], H, G, d, 0, 1, None, None, zeros[:4], pages, zeros[:4] - 1, ps)) == 1


@pytest.mark.parametrize("size", ["64", "128"])
def test_native_prompt_steps_count_what_the_parts_do(size, tmp_path):
    """Both launch the same kernels: prompts alone, behind cached tokens (shares of keys and their join) and beside single tokens."""
    from qwen_decoder_b200.engine import StepEntry
    path, got = folder(size, tmp_path, projection_dtype="float8_e4m3", max_position_embeddings=8192), []
    for native in (True, False):
        runner = runner_of(path, num_pages=600)
        if not native:
            runner.model.native_prompt = None
        a, b, counts = runner.open("a"), runner.open("b"), []
        for entries in ([(a, 4000)], [(a, 3)], [(a, 1), (b, 300)], [(a, 5), (b, 1)]):
            count = kernels.launches()
            runner.step([StepEntry(c, [7] * n, [n - 1]) for c, n in entries])
            counts.append(kernels.launches() - count)
        got.append(counts)
    assert got[0] == got[1]


@pytest.mark.parametrize("H,G,d", [(16, 2, 128), (28, 4, 128), (14, 2, 64), (11, 1, 64)])
@pytest.mark.parametrize("tokens,before,window,columns", [([130], [0], 0, 0), ([20, 1, 37], [0, 200, 3], 0, 0), ([300, 2], [100, 511], 100, 0), ([37], [4000], 0, 0),
                                                          ([3, 40], [9000, 10], 0, 0), ([5, 9], [30, 200], 0, 3000)])
def test_portions_weights_are_float16(guard_regions, H, G, d, tokens, before, window, columns):
    """Where scales are near one another weights are off by half a step of float16; on scratch of exactly the size asked for, no numbers before."""
    gen, ps, T = torch.Generator().manual_seed(43), 16, sum(tokens)
    pages, table = a_cache(gen, [b + t for b, t in zip(before, tokens)], G, ps, d)
    if columns:
        table = torch.cat([table, torch.full((len(tokens), columns), -1, dtype=torch.int32)], 1)
    q = torch.randn((T, H * d), generator=gen).bfloat16()
    reqs = [r for r, t in enumerate(tokens) for _ in range(t)]
    positions = [b + i for b, t in zip(before, tokens) for i in range(t)]
    want, bound = plain.attention(q, pages, table, reqs, positions, H, G, d, ps, d ** -0.5, window, plain.FP16_HALF_STEP)
    lib, LL, R, keys = kernels.library("attention_fp8_chunk"), ctypes.c_longlong, len(tokens), table.shape[1] * ps
    lib.qd_prefill_attention_fp8_scratch.restype = LL
    floats = lib.qd_prefill_attention_fp8_scratch(T, R, H, G, d, window, keys, kernels.sm_count())
    assert (floats > 0) == (columns > 0 or keys > 1000)
    scratch = torch.full((max(floats, 4),), math.nan, device=DEV)
    args = q.to(DEV), torch.empty((T, H * d), dtype=torch.bfloat16, device=DEV), pages.to(DEV), table.to(DEV), int32([0] + tokens).cumsum(0).to(torch.int32), int32(before)
    qd, out, pd, td, cu, start = args
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    code = lib.qd_prefill_attention_fp8(at(qd), LL(H * d), at(out), LL(H * d), at(pd), LL(len(pd)), at(td), table.shape[1], at(cu), at(start), R, T, T, H, G, d, ps,
                                        ctypes.c_float(d ** -0.5), window, keys, at(scratch) if floats else None, kernels.sm_count(),
                                        ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert code == 0
    kernels.check_status()
    off = (out.cpu().double() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    other = torch.empty_like(out)
    kernels.prefill_attention_fp8(qd, other, *args[2:], H, G, d, ps, d ** -0.5, window)
    assert torch.equal(out, other)


FIRST = """
import sys, torch
sys.path[:0] = {paths!r}
import plain_fp8_cache as plain
from qwen_decoder_b200 import kernels
H, G, d, ps, DEV = 4, 2, 64, 16, "cuda:0"
pages = plain.filled_pages(torch.Generator().manual_seed(0), 400, G, ps, d).to(DEV)
i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)
table, zeros, positions, slots = torch.arange(400, dtype=torch.int32, device=DEV).view(1, 400), i32([0, 0, 0]), i32([3, 50, 6000]), i32([1, 2, 3])
x, out = torch.randn((3, 8 * d), device=DEV).bfloat16(), torch.zeros((3, H * d), dtype=torch.bfloat16, device=DEV)
q, f, z, cu = x[:, :H * d], torch.full((3,), 0.5, device=DEV), torch.randn((3, 5000), device=DEV), i32([0, 3])
call = {{"write": lambda: kernels.rope_kv_write_fp8(x, None, out, H, G, d, 0, 1, None, None, positions, pages, slots, ps),
         "decode": lambda: kernels.decode_attention_fp8(q, out, pages, table, zeros, positions, H, G, d, ps, 0.1),
         "prefill": lambda: kernels.prefill_attention_fp8(q, out, pages, table, cu, positions[2:], H, G, d, ps, 0.1),
         "sample": lambda: kernels.sample_nucleus(z, f, zeros, f, f, f, out[0, :6].view(torch.int32))}}[sys.argv[1]]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call()
out.zero_()
graph.replay()
first = out.clone()
call()
assert torch.equal(first, out) and (sys.argv[1] == "sample" or float(out.float().abs().sum()) > 0)
kernels.check_status()
print("captured first")
"""


@pytest.mark.parametrize("which", ["write", "decode", "prefill", "sample"])
def test_a_process_first_call_may_be_captured(which):
    here = os.path.dirname(os.path.abspath(__file__))
    got = subprocess.run([sys.executable, "-c", FIRST.format(paths=[os.path.dirname(here), here]), which], capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "captured first" in got.stdout, got.stderr[-2000:]


def test_a_wait_of_single_tokens_that_runs_out():
    kernels.check_status()
    kernels.wait_probe("attention_fp8_decode")
    with pytest.raises(kernels.KernelError, match="attention_fp8_decode"):
        kernels.check_status()
    kernels.check_status()
