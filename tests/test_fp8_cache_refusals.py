"""What the entry points of the cache in 8 bits and of tokens from the nucleus refuse, before anything is launched."""
import pytest
import torch

from qwen_decoder_b200 import kernels
from qwen_decoder_b200.kernels import KernelError

i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)


def test_pages():
    pages = kernels.fp8_pages(3, 2, 16, 64, "cpu")
    assert tuple(pages.shape) == (3, 2 * 16 * 130) == (3, kernels.fp8_page_bytes(2, 16, 64))
    numbers, scales = kernels.fp8_page_views(pages, 2, 16, 64)
    assert tuple(numbers.shape) == (3, 2, 2, 16, 64) and tuple(scales.shape) == (3, 2, 16, 2)
    numbers.view(torch.uint8)[1, 1, 0, 3, 5] = 9
    scales.view(torch.uint8)[1, 1, 4, 1] = 8
    assert int(pages[1, 2 * 16 * 64 + 3 * 64 + 5]) == 9 and int(pages[1, 4 * 16 * 64 + 16 * 2 + 4 * 2 + 1]) == 8


@pytest.mark.parametrize("bad", [(torch.zeros(3, 4160), 2, 16, 64), (torch.zeros(4160, dtype=torch.uint8), 2, 16, 64), (torch.zeros(3, 4161, dtype=torch.uint8), 2, 16, 64),
                                 (torch.zeros(3, 8320, dtype=torch.uint8)[:, ::2], 2, 16, 64), (torch.zeros(3, 4160, dtype=torch.uint8), -2, -16, 64),
                                 (torch.zeros(3, 0, dtype=torch.uint8), 0, 16, 64), (torch.zeros(3, 4160, dtype=torch.uint8), 2, 1 << 31, 64), (None, 2, 16, 64)])
def test_page_views(bad):
    with pytest.raises((KernelError, TypeError)):
        kernels.fp8_page_views(*bad)


def test_page_views_of_rows_apart():
    whole = torch.arange(6 * 4160, dtype=torch.int64).remainder(251).to(torch.uint8).view(6, 4160)
    numbers, scales = kernels.fp8_page_views(whole[1::2], 2, 16, 64)
    assert torch.equal(numbers.view(torch.uint8).flatten(1), whole[1::2, :4096]) and torch.equal(scales.view(torch.uint8).flatten(1), whole[1::2, 4096:])


@pytest.mark.parametrize("H,G,d,ps,ok", [(16, 2, 128, 16, True), (14, 2, 64, 48, True), (17, 1, 128, 16, False), (16, 2, 96, 16, False), (16, 3, 64, 16, False),
                                         (16, 2, 64, 8, False), (16, 2, 64, 0, False), (16, 1, 64, 16, True), (16, 2, 64, 1 << 15, False)])
def test_supported(H, G, d, ps, ok):
    assert kernels.fp8_cache_supported(H, G, d, ps) == ok


def write_args(**kw):
    a = dict(qkv=bf16(3, 512), bias=None, q_out=bf16(3, 256), H=4, G=2, d=64, rotary_dim=64, pairing=1, cos=torch.zeros(9, 32), sin=torch.zeros(9, 32),
             positions=i32(3), pages=kernels.fp8_pages(2, 2, 16, 64, "cpu"), slot_map=i32(3), page_size=16, write_kv=True)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(qkv=bf16(3, 500)), dict(qkv=torch.zeros(3, 512, dtype=torch.float16)), dict(qkv=torch.zeros(0, 3, 512)), dict(qkv=bf16(2, 3, 512)), dict(qkv=bf16(3, 1024)[:, ::2]),
    dict(qkv=bf16(3, 520)[:, :512]), dict(bias=torch.zeros(511)), dict(bias=bf16(512)), dict(q_out=bf16(4, 256)), dict(q_out=torch.zeros(3, 256)), dict(q_out=bf16(3, 264)[:, :256]),
    dict(G=3), dict(d=96), dict(page_size=8), dict(rotary_dim=72), dict(rotary_dim=24), dict(rotary_dim=128), dict(rotary_dim=-16), dict(pairing=2), dict(cos=None),
    dict(cos=torch.zeros(9, 16)), dict(sin=torch.zeros(8, 32)), dict(cos=torch.zeros(9, 32, dtype=torch.float64)), dict(pages=torch.zeros(2, 4160)), dict(pages=None),
    dict(pages=kernels.fp8_pages(2, 2, 16, 128, "cpu")), dict(pages=kernels.fp8_pages(2, 2, 32, 64, "cpu")[:, ::2]), dict(slot_map=None)])
def test_write(bad):
    with pytest.raises(KernelError):
        kernels.rope_kv_write_fp8(**write_args(**bad))


def test_write_needs_a_device():
    with pytest.raises(KernelError, match="CUDA"):
        kernels.rope_kv_write_fp8(**write_args())


def decode_args(**kw):
    a = dict(q=bf16(3, 256), out=bf16(3, 256), pages=kernels.fp8_pages(2, 2, 16, 64, "cpu"), block_table=i32(2, 5), token_req=i32(3), positions=i32(3), H=4, G=2, d=64,
             page_size=16, scale=0.1, window=0, max_keys=None)
    a.update(kw)
    return a


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(3, 256)), dict(q=bf16(3, 255)), dict(q=bf16(3, 260)[:, :256]), dict(q=bf16(3, 512)[:, ::2]), dict(out=bf16(2, 256)), dict(out=bf16(3, 264)[:, 4:260]),
    dict(H=34), dict(G=3), dict(d=32), dict(page_size=24), dict(pages=torch.zeros(2, 4160)), dict(block_table=i32(10)), dict(block_table=i32(0, 4)), dict(window=-1),
    dict(window=1 << 40)])
def test_decode(bad):
    with pytest.raises(KernelError):
        kernels.decode_attention_fp8(**decode_args(**bad))


def test_decode_needs_a_device():
    with pytest.raises(KernelError, match="CUDA"):
        kernels.decode_attention_fp8(**decode_args())


def test_sample():
    f = lambda n: torch.zeros(n)
    good = dict(logits=torch.zeros(3, 10), temperature=f(3), top_k=i32(3), top_p=f(3), min_p=f(3), draws=f(3), out=i32(3))
    for bad in (dict(logits=bf16(3, 10)), dict(logits=torch.zeros(10)), dict(logits=torch.zeros(10, 3).t()), dict(logits=torch.zeros(3, 0)), dict(temperature=f(2)),
                dict(top_k=f(3)), dict(top_p=f(6)[::2]), dict(min_p=torch.zeros(3, dtype=torch.float64)), dict(draws=f((3, 1))), dict(out=torch.zeros(3, dtype=torch.int64))):
        with pytest.raises(KernelError):
            kernels.sample_nucleus(**{**good, **bad})
    with pytest.raises(KernelError, match="CUDA"):
        kernels.sample_nucleus(**good)


@pytest.mark.parametrize("bad", [
    dict(q=torch.zeros(3, 256)), dict(q=bf16(3, 255)), dict(out=bf16(2, 256)), dict(H=34), dict(d=32), dict(page_size=24), dict(pages=torch.zeros(2, 4160)),
    dict(block_table=i32(10)), dict(block_table=i32(2, 0)), dict(window=-1), dict(n_tokens=4)])
def test_prefill(bad):
    a = dict(q=bf16(3, 256), out=bf16(3, 256), pages=kernels.fp8_pages(2, 2, 16, 64, "cpu"), block_table=i32(2, 5), cu_tokens=i32(3), start_pos=i32(2), H=4, G=2, d=64,
             page_size=16, scale=0.1)
    with pytest.raises(KernelError):
        kernels.prefill_attention_fp8(**{**a, **bad})
    with pytest.raises(KernelError, match="CUDA"):
        kernels.prefill_attention_fp8(**a)
