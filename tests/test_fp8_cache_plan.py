"""How launches of the attention over a cache in 8 bits are cut, on the host alone."""
import ctypes

import pytest

from qwen_decoder_b200 import kernels

SMS = 148
HEADS = [(28, 4, 128), (16, 2, 128), (14, 2, 64), (40, 8, 128), (7, 1, 128), (16, 1, 64)]


def decode_scratch(*sizes):
    f = kernels.library("attention_fp8_decode").qd_decode_attention_fp8_scratch
    f.restype = ctypes.c_longlong
    return f(*sizes)


def prefill_scratch(*sizes):
    f = kernels.library("attention_fp8_chunk").qd_prefill_attention_fp8_scratch
    f.restype = ctypes.c_longlong
    return f(*sizes)


@pytest.mark.parametrize("H,G,d", HEADS)
@pytest.mark.parametrize("window", [0, 1500])
def test_scratch_of_single_tokens_holds_every_round(H, G, d, window):
    """A call goes in rounds of 1,024 tokens, each planned by itself: what is left over may be dealt out where a full round goes in clusters."""
    more = 0
    for keys in (1000, 1024, 1025, 1200, 1500, 2047, 2048, 2049, 2100, 9000):
        of_round = [decode_scratch(n, H, G, d, window, keys, SMS) for n in range(1025)]
        for T in list(range(1, 1300)) + list(range(1900, 2300)) + list(range(2950, 3000)):
            asked = decode_scratch(T, H, G, d, window, keys, SMS)
            rounds = ([1024] if T >= 1024 else []) + [T % 1024]
            assert asked >= max(of_round[n] for n in rounds), (T, keys)
            more += T > 1024 and of_round[T % 1024] > of_round[1024]
    assert more                                            # (such calls are among these)


@pytest.mark.parametrize("H,G,d", HEADS)
def test_a_window_past_all_keys_is_none(H, G, d):
    for window in (40000, 1 << 30, 2 ** 31 - 1):
        for T, keys in ((1, 32000), (18, 2000), (37, 32037), (300, 700)):
            assert prefill_scratch(T, 1, H, G, d, window, keys, SMS) == prefill_scratch(T, 1, H, G, d, 0, keys, SMS)
            assert decode_scratch(T, H, G, d, window, keys, SMS) == decode_scratch(T, H, G, d, 0, keys, SMS)


def test_a_kernel_built_otherwise_is_no_refusal_of_sizes():
    with pytest.raises(kernels.KernelError, match="built with other registers"):
        kernels._check(kernels.ERR_BUILD, "prefill_attention_fp8")
    with pytest.raises(kernels.KernelError, match="sizes or types"):
        kernels._check(kernels.ERR_UNSUPPORTED, "prefill_attention_fp8")
