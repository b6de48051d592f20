"""What the entry points of the operators in 8 bits and of the log probabilities refuse, before anything is launched."""
import pytest
import torch

from qwen_decoder_b200 import kernels
from qwen_decoder_b200.kernels import Fp8Rows, KernelError, fp8_rows


def rows(R, K):
    return fp8_rows(R, K, "cpu")


@pytest.mark.parametrize("R,K,q,s", [(3, 128, (128, 1), (4, 1)), (3, 100, (112, 1), (4, 1)), (2, 1300, (1312, 1), (12, 1)), (1, 1, (16, 1), (4, 1))])
def test_room_for_rows(R, K, q, s):
    out = rows(R, K)
    assert tuple(out.q.shape) == (R, K) and out.q.stride() == q and tuple(out.s.shape) == (R, -(-K // 128)) and out.s.stride()[:1] == s[:1]
    assert kernels._host_calls().check_rows(out, "out") == (R, K)


BAD_ROWS = {
    "type of q": lambda: Fp8Rows(torch.zeros(2, 256), rows(2, 256).s),
    "type of s": lambda: Fp8Rows(rows(2, 256).q, torch.zeros(2, 2)),
    "rows of s": lambda: Fp8Rows(rows(2, 256).q, rows(3, 256).s),
    "blocks of s": lambda: Fp8Rows(rows(2, 256).q, rows(2, 512).s),
    "dimensions": lambda: Fp8Rows(rows(2, 256).q[0], rows(2, 256).s),
    "distance of q's rows": lambda: Fp8Rows(torch.empty(2, 264, dtype=torch.float8_e4m3fn)[:, :256], rows(2, 256).s),
    "address of q": lambda: Fp8Rows(torch.empty(2, 272, dtype=torch.float8_e4m3fn)[:, 4:260], rows(2, 256).s),
    "order of q": lambda: Fp8Rows(torch.empty(256, 16, dtype=torch.float8_e4m3fn).t()[:2], rows(2, 256).s),
    "distance of s's rows": lambda: Fp8Rows(rows(2, 256).q, torch.empty(2, 3, dtype=torch.float8_e8m0fnu)[:, :2]),
}


@pytest.mark.parametrize("what", sorted(BAD_ROWS))
def test_rows_that_do_not_fit(what):
    bad, good = BAD_ROWS[what](), rows(2, 256)
    with pytest.raises(KernelError):
        kernels.gemm_fp8(bad, good, None, torch.empty(2, 2))
    with pytest.raises(KernelError):
        kernels.gemm_fp8(good, bad, None, torch.empty(2, 2))
    with pytest.raises(KernelError):
        kernels.quantize_fp8(torch.zeros(2, 256), bad)


def test_products():
    x, w = rows(3, 256), rows(8, 256)
    for out in (torch.empty(3, 7), torch.empty(3, 8, dtype=torch.float16), torch.empty(8, 3).t(), torch.empty(24)):
        with pytest.raises(KernelError, match="out must be"):
            kernels.gemm_fp8(x, w, None, out)
    with pytest.raises(KernelError, match="features"):
        kernels.gemm_fp8(rows(3, 128), w, None, torch.empty(3, 8))
    for bias in (torch.zeros(7), torch.zeros(8, dtype=torch.bfloat16), torch.zeros(16)[::2]):
        with pytest.raises(KernelError, match="bias"):
            kernels.gemm_fp8(x, w, bias, torch.empty(3, 8))
    with pytest.raises(KernelError, match="as many rows"):
        kernels.gemm_fp8_gated(x, rows(7, 256), None, rows(3, 3))
    with pytest.raises(KernelError, match="fit"):
        kernels.gemm_fp8_gated(x, w, None, rows(3, 8))
    with pytest.raises(KernelError, match="act"):
        kernels.gemm_fp8_gated(x, w, None, rows(3, 4), kernels.ACT_CLAMPED)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.gemm_fp8(x, w, None, torch.empty(3, 8), (1, 64, 1))


def test_sources():
    out = rows(3, 256)
    for x in (torch.zeros(3, 255), torch.zeros(3, 256, dtype=torch.float16), torch.zeros(2, 3, 256, dtype=torch.bfloat16), torch.zeros(256, 3).t(),
              torch.zeros(0, 3, 256), torch.zeros(256)):
        with pytest.raises(KernelError):
            kernels.quantize_fp8(x, out)
    with pytest.raises(KernelError):
        kernels.gate_fp8(torch.zeros(3, 256), out)
    with pytest.raises(KernelError, match="bias"):
        kernels.gate_fp8(torch.zeros(3, 512), out, torch.zeros(256))
    w = torch.ones(256)
    for bad in (dict(x=torch.zeros(3, 256, dtype=torch.bfloat16)), dict(x=torch.zeros(4, 256)), dict(weight=torch.ones(255)),
                dict(delta=torch.zeros(2, 256)), dict(delta_scale=torch.zeros(3)), dict(rows=torch.zeros(3, dtype=torch.int64)),
                dict(rows=torch.zeros(2, dtype=torch.int32)), dict(delta=torch.zeros(3, 512)[:, ::2])):
        args = dict(x=torch.zeros(3, 256), delta=None, weight=w, out=out, eps=1e-6)
        args.update(bad)
        with pytest.raises(KernelError):
            kernels.add_rmsnorm_fp8(**args)


def test_log_probabilities():
    z, t = torch.zeros(3, 10), torch.zeros(3, dtype=torch.int32)
    for args in ((z.half(), t), (z[0], t), (torch.zeros(10, 3).t(), t), (z, t.long()), (z, t[:2]), (z, t, 11), (z, t, -1), (torch.zeros(3, 50), t, 33),
                 (torch.zeros(3, 0), t), (z, torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(KernelError):
            kernels.token_logprobs(*args)
    with pytest.raises(KernelError, match="CUDA"):
        kernels.token_logprobs(z, t, 2)
