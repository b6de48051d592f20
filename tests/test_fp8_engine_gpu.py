"""Models whose projections are in 8 bits, through the step function and the engine: every norm and product of a step against float64 on
its own inputs, attention behind them, the whole beside the stored model; log probabilities of generated and of given tokens."""
import dataclasses
import functools

import pytest
import torch

import plain_model
import test_fp8_gpu as kernel_tests
from tiny_configs import SEEDS, TINY

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BOTH = {"projection_dtype": "float8_e4m3", "output_projection_dtype": "float8_e4m3"}
PROMPT = [(37 * i * i + 11 * i + 5) % 290 for i in range(150)]


def folder(name, path, std=0.08, **keys):
    from qwen_decoder_b200.config import Qwen2Config
    from qwen_decoder_b200.weights import write_random_model
    return write_random_model(Qwen2Config.from_dict(dict(TINY[name], **keys)), str(path), SEEDS[name], dtype=torch.bfloat16, std=std)


def runner_of(path, **kw):
    from qwen_decoder_b200.engine import ModelRunner
    return ModelRunner.from_folder(path, dtype="bfloat16", device=DEV, num_pages=64, **kw)


def logits_of(runner, tokens, cuts):
    from qwen_decoder_b200.engine import StepEntry
    rc, out, at = runner.open("r"), [], 0
    for n in cuts:
        part = tokens[at:at + n]
        out.append(runner.step([StepEntry(rc, part, list(range(len(part))))]).clone())
        at += n
    assert at == len(tokens)
    runner.close(rc)
    runner.check_status()
    return torch.cat(out).double().cpu()


class Watch:
    """Stands around the entry points in 8 bits: every call of a step is checked against float64 on its own inputs, with the bounds of the
    operators' own tests, and what goes from one into the next is written down.  (End to end nothing so tight can be said: a difference in
    the last bit before a rounding to 8 bits may tip a number into the next step, an eighth of it, and every rounding after that differs.)"""

    def __init__(self, monkeypatch):
        from qwen_decoder_b200 import kernels
        self.calls = []
        for name in ("add_rmsnorm_fp8", "quantize_fp8", "gemm_fp8", "gemm_fp8_gated"):
            monkeypatch.setattr(kernels, name, functools.partial(getattr(self, name), getattr(kernels, name)))

    def add_rmsnorm_fp8(self, real, x, delta, weight, out, eps, rows=None, write_back=True, delta_scale=None):
        before = x.double()
        d = delta.double() if delta is not None else torch.zeros_like(before)
        d = d.sum(0) if d.dim() == 3 else d
        real(x, delta, weight, out, eps, rows=rows, write_back=write_back, delta_scale=delta_scale)
        sums, off = before + d, 4 * 2.0 ** -24 * (before.abs() + d.abs())
        if write_back:
            assert ((x.double() - sums).abs() <= off).all()
        if rows is not None:
            sums, off = sums[rows.long()], off[rows.long()]
        inv = torch.rsqrt(sums.square().mean(1, keepdim=True) + eps)
        y = sums * inv * weight.double()
        kernel_tests.check_rows(out, y, 2.0 ** -17 * y.abs() + (off * inv + sums.abs() * inv * inv * off.square().mean(1, keepdim=True).sqrt())
                                * weight.double().abs())
        self.calls.append(("norm", delta.data_ptr() if delta is not None else 0, out.q.data_ptr()))

    def quantize_fp8(self, real, x, out):
        real(x, out)
        kernel_tests.check_rows(out, x.double(), torch.zeros_like(x, dtype=torch.float64))
        self.calls.append(("rows", x.data_ptr(), out.q.data_ptr()))

    def gemm_fp8(self, real, x, w, bias, out, plan=None, resident=False):
        real(x, w, bias, out, plan, resident)
        want = kernel_tests.value(x) @ kernel_tests.value(w).T + (0 if bias is None else bias.double())
        close = (2.0 ** -8 if out.dtype == torch.bfloat16 else 2.0 ** -23) * want.abs() + kernel_tests.sums_off(x, w)
        assert ((out.double() - want).abs() <= close).all()
        self.calls.append(("product", x.q.data_ptr(), out.data_ptr()))

    def gemm_fp8_gated(self, real, x, w, bias, out, act=0, plan=None, resident=False):
        real(x, w, bias, out, act, plan, resident)
        z, F = kernel_tests.value(x) @ kernel_tests.value(w).T, out.shape[1]
        off = kernel_tests.sums_off(x, w) + 2.0 ** -23 * z.abs()
        g, u = z[:, :F], z[:, F:]
        kernel_tests.check_rows(out, kernel_tests.gated(g, u, act), 1.2 * off[:, :F] * u.abs() + (g.abs() + off[:, :F]) * off[:, F:]
                                + 2.0 ** -20 * (g * u).abs())
        self.calls.append(("gated", x.q.data_ptr(), out.q.data_ptr()))


@pytest.mark.parametrize("output", [False, True])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_every_product_and_norm_of_a_step(name, output, tmp_path, monkeypatch):
    runner = runner_of(folder(name, tmp_path, **(BOTH if output else {"projection_dtype": "float8_e4m3"})), use_graphs=False)
    runner.model.native_prompt = None                      # (the entry points stand between the parts alone)
    watch = Watch(monkeypatch)
    for cuts in ([100], [40, 1, 59], [17, 3, 16, 64], [96] + [1] * 4):
        logits_of(runner, PROMPT[:100], cuts)
        calls = watch.calls
        watch.calls = []
        layer = ["norm", "product", "rows", "product", "norm", "gated", "product"]
        step = layer * TINY[name]["num_hidden_layers"] + (["norm", "product"] if output else [])
        assert [c[0] for c in calls] == step * len(cuts)
        for i, (kind, took, gave) in enumerate(calls):
            if kind == "product" and calls[i - 1][0] in ("norm", "rows", "gated") or kind == "gated":
                assert took == calls[i - 1][2]             # each takes what the one before left ...
            if kind == "norm" and i % len(step):
                assert took == calls[i - 1][2]             # ... and the norm adds the branch's product to the sum


def test_attention_behind_products_in_8_bits(tmp_path, monkeypatch):
    """Attention's output, of portions and of single tokens, against float64 from the same q, k and v."""
    from qwen_decoder_b200 import kernels
    from qwen_decoder_b200.parts.fp8 import GQAttentionFp8
    path = folder("D", tmp_path, projection_dtype="float8_e4m3")
    runner = runner_of(path, use_graphs=False)
    runner.model.native_prompt = None
    cfg, w = plain_model.read_folder(path)
    mixer = runner.model.layers[0].mixer
    qkv, attn = [], []
    real_product, real_out = type(mixer.qkv)._product, GQAttentionFp8._out_product

    def product(self, x, bias, dtype):
        out = real_product(self, x, bias, dtype)
        if self is mixer.qkv:
            qkv.append(out.double() + (mixer.qkv.bias.double() if bias is None else 0))
        return out

    def out_product(self, a):
        if self is mixer:
            attn.append(a.double())
        return real_out(self, a)

    monkeypatch.setattr(type(mixer.qkv), "_product", product)
    monkeypatch.setattr(GQAttentionFp8, "_out_product", out_product)
    H, G, d = cfg["num_attention_heads"], cfg["num_key_value_heads"], plain_model.head_dim_of(cfg)
    pairing = cfg.get("rope_pairing", "half")
    for cuts in ([100], [50, 10, 36] + [1] * 4):
        qkv.clear(), attn.clear()
        logits_of(runner, PROMPT[:100], cuts)
        z, got, at = torch.cat(qkv).cpu(), torch.cat(attn).cpu(), torch.arange(100)
        q = plain_model.rope(z[:, :H * d], at, H, d, cfg["rope_theta"], pairing)
        k = plain_model.rope(z[:, H * d:(H + G) * d], at, G, d, cfg["rope_theta"], pairing)
        v = z[:, (H + G) * d:]
        want = plain_model.attention(q, k, v, H, G, d)
        # q and k may be rounded to bfloat16 twice each (2^-8), weights and results once (2^-9): a score is off by 2^-7 of its terms' sizes
        # at most, a weight by e^(2 * that)
        sizes = torch.einsum("thd,shd->tsh", q.view(100, H, d).abs(), k.view(100, G, d).abs().repeat_interleave(H // G, 1)).amax() / d ** 0.5
        assert float((got - want).abs().max()) <= (2 * 2.0 ** -7 * float(sizes) + 3 * 2.0 ** -9) * float(v.abs().max())


@pytest.mark.parametrize("output", [False, True])
@pytest.mark.parametrize("name", ["A", "B", "C", "D"])
def test_prompt_steps_from_native_code_are_the_parts(name, output, tmp_path):
    """The same launches: the same bits, of few and of many tokens, beside single tokens of other requests, with nothing wanted."""
    from qwen_decoder_b200.engine import StepEntry
    path = folder(name, tmp_path, **(BOTH if output else {"projection_dtype": "float8_e4m3"}))
    got = []
    for native in (True, False):
        runner = runner_of(path, use_graphs=False)
        assert runner.model.native_prompt is not None
        if not native:
            runner.model.native_prompt = None
        out = [logits_of(runner, PROMPT[:n], cuts) for n, cuts in ((100, [100]), (74, [40, 17, 3, 1, 13]), (2, [2]), (16, [16]))]
        a, b = runner.open("a"), runner.open("b")
        runner.step([StepEntry(a, PROMPT[:30], [])])
        for n in (1, 9, 33):
            out.append(runner.step([StepEntry(a, [7], [0]), StepEntry(b, PROMPT[:n + 1], [0, n])]).double().cpu())
        if native:
            assert runner.model.native_prompt.steps >= 10
        got.append(out)
    for x, y in zip(*got):
        assert torch.isfinite(x).all() and torch.equal(x, y)


@pytest.mark.parametrize("tokens", [5, 100])
def test_only_the_output_projection_in_8_bits(tokens, tmp_path):
    """Layers in 16 bits launched from native code, whose last norm leaves rows in 8 bits: those that the model in 16 bits takes."""
    from qwen_decoder_b200.engine import StepEntry
    path = folder("B", tmp_path)
    rows = []
    for projections in (None, {"output_projection_dtype": "float8_e4m3"}):
        runner = runner_of(path, projections=projections)
        real = runner.model._logits
        runner.model._logits = lambda h: (rows.append(h), real(h))[1]
        assert runner.model.native_prompt is not None
        rc = runner.open("r")
        runner.step([StepEntry(rc, PROMPT[:tokens], [0, tokens - 1])])
        assert runner.model.native_prompt.steps == 1
    plain, rounded = rows
    y = plain.double()
    kernel_tests.check_rows(rounded, y, 2.0 ** -8 * y.abs())          # (y is rounded to bfloat16 itself)


def test_weights_in_8_bits_are_near_the_ones_in_16(tmp_path):
    """The whole rounding: both operands of every product to 4 significant bits, 2.6 % of each, against the model as it is stored."""
    path = folder("B", tmp_path)
    cfg, w = plain_model.read_folder(path)
    exact = plain_model.forward(cfg, w, PROMPT[:60])
    got = logits_of(runner_of(path, projections=BOTH), PROMPT[:60], [60])
    off = float((got - exact).norm() / exact.norm())
    assert 0.005 < off < 0.2, off                         # rounded, and not far


def test_replayed_steps_are_the_steps(tmp_path):
    path = folder("D", tmp_path, **BOTH)
    a = logits_of(runner_of(path), PROMPT[:60], [50] + [1] * 10)
    b = logits_of(runner_of(path, use_graphs=False), PROMPT[:60], [50] + [1] * 10)
    assert torch.equal(a, b)


def test_generation_with_log_probabilities(tmp_path):
    from qwen_decoder_b200.engine import Engine, SamplingParams
    path = folder("B", tmp_path)
    engine = Engine(path, device=DEV, num_pages=64, **BOTH)
    prompts = [PROMPT[:30], PROMPT[5:50], PROMPT[7:9]]
    params = [SamplingParams(max_new_tokens=12, logprobs=5), SamplingParams(max_new_tokens=9), SamplingParams(max_new_tokens=7, logprobs=0)]
    reqs = [engine.add_request(p, sp) for p, sp in zip(prompts, params)]
    # the logits that each token was drawn from, by the request and the token's place
    seen, real = {}, engine._launch

    def launch(plan, device_tokens=None):
        places = [(e.request.request_id, e.request.cache.num_tokens + len(e.tokens)) for e in plan.entries if e.samples]
        step = engine.runner.step

        def recorded(*a, **kw):
            out = step(*a, **kw)
            for place, row in zip(places, out[0]):
                seen[place] = row.clone()
            return out
        engine.runner.step = recorded
        try:
            return real(plan, device_tokens)
        finally:
            del engine.runner.step
    engine._launch = launch
    while engine.has_work():
        engine.step()
    assert [len(r.logprobs) for r in reqs] == [12, 0, 7]
    plain = Engine(path, device=DEV, num_pages=64, **BOTH).generate(prompts, [dataclasses.replace(p, logprobs=None) for p in params])
    assert [r.output for r in reqs] == plain              # who asks for them gets the same tokens
    for r in (reqs[0], reqs[2]):
        assert [p.token for p in r.logprobs] == r.output
        lp = torch.log_softmax(torch.stack([seen[r.request_id, len(r.prompt) + i] for i in range(len(r.output))]).double(), 1)
        for i, p in enumerate(r.logprobs):
            # (the bounds of the kernel's own tests at this vocabulary)
            assert p.logprob == pytest.approx(float(lp[i, p.token]), abs=1e-5)
            assert p.entropy == pytest.approx(float(-(lp[i].exp() * lp[i]).sum()), abs=3e-5)
            assert len(p.top) == r.params.logprobs
            if p.top:
                assert p.top[0] == (p.token, p.logprob) and all(a[1] >= b[1] for a, b in zip(p.top, p.top[1:]))      # greedy


def test_scores_of_given_tokens(tmp_path):
    from qwen_decoder_b200.engine import Engine, StepError
    path = folder("D", tmp_path)
    engine = Engine(path, device=DEV, num_pages=64, max_prefill_tokens_per_step=16)
    prompts = [PROMPT[:50], PROMPT[:2], PROMPT[:1], PROMPT[:17]]
    scores = engine.score(prompts, top=3)
    assert [len(s) for s in scores] == [49, 1, 0, 16]
    logits = logits_of(engine.runner, PROMPT[:49], [16, 16, 16, 1])        # the same portions
    lp = torch.log_softmax(logits, 1)
    for i, s in enumerate(scores[0]):
        assert s.token == PROMPT[i + 1]
        assert s.logprob == pytest.approx(float(lp[i, s.token]), abs=1e-5) and len(s.top) == 3
        assert s.entropy == pytest.approx(float(-(lp[i].exp() * lp[i]).sum()), abs=3e-5)
        best = torch.topk(lp[i], 3)
        assert [t for t, _ in s.top] == best.indices.tolist() and [p for _, p in s.top] == pytest.approx(best.values.tolist(), abs=1e-5)
    assert scores[3] == scores[0][:16]
    pages = engine.runner.cache.free_pages()
    with pytest.raises(StepError):
        engine.score([[5, 100000]])
    with pytest.raises(ValueError, match="most probable"):
        engine.score([[5, 6]], top=33)
    assert engine.runner.cache.free_pages() == pages       # nothing is kept


def test_refusals(tmp_path):
    from qwen_decoder_b200.engine import Engine, ModelRunner, SamplingParams
    path = folder("A", tmp_path)
    with pytest.raises(ValueError, match="bfloat16"):
        ModelRunner.from_folder(path, dtype="float32", device=DEV, num_pages=4, projections=BOTH)
    with pytest.raises(ValueError, match="projections"):
        ModelRunner.from_folder(path, device=DEV, num_pages=4, projections={"projection_dtype": "int8"})
    engine = Engine(path, device=DEV, num_pages=4)
    with pytest.raises(ValueError, match="most probable"):
        engine.add_request([1, 2], SamplingParams(logprobs=40))
