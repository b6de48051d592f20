"""Models whose keys and values are cached in 8 bits, and tokens by top-p and min-p, through the step function, the engine and the command line."""
import functools

import pytest
import torch

import plain_fp8_cache as plain
from tiny_configs import TINY

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
SIZES = {"64": dict(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2, head_dim=64),
         "128": dict(hidden_size=256, intermediate_size=512, num_attention_heads=7, num_key_value_heads=1, head_dim=128)}
PROMPT = [(37 * i * i + 11 * i + 5) % 290 for i in range(400)]


def folder(size, path, **keys):
    from qwen_decoder_b200.config import Qwen2Config
    from qwen_decoder_b200.weights import write_random_model
    return write_random_model(Qwen2Config.from_dict(dict(TINY["B"], num_hidden_layers=3, **SIZES[size], **keys)), str(path), 5, dtype=torch.bfloat16, std=0.08)


def runner_of(path, **kw):
    from qwen_decoder_b200.engine import ModelRunner
    kw = dict(dict(num_pages=128, projections={"cache_dtype": "float8_e4m3"}), **kw)
    return ModelRunner.from_folder(path, dtype="bfloat16", device=DEV, **kw)


class Watch:
    """Around the entry points: every call of a step against float64 on its own inputs."""

    def __init__(self, monkeypatch):
        from qwen_decoder_b200 import kernels
        self.calls = []
        for name in ("rope_kv_write_fp8", "decode_attention_fp8", "prefill_attention_fp8"):
            monkeypatch.setattr(kernels, name, functools.partial(getattr(self, name), getattr(kernels, name)))

    def rope_kv_write_fp8(self, real, qkv, bias, q, H, G, d, rot, pairing, cos, sin, positions, pages, slots, ps, write=True):
        real(qkv, bias, q, H, G, d, rot, pairing, cos, sin, positions, pages, slots, ps, write)
        x = qkv.double().cpu()
        x = x.sum(0) if x.dim() == 3 else x
        x = (x if bias is None else x + bias.double().cpu()).view(-1, H + 2 * G, d)
        at, half = positions.long().cpu(), rot // 2
        c, s = cos.double().cpu()[at][:, None], sin.double().cpu()[at][:, None]
        y = x.clone()
        a, b = (x[:, :H + G, :half], x[:, :H + G, half:rot]) if pairing else (x[:, :H + G, 0:rot:2], x[:, :H + G, 1:rot:2])
        if pairing:
            y[:, :H + G, :half], y[:, :H + G, half:rot] = a * c - b * s, a * s + b * c
        else:
            y[:, :H + G, 0:rot:2], y[:, :H + G, 1:rot:2] = a * c - b * s, a * s + b * c
        rows = plain.page_rows(pages.cpu(), G, ps, d)
        for t, slot in enumerate(slots.tolist()):
            want = y[t, H:].view(2, G, d)
            step = (plain.E4M3_HALF_STEP * want.abs()).clamp(min=0) + 2.0 ** -10 * plain.scale_of(want).unsqueeze(-1)
            assert bool(((rows[slot // ps, :, :, slot % ps] - want).abs() <= step).all())
        off = (q.cpu().double().view(-1, H, d) - y[:, :H]).abs()
        assert bool((off <= plain.BF16_HALF_STEP * y[:, :H].abs() + 2.0 ** -18 * x[:, :H].abs().amax(-1, keepdim=True)).all())
        self.calls.append("write")

    def _attention(self, q, out, pages, table, reqs, positions, H, G, d, ps, scale, window, step):
        want, bound = plain.attention(q.cpu(), pages.cpu(), table.cpu(), reqs, positions, H, G, d, ps, scale, window, step)
        assert bool(((out.cpu().double() - want).abs() <= bound).all())

    def decode_attention_fp8(self, real, q, out, pages, table, reqs, positions, H, G, d, ps, scale, window=0, max_keys=None):
        real(q, out, pages, table, reqs, positions, H, G, d, ps, scale, window, max_keys)
        self._attention(q, out, pages, table, reqs.tolist(), positions.tolist(), H, G, d, ps, scale, window, plain.FP16_HALF_STEP)
        self.calls.append("decode")

    def prefill_attention_fp8(self, real, q, out, pages, table, cu, start, H, G, d, ps, scale, window=0, max_keys=None, n_tokens=None):
        real(q, out, pages, table, cu, start, H, G, d, ps, scale, window, max_keys, n_tokens)
        cu, start = cu.tolist(), start.tolist()
        reqs = [r for r in range(len(start)) for _ in range(cu[r + 1] - cu[r])]
        positions = [start[r] + i for r in range(len(start)) for i in range(cu[r + 1] - cu[r])]
        self._attention(q[cu[0]:cu[-1]], out[cu[0]:cu[-1]], pages, table, reqs, positions, H, G, d, ps, scale, window, plain.BF16_HALF_STEP)
        self.calls.append("prefill")


@pytest.mark.parametrize("size", sorted(SIZES))
@pytest.mark.parametrize("keys", [{}, {"projection_dtype": "float8_e4m3"}, {"rope_pairing": "adjacent", "attention_bias": False}])
def test_every_call_of_a_step(size, keys, tmp_path, monkeypatch):
    from qwen_decoder_b200.engine import StepEntry
    runner = runner_of(folder(size, tmp_path, **keys), use_graphs=False)
    runner.model.native_prompt = None                       # (the entry points stand between the parts alone)
    watch = Watch(monkeypatch)
    a, b = runner.open("a"), runner.open("b")
    runner.step([StepEntry(a, PROMPT[:150], [149])])
    runner.step([StepEntry(a, PROMPT[150:151], [0]), StepEntry(b, PROMPT[:7], [6])])
    runner.step([StepEntry(a, PROMPT[151:190], [0]), StepEntry(b, PROMPT[7:8], [0])])
    runner.step([StepEntry(a, PROMPT[190:191], [0]), StepEntry(b, PROMPT[8:9], [0])])
    steps = [["write", "prefill"], ["write", "decode", "prefill"], ["write", "decode", "prefill"], ["write", "decode"]]
    assert watch.calls == [c for s in steps for c in s * 3]
    runner.check_status()


@pytest.mark.parametrize("size", sorted(SIZES))
def test_native_prompt_steps_are_the_parts(size, tmp_path):
    """With products in 8 bits both paths call the same kernels with the same arguments."""
    from qwen_decoder_b200.engine import StepEntry
    path = folder(size, tmp_path, projection_dtype="float8_e4m3")
    got = []
    for native in (True, False):
        runner = runner_of(path)
        if not native:
            runner.model.native_prompt = None
        a, b = runner.open("a"), runner.open("b")
        out = [runner.step([StepEntry(a, PROMPT[:150], [3, 149])])]
        out.append(runner.step([StepEntry(a, PROMPT[150:151], [0]), StepEntry(b, PROMPT[:300], [299])]))
        out.append(runner.step([StepEntry(a, PROMPT[151:160], [8]), StepEntry(b, PROMPT[300:301], [0])]))
        assert (runner.model.native_prompt is not None and runner.model.native_prompt.steps == 3) == native
        got.append(torch.cat(out).clone())
    assert torch.equal(*got)


@pytest.mark.parametrize("size", sorted(SIZES))
@pytest.mark.parametrize("keys", [{}, {"projection_dtype": "float8_e4m3"}])
def test_replayed_steps_are_eager_ones(size, keys, tmp_path):
    """Single tokens of one, two and four requests, replayed and launched one by one: the same kernels on the same shares of keys, the same bits."""
    from qwen_decoder_b200.engine import StepEntry
    path, got = folder(size, tmp_path, **keys), []
    for graphs in (True, False):
        runner, out = runner_of(path, use_graphs=graphs), []
        for n in (1, 2, 4):
            rcs = [runner.open((n, i)) for i in range(n)]
            for i, rc in enumerate(rcs):
                runner.step([StepEntry(rc, PROMPT[:150 - 40 * i], [])])
            for i in range(5):
                out.append(runner.step([StepEntry(rc, PROMPT[200 + i + j:201 + i + j], [0]) for j, rc in enumerate(rcs)]).clone())
            for rc in rcs:
                runner.close(rc)
        assert bool(runner._graphs) == graphs
        runner.check_status()
        got.append(torch.cat(out))
    assert torch.equal(*got)


def test_the_engine(tmp_path, capsys):
    """generate with a cache in 8 bits: more pages in the same memory, prefix cache, preemption, running ahead; the same tokens whichever."""
    from qwen_decoder_b200.cache import CacheManager
    from qwen_decoder_b200.engine import Engine, SamplingParams
    path = folder("64", tmp_path, projection_dtype="float8_e4m3")
    prompts = [PROMPT[i:i + 20 + 9 * i] for i in range(6)]
    params = SamplingParams(max_new_tokens=12, ignore_eos=True)
    outs = []
    for kw in (dict(), dict(run_ahead=False, use_graphs=False), dict(enable_prefix_cache=True)):
        engine = Engine(path, cache_dtype="float8_e4m3", device=DEV, num_pages=64, max_prefill_tokens_per_step=64, **kw)
        outs.append(engine.generate(prompts, params))
    assert all(len(o) == 12 for o in outs[0])
    bf16 = Engine(path, device=DEV, num_pages=4)
    per = [CacheManager.bytes_per_page(e.runner.layout, 16, torch.bfloat16) for e in (engine, bf16)]
    assert engine.runner.cache.kv[0].dtype == torch.uint8 and per[0] * 128 == per[1] * 65
    few = Engine(path, cache_dtype="float8_e4m3", device=DEV, num_pages=9, max_prefill_tokens_per_step=64)
    assert [len(o) for o in few.generate(prompts, params)] == [12] * 6
    from qwen_decoder_b200.engine import cli
    assert cli.main([path, "4", "--cache-dtype", "float8_e4m3", "--prompt-ids", "5,17,3", "--max-new-tokens", "4", "--ignore-eos", "--temperature", "0.8",
                     "--top-p", "0.9", "--min-p", "0.01", "--num-pages", "16"]) == 0
    assert "[0] (length)" in capsys.readouterr().out


# ---- tokens by top-p and min-p -----------------------------------------------------------------------------------------

def test_sampling_of_steps(tmp_path):
    """Eager and replayed steps draw what the plain sampler draws from their logits; rows without top-p and min-p what they draw without them."""
    from qwen_decoder_b200.engine import StepEntry
    runner = runner_of(folder("64", tmp_path), projections=None)
    how = [(0.8, 0, 0.31, 0.9, 0.0), (0.0, 0, 0.2, 0.5, 0.1), (0.7, 30, 0.77, 1.0, 0.0), (1.3, 0, 0.12, 1.0, 0.05), (0.9, 12, 0.99, 0.8, 0.02)]
    f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
    for n, graphs in ((1, True), (40, True), (3, False)):
        runner.use_graphs = graphs
        rcs = [runner.open((n, i)) for i in range(len(how))]
        for rc, i in zip(rcs, range(len(how))):
            runner.step([StepEntry(rc, PROMPT[i:i + n], [])])
        entries = [StepEntry(rc, PROMPT[100 + i:101 + i], [0]) for i, rc in enumerate(rcs)]
        cols = [list(c) for c in zip(*how)]
        logits, tokens = runner.step(entries, sampling=(cols[0], cols[1], cols[2], cols[3], cols[4]))
        z = logits.cpu()
        for r, (t, k, u, p, m) in enumerate(how):
            want, margin = plain.sample(z[r], f32(t), k, f32(p), f32(m), f32(u))
            assert margin < 1e-6 or int(tokens[r]) == want, (r, int(tokens[r]), want)
        z = logits.clone()
        alone = runner.sampler.sample(z, cols[0], cols[1], cols[2])
        assert int(alone[1]) == int(tokens[1]) and int(alone[2]) == int(tokens[2])
        for rc in rcs:
            runner.close(rc)


def test_requests_do_not_depend_on_their_batch(tmp_path):
    from qwen_decoder_b200.engine import Engine, SamplingParams
    path = folder("128", tmp_path)
    params = [SamplingParams(temperature=0.9, top_p=0.8, max_new_tokens=10, ignore_eos=True, seed=3), SamplingParams(temperature=0.9, max_new_tokens=10, ignore_eos=True, seed=3),
              SamplingParams(temperature=1.2, min_p=0.1, top_k=25, max_new_tokens=10, ignore_eos=True, seed=4), SamplingParams(max_new_tokens=10, ignore_eos=True)]
    engine = Engine(path, device=DEV, num_pages=64, dtype="bfloat16")
    seen = []
    for group in (params, params[:2], params[:1]):
        engine._next_id = 0                                   # (a request's draws go by its key)
        seen.append(engine.generate([PROMPT[:9]] * len(group), group))
    assert len(set(map(tuple, seen[0]))) > 1
    with pytest.raises(ValueError, match="top_p"):
        engine.add_request([1], SamplingParams(top_p=0.0))
    with pytest.raises(ValueError, match="min_p"):
        engine.add_request([1], SamplingParams(min_p=1.5))
