"""Scores and log probabilities beside other work: scores asked for while requests are under way, prefix caching, steps launched ahead."""
import dataclasses

import pytest
import torch

from test_fp8_engine_gpu import BOTH, DEV, PROMPT, folder

pytestmark = pytest.mark.gpu


def finish(engine):
    while engine.has_work():
        engine.step()


@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("keys", [{}, BOTH])
def test_scores_while_requests_are_under_way(keys, prefix, tmp_path):
    """They change no request's tokens, and are what an idle engine gives."""
    from qwen_decoder_b200.engine import Engine, SamplingParams
    path = folder("B", tmp_path)
    make = lambda: Engine(path, device=DEV, num_pages=96, enable_prefix_cache=prefix, max_prefill_tokens_per_step=16, **keys)  # noqa: E731
    prompts = [PROMPT[:40], PROMPT[:33], PROMPT[60:62]]
    params = [SamplingParams(max_new_tokens=14, temperature=0.8, top_k=5, seed=3, logprobs=2), SamplingParams(max_new_tokens=10),
              SamplingParams(max_new_tokens=12, logprobs=0)]
    given = [PROMPT[:50], PROMPT[20:37]]
    alone = make()
    want = [alone.add_request(p, sp) for p, sp in zip(prompts, params)]
    finish(alone)
    scores = alone.score(given, top=4)
    engine = make()
    reqs = [engine.add_request(p, sp) for p, sp in zip(prompts, params)]
    steps = 0
    while engine.has_work():
        engine.step()
        steps += 1
        if steps in (1, 3, 6, 9):
            between = engine.score(given, top=4)
            for a, b in zip(between, scores):
                assert [p.token for p in a] == [p.token for p in b]
                assert [p.logprob for p in a] == pytest.approx([p.logprob for p in b], abs=1e-5)
    assert steps >= 10
    assert [r.output for r in reqs] == [r.output for r in want]
    assert [r.logprobs for r in reqs] == [r.logprobs for r in want]
    assert [len(r.logprobs) for r in reqs] == [14, 0, 12]


def test_log_probabilities_of_steps_launched_ahead(tmp_path):
    """Also of requests that end on a stop token: as many as output tokens, the same as of steps one after the other."""
    from qwen_decoder_b200.engine import Engine, SamplingParams
    path = folder("B", tmp_path)
    first = Engine(path, device=DEV, num_pages=64).generate([PROMPT[:20]], SamplingParams(max_new_tokens=12, ignore_eos=True))[0]
    stop = first[6]
    results = []
    for ahead in (True, False):
        engine = Engine(path, device=DEV, num_pages=64, run_ahead=ahead)
        params = SamplingParams(max_new_tokens=12, ignore_eos=True, logprobs=3)
        reqs = [engine.add_request(PROMPT[:20], dataclasses.replace(params, ignore_eos=False, stop_ids=(stop,))), engine.add_request(PROMPT[3:9], params)]
        finish(engine)
        for r in reqs:
            assert [p.token for p in r.logprobs] == r.output and all(len(p.top) == 3 for p in r.logprobs)
        results.append([(r.output, r.logprobs) for r in reqs])
    assert results[0] == results[1] and len(results[0][0][0]) < 12
