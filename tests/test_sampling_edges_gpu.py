"""Tokens by top-p and min-p where the settings are at an end of their range."""
import math

import pytest
import torch

from test_sampling_nucleus_gpu import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [math.inf, 3e38, 1e35, 1e10])
def test_high_temperatures(guard_regions, temperature):
    """All tokens alike: of a row of 5,000, and of the 50 and the 300 largest."""
    gen = torch.Generator().manual_seed(13)
    z = torch.randn((4, 5000), generator=gen) * 2.5
    for k in (0, 50, 300):
        check(z, [temperature] * 4, [k] * 4, [0.999, 0.7, 1.0, 0.5], [0.0, 0.0, 0.5, 0.9], torch.rand(4, generator=gen).tolist())


def test_padding_of_a_captured_step_has_no_top_p(tmp_path):
    """Rows that pad a batch are nobody's: neither top-p nor min-p, so that their logits are not gone through for them."""
    from qwen_decoder_b200.engine import StepEntry
    from test_fp8_cache_engine_gpu import folder, runner_of
    runner = runner_of(folder("64", tmp_path), projections=None)
    opened = [runner.open(c) for c in "abc"]
    runner.step([StepEntry(c, [5, 6, 7], [2]) for c in opened])
    for top_ps, min_ps in (([0.5, 0.9, 1.0], [0.0, 0.1, 0.0]), ([1.0, 1.0, 0.25], [0.0, 0.5, 0.0])):
        runner.step([StepEntry(c, [9], [0]) for c in opened], sampling=([0.8] * 3, [0, 5, 7], [0.3] * 3, top_ps, min_ps))
        graph, = (g for g in runner._graphs.values() if g.nucleus)
        assert torch.equal(graph.top_ps.cpu(), torch.tensor(top_ps + [1.0])) and torch.equal(graph.min_ps.cpu(), torch.tensor(min_ps + [0.0]))


def test_top_p_or_min_p_alone():
    """Either list without the other: the other's rows have none."""
    from qwen_decoder_b200.sampling import Sampler
    gen = torch.Generator().manual_seed(14)
    z, sampler = (torch.randn((3, 4000), generator=gen) * 2.5).cuda(), Sampler("cuda:0")
    args = z, [0.9, 0.0, 1.3], [0, 0, 40], [0.3, 0.5, 0.99]
    p, m, ones, zeros = [0.5, 0.5, 1.0], [0.2, 0.1, 0.3], [1.0] * 3, [0.0] * 3
    assert torch.equal(sampler.sample(*args, min_ps=m), sampler.sample(*args, ones, m))
    assert torch.equal(sampler.sample(*args, top_ps=p), sampler.sample(*args, p, zeros))
    assert torch.equal(sampler.sample(*args), sampler.sample(*args, ones, zeros))
