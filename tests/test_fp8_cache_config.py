"""A cache in 8 bits in configurations, descriptions and the cache manager."""
import pytest
import torch

from tiny_configs import TINY
from qwen_decoder_b200.cache import CacheManager, PagedKV
from qwen_decoder_b200.cache.manager import CacheLayout
from qwen_decoder_b200.config import Qwen2Config, describe_model
from qwen_decoder_b200.config.model_config import ConfigError
from qwen_decoder_b200.engine.runner import with_projections
from qwen_decoder_b200.parts.model import build_model


def test_configuration():
    d = dict(TINY["A"], num_attention_heads=4, num_key_value_heads=2, head_dim=64)
    cfg = Qwen2Config.from_dict(dict(d, cache_dtype="float8_e4m3"))
    assert cfg.to_dict()["cache_dtype"] == "float8_e4m3" and "cache_dtype" not in Qwen2Config.from_dict(d).to_dict()
    assert describe_model(cfg).layers[0].mixer.params["cache_dtype"] == "float8_e4m3"
    assert "cache_dtype" not in describe_model(Qwen2Config.from_dict(d)).layers[0].mixer.params
    assert with_projections(Qwen2Config.from_dict(d), {"cache_dtype": "float8_e4m3", "projection_dtype": None}) == cfg
    layout = build_model(describe_model(cfg)).cache_layout()
    assert layout.groups[0].need == PagedKV(2, 64, numbers="float8_e4m3")
    for bad in ("float8_e5m2", "int8", 8):
        with pytest.raises(ConfigError, match="cache_dtype"):
            Qwen2Config.from_dict(dict(d, cache_dtype=bad))
    with pytest.raises(ValueError, match="cache_dtype"):
        with_projections(Qwen2Config.from_dict(d), {"cache_dtype": "int8"})


def test_models_that_have_none():
    import veterax_configs
    from qwen_decoder_b200.config import registry
    with pytest.raises(ValueError, match="cache_dtype"):
        with_projections(object(), {"cache_dtype": "float8_e4m3"})
    with pytest.raises(ValueError, match="cache_dtype"):
        build_model(describe_model(Qwen2Config.from_dict(dict(TINY["A"], head_dim=32, cache_dtype="float8_e4m3"))))


def test_refused_with_float32():
    d = dict(TINY["A"], num_attention_heads=4, num_key_value_heads=2, head_dim=64, cache_dtype="float8_e4m3")
    model = build_model(describe_model(Qwen2Config.from_dict(d)))
    with pytest.raises(ValueError, match="bfloat16"):
        model.layers[0].mixer.bind(None, torch.float32, torch.device("cpu"))


def test_manager():
    kv8, kv = PagedKV(2, 64, numbers="float8_e4m3"), PagedKV(2, 64)
    layout = CacheLayout.from_needs([kv8, kv, kv8], [None, None, None])
    assert len(layout.groups) == 2                      # pages of their own
    assert CacheManager.bytes_per_page(layout, 16, torch.bfloat16) == 2 * 2 * 16 * 130 + 2 * 2 * 16 * 64 * 2
    m = CacheManager(layout, 5, 16, 2, dtype=torch.bfloat16, device="cpu")
    assert tuple(m.kv[0].shape) == (2, 6, 2 * 16 * 130) and m.kv[0].dtype == torch.uint8
    assert tuple(m.kv[1].shape) == (1, 6, 2, 2, 16, 64) and m.kv[1].dtype == torch.bfloat16
    with pytest.raises(ValueError, match="16"):
        CacheManager(layout, 5, 8, 2, device="cpu")
    with pytest.raises(ValueError):
        PagedKV(2, 64, numbers="int8")
    with pytest.raises(ValueError):
        PagedKV(2, 64, v_dim=32, numbers="float8_e4m3")


def test_rows_that_top_p_and_min_p_leave_alone():
    """What rounds to 1 (0) where the kernels read it is no top-p (min-p) for anybody: one of the two kernels has each row."""
    from qwen_decoder_b200.sampling import without_nucleus
    top_p, min_p = [1.0, 1.0 - 1e-12, 0.99999999, 0.9999999, 1.0, 1.0, 0.5], [0.0, 0.0, 0.0, 0.0, 1e-60, 1e-30, 0.0]
    assert without_nucleus([0.8] * 7, top_p, min_p) == [0.8, 0.8, 0.8, 0.0, 0.8, 0.0, 0.0]
    for p, m, t in zip(top_p, min_p, without_nucleus([0.8] * 7, top_p, min_p)):
        on_device = torch.tensor([p, m], dtype=torch.float32)
        assert (t == 0.0) == bool(on_device[0] < 1 or on_device[1] > 0)
