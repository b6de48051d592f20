from .sampler import Sampler, uniform_draw, without_nucleus

__all__ = ["Sampler", "uniform_draw", "without_nucleus"]
