from .sampler import DeviceSampler, Filters

__all__ = ["DeviceSampler", "Filters"]
