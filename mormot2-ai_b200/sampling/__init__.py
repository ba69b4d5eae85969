"""Choosing the next token: settings (``Sampling``) and the device sampler; what a model says of
given tokens (``token_scores``)."""
from .settings import Sampling, sampling_from_config
from .device import DeviceSampler
from .scores import Scores, token_scores

__all__ = ["Sampling", "sampling_from_config", "DeviceSampler", "Scores", "token_scores"]
