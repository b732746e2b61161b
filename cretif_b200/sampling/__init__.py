"""Sampling: parameters, the device sampler, and the verification of drafted tokens."""
from .sampler import DraftVerifier, Sampler, SamplingParams, uniform01

__all__ = ["DraftVerifier", "Sampler", "SamplingParams", "uniform01"]
