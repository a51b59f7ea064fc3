from .sampler import NonFiniteLogitsError, Sampler, StagedDrafts, StagedSample

__all__ = ["NonFiniteLogitsError", "Sampler", "StagedDrafts", "StagedSample"]
