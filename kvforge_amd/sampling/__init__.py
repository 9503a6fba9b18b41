from kvforge_amd.sampling.params import BeamParams, SamplingParams
from kvforge_amd.sampling.rng import uniform

__all__ = ["BeamParams", "SamplingParams", "uniform"]
