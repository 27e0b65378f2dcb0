from .beams import BeamSelector
from .sampler import Sampler, pack_sampling

__all__ = ["BeamSelector", "Sampler", "pack_sampling"]
