from .config import CoreMode, LSSOConfig
from .layers import CausalMixer, GatedFeedForward, GroupNorm, ResidualDropout, TokenEmbedding
from .model import LSSO
from .reference import rotary_amplitude, rotary_frequencies

__all__ = [
    "CausalMixer",
    "CoreMode",
    "GatedFeedForward",
    "GroupNorm",
    "LSSO",
    "LSSOConfig",
    "ResidualDropout",
    "TokenEmbedding",
    "rotary_amplitude",
    "rotary_frequencies",
]
