from .config import CoreMode, LSSOConfig
from .layers import GatedFeedForward, ResidualDropout, TokenEmbedding
from .model import LSSO

__all__ = ["CoreMode", "GatedFeedForward", "LSSO", "LSSOConfig", "ResidualDropout", "TokenEmbedding"]
