from .embedding import Embedding
from .experts import Experts
from .linear import Linear
from .module import Parameter

__all__ = ["Parameter", "Linear", "Embedding"]     # the names of the reference; Experts is ours
