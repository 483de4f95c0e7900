from .muon import Muon
from .selective_adam import SelectiveAdam

__all__ = ["Muon", "SelectiveAdam"]
