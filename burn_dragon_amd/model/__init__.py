from .attention import Attention
from .bdh import BDH, DecodeGraph
from .config import BDHConfig, FusedKernelConfig
from .state import LayerState, LayerVizState, ModelState, SharedState

__all__ = ["Attention", "BDH", "DecodeGraph", "BDHConfig", "FusedKernelConfig", "LayerState", "LayerVizState", "ModelState",
           "SharedState"]
