from .block import OmniMoEBlock, RMSNorm
from .omni_moe import OmniMoE, OmniMoEConfig

__all__ = ["OmniMoE", "OmniMoEConfig", "OmniMoEBlock", "RMSNorm"]
