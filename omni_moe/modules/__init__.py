from omni_moe_b200.modules import OmniMoE, OmniMoEBlock, OmniMoEConfig, RMSNorm  # noqa: F401
