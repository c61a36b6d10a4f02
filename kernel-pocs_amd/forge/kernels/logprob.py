"""Token log-probabilities, preference and policy losses (no reference
counterpart; beside forge.kernels.cross_entropy)."""
from kernels.logprob import (
    ForgePolicyLossFunction,
    ForgePreferenceLossFunction,
    ForgeTokenLogpsFunction,
    PolicyLossOutput,
    PreferenceLossOutput,
    forge_policy_loss,
    forge_preference_loss,
    forge_token_logps,
)

__all__ = [
    "ForgePolicyLossFunction",
    "ForgePreferenceLossFunction",
    "ForgeTokenLogpsFunction",
    "PolicyLossOutput",
    "PreferenceLossOutput",
    "forge_policy_loss",
    "forge_preference_loss",
    "forge_token_logps",
]
