"""Token log-probabilities, preference loss and policy loss from logits."""
from .policy import ForgePolicyLossFunction, PolicyLossOutput, forge_policy_loss  # noqa: F401
from .preference import ForgePreferenceLossFunction, PreferenceLossOutput, forge_preference_loss  # noqa: F401
from .token_logps import ForgeTokenLogpsFunction, forge_token_logps  # noqa: F401
