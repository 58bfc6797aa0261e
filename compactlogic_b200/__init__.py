"""compactlogic_b200 — the CompactLogic logic-layer hot path on hand-written sm_100a kernels.

Drop-in for the reference package: ``from compactlogic_b200 import *`` provides the same
LogicLayer / ConvLayer / GroupSum / hooks API (compactlogic/__init__.py:1).
"""
from .compactlogic import *  # noqa: F401,F403
from .compactlogic import __all__ as _api
from .packed import PackedLogicNet, packed_from_state_dict  # noqa: F401
from .training import (LogicDropout, LogicLayerNorm, PolicyLoss, action_log_probs, dropout, layer_norm,  # noqa: F401
                       policy_loss)

# The function names dropout and layer_norm are attributes of the package but not part of a star import, where they would
# hide torch.nn.functional's.
__all__ = list(_api) + ["PackedLogicNet", "packed_from_state_dict", "LogicDropout", "LogicLayerNorm",
                           "action_log_probs", "policy_loss"]
