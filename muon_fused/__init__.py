"""B200-native (sm_100a) Newton-Schulz engine for the Muon optimizer.

Drop-in for StarrickLiu/fused-muon's public surface (muon_fused/__init__.py:1-4):
``FusedMuon``, ``fused_newton_schulz`` and ``__version__``.  Beside them stand
the other operators of the step: ``fused_newton_schulz_heads``,
``fused_adamw`` and ``fused_normed_update``.
"""

from muon_fused.optimizer import FusedMuon
from muon_fused.ns_step import (fused_newton_schulz, fused_newton_schulz_heads, workspace_size,
                                workspace_size_heads)
from muon_fused.step_ops import fused_adamw, fused_normed_update

__version__ = "0.1.0"
__all__ = ["FusedMuon", "fused_adamw", "fused_newton_schulz", "fused_newton_schulz_heads",
           "fused_normed_update", "workspace_size", "workspace_size_heads"]
