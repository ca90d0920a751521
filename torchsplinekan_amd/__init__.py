"""torchsplinekan_amd -- B-spline KAN layers with a native MI355X (gfx950) backend.

Drop-in for the torch-spline-kan hot path: ``KANLinear`` / ``KAN`` with the
same API, backed by ``torchsplinekan_amd._C`` (the replacement of
``spline_kan._C``), whose device work runs in libkan_hip.so.
"""

from .kan_linear import KANLinear
from .kan import KAN
from .pruning import PruneResult, prune_nodes
from .experts import KANExperts, KANExpertStack
from .act8 import Activation8, checkpoint_8bit, quantize_activation
from .grouped import grouped_linear
from .gated import gated_linear
from .losses import linear_cross_entropy, linear_distillation
from .residual import residual_norm
from .layernorm import layer_norm

__version__ = "0.1.0"

__all__ = ["KANLinear", "KAN", "PruneResult", "prune_nodes", "Activation8", "checkpoint_8bit",
           "quantize_activation", "grouped_linear", "gated_linear", "residual_norm", "layer_norm",
           "linear_cross_entropy", "linear_distillation", "KANExperts", "KANExpertStack",
           "__version__"]
