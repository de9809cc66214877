"""luma_amd -- LUMA (Log-space Unbiased Momentum AdamW) optimizer step for MI355X.

Drop-in for ``luma_optimizer``: ``from luma_amd import LUMA``.  The step runs
in hand-written HIP kernels (gfx950) behind the C ABI of include/luma.h; see
``luma_amd.optimizer``.
"""

from luma_amd import functional  # noqa: F401  (registers torch.ops.luma_amd.luma_step)
from luma_amd.clip import clip_grad_norm_, clip_grads_with_norm_, get_total_norm  # noqa: F401
from luma_amd.config import get_kernel_config
from luma_amd.loss import linear_cross_entropy  # noqa: F401
from luma_amd.optimizer import LUMA
from luma_amd.policy import policy_loss  # noqa: F401
from luma_amd.residual import add_layer_norm, dropout, layer_norm  # noqa: F401

# (the reference's names; the operators beside the step are imported by name)
__all__ = ["LUMA", "get_kernel_config"]
__version__ = "0.1.0"
