"""psgd_pro_amd: the PSGD-Kron preconditioner update + gradient apply on MI355X (gfx950) HIP kernels.

    from psgd_pro_amd import KronWhiten, make_ops

KronWhiten is a drop-in for the reference optimizer (psgd_pro.KronWhiten / psgd_pro_fast.KronWhiten); make_ops /
HipOps is the drop-in for its arithmetic plugin (kernels/ops.py make_ops). linear_cross_entropy, residual_norm,
qk_norm_rope, window_attention and dropout are operators of the training step in front of the optimizer, AdamW
(adamw_step) the step of what a Kron preconditioner does not suit. All run on libpsgdk.so, built with
`python -m psgd_pro_amd.build`.
"""
from .adamw import AdamW, adamw_state, adamw_step
from .attention import qk_norm_rope, window_attention
from .kron import KronWhiten
from .ops import EagerOps, HipOps, make_ops
from .train import dropout, linear_cross_entropy, residual_norm

__all__ = ["KronWhiten", "EagerOps", "HipOps", "make_ops", "AdamW", "adamw_state", "adamw_step", "dropout",
           "linear_cross_entropy", "qk_norm_rope", "residual_norm", "window_attention"]
