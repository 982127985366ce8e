"""Public operator API: drop-in for ``coda.kernels.functional`` (README.md:45-49 of the reference)."""

from . import cross_entropy, qknorm_rope, sigmoid, sigmoid_glu, swiglu
from .cross_entropy import linear_cross_entropy, linear_cross_entropy_forward
from .cross_entropy_pieces import linear_cross_entropy_pieces
from .dropout import dropout
from .linear_e4m3 import linear_e4m3
from .qknorm_rope import linear_qknorm_rope
from .rms_norm import add_rms_norm, add_rms_norm_e4m3, quantize_e4m3, rms_norm, rms_norm_e4m3
from .sigmoid import linear_sigmoid
from .sigmoid_glu import linear_sigmoid_glu
from .swiglu import linear_swiglu

__all__ = [
    "linear_swiglu",
    "linear_sigmoid",
    "linear_sigmoid_glu",
    "linear_cross_entropy",
    "linear_cross_entropy_forward",
    "linear_qknorm_rope",
    "linear_cross_entropy_pieces",
    "rms_norm",
    "add_rms_norm",
    "dropout",
    "rms_norm_e4m3",
    "add_rms_norm_e4m3",
    "quantize_e4m3",
    "linear_e4m3",
    "swiglu",
    "sigmoid",
    "cross_entropy",
    "qknorm_rope",
]
