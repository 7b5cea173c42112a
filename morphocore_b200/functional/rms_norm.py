import torch

from ._ops import ops
from .activation8 import Activation8, keeping_8bit

_OUTPUTS = {"float": (True, False), "8bit": (False, True), "both": (True, True)}


def rms_norm(x: torch.Tensor, weight: torch.Tensor = None, residual: torch.Tensor = None, eps: float = 1e-6, dim: int = -3,
             output: str = "float"):
    """Root-mean-square norm over the channels, after the addition of a residual, on the GPU.

    s = x + residual (rounded to the tensors' type; s = x without a residual),
    y = s / sqrt(mean_c s^2 + eps) * weight[c].

    x : float32, float64, float16 or bfloat16, CUDA; (N, C, H, W) or (C, H, W) with the default `dim`.
    weight : (C,), optional, in the type of x, or float32 beside an x in half precision (it then enters, and gets its gradient, unrounded).
    residual : like x, optional, in its type.
    dim : the dimension that is normalised, at most 16384 long: -3 for the channels of feature maps, -1 for rows of channels.
    output : 'float' for y; '8bit' for its 8-bit form (an `Activation8` with a row for every plane of what follows `dim`, or for
        the channels where a single element follows), which `decode_8bit` reads; 'both' for y and that form, to be handed to the layer
        behind the norm (`checkpoint_8bit(layer, y, ..., packed=...)`).
    Returns y, the 8-bit form, or both of them; with a residual also s: (y, s), (packed, s) or (y, packed, s).

    The mean and the factor are held in double. In float32 y is rounded once, in half precision from that float32, so that y and its codes
    do not depend on strides or alignment; in float64 the last place may.
    Differentiable once in x, residual and weight; the 8-bit form has no gradient, so 'float' or 'both' in training.
    """
    try:
        want_y, want_codes = _OUTPUTS[output]
    except (KeyError, TypeError):
        raise ValueError(f"Unknown output: {output}. Expected one of {sorted(_OUTPUTS)}.") from None
    out = list(ops.rms_norm(x, residual, weight, eps, dim, want_y, want_codes, keeping_8bit()))
    result = [out.pop(0)] if want_y else []
    total = [out.pop(0)] if residual is not None else []
    if want_codes:
        result.append(Activation8(*out, x.dtype))
    result += total
    return result[0] if len(result) == 1 else tuple(result)
