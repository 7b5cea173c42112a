"""Activations in 8 bits: the format, and layers that keep their input in it for the backward pass."""
import threading
from typing import NamedTuple

import torch

from ._ops import ops


class Activation8(NamedTuple):
    """A tensor in 8 bits: what `encode_8bit`, and `rms_norm` with an 8-bit output, return.

    codes : int8, in the tensor's shape.
    scales : float32 (float64 for a float64 tensor), (leading dimensions..., blocks of a row): the dimensions that it does not have
        make up a row, which is cut into blocks of 128 elements, the last one shorter.
    dtype : the type that it was encoded from, and is decoded to.

    With m the largest finite magnitude of a block, scale = m / 126 and code = round(x * (126 / m)); a finite value comes back within
    half a scale. -128 stands for NaN, -127 and 127 for the infinities. A block without a magnitude of 2^-100 (2^-900) or more
    is stored as zeros.
    """
    codes: torch.Tensor
    scales: torch.Tensor
    dtype: torch.dtype

    @property
    def shape(self) -> torch.Size:
        return self.codes.shape

    @property
    def nbytes(self) -> int:
        return self.codes.nbytes + self.scales.nbytes


def encode_8bit(x: torch.Tensor, row_dims: int = 2) -> Activation8:
    """The 8-bit form of `x` (float32, float64, float16 or bfloat16, CUDA): 1.03 bytes an element where rows are long.

    row_dims : trailing dimensions that make up a row; no block crosses from one row to the next. 2 for feature maps (one plane
        of H x W pixels a row), 1 for rows of channels. Not differentiable: no gradient flows through the codes.
    """
    codes, scales = ops.encode_8bit(x, min(row_dims, x.dim()) if x.dim() else row_dims)
    return Activation8(codes, scales, x.dtype)


def decode_8bit(packed: Activation8) -> torch.Tensor:
    """The values that an activation in 8 bits stands for, in the type it was encoded from."""
    return ops.decode_8bit(packed.codes, packed.scales, packed.dtype)


class _Mode(threading.local):
    """What `checkpoint_8bit` asks of the layers that are called under it, in the calling thread."""
    active = False
    packed = None     # the 8-bit form that the caller has of `packed_of`, at that tensor's `version`
    packed_of = None
    version = None


_mode = _Mode()


def keeping_8bit() -> bool:
    """Whether the layers called now keep their input in 8 bits."""
    return _mode.active


def _version(x):
    """A tensor's count of changes in place, None for what has none."""
    return x._version if isinstance(x, torch.Tensor) and not x.is_inference() else None


def kept_codes(x: torch.Tensor = None) -> tuple:
    """Codes and scales that the caller has for `x`, the input of the layer called now, or (None, None): they are those of one tensor, and
    a layer that is called on another one, or on what has become of it, encodes its own. Without `x`, those of whatever tensor."""
    if _mode.packed is None or (x is not None and (x is not _mode.packed_of or _version(x) != _mode.version)):
        return None, None
    return _mode.packed.codes, _mode.packed.scales


def checkpoint_8bit(function, *args, packed: Activation8 = None, **kwargs):
    """`function(*args, **kwargs)`, with what its layers keep for the backward pass in 8 bits.

    function : an operation of `morphocore_b200.functional` or any callable that uses them, a module of `morphocore_b200.nn` or a whole
        model. Its outputs are those of the plain call. Every dilation, erosion, smorph (and what is composed of them) and rms_norm
        in it then keeps its input as an `Activation8`, a quarter of a float32 tensor, and its backward pass gives the
        gradients at the values that the codes stand for. Dilations and erosions with a 'max' or 'min' merge and save_indices=True
        keep their winning indices alone, and their gradients are the exact ones; pass save_indices=False to keep the 8-bit input
        instead. Under torch.no_grad() nothing is kept, and nothing encoded.
    packed : the 8-bit form of the layer's input, where the caller has it already (`rms_norm` with output='both' has written it), so
        that the layer need not encode it again. For a single dilation, erosion, smorph or sigma_layer, or a module of one; it must
        be the 8-bit form of the very input. Other layers that run meanwhile, in a module derived from one of these or in a hook, encode
        their own inputs.

    The input may be changed in place, or freed, before the backward pass.
    """
    if packed is not None and not getattr(function, "takes_packed", False):
        raise ValueError("packed is the input of one layer: dilation, erosion, smorph, sigma_layer or a module of one of them")
    x = args[0] if args else kwargs.get("x")
    before = _mode.active, _mode.packed, _mode.packed_of, _mode.version
    _mode.active, _mode.packed, _mode.packed_of, _mode.version = True, packed, x, _version(x)
    try:
        return function(*args, **kwargs)
    finally:
        _mode.active, _mode.packed, _mode.packed_of, _mode.version = before
