from .activation8 import Activation8, checkpoint_8bit, decode_8bit, encode_8bit
from .dilation import dilation
from .erosion import erosion
from .compositions import opening, closing, sigma_layer
from .rms_norm import rms_norm
from .smorph import smorph

__all__ = ['dilation', 'erosion', 'opening', 'closing', 'sigma_layer', 'smorph', 'rms_norm', 'Activation8', 'encode_8bit', 'decode_8bit',
           'checkpoint_8bit']
