"""Layers (reference: morphocore/nn/__init__.py)."""
from .dilation import Dilation
from .erosion import Erosion
from .opening import Opening
from .closing import Closing
from .sigma_layer import SigmaLayer
from .smorph import SMorph
from .stack import MorphoStack
from .rms_norm import RMSNorm
from .channel_mixer import ChannelMixer
from .token_mixer import TokenMixer
from .checkpoint8 import Checkpoint8
from .morpho_module import MorphoModule
from .alpha_module import AlphaModule

__all__ = ['Dilation', 'Erosion', 'Opening', 'Closing', 'SigmaLayer', 'SMorph', 'MorphoStack', 'RMSNorm', 'ChannelMixer', 'TokenMixer', 'Checkpoint8', 'MorphoModule', 'AlphaModule']
