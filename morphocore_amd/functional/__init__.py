"""Functional operators (reference: morphocore/functional/__init__.py)."""
from .dilation import dilation
from .erosion import erosion
from .opening import opening
from .closing import closing
from .sigma_layer import sigma_layer
from .smorph import smorph
from .stack import morpho_stack
from .checkpoint8 import Packed8, checkpoint8, pack8, unpack8
from .rms_norm import Normed8, rms_norm, rms_norm8
from .gated_silu import Gated8, gated_silu, gated_silu8
from .linear8 import grad_weight8, linear8
from .merge_enum import MorphoMerge, MorphoPadding, str_to_merge, str_to_padding
from ._ops import ops

__all__ = ['dilation', 'erosion', 'opening', 'closing', 'sigma_layer', 'smorph', 'morpho_stack', 'MorphoMerge', 'MorphoPadding', 'str_to_merge',
           'str_to_padding', 'Packed8', 'pack8', 'unpack8', 'checkpoint8', 'Normed8', 'rms_norm', 'rms_norm8', 'Gated8', 'gated_silu', 'gated_silu8',
           'linear8', 'grad_weight8', 'ops']
