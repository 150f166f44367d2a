"""Selective state mixer: short causal convolution + selective scan, over whole sequences
(training, prompts) and one token at a time, and the mixer built from them."""
from .conv import short_conv, short_conv_step
from .mixer import MixerCache, SelectiveStateMixer
from .scan import selective_state_scan, selective_state_step

__all__ = ["MixerCache", "SelectiveStateMixer", "selective_state_scan", "selective_state_step", "short_conv",
           "short_conv_step"]
