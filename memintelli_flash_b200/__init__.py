"""memintelli_flash_b200: B200 (sm_100a) kernels for Memintelli's CIM bit-sliced matmul.

Drop-in for the hot path of the reference package:
``memintelli.pimpy`` (SlicedData, DPETensor, SNR/RE/ABSE, dot_high_dim) and
``memintelli.NN_layers`` (LinearMem, Conv2dMem).  Beside it, what tuning a language model
on such layers needs: ``NN_layers.EmbeddingScaled`` and ``tuning`` (policy and preference
losses, token log-probabilities, gradient clipping).
"""
from . import pimpy, NN_layers, tuning
from .pimpy import SlicedData, DPETensor, SNR, RE, ABSE, dot_high_dim
from .NN_layers import LinearMem, Conv2dMem, EmbeddingScaled

__version__ = "0.1.0"
