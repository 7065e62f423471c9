"""B200 counterparts of ``memintelli.NN_layers`` (LinearMem, Conv2dMem)."""
from .linear import LinearMem
from .convolution import Conv2dMem
from .embedding import EmbeddingScaled, embedding_scaled, embedding_scaled_grad
from .functions import linear_mem_func, conv2d_mem_func, LinearMemRunc, Conv2dMemRunc

__all__ = ['LinearMem', 'Conv2dMem', 'EmbeddingScaled', 'embedding_scaled', 'embedding_scaled_grad',
           'linear_mem_func', 'conv2d_mem_func', 'LinearMemRunc', 'Conv2dMemRunc']
