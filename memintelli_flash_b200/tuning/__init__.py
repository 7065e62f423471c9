"""Operators of a language-model tuning step around the crossbar layers: token log-probabilities, the clipped policy
loss and the paired preference loss with the gradient of their logits, and global gradient-norm clipping.  The token
embedding is in ``NN_layers`` (``EmbeddingScaled``)."""
from .losses import (PolicyLoss, PreferenceLoss, policy_loss, policy_loss_grad, preference_loss,
                     preference_loss_grad, token_logprobs)
from .grad_clip import clip_grad_norm_, grad_norm

__all__ = ['token_logprobs', 'policy_loss', 'policy_loss_grad', 'PolicyLoss', 'preference_loss',
           'preference_loss_grad', 'PreferenceLoss', 'grad_norm', 'clip_grad_norm_']
