"""``deepspeed.runtime.utils``: the helpers pipeline scripts and ``PipelineModule`` use
(reference ``deepspeed/runtime/utils.py:51-61,470-551``)."""
import random

import torch

from bamboo_b200 import post_training
from bamboo_b200.partition import partition_balanced, partition_uniform

__all__ = ["set_random_seed", "partition_uniform", "partition_balanced", "clip_grad_norm_"]


def set_random_seed(seed):
    """Seed ``random``, ``numpy`` and ``torch`` alike."""
    import numpy
    random.seed(seed)
    numpy.random.seed(seed)
    torch.manual_seed(seed)


def clip_grad_norm_(parameters, max_norm, norm_type=2, mpu=None):
    """Scale the gradients in place to a global 2-norm of at most ``max_norm``; returns the norm before as a float (reference
    ``deepspeed/runtime/utils.py:141-192``; ``bamboo_b200.post_training.clip_grad_norm_`` returns it without reading the device)."""
    if norm_type != 2 or mpu is not None:
        raise NotImplementedError("the 2-norm over one rank's gradients; a pipeline clips over its stages with `gradient_clipping`")
    parameters = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = [p.grad if getattr(p, "main_grad", None) is None else p.main_grad for p in parameters]
    return float(post_training.clip_grad_norm_([g for g in grads if g is not None], max_norm))
