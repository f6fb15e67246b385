"""Embedding lookup with scaling (csrc/kernels/embedding.hip): one pass over
the named rows forward; backward sorts the tokens by id and sums each id's
rows in order, so the gradient has the same bits each time. Eager fallback
off the GPU."""
import torch
import torch.nn as nn
import torch.nn.functional as F

_SUPPORTED = (torch.float32, torch.float16, torch.bfloat16)


def embedding(ids, weight, scale=1.0, padding_idx=None):
    """scale * weight[ids], of ids' shape with weight's rows behind it.

    ids: int32 or int64 of any shape; weight: [V, D]; scale: a number (a
    tensor is refused: it would get no gradient). The row `padding_idx`
    is looked up like any other and gets no gradient. Sums in the gradient are
    in fp32, rounded once to weight's type.

    On the GPU an id outside [0, V) gives a row of NaN and no gradient (a
    check would wait for the GPU); on the CPU it raises IndexError. A call on
    the GPU takes fewer than 2^26 ids. The gradient is not differentiable
    again. A trace holds the call as the operator axon::embedding.
    """
    if isinstance(scale, torch.Tensor):
        raise TypeError("embedding: scale must be a number")
    if weight.is_cuda and weight.dtype in _SUPPORTED:
        from axon import _core

        return _core.embedding(ids, weight, scale, padding_idx)
    if weight.dim() != 2:
        raise ValueError("embedding: weight must be [V, D], got "
                         f"{tuple(weight.shape)}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError("embedding: ids must be int32 or int64, got "
                        f"{ids.dtype}")
    if padding_idx is not None and not (
            -weight.size(0) <= padding_idx < weight.size(0)):
        raise ValueError(f"embedding: padding_idx {padding_idx} outside "
                         f"the {weight.size(0)} rows")
    y = F.embedding(ids, weight, padding_idx)
    return y if scale == 1.0 else y * scale


class FusedEmbedding(nn.Embedding):
    """nn.Embedding with the CDNA4 kernels, and a factor for its rows. Same
    state dict. max_norm, scale_grad_by_freq and sparse take torch's path."""

    def __init__(self, *args, scale=1.0, **kwargs):
        super().__init__(*args, **kwargs)
        self.scale = float(scale)

    def forward(self, input):
        if self.max_norm is None and not (self.scale_grad_by_freq or
                                          self.sparse):
            return embedding(input, self.weight, self.scale, self.padding_idx)
        y = super().forward(input)
        return y if self.scale == 1.0 else y * self.scale
