"""Calls of the language-model operators that their users made before, or that
the documentation allows, off the GPU."""
import pytest
import torch


def test_traced_clipping_on_the_cpu():
    from axon.optim import clip_grad_norm_

    p = torch.nn.Parameter(torch.zeros(5))
    p.grad = torch.ones(5)
    traced = torch.jit.trace(lambda x: x + clip_grad_norm_([p], 1.0),
                             (torch.zeros(1),), check_trace=False)
    assert traced(torch.zeros(1)).shape == (1,)
