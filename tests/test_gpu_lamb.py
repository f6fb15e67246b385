"""FusedLAMB's trust ratio on the GPU against the formula in 64 bits."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="needs a GPU")]


@pytest.mark.parametrize("shape", [(1,), (40,), (64, 65), (20000,)])
def test_lamb_trust_ratio(shape):
    from axon.optim import FusedLAMB

    g = torch.Generator(device="cuda").manual_seed(1)
    p = torch.nn.Parameter(torch.randn(shape, generator=g, device="cuda"))
    p.grad = torch.randn(shape, generator=g, device="cuda")
    w, d = p.detach().double(), p.grad.double()
    lr, wd, eps, b2 = 0.01, 0.1, 1e-6, 0.999
    FusedLAMB([p], lr=lr, weight_decay=wd, eps=eps).step()
    u = d / ((d * d * (1 - b2)).sqrt() / math.sqrt(1 - b2) + eps) + wd * w
    step = lr * (w.norm() / u.norm()) * u
    # 1 - 0.999 in fp32 is off by 2^-23 / 1e-3, its root by half of that
    # (6e-5), which the update and its norm both carry; the sums of squares
    # of up to 20000 values add less than 1e-4.
    err = (p.detach().double() - (w - step)).abs()
    assert (err <= 3e-4 * step.abs() + 2.0 ** -23 * w.abs()).all()
