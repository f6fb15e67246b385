"""GPU tests of the clipped steps: parameters on several devices, steps after
the first against the formulas, and refusals that change nothing."""
import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="needs a GPU")]

DEV = "cuda:0"


@pytest.mark.parametrize("first", ["cpu", DEV])
@pytest.mark.parametrize("name", ["SGD", "Adam", "AdamW", "LAMB"])
def test_groups_on_two_devices(name, first):
    """One group on the CPU, one on the GPU, in either order: each step equals
    that of the same parameters in one optimizer on the CPU."""
    import axon.optim

    other = DEV if first == "cpu" else "cpu"
    g = torch.Generator().manual_seed(0)
    start = [torch.randn(s, generator=g) for s in ((40, 3), (7,), (100,))]

    def make(devices):
        ps = [torch.nn.Parameter(v.clone().to(d))
              for v, d in zip(start, devices)]
        kw = dict(momentum=0.9) if name == "SGD" else {}
        return ps, getattr(axon.optim, "Fused" + name)(
            [{"params": ps[:1]}, {"params": ps[1:]}], lr=0.05,
            weight_decay=0.1, max_grad_norm=0.5, **kw)

    a, one = make(["cpu"] * 3)
    b, two = make([first, other, other])
    for _ in range(3):
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape, generator=g)
            q.grad = p.grad.to(q.device)
        one.step()
        two.step()
        assert abs(float(one.grad_norm) - float(two.grad_norm)) \
            <= 2.0 ** -23 * float(one.grad_norm)
    for p, q in zip(a, b):
        # Three steps of 0.05 on weights of up to 4: each step's direction
        # carries the corrections 1 - b^t, 6e-5 off at the first step as the
        # kernel takes them in fp32, times a direction of at most 4.
        assert (p - q.cpu()).abs().max() <= 3 * 0.05 * 4 * 1e-4 + 1e-6
        if name != "SGD":
            assert float(two.state[q]["step"]) == 3.0
