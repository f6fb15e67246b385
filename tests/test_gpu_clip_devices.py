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


@pytest.mark.parametrize("clip", [None, 0.5])
@pytest.mark.parametrize("name", ["SGD", "Adam", "AdamW", "LAMB"])
def test_a_refused_step_changes_nothing(name, clip):
    """A parameter that no kernel takes, behind others that are fine: before
    and after the state is there."""
    import axon.optim

    kw = dict(momentum=0.9) if name == "SGD" else {}
    ps = [torch.nn.Parameter(torch.ones(5, device=DEV, dtype=t))
          for t in (torch.float32, torch.bfloat16, torch.float64)]
    opt = getattr(axon.optim, "Fused" + name)(
        [{"params": ps[:1]}, {"params": ps[1:]}], lr=0.1, max_grad_norm=clip,
        **kw)

    def refused():
        for p in ps:
            p.grad = torch.full_like(p, 0.25)
        before = [p.detach().clone() for p in ps]
        state = {p: {k: v.clone() for k, v in s.items()}
                 for p, s in opt.state.items()}
        with pytest.raises(RuntimeError, match="bfloat16 parameters only"):
            opt.step()
        assert all(torch.equal(p, b) for p, b in zip(ps, before))
        assert set(opt.state) == set(state)
        for p, s in state.items():
            assert set(opt.state[p]) == set(s)
            assert all(torch.equal(opt.state[p][k], v) for k, v in s.items())

    refused()
    for p in ps[:2]:
        p.grad = torch.full_like(p, 0.25)
    ps[2].grad = None
    opt.step()
    opt.step()
    assert not torch.equal(ps[0].detach(), torch.ones(5, device=DEV))
    refused()


@pytest.mark.parametrize("name", ["SGD", "Adam", "AdamW", "LAMB"])
@pytest.mark.parametrize("now", [torch.float32, torch.float16])
def test_state_of_another_type_is_refused(name, now):
    """A model cast after its optimizer's first step: the kernels read state
    as the parameter's type, past its end if that is wider."""
    import axon.optim

    layer = torch.nn.Linear(8, 4).to(DEV, torch.bfloat16)
    kw = dict(momentum=0.9) if name == "SGD" else {}
    opt = getattr(axon.optim, "Fused" + name)(layer.parameters(), lr=0.1, **kw)
    for p in layer.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    layer.to(now)
    for p in layer.parameters():
        p.grad = torch.ones_like(p)
    before = [p.detach().clone() for p in layer.parameters()]
    state = {p: {k: v.clone() for k, v in s.items()}
             for p, s in opt.state.items()}
    with pytest.raises(RuntimeError, match="state"):
        opt.step()
    assert all(torch.equal(p, b)
               for p, b in zip(layer.parameters(), before))
    for p, s in state.items():
        assert all(torch.equal(opt.state[p][k], v) for k, v in s.items())
    opt.load_state_dict(opt.state_dict())  # brings the state to the new type
    opt.step()
    assert all(not torch.equal(p, b)
               for p, b in zip(layer.parameters(), before))


def test_core_refuses_lists_that_do_not_match():
    """The launchers themselves: state of another type, shape or device."""
    from axon import _core

    p, g = (torch.ones(4, 6, device=DEV) for _ in range(2))
    bad = [torch.ones(4, 6, device=DEV, dtype=torch.bfloat16),
           torch.ones(2, 6, device=DEV), torch.ones(4, 6)]
    for m in bad:
        for gs, ms, vs in (([m], [g], [g]), ([g], [m], [g]), ([g], [g], [m])):
            with pytest.raises(RuntimeError, match="fused optimizer"):
                _core.fused_adam([p], gs, ms, vs, 0.1, 0.9, 0.99, 1e-8, 0.0, 1,
                                 False)
            with pytest.raises(RuntimeError, match="fused optimizer"):
                _core.fused_lamb([p], gs, ms, vs, 0.1, 0.9, 0.99, 1e-8, 0.0, 1)
        with pytest.raises(RuntimeError, match="fused optimizer"):
            _core.fused_sgd([p], [g], [m], 0.1, 0.9, 0.0, 0.0, False, False)
    with pytest.raises(RuntimeError, match="fused optimizer"):
        _core.fused_sgd([p, p], [g], [g, g], 0.1, 0.9, 0.0, 0.0, False, False)
    with pytest.raises(RuntimeError, match="fused optimizer"):
        _core.fused_sgd([p], [g], [], 0.1, 0.9, 0.0, 0.0, False, False)
    with pytest.raises(RuntimeError, match="fused optimizer"):
        _core.fused_adam([p], [g], [g], [], 0.1, 0.9, 0.99, 1e-8, 0.0, 1,
                         False)
    assert torch.equal(p, torch.ones(4, 6, device=DEV))
