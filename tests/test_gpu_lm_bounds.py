"""GPU tests of the language-model operators where a bound has to be tight to
say anything: classes masked by the type's lowest value, streams that the host
is far ahead of, clipped steps after the first. U = 2^-24 for each fp32
operation in the chain, half a step of the type for a rounding to it."""
import pytest
import torch

from test_gpu_lm import DEV, TYPES, U, _close, _rounded

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="needs a GPU")]


def _masked(n, vocab, dtype, low):
    """Logits of which classes are masked in several ways, and their labels,
    which are not masked."""
    g = torch.Generator(device=DEV).manual_seed(n + vocab)
    x = (torch.randn(n, vocab, generator=g, device=DEV) * 3).to(dtype)
    t = torch.full((n,), vocab // 2, device=DEV)
    at = torch.arange(vocab, device=DEV)
    keep = [at < vocab // 2 + 1,        # the last ones masked
            at >= vocab // 2,           # the first ones masked
            at % 2 == vocab // 2 % 2,   # every second one
            at == vocab // 2,           # all but the label
            at % 64 == vocab // 2 % 64,
            at < 0]                     # all alike
    mask = torch.stack([keep[i % len(keep)] for i in range(n)])
    return torch.where(mask, x, low), t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab", [
    (12, 37), (12, 1100), (2100, 1281), (12, 3001), (600, 9001), (6, 40007),
])
def test_classes_masked_by_the_lowest_value(n, vocab, dtype):
    """A masked class adds exactly 0 to the sum of a row that has others, and
    neither its distance nor its rescaling adds a rounding."""
    from axon.ops import cross_entropy

    x, t = _masked(n, vocab, dtype, torch.finfo(dtype).min)
    x.requires_grad_()
    loss = cross_entropy(x, t, reduction="none")
    dloss = torch.linspace(0.5, 2.0, n, device=DEV)
    (grad,) = torch.autograd.grad(loss, x, dloss)

    z = x.detach().double()
    top = z.amax(1, keepdim=True)
    # exp gives 0 in fp32 below -104 (2^-150).
    live = z - top > -110.0
    d = torch.where(live, z - top, 0.0)
    e = torch.where(live, d.exp(), 0.0)
    s = e.sum(1, keepdim=True)
    p, ln = e / s, s.log()
    gap = top - z.gather(1, t[:, None])
    row = (ln + gap)[:, 0]
    # exp: its difference, the factor log2 e and its product (3 |d|), 1 ulp;
    # additions of a thread (V / 16 values of a short row, up to 1280, V / 64
    # of others) and of 10 joins, each with a rescaling, whose arguments add
    # up to the range of the live values.
    steps = min(vocab / 16, 80) + vocab / 64 + 16
    reach = d.abs().amax(1, keepdim=True)
    lost = (p * d.abs()).sum(1, keepdim=True)
    s_rel = U * (2 + 3 * lost + 3 * steps + 3 * reach)
    tol = (s_rel + U * (6 * ln.abs() + 8 * gap.abs() + 4))[:, 0] \
        + 4 * U * row.abs()
    assert tol.max() <= 3e-4  # the bound says something
    _close(loss.detach(), row, tol, "loss")

    onehot = torch.zeros_like(z).scatter_(1, t[:, None], 1.0)
    want = (p - onehot) * dloss.double()[:, None]
    p_tol = p * (s_rel + U * (10 + 3 * d.abs())) + 4 * U * onehot + 2.0 ** -126
    gtol = p_tol * dloss.double()[:, None] * (1 + torch.finfo(dtype).eps) \
        + _rounded(want, dtype, 3)
    _close(grad, want, gtol, "grad")
    # Exactly nothing where a class is masked in a row that has others.
    some = live.any(1) & ~live.all(1)
    assert not grad[some][~live[some]].any()


def test_a_stream_far_behind_the_host():
    """Inputs that are NaN until the stream's last launch before the calls,
    behind milliseconds of work: a call on another stream would read them."""
    from axon.ops import cross_entropy, embedding
    from axon.optim import FusedAdamW, clip_grad_norm_, grad_norm

    g = torch.Generator(device=DEV).manual_seed(2)
    base = torch.randn(64, 5000, generator=g, device=DEV)
    t = torch.randint(5000, (64,), generator=g, device=DEV)
    ids = torch.randint(64, (3000,), generator=g, device=DEV)
    big = torch.randn(8192, 8192, generator=g, device=DEV)

    def work(x, params, opt, busy):
        x.fill_(float("nan"))
        for p in params:
            p.grad.fill_(float("nan"))
        torch.cuda.synchronize()
        if busy:
            for _ in range(3):
                big @ big
            # The host is ahead: this has not run yet.
            assert not torch.cuda.current_stream().query()
        x.copy_(base)
        for p in params:
            p.grad.copy_(base)
        leaf = x.detach().requires_grad_()
        loss = cross_entropy(leaf, t)
        (dx,) = torch.autograd.grad(loss, leaf)
        y = embedding(ids, leaf, scale=3.0)
        (dw,) = torch.autograd.grad(y, leaf, y.detach())
        norm = grad_norm([x, dx])
        opt.step()
        clipped = clip_grad_norm_(params, 0.5)
        if busy:
            assert not torch.cuda.current_stream().query()
        return [loss.detach(), dx, y.detach(), dw, norm, clipped,
                opt.grad_norm] + [p.detach() for p in params] + \
            [p.grad for p in params]

    def fresh():
        params = [torch.nn.Parameter(torch.ones(64, 5000, device=DEV))]
        params[0].grad = torch.ones(64, 5000, device=DEV)
        opt = FusedAdamW(params, lr=0.1, max_grad_norm=1.0)
        opt.step()  # the state is there: the next one reads it in one call
        return torch.empty_like(base), params, opt

    want = work(*fresh(), busy=False)
    torch.cuda.synchronize()
    assert all(torch.isfinite(w).all() for w in want)
    side = torch.cuda.Stream()
    args = fresh()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        big @ big  # the library's workspace for this stream
        got = work(*args, busy=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["Adam", "AdamW", "LAMB"])
def test_clipped_steps_after_the_first(name, dtype, monkeypatch):
    """The step that reads a whole group in one call, with the factor, against
    the formulas in 64 bits on the state that it found: clipped and unclipped
    steps, two groups, a tensor of odd length."""
    import axon.optim
    from axon import _core

    lr, wd, b1, b2 = 0.01, 0.1, 0.9, 0.999
    eps = 1e-6 if name == "LAMB" else 1e-8
    g = torch.Generator(device=DEV).manual_seed(11)
    ps = [torch.nn.Parameter(torch.randn(s, generator=g, device=DEV).to(dtype))
          for s in ((33, 65), (5,), (20001,), (3, 1000))]
    opt = getattr(axon.optim, "Fused" + name)(
        [{"params": ps[:2]}, {"params": ps[2:]}], lr=lr, weight_decay=wd,
        max_grad_norm=1.5)
    calls = []
    whole = _core.fused_adam_group
    monkeypatch.setattr(_core, "fused_adam_group",
                        lambda *a: calls.append(whole(*a)) or calls[-1])
    for t in range(1, 5):
        std = 1e-4 if t == 3 else 0.3  # the third one stays within the bound
        for p in ps:
            p.grad = (torch.randn(p.shape, generator=g, device=DEV)
                      * std).to(dtype)
        norm = torch.stack([p.grad.double().norm() for p in ps]).norm()
        factor = (1.5 / (norm + 1e-6)).clamp(max=1.0)
        assert (float(factor) == 1.0) == (t == 3)
        old = [(p.detach().double(), p.grad.double() * factor,
                *((opt.state[p][k].double() for k in ("exp_avg", "exp_avg_sq"))
                  if t > 1 else (p.detach().double() * 0,) * 2)) for p in ps]
        opt.step()
        _close(opt.grad_norm, norm, norm * 1.01 * U)
        for p, (w, c, m, v) in zip(ps, old):
            # The factor takes 6 roundings at most, h one more product and sum.
            h, dh = c, 8 * U * c.abs()
            if name == "Adam":
                h = c + wd * w
                dh = 8 * U * (c.abs() + wd * w.abs())
            # Its betas are fp32 values: 0.9 and 0.999 within u, 1 - 0.9 then
            # within 2^-24 / 0.1, 1 - 0.999 within 2^-24 / 0.001 (6e-5).
            dm = 4 * U * (b1 * m.abs() + h.abs()) + (1 - b1) * dh
            dv = 4 * U * b2 * v + 6.1e-5 * (1 - b2) * h * h \
                + 2 * (1 - b2) * h.abs() * dh
            m = b1 * m + (1 - b1) * h
            v = b2 * v + (1 - b2) * h * h
            st = opt.state[p]
            assert float(st["step"]) == t
            _close(st["exp_avg"], m, dm * 1.01 + _rounded(m, dtype, 2))
            _close(st["exp_avg_sq"], v, dv * 1.01 + _rounded(v, dtype, 2))
            # The corrections: 1 - 0.9^t within (t + 2) u / 0.1 of itself, and
            # 1 - 0.999^t within (t + 2) u / (t 0.001) (1.8e-4), its root
            # within 9e-5.
            c1, c2 = 1 - b1 ** t, (1 - b2 ** t) ** 0.5
            den = v.sqrt() / c2 + eps
            u = m / c1 / den
            du = dm / c1 / den + u.abs() * (1e-4 + 0.5 * dv / v.clamp(
                min=1e-300) + 10 * U)
            if name == "LAMB":
                step = u + wd * w
                ratio = w.norm() / step.norm()
                # The norms: 80 additions of a thread, a block's, the blocks';
                # the update's own error, in the direction of all.
                dr = 100 * U + float(du.norm() / step.norm())
                du = du + step.abs() * dr
            else:
                w = w * (1 - lr * wd) if name == "AdamW" else w
                step, ratio = u, 1.0
            want = w - lr * ratio * step
            _close(p.detach(), want,
                   1.01 * lr * ratio * du + _rounded(want, dtype, 4), name)
    assert calls == [False, False] + [True] * 6
