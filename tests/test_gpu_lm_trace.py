"""The language-model operators under tracing and torch's function transforms:
a trace holds the operator itself, on its inputs, or the call is refused."""
import io

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="needs a GPU")]

DEV = "cuda:0"


def _ids(seed, shape, most):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(most, shape, generator=g, device=DEV)


def _values(seed, shape, dtype=torch.float32):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randn(shape, generator=g, device=DEV).to(dtype)


def _saved(traced):
    """The trace as it comes back from a file."""
    f = io.BytesIO()
    torch.jit.save(traced, f)
    f.seek(0)
    return torch.jit.load(f)


def test_traced_embedding():
    from axon.ops import embedding

    def f(ids, w):
        return embedding(ids, w, scale=2.5, padding_idx=-1)

    traced = torch.jit.trace(f, (_ids(0, (3, 5), 20), _values(0, (20, 9))))
    graph = str(traced.graph)
    assert "axon::embedding" in graph and "aten::empty" not in graph
    for again in (traced, _saved(traced)):
        for seed, shape in ((1, (3, 5)), (2, (7,)), (3, (2, 1, 4))):
            ids = _ids(seed, shape, 20)
            w = _values(seed, (20, 9)).requires_grad_()
            got, want = again(ids, w), f(ids, w)
            assert torch.equal(got, want)
            dy = _values(seed + 9, want.shape)
            assert torch.equal(torch.autograd.grad(got, w, dy)[0],
                               torch.autograd.grad(want, w, dy)[0])


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("shape", [(7, 33), (2, 5, 33), (2, 3, 4, 33)])
def test_traced_cross_entropy(shape, reduction):
    from axon.ops import cross_entropy

    def f(x, t):
        return cross_entropy(x, t, label_smoothing=0.1, reduction=reduction)

    def inputs(seed):
        t = _ids(seed, shape[:-1], shape[-1])
        t.view(-1)[seed % 3] = -100
        return _values(seed, shape, torch.bfloat16).requires_grad_(), t.int()

    traced = torch.jit.trace(f, inputs(0))
    graph = str(traced.graph)
    assert "axon::cross_entropy" in graph and "aten::empty" not in graph
    for again in (traced, _saved(traced)):
        for seed in (1, 2):
            x, t = inputs(seed)
            got, want = again(x, t), f(x, t)
            assert got.dtype == torch.float32 and torch.equal(got, want)
            dy = _values(seed + 9, want.shape)
            assert torch.equal(torch.autograd.grad(got, x, dy)[0],
                               torch.autograd.grad(want, x, dy)[0])


def test_traced_model():
    """Lookup, product and loss as one traced module, without gradients."""
    from axon.ops import FusedEmbedding, cross_entropy

    class Model(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.embed = FusedEmbedding(50, 16, scale=4.0)
            self.head = torch.nn.Linear(16, 50, bias=False)

        def forward(self, ids):
            return cross_entropy(self.head(self.embed(ids)), ids)

    torch.manual_seed(0)
    model = Model().to(DEV)
    with torch.no_grad():
        traced = torch.jit.trace(model, (_ids(0, (2, 8), 50),))
        for seed in (1, 2):
            ids = _ids(seed, (2, 8), 50)
            assert torch.equal(traced(ids), model(ids))


def test_traced_norm():
    from axon.optim import clip_grad_norm_, grad_norm

    traced = torch.jit.trace(lambda a, b: grad_norm([a, b], 1.0),
                             (_values(0, (9,)), _values(1, (300, 7))))
    for seed in (2, 3):
        a, b = _values(seed, (9,)), _values(seed + 5, (300, 7))
        assert torch.equal(traced(a, b), grad_norm([a, b], 1.0))

    # What is read from .grad, or written there, has no place in a trace.
    p = torch.nn.Parameter(torch.zeros(5, device=DEV))
    for nonfinite in (False, True):
        p.grad = torch.ones(5, device=DEV)

        def clip(x):
            return x + clip_grad_norm_([p], 1.0, error_if_nonfinite=nonfinite)

        with pytest.raises((NotImplementedError, RuntimeError),
                           match="traced"):
            torch.jit.trace(clip, (torch.zeros(1, device=DEV),))
        assert torch.equal(p.grad, torch.ones(5, device=DEV))


def test_fx_graphs():
    """Graphs of the operators, forward and with the gradients."""
    from torch.fx.experimental.proxy_tensor import make_fx

    from axon.ops import cross_entropy, embedding
    from axon.optim import grad_norm

    def f(ids, w, t):
        x = embedding(ids, w, scale=3.0)
        loss = cross_entropy(x, t)
        (dw,) = torch.autograd.grad(loss, w)
        return x, loss, dw, grad_norm([dw])

    def inputs(seed):
        return (_ids(seed, (6,), 20), _values(seed, (20, 9)).requires_grad_(),
                _ids(seed + 5, (6,), 9))

    graph = make_fx(f)(*inputs(0))
    for seed in (1, 2):
        for got, want in zip(graph(*inputs(seed)), f(*inputs(seed))):
            assert torch.equal(got, want)


def test_function_transforms():
    """vmap and torch.func.grad give the plain calls' results."""
    from axon.ops import cross_entropy, embedding

    ids, w = _ids(0, (4, 6), 20), _values(0, (20, 9))
    got = torch.func.vmap(lambda i: embedding(i, w, scale=2.0))(ids)
    assert torch.equal(got, embedding(ids, w, scale=2.0))
    x, t = _values(1, (4, 6, 9)), _ids(1, (4, 6), 9)
    got = torch.func.vmap(cross_entropy)(x, t)
    want = torch.stack([cross_entropy(a, b) for a, b in zip(x, t)])
    assert torch.equal(got, want)
    got = torch.func.grad(lambda v: cross_entropy(v, t[0]))(x[0])
    leaf = x[0].clone().requires_grad_()
    assert torch.equal(got, torch.autograd.grad(cross_entropy(leaf, t[0]),
                                                leaf)[0])
    got = torch.func.grad(
        lambda v: embedding(ids, v, scale=2.0).square().sum())(w)
    leaf = w.clone().requires_grad_()
    embedding(ids, leaf, scale=2.0).square().sum().backward()
    assert torch.equal(got, leaf.grad)


def test_second_derivatives_are_refused():
    """Under torch's graph and under its function transforms: an error, never
    zeros. What does not depend on the gradient again is no error."""
    from axon.ops import cross_entropy, embedding

    x, t = _values(0, (6, 9)), _ids(0, (6,), 9)
    w, ids = _values(1, (20, 9)), _ids(1, (6,), 20)

    def loss(v):
        return cross_entropy(v, t)

    def cubes(v):
        return embedding(ids, v).pow(3).sum()

    grad = torch.func.grad
    for f, v in ((loss, x), (cubes, w)):
        with pytest.raises(RuntimeError, match="not differentiable again"):
            grad(lambda u: grad(f)(u).square().sum())(v)
        with pytest.raises(NotImplementedError):
            torch.func.jvp(f, (v,), (torch.ones_like(v),))
        with pytest.raises(NotImplementedError):
            torch.func.jvp(grad(f), (v,), (torch.ones_like(v),))
        leaf = v.clone().requires_grad_()
        (g,) = torch.autograd.grad(f(leaf), leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="not differentiable again"):
            g.sum().backward()
    dy = _values(2, (6, 9))
    with pytest.raises(NotImplementedError):
        torch.func.jvp(lambda d: torch.func.vjp(
            lambda v: embedding(ids, v), w)[1](d)[0], (dy,), (dy,))
    leaf = w.clone().requires_grad_()
    (g,) = torch.autograd.grad(embedding(ids, leaf), leaf, dy,
                               create_graph=True)
    assert not g.requires_grad


def test_gradients_of_each_sample():
    from axon.ops import cross_entropy, embedding

    x, t = _values(0, (6, 9)), _ids(0, (6,), 9)
    got = torch.func.vmap(torch.func.grad(cross_entropy))(x, t)
    leaf = x.clone().requires_grad_()
    cross_entropy(leaf, t, reduction="sum").backward()
    assert torch.equal(got, leaf.grad)
    w, ids = _values(1, (3, 20, 9)), _ids(1, (6,), 20)
    got = torch.func.vmap(torch.func.grad(
        lambda v: embedding(ids, v).square().sum()))(w)
    for one, v in zip(got, w):
        leaf = v.clone().requires_grad_()
        embedding(ids, leaf).square().sum().backward()
        assert torch.equal(one, leaf.grad)


def test_modes_and_hooks_around_the_calls():
    """Clipping in an fx trace is refused; a mode that only watches, saved
    tensors on the CPU and recomputed ones change nothing."""
    from torch.fx.experimental.proxy_tensor import make_fx
    from torch.utils.checkpoint import checkpoint
    from torch.utils.flop_counter import FlopCounterMode

    from axon.ops import cross_entropy, embedding
    from axon.optim import FusedAdamW, clip_grad_norm_

    p = torch.nn.Parameter(torch.zeros(5, device=DEV))
    p.grad = torch.ones(5, device=DEV)
    opt = FusedAdamW([p], max_grad_norm=1.0)
    for f in (lambda x: x + clip_grad_norm_([p], 1.0),
              lambda x: (opt.step(), x)[1]):
        with pytest.raises(NotImplementedError, match="traced"):
            make_fx(f)(torch.zeros(1, device=DEV))
    assert torch.equal(p.grad, torch.ones(5, device=DEV))
    assert torch.equal(p.detach(), torch.zeros(5, device=DEV))

    ids, w = _ids(0, (6,), 20), _values(0, (20, 9))
    t = _ids(1, (6,), 9)

    def loss(leaf):
        return cross_entropy(embedding(ids, leaf, scale=2.0), t)

    def grad(run):
        leaf = w.clone().requires_grad_()
        run(leaf).backward()
        return leaf.grad

    want = grad(loss)
    assert torch.equal(grad(lambda v: checkpoint(
        loss, v, use_reentrant=False)), want)
    with FlopCounterMode(display=False):
        assert torch.equal(grad(loss), want)
    with torch.autograd.graph.save_on_cpu():
        assert torch.equal(grad(loss), want)
