"""The language-model operators off the GPU: the formulas, refusals, and how
the optimizers and models use them."""
import copy
import math
import pickle

import pytest
import torch
import torch.nn.functional as F

from axon.ops import FusedEmbedding, cross_entropy, embedding
from axon.optim import (FusedAdam, FusedAdamW, FusedLAMB, FusedSGD,
                        clip_grad_norm_, grad_norm)

from conftest import run_distributed


def test_embedding_matches_torch():
    torch.manual_seed(0)
    w = torch.randn(9, 5, requires_grad=True)
    ids = torch.randint(9, (3, 4))
    y = embedding(ids, w, scale=2.5, padding_idx=-9)
    assert torch.equal(y, F.embedding(ids, w) * 2.5)
    y.sum().backward()
    want = torch.bincount(ids.flatten(), minlength=9)[:, None] * 2.5
    want[0] = 0
    assert torch.allclose(w.grad, want.expand(9, 5))
    assert embedding(ids.int(), w).shape == (3, 4, 5)
    m = FusedEmbedding(9, 5, padding_idx=1, scale=3.0)
    ref = torch.nn.Embedding(9, 5, padding_idx=1)
    ref.load_state_dict(m.state_dict())
    assert torch.equal(m(ids), ref(ids) * 3.0)
    table = torch.randn(4, 3)
    assert torch.equal(FusedEmbedding.from_pretrained(table)(ids % 4),
                       table[ids % 4])
    assert FusedEmbedding(9, 5, None, 2.0).max_norm == 2.0  # as nn.Embedding
    sparse = FusedEmbedding(9, 5, sparse=True)
    sparse(ids).sum().backward()
    assert sparse.weight.grad.is_sparse


def test_embedding_refusals():
    w = torch.randn(4, 3)
    ids = torch.tensor([0, 1])
    with pytest.raises(ValueError):
        embedding(ids, w[0])
    with pytest.raises(TypeError):
        embedding(ids.float(), w)
    with pytest.raises(TypeError):
        embedding(ids, w, scale=torch.tensor(2.0))
    for bad in (4, -5):
        with pytest.raises(ValueError):
            embedding(ids, w, padding_idx=bad)
    with pytest.raises(IndexError):
        embedding(torch.tensor([4]), w)


@pytest.mark.parametrize("reduction", ["none", "mean", "sum"])
@pytest.mark.parametrize("eps", [0.0, 0.1])
def test_cross_entropy_matches_torch(reduction, eps):
    torch.manual_seed(1)
    x = torch.randn(3, 4, 7, requires_grad=True)
    t = torch.randint(7, (3, 4))
    t[1, 2] = -100
    got = cross_entropy(x, t, label_smoothing=eps, reduction=reduction)
    want = F.cross_entropy(x.transpose(1, 2), t, label_smoothing=eps,
                           reduction=reduction)
    assert torch.allclose(got, want)
    half = cross_entropy(x.detach().bfloat16(), t, label_smoothing=eps,
                         reduction=reduction)
    assert half.dtype == torch.float32
    assert cross_entropy(x.double(), t).dtype == torch.float64
    assert torch.equal(cross_entropy(x, t.int()), cross_entropy(x, t))
    assert torch.isnan(cross_entropy(x, torch.full((3, 4), -100)))


def test_cross_entropy_refusals():
    x, t = torch.randn(4, 7), torch.zeros(4, dtype=torch.long)
    for kw in (dict(reduction="max"), dict(label_smoothing=1.5),
               dict(label_smoothing=-0.1)):
        with pytest.raises(ValueError):
            cross_entropy(x, t, **kw)
    with pytest.raises(ValueError):
        cross_entropy(x, t[:3])
    with pytest.raises(ValueError):
        cross_entropy(x[:, :0], t)
    with pytest.raises(TypeError):
        cross_entropy(x, torch.zeros(4))
    with pytest.raises(IndexError):
        cross_entropy(x, t + 7)


@pytest.mark.parametrize("kind", [2.0, 1, math.inf])
def test_clip_matches_torch(kind):
    def params():
        torch.manual_seed(2)
        ps = [torch.nn.Parameter(torch.zeros(s)) for s in [(3, 4), (7,), (0,)]]
        for p in ps:
            p.grad = torch.randn(p.shape)
        return ps + [torch.nn.Parameter(torch.zeros(2))]

    for bound in (0.5, 100.0):
        a, b = params(), params()
        got = clip_grad_norm_(iter(a), bound, norm_type=kind)
        # torch has no maximum over an empty gradient.
        want = torch.nn.utils.clip_grad_norm_([p for p in b if p.numel()],
                                              bound, norm_type=kind)
        assert torch.allclose(got, want)
        for p, q in zip(a[:3], b):
            assert torch.allclose(p.grad, q.grad)
    a = params()
    assert torch.allclose(grad_norm([p.grad for p in a[:3]], kind),
                          torch.nn.utils.clip_grad_norm_(a[:2], 1e9, kind))


def test_clip_edges():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(clip_grad_norm_([p], 1.0)) == 0.0
    assert float(clip_grad_norm_([], 1.0)) == 0.0
    p.grad = torch.tensor([3.0, 4.0, 0.0])
    q = torch.nn.Parameter(torch.zeros(3))
    q.grad = p.grad
    assert float(clip_grad_norm_([p, q, p], 1.0)) == 5.0  # counts once
    assert torch.allclose(p.grad, torch.tensor([0.6, 0.8, 0.0]))
    p.grad = torch.tensor([3.0, math.inf, 0.0])
    with pytest.raises(RuntimeError):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert p.grad[0] == 3.0
    for kw in (dict(max_norm=-1.0), dict(max_norm=math.nan),
               dict(max_norm=1.0, norm_type=3)):
        with pytest.raises(ValueError):
            clip_grad_norm_([p], **kw)
    with pytest.raises(ValueError):
        FusedAdamW([p], max_grad_norm=-1.0)


@pytest.mark.parametrize("make", [
    lambda ps, **kw: FusedSGD(ps, lr=0.1, momentum=0.9, dampening=0.5, **kw),
    lambda ps, **kw: FusedAdam(ps, lr=0.1, weight_decay=0.1, **kw),
    lambda ps, **kw: FusedAdamW(ps, lr=0.1, **kw),
    lambda ps, **kw: FusedLAMB(ps, lr=0.1, **kw)])
def test_clipped_step_is_clip_then_step(make):
    """max_grad_norm over all groups of the optimizer is clip_grad_norm_ and
    a step; p.grad stays as it was."""
    def params():
        torch.manual_seed(3)
        return [torch.nn.Parameter(torch.randn(s)) for s in [(4, 5), (6,)]]

    a, b = params(), params()
    groups = [{"params": [a[0]]}, {"params": [a[1]], "lr": 0.05}]
    one = make(groups, max_grad_norm=1.0)
    two = make([{"params": [b[0]]}, {"params": [b[1]], "lr": 0.05}])
    for step in range(3):
        torch.manual_seed(10 + step)
        for p, q in zip(a, b):
            p.grad = torch.randn(p.shape) * 3
            q.grad = p.grad.clone()
        raw = [p.grad.clone() for p in a]
        norm = clip_grad_norm_(b, 1.0)
        one.step()
        two.step()
        assert torch.equal(one.grad_norm, norm)
        assert all(torch.equal(p.grad, r) for p, r in zip(a, raw))
        for p, q in zip(a, b):
            assert torch.allclose(p, q, rtol=1e-6, atol=1e-7)


def test_max_grad_norm_is_kept_by_copies_not_by_state():
    p = torch.nn.Parameter(torch.ones(2))
    opt = FusedAdamW([p], max_grad_norm=0.25)
    assert copy.deepcopy(opt).max_grad_norm == 0.25
    assert pickle.loads(pickle.dumps(opt)).max_grad_norm == 0.25
    opt.load_state_dict(FusedAdamW([p]).state_dict())
    assert opt.max_grad_norm == 0.25
    torch.optim.AdamW([p]).load_state_dict(opt.state_dict())
    opt.step()  # no gradients: nothing to do
    assert opt.grad_norm is None


def _clip_of_averages(rank, size):
    """Each rank has other gradients; the norm is that of their average."""
    import axon as hvd

    p = torch.nn.Parameter(torch.zeros(3))
    opt = hvd.DistributedOptimizer(
        FusedSGD([p], lr=1.0, max_grad_norm=1.0), named_parameters=[("p", p)])
    (p * torch.tensor([6.0, 8.0, 0.0]) * (2 * rank)).sum().backward()
    opt.step()
    assert abs(float(opt.grad_norm) - 10.0) < 1e-5
    assert torch.allclose(p, torch.tensor([-0.6, -0.8, 0.0]))


def test_clipping_under_distributed_optimizer_ws2():
    run_distributed(_clip_of_averages, 2)


def test_llama_loss_is_the_shifted_loss():
    from axon.models.llama import LlamaForCausalLM, llama_tiny_config

    torch.manual_seed(4)
    model = LlamaForCausalLM(llama_tiny_config())
    ids = torch.randint(256, (2, 9))
    want = F.cross_entropy(model(ids)[:, :-1].reshape(-1, 256),
                           ids[:, 1:].reshape(-1))
    assert torch.allclose(model.lm_loss(ids), want)
    assert torch.isnan(model.lm_loss(ids[:, :1]))  # no label at all
