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


def test_mlm_loss_takes_flat_labels():
    """As many labels as positions, in any shape, as before: one value."""
    from axon.models.bert import BertForPreTraining, bert_tiny_config

    torch.manual_seed(0)
    model = BertForPreTraining(bert_tiny_config())
    ids = torch.randint(128, (2, 32))
    labels = torch.where(torch.rand(2, 32) < 0.3, ids, -100)
    want = model.mlm_loss(ids, labels)
    for flat in (labels.view(-1), labels.view(-1, 1)):
        assert torch.equal(model.mlm_loss(ids, flat), want)
    with pytest.raises((ValueError, RuntimeError)):
        model.mlm_loss(ids, labels[:1])


@pytest.mark.parametrize("kind", [1.0, 2.0, float("inf")])
def test_norm_of_complex_gradients(kind):
    """The norm of the absolute values, and gradients scaled by it."""
    from axon.optim import clip_grad_norm_, grad_norm

    torch.manual_seed(1)
    z = torch.randn(30, dtype=torch.complex64)
    x = torch.randn(7)
    size = torch.cat([z.to(torch.complex128).abs(), x.double().abs()])
    want = torch.linalg.vector_norm(size, kind)
    # 64-bit sums (and square roots); one rounding to fp32.
    assert abs(grad_norm([z, x], kind).double() - want) <= 2.0 ** -23 * want
    assert grad_norm([z, x], kind).dtype == torch.float32
    assert grad_norm([z.to(torch.complex128)], kind).dtype == torch.float64
    p, q = torch.nn.Parameter(z.clone()), torch.nn.Parameter(x.clone())
    p.grad, q.grad = z.clone(), x.clone()
    clip_grad_norm_([p, q], 0.5, kind)
    factor = 0.5 / (want + 1e-6)
    # The factor's rounding to fp32, the product's: 2 u each, twice for the
    # complex one's parts.
    for got, start in ((p.grad, z), (q.grad, x)):
        wide = start.to(torch.complex128)
        assert ((got.to(torch.complex128) - wide * factor).abs()
                <= 8 * 2.0 ** -24 * wide.abs() * factor).all()


@pytest.mark.parametrize("name", ["SGD", "Adam", "AdamW", "LAMB"])
def test_norm_of_a_step_without_gradients(name):
    """There is none, and not an earlier step's."""
    import axon.optim

    p = torch.nn.Parameter(torch.ones(4))
    opt = getattr(axon.optim, "Fused" + name)([p], lr=0.1, max_grad_norm=1.0)
    p.grad = torch.ones(4)
    opt.step()
    assert float(opt.grad_norm) == 2.0
    opt.zero_grad(set_to_none=True)
    before = p.detach().clone()
    opt.step()
    assert opt.grad_norm is None and torch.equal(p.detach(), before)
