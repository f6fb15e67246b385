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
