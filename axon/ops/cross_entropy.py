"""Cross entropy over the last dimension (csrc/kernels/cross_entropy.hip): the
logits are read in their own type, once for the loss and once for the
gradient; no fp32 copy of them and no softmax is stored. Eager fallback off
the GPU."""
import torch
import torch.nn.functional as F

_SUPPORTED = (torch.float32, torch.float16, torch.bfloat16)


def cross_entropy(logits, target, ignore_index=-100, label_smoothing=0.0,
                  reduction="mean"):
    """F.cross_entropy with the classes in the LAST dimension.

    logits: [..., V]; target: int32 or int64 of the shape before V. Rows with
    `ignore_index` count neither in the loss nor in the mean; a mean over no
    rows is NaN. Statistics and loss are fp32 whatever the logits' type (the
    loss is returned in fp32; float64 logits keep theirs), and the gradient
    is rounded once to the logits' type.

    On the GPU a label outside [0, V) that is not ignore_index makes the loss
    and its row's gradient NaN (a check would wait for the GPU); on the CPU it
    raises IndexError. A call on the GPU takes up to 2^24 - 256 rows, 2^26 -
    256 of up to 1024 vectors of 16 bytes. The gradient is not differentiable
    again. A trace holds the call as the operator axon::cross_entropy.
    """
    if logits.is_cuda and logits.dtype in _SUPPORTED:
        from axon import _core

        return _core.cross_entropy(logits, target, ignore_index,
                                   label_smoothing, reduction)
    if reduction not in ("none", "mean", "sum"):
        raise ValueError(f"cross_entropy: reduction {reduction!r}, expected "
                         "'none', 'mean' or 'sum'")
    if not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("cross_entropy: label_smoothing outside [0, 1]: "
                         f"{label_smoothing}")
    if target.dtype not in (torch.int32, torch.int64):
        raise TypeError("cross_entropy: target must hold class numbers "
                        f"(int32 or int64), got {target.dtype}")
    if (logits.dim() < 1 or logits.size(-1) == 0 or
            target.shape != logits.shape[:-1]):
        raise ValueError(f"cross_entropy: logits {tuple(logits.shape)} and "
                         f"target {tuple(target.shape)}: one label for each "
                         "row of classes")
    if logits.dtype in (torch.float16, torch.bfloat16):
        logits = logits.float()
    loss = F.cross_entropy(logits.reshape(-1, logits.size(-1)),
                           target.reshape(-1).long(),
                           ignore_index=ignore_index,
                           label_smoothing=label_smoothing,
                           reduction=reduction)
    return loss.view(target.shape) if reduction == "none" else loss
