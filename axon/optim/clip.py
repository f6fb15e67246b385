"""The norm over all gradients, and clipping by it (csrc/kernels/grad_norm.hip):
one launch for up to 192 tensors reads the gradients, and one scales them where
the norm is over its bound; nothing waits for the GPU. Eager fallback off the
GPU."""
import math

import torch

_SUPPORTED = (torch.float32, torch.float16, torch.bfloat16)
_TYPES = {1.0: 1, 2.0: 2, math.inf: 0}


def _checked_type(norm_type):
    norm_type = float(norm_type)
    if norm_type not in _TYPES:
        raise ValueError(f"norm_type {norm_type}: expected 1, 2 or inf")
    return norm_type


def _checked_max(max_norm):
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be >= 0, got {max_norm}")
    return max_norm


def _fast_path(tensors):
    dev = tensors[0].device
    return dev.type == "cuda" and all(
        t.device == dev and t.dtype in _SUPPORTED and
        t.layout == torch.strided for t in tensors)


def _once(tensors):
    seen, kept = set(), []
    for t in tensors:
        key = (t.data_ptr(), t.shape, t.stride(), t.dtype, t.device)
        if t.numel() == 0 or key not in seen:
            seen.add(key)
            kept.append(t)
    return kept


def _norm_eager(tensors, norm_type):
    norms = [torch.linalg.vector_norm(
                 t.detach().to(torch.complex128 if t.is_complex()
                               else torch.float64), norm_type)
             for t in _once(tensors) if t.numel()]
    if not norms:
        return torch.zeros((), device=tensors[0].device)
    norms = torch.stack([n.to(norms[0].device) for n in norms])
    total = torch.linalg.vector_norm(norms, norm_type)
    wide = any(t.dtype in (torch.float64, torch.complex128) for t in tensors)
    return total if wide else total.float()


def norm_and_factor(tensors, max_norm, norm_type=2.0):
    """The norm over `tensors` (one at least) and the factor that clips it,
    min(1, max_norm / (norm + 1e-6)): two 0-dim tensors."""
    if _fast_path(tensors):
        from axon import _core

        out = _core.grad_norm(tensors, _TYPES[norm_type], max_norm)
        return out[0], out[1]
    norm = _norm_eager(tensors, norm_type)
    return norm, (max_norm / (norm + 1e-6)).clamp(max=1.0)


@torch.no_grad()
def grad_norm(tensors, norm_type=2.0):
    """The norm over all values of `tensors` (gradients, say) as one vector: a
    0-dim fp32 tensor (fp64 if one of them is). norm_type: 1, 2 or inf. Sums
    are in 64 bits. A tensor given twice counts once; none at all give 0."""
    norm_type = _checked_type(norm_type)
    tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    if not tensors:
        return torch.tensor(0.0)
    return norm_and_factor(tensors, math.inf, norm_type)[0]


@torch.no_grad()
def clip_grad_norm_(parameters, max_norm, norm_type=2.0,
                    error_if_nonfinite=False):
    """Scale the gradients in place by min(1, max_norm / (norm + 1e-6)), with
    the norm over all of them (torch.nn.utils.clip_grad_norm_). Returns the
    norm before clipping, a 0-dim fp32 tensor on the gradients' device.

    norm_type: 1, 2 or inf. A gradient that several parameters share counts
    once and is scaled once; on the GPU, gradients that share memory in part
    are refused.
    A norm of inf or NaN makes the factor 0 or NaN as in torch;
    error_if_nonfinite raises instead (and waits for the GPU). On the GPU a
    call cannot be traced (NotImplementedError): the gradients are no arguments.

    Under DistributedOptimizer the gradients are averaged first:

        opt.synchronize()
        axon.optim.clip_grad_norm_(model.parameters(), 1.0)
        with opt.skip_synchronize():
            opt.step()

    or give the fused optimizer max_grad_norm, and step() does both. Under a
    GradScaler, unscale the gradients first (scaler.unscale_(opt)), either way.
    """
    norm_type, max_norm = _checked_type(norm_type), _checked_max(max_norm)
    parameters = ([parameters] if isinstance(parameters, torch.Tensor)
                  else list(parameters))
    if not error_if_nonfinite:
        from axon import _core

        out = _core.param_grad_norm([parameters], _TYPES[norm_type], max_norm,
                                    True)
        if out is None:
            return torch.tensor(0.0)
        if out is not False:
            return out[0]
    grads = [g for g in (p.grad for p in parameters) if g is not None]
    if not grads:
        return torch.tensor(0.0)
    norm, factor = norm_and_factor(grads, max_norm, norm_type)
    if error_if_nonfinite and not torch.isfinite(norm):
        raise RuntimeError(f"the norm of order {norm_type} over all gradients "
                           f"is {float(norm)}; the gradients are unchanged")
    if _fast_path(grads):
        from axon import _core

        _core.grad_scale_(grads, factor)
        return norm
    for g in _once(grads):
        g.mul_(factor.to(g.device))
    return norm
