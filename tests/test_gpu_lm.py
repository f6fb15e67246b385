"""GPU tests of the language-model operators: embedding, cross entropy and the
gradient norm, against plain formulas in 64 bits. Tolerances are bounds from
the arithmetic: u = 2^-24 for each fp32 operation in the chain, half a step of
the result's type for its one rounding."""
import math

import pytest
import torch

pytestmark = [pytest.mark.gpu,
              pytest.mark.skipif(not torch.cuda.is_available(),
                                 reason="needs a GPU")]

DEV = "cuda:0"
U = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _close(got, want, tol, what=""):
    """|got - want| <= tol where want is finite, the same inf and NaN where
    it is not. tol: of want's shape."""
    got = got.double()
    assert got.shape == want.shape, what
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    odd = ~fine & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd]), what
    over = ((got - want).abs() - tol)[fine]
    assert over.numel() == 0 or over.max() <= 0, (what, float(over.max()))


def _rounded(want, dtype, chain):
    """The bound for a value that `chain` fp32 roundings lead to and that is
    then rounded to dtype: half a step, of the least normal's at least."""
    f = torch.finfo(dtype)
    return want.abs() * (chain * U + f.eps / 2 * (1 + chain * U)) + \
        f.smallest_normal * f.eps / 2


# ------------------------------------------------------------- embedding

def _ids(kind, n, vocab, g):
    if kind == "same":
        return torch.full((n,), vocab - 1, device=DEV)
    if kind == "falling":
        return (vocab - 1 - torch.arange(n, device=DEV) % vocab)
    ids = torch.randint(vocab, (n,), generator=g, device=DEV)
    if kind == "skewed":  # half of the tokens are one word
        half = torch.rand(n, generator=g, device=DEV) < 0.5
        ids = torch.where(half, vocab // 2, ids)
    return ids


def _embedding_wanted(ids, w, dy, scale, padding):
    """(out, dw, their bounds) in 64 bits."""
    vocab = w.size(0)
    flat = ids.reshape(-1).long()
    known = (flat >= 0) & (flat < vocab)
    out = w.double()[flat.clamp(0, vocab - 1)] * scale
    out[~known] = math.nan
    part = known if padding is None else known & (flat != padding)
    d = dy.double().reshape(len(flat), -1)[part]
    to = flat[part]
    dw = torch.zeros(w.shape, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(dw).index_add_(0, to, d.abs()) * abs(scale)
    dw.index_add_(0, to, d * scale)
    count = torch.bincount(to, minlength=vocab)[:, None]
    f = torch.finfo(w.dtype)
    # count - 1 additions, in any order, and the factor's product.
    tol = size * (count + 1) * U + _rounded(dw, w.dtype, 2)
    tol += size * (count + 1) * U * f.eps
    return (out.reshape(*ids.shape, -1), dw,
            _rounded(out, w.dtype, 1).reshape(*ids.shape, -1), tol)


def _embedding_case(n, vocab, dim, dtype, kind, scale, padding, seed=0):
    from axon.ops import embedding

    g = torch.Generator(device=DEV).manual_seed(seed)
    ids = _ids(kind, n, vocab, g)
    w = torch.randn(vocab, dim, generator=g, device=DEV).to(dtype)
    w.requires_grad_()
    dy = torch.randn(n, dim, generator=g, device=DEV).to(dtype)
    out = embedding(ids, w, scale=scale, padding_idx=padding)
    assert out.dtype == dtype
    out.backward(dy)
    want, dw, tol, dtol = _embedding_wanted(ids, w.detach(), dy, scale,
                                            padding)
    _close(out.detach(), want, tol, "out")
    assert w.grad.dtype == dtype
    _close(w.grad, dw, dtol, "grad")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab,dim", [
    (1, 1, 1), (1, 7, 3), (3, 2, 16), (63, 5, 65), (300, 10, 33),
    (2047, 700, 8), (2049, 50, 24), (2500, 129, 1032), (5000, 3, 130),
    (33000, 999, 12), (40, 20000, 17),
])
def test_embedding(n, vocab, dim, dtype):
    _embedding_case(n, vocab, dim, dtype, "uniform", 1.0, None)
    _embedding_case(n, vocab, dim, dtype, "skewed", 22.5, 0, seed=1)


@pytest.mark.parametrize("kind", ["same", "falling", "skewed"])
@pytest.mark.parametrize("n", [256, 4097, 32769, 70000])
def test_embedding_orders(kind, n):
    _embedding_case(n, 37, 40, torch.bfloat16, kind, 0.5, None)
    _embedding_case(n, 37, 40, torch.float32, kind, -3.0, 18)


def test_embedding_no_tokens():
    from axon.ops import embedding

    w = torch.randn(5, 8, device=DEV, requires_grad=True)
    one = embedding(torch.tensor(3, device=DEV), w)  # a single id
    assert torch.equal(one, w[3])
    empty = torch.zeros(0, 8, device=DEV, requires_grad=True)
    rows = embedding(torch.tensor([0, 1], device=DEV), empty)  # no table
    assert rows.isnan().all()
    rows.sum().backward()
    assert empty.grad.shape == (0, 8)

    w = torch.randn(5, 8, device=DEV, requires_grad=True)
    out = embedding(torch.zeros(2, 0, dtype=torch.long, device=DEV), w)
    assert out.shape == (2, 0, 8)
    out.sum().backward()
    assert torch.equal(w.grad, torch.zeros_like(w))


def test_embedding_ids_outside():
    """NaN rows, no gradient, and nothing read or written outside."""
    from axon.ops import embedding

    ids = torch.tensor([3, -1, 0, 10, 1 << 40, -(1 << 40), 3, 9], device=DEV)
    for dtype in TYPES:
        w = torch.randn(10, 9, device=DEV).to(dtype).requires_grad_()
        dy = torch.randn(8, 9, device=DEV).to(dtype)
        out = embedding(ids, w, scale=2.0)
        out.backward(dy)
        want, dw, tol, dtol = _embedding_wanted(ids, w.detach(), dy, 2.0, None)
        _close(out.detach(), want, tol)
        _close(w.grad, dw, dtol)


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_layouts(dtype):
    """int32 ids of two dimensions and odd strides, rows of a wider matrix,
    a transposed weight, an expanded gradient, a negative padding_idx."""
    from axon.ops import embedding

    g = torch.Generator(device=DEV).manual_seed(3)
    ids = torch.randint(11, (6, 10), generator=g, device=DEV,
                        dtype=torch.int32)[:, ::2]
    wide = torch.randn(11, 50, generator=g, device=DEV).to(dtype)
    for w in (wide[:, 3:20], wide[:, ::2], wide.t()[:11].contiguous().t()):
        leaf = w.detach().clone().requires_grad_()
        view = torch.empty_strided(w.shape, w.stride(), dtype=dtype,
                                   device=DEV)
        view.copy_(w)
        view.requires_grad_()
        out = embedding(ids, view, scale=1.5, padding_idx=-1)
        dy = torch.randn(1, 1, w.size(1), generator=g, device=DEV).to(
            dtype).expand(out.shape)
        out.backward(dy)
        want, dw, tol, dtol = _embedding_wanted(ids, leaf.detach(), dy, 1.5,
                                                10)
        _close(out.detach(), want, tol)
        _close(view.grad, dw, dtol)


def test_embedding_module_and_same_bits():
    from axon.ops import FusedEmbedding

    torch.manual_seed(0)
    ref = torch.nn.Embedding(50, 24, padding_idx=4).to(DEV)
    mine = FusedEmbedding(50, 24, padding_idx=4).to(DEV)
    mine.load_state_dict(ref.state_dict())
    ids = torch.randint(50, (8, 300), device=DEV)
    assert torch.equal(mine(ids), ref(ids))
    dy = torch.randn(8, 300, 24, device=DEV)
    grads = []
    for _ in range(3):
        mine.zero_grad()
        mine(ids).backward(dy)
        grads.append(mine.weight.grad.clone())
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])
    assert not grads[0][4].any()


# --------------------------------------------------------- cross entropy

def _loss_wanted(x, target, dloss, eps, ignore, reduction):
    """Row losses (or their mean/sum), gradient, and bounds, in 64 bits."""
    vocab = x.size(-1)
    z = x.double().reshape(-1, vocab)
    t = target.reshape(-1)
    n = len(t)
    used = t != ignore
    known = (t >= 0) & (t < vocab)
    at = t.clamp(0, vocab - 1)[:, None]
    top = z.amax(1, keepdim=True)
    d = z - top
    e = d.exp()
    s = e.sum(1, keepdim=True)
    p = e / s
    ln = s.log()
    gap = top - z.gather(1, at)
    row = (1 - eps) * (ln + gap)
    if eps:
        row = row + eps * (ln + top - z.mean(1, keepdim=True))
    row = torch.where(known[:, None], row, math.nan)[:, 0]
    row = torch.where(used, row, 0.0)
    onehot = torch.zeros_like(z).scatter_(1, at, 1.0)
    g = p - (1 - eps) * onehot - eps / vocab
    g = torch.where(known[:, None], g, math.nan)
    count = int(used.sum())
    if reduction == "none":
        per_row, loss = dloss.double().reshape(-1), row
    else:
        per_row = dloss.double().reshape(1).expand(n)
        loss = row.sum()
        if reduction == "mean":
            per_row = per_row / max(count, 1)
            loss = loss / count if count else loss * math.nan
    grad = torch.where(used[:, None], g * per_row[:, None], 0.0)
    # Roundings: exp (argument: its difference, the factor log2 e and its
    # product; the result: 1 ulp = 2 u), the additions of one thread and of
    # the joins, a rescaling at each step whose arguments add up to the range.
    fine = lambda v: torch.where(torch.isfinite(v), v, 0.0)  # noqa: E731
    # A thread has V / 16 values of a short row (up to 1280), V / 64 of others.
    steps = min(vocab / 16, 80) + vocab / 64 + 16
    reach = fine(d).abs().amax(1, keepdim=True)
    lost = fine(p * fine(d).abs()).sum(1, keepdim=True)
    s_rel = U * (2 + 3 * lost + 3 * steps + 3 * reach)
    size = fine(z).abs().mean(1, keepdim=True)
    row_tol = s_rel + U * (6 * fine(ln).abs() + 4 * fine(gap).abs() + 4)
    if eps:
        row_tol = row_tol + U * (steps + 4) * (size + fine(top).abs())
    row_tol = row_tol[:, 0]
    row_tol = row_tol + 4 * U * fine(row).abs()
    if reduction == "none":
        tol = row_tol
    else:
        tol = torch.where(used, row_tol, 0.0).sum()
        tol = tol / max(count, 1) if reduction == "mean" else tol
        tol = tol + 2 * U * fine(loss).abs()
    p_tol = p * (s_rel + U * (6 + 3 * fine(d).abs())) + 4 * U * onehot + \
        4 * U * eps / vocab + 4 * U * p
    # The GPU's exp2 gives 0 below the least normal value, 2^-126; S >= 1.
    p_tol = p_tol + 2.0 ** -126
    exact = _rounded(grad, x.dtype, 3)
    gtol = torch.where(torch.isfinite(p_tol), p_tol, 0.0) * \
        per_row.abs()[:, None] * (1 + torch.finfo(x.dtype).eps) + exact
    return (loss, grad.reshape(x.shape), tol, gtol.reshape(x.shape))


def _loss_check(x, target, eps=0.0, ignore=-100, reduction="mean",
                dloss=None):
    from axon.ops import cross_entropy

    x.requires_grad_()
    loss = cross_entropy(x, target, ignore_index=ignore, label_smoothing=eps,
                         reduction=reduction)
    assert loss.dtype == torch.float32
    if dloss is None:
        dloss = torch.full(loss.shape, 1.0, device=DEV)
    (grad,) = torch.autograd.grad(loss, x, dloss)
    assert grad.dtype == x.dtype
    want, g, tol, gtol = _loss_wanted(x.detach(), target, dloss, eps, ignore,
                                      reduction)
    _close(loss.detach().reshape(want.shape), want, tol, "loss")
    _close(grad, g, gtol, "grad")
    return loss, grad


def _logits(n, vocab, dtype, seed=0, std=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(n, vocab, generator=g, device=DEV) * std).to(dtype)
    t = torch.randint(vocab, (n,), generator=g, device=DEV)
    return x, t, g


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,vocab", [
    (1, 1), (1, 2), (5, 7), (64, 10), (33, 255), (9, 1000), (4, 1024),
    (4, 1025), (3, 4099), (130, 2051), (1, 50001), (2, 131072), (700, 8191),
    (2100, 1281), (2100, 2600), (2500, 8200), (513, 641), (20, 1280),
])
def test_cross_entropy(n, vocab, dtype):
    x, t, g = _logits(n, vocab, dtype)
    t[torch.rand(n, generator=g, device=DEV) < 0.2] = -100
    _loss_check(x, t)
    x, t, g = _logits(n, vocab, dtype, seed=1)
    weights = torch.randn(n, generator=g, device=DEV)
    _loss_check(x, t, eps=0.1, reduction="none", dloss=weights)
    x, t, g = _logits(n, vocab, dtype, seed=2)
    _loss_check(x, t, reduction="sum", ignore=0,
                dloss=torch.tensor(-2.5, device=DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [37, 3001, 40007])
def test_cross_entropy_odd_values(dtype, vocab):
    """Classes masked by -inf or by the type's lowest value, rows of nothing
    else, inf, NaN, rows all ignored, confident rows."""
    low = torch.finfo(dtype).min
    x, t, g = _logits(12, vocab, dtype)
    t[:] = 5
    x[0, 6:] = -math.inf            # masked classes
    x[1, 6:] = low
    x[2] = -math.inf                # nothing left: NaN
    x[3] = low                      # all alike
    x[4, 9] = math.inf              # NaN
    x[5, 8] = math.nan
    x[6, 5] = -math.inf             # the label itself is masked: inf
    x[7, 5] = 500.0                 # certain
    x[8] = 0.0
    x[9, :6], x[9, 6:] = -math.inf, 1.0
    t[10] = -100
    x[10] = math.nan                # ignored: not read
    x[11, -1] = -math.inf
    for reduction in ("none",):
        _loss_check(x.clone(), t, reduction=reduction)
    keep = torch.tensor([0, 1, 3, 7, 8, 11], device=DEV)
    _loss_check(x[keep].contiguous(), t[keep])
    _loss_check(x[8:11].clone(), torch.full((3,), -100, device=DEV))
    _loss_check(x[[3, 8]].clone(), t[[3, 8]], eps=0.3)


def test_cross_entropy_labels_outside():
    for vocab in (50, 2000):
        x, t, _ = _logits(6, vocab, torch.bfloat16)
        t[1], t[4], t[5] = vocab, -1, 1 << 40
        _loss_check(x, t, reduction="none")


@pytest.mark.parametrize("dtype", TYPES)
def test_cross_entropy_layouts(dtype):
    """Leading shapes, rows with strides, a slice that skips the last row of
    each sequence, a transposed matrix, int32 labels, one row alone."""
    from axon.ops import cross_entropy

    g = torch.Generator(device=DEV).manual_seed(5)
    base = torch.randn(3, 8, 70, generator=g, device=DEV).to(dtype)
    t = torch.randint(60, (3, 8), generator=g, device=DEV)
    for x, y in [(base[:, :-1, :61], t[:, 1:]), (base[:, ::2, 5:66], t[:, ::2]),
                 (base.transpose(0, 1)[..., :60], t.t()),
                 (base[0].t()[:60].t(), t[0]), (base[1, 2, :60], t[1, 2]),
                 (base[:1, :1].expand(3, 8, 70), t)]:
        view = x.detach()
        view.requires_grad_()
        loss = cross_entropy(view, y.to(torch.int32), reduction="none")
        assert loss.shape == y.shape
        dloss = torch.rand(y.shape, generator=g, device=DEV)
        (grad,) = torch.autograd.grad(loss, view, dloss)
        want, gw, tol, gtol = _loss_wanted(x, y, dloss, 0.0, -100, "none")
        _close(loss.detach().reshape(-1), want, tol)
        _close(grad, gw, gtol)
    x4 = base.reshape(3, 2, 4, 70)
    assert torch.equal(cross_entropy(x4, t.view(3, 2, 4), reduction="none"),
                       cross_entropy(base, t, reduction="none").view(3, 2, 4))
    # The gradient of a sum has one value for all rows.
    x = base[0].clone().requires_grad_()
    cross_entropy(x, t[0], reduction="none").sum().backward()
    y = base[0].clone().requires_grad_()
    cross_entropy(y, t[0], reduction="sum").backward()
    assert torch.equal(x.grad, y.grad)
    none = cross_entropy(base[:0].requires_grad_(), t[:0], reduction="sum")
    assert float(none.detach()) == 0.0


def test_cross_entropy_long_offsets():
    """Rows that start past 2^31 values."""
    from axon.ops import cross_entropy

    rows, vocab = 2, 70000
    big = torch.zeros(1 << 31, device=DEV, dtype=torch.bfloat16)
    x = torch.as_strided(big, (rows, vocab), ((1 << 31) - vocab, 1))
    x.copy_(torch.randn(rows, vocab, device=DEV))
    t = torch.tensor([3, vocab - 1], device=DEV)
    want, _, tol, _ = _loss_wanted(x, t, torch.ones(2, device=DEV), 0.0, -100,
                                   "none")
    _close(cross_entropy(x, t, reduction="none"), want, tol)


def test_cross_entropy_differences():
    """The gradient against central differences of the 64-bit loss."""
    x, t, _ = _logits(4, 30, torch.float32, std=1.0)
    _, grad = _loss_check(x, t, eps=0.1)
    z = x.detach().double()
    h = 1e-5
    for i, j in [(0, 0), (1, int(t[1])), (3, 29)]:
        up, down = z.clone(), z.clone()
        up[i, j] += h
        down[i, j] -= h
        f = lambda v: torch.nn.functional.cross_entropy(  # noqa: E731
            v, t, label_smoothing=0.1)
        # h^2 / 6 times a third derivative of at most 1, and 64-bit noise.
        assert abs(float((f(up) - f(down)) / (2 * h)) -
                   float(grad[i, j])) < 1e-9 + 1e-10 + 40 * U


def test_cross_entropy_twice_backward():
    """A second backward pass over a kept graph gives the same gradient, and
    a loss changed in place by its user does not reach it."""
    from axon.ops import cross_entropy

    x, t, _ = _logits(10, 100, torch.bfloat16)
    x.requires_grad_()
    loss = cross_entropy(x, t)
    (a,) = torch.autograd.grad(loss, x, retain_graph=True)
    a0 = a.clone()
    a.zero_()
    (b,) = torch.autograd.grad(loss, x, retain_graph=True)
    assert torch.equal(a0, b)
    loss2 = cross_entropy(x, t)
    loss2.div_(1.0)
    (c,) = torch.autograd.grad(loss2, x)
    assert torch.equal(a0, c)


# ---------------------------------------------------------- gradient norm

def _params(shapes, dtypes, seed=0, std=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    ps = []
    for shape, dtype in zip(shapes, dtypes):
        p = torch.nn.Parameter(torch.zeros(shape, device=DEV, dtype=dtype))
        p.grad = (torch.randn(shape, generator=g, device=DEV) * std).to(dtype)
        ps.append(p)
    return ps


def _clip_wanted(grads, max_norm, kind):
    gs = [g.double() for g in grads]
    if kind == 2:
        norm = sum((g ** 2).sum() for g in gs).sqrt()
    elif kind == 1:
        norm = sum(g.abs().sum() for g in gs)
    else:
        norm = torch.stack([g.abs().max() for g in gs if g.numel()]).max()
    c = (max_norm / (norm + 1e-6)).clamp(max=1.0)
    return norm, [g * c for g in gs]


def _clip_check(ps, max_norm, kind=2.0):
    from axon.optim import clip_grad_norm_

    grads = [p.grad.clone() for p in ps]
    norm, want = _clip_wanted(grads, max_norm, kind)
    got = clip_grad_norm_(ps, max_norm, norm_type=kind)
    assert got.dtype == torch.float32 and got.dim() == 0
    # 64-bit sums; one rounding to fp32.
    _close(got, norm, norm * 1.01 * U + 1e-45)
    for p, w in zip(ps, want):
        # The factor: the norm, the sum with 1e-6, the quotient (1 ulp at
        # most: 2 u); then the product.
        _close(p.grad, w, _rounded(w, p.dtype, 6))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [2.0, 1.0, math.inf])
def test_clip(dtype, kind):
    shapes = [(1,), (3,), (0,), (16384,), (16385,), (257, 65), (7, 9, 11),
              (70001,), ()]
    _clip_check(_params(shapes, [dtype] * 9), 0.7, kind)
    ps = _params(shapes, [dtype] * 9)
    before = [p.grad.clone() for p in ps]
    _clip_check(ps, 1e6, kind)  # within the bound: the bits stay
    assert all(torch.equal(p.grad, b) for p, b in zip(ps, before))


def test_clip_many_and_mixed():
    """More tensors than one table holds, of three types, views of one
    buffer at odd places."""
    flat = torch.randn(60000, device=DEV)
    ps, at = [], 0
    for i in range(450):
        n = 1 + (i * 37) % 211
        dtype = TYPES[i % 3]
        p = torch.nn.Parameter(torch.zeros(n, device=DEV, dtype=dtype))
        if dtype == torch.float32:
            p.grad = flat[at:at + n]
        else:
            p.grad = flat[at:at + n].to(dtype)
        at += n
        ps.append(p)
    tail = flat[at:].clone()
    _clip_check(ps, 3.0)
    assert torch.equal(flat[at:], tail)


def test_clip_layouts_and_sharing():
    """channels_last and transposed gradients, interleaved columns of one
    matrix, a gradient that two parameters share."""
    a = torch.nn.Parameter(torch.zeros(4, 6, 5, 3, device=DEV))
    a.grad = torch.randn(4, 6, 5, 3, device=DEV).to(
        memory_format=torch.channels_last)
    b = torch.nn.Parameter(torch.zeros(9, 31, device=DEV))
    b.grad = torch.randn(31, 9, device=DEV).t()
    both = torch.randn(50, 20, device=DEV)
    c = torch.nn.Parameter(torch.zeros(50, 8, device=DEV))
    c.grad = both[:, :8]
    d = torch.nn.Parameter(torch.zeros(50, 12, device=DEV))
    d.grad = both[:, 8:]
    _clip_check([a, b, c, d], 2.0)
    e = torch.nn.Parameter(torch.zeros(50, device=DEV))
    e.grad = torch.randn(50, device=DEV)
    f = torch.nn.Parameter(torch.zeros(50, device=DEV))
    f.grad = e.grad
    before = e.grad.double()
    from axon.optim import clip_grad_norm_

    norm = clip_grad_norm_([e, f, e], 0.5)
    _close(norm, before.norm(), before.norm() * 1.01 * U)
    _close(e.grad, before * 0.5 / (before.norm() + 1e-6),
           _rounded(before, torch.float32, 6))


def test_clip_extremes():
    """Squares past fp32's range both ways, inf, NaN, a bound of zero."""
    from axon.optim import clip_grad_norm_, grad_norm

    for std in (1e30, 1e-30):
        ps = _params([(1000,), (77,)], [torch.float32, torch.bfloat16],
                     std=std)
        _clip_check(ps, 1.0)
    for bad in (math.inf, -math.inf, math.nan):
        for kind in (2.0, 1.0, math.inf):
            ps = _params([(100,), (5,)], [torch.float32, torch.float16])
            ref = [p.grad.clone() for p in ps]
            ps[0].grad[17] = bad
            ref[0][17] = bad
            with pytest.raises(RuntimeError):
                clip_grad_norm_(ps, 1.0, kind, error_if_nonfinite=True)
            assert torch.equal(ps[1].grad, ref[1])
            norm = clip_grad_norm_(ps, 1.0, kind)
            if math.isnan(bad):
                assert math.isnan(float(norm))
                assert all(p.grad.isnan().all() for p in ps)
            else:
                assert float(norm) == math.inf
                assert math.isnan(float(ps[0].grad[17]))
                assert not ps[1].grad.any()
    ps = _params([(100,)], [torch.float32])
    clip_grad_norm_(ps, 0.0, error_if_nonfinite=True)
    assert not ps[0].grad.any()
    assert float(grad_norm([])) == 0.0
    assert float(grad_norm([torch.zeros(0, device=DEV)])) == 0.0


def test_clip_tells_autograd():
    """What was saved before the gradients were scaled is known as stale."""
    from axon.optim import clip_grad_norm_

    p = torch.nn.Parameter(torch.zeros(8, device=DEV))
    p.grad = torch.ones(8, device=DEV)
    w = torch.ones(8, device=DEV, requires_grad=True)
    out = (w * p.grad).sum()
    clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward()


def test_clip_refusals_gpu():
    from axon.optim import clip_grad_norm_

    flat = torch.randn(100, device=DEV)
    ps = [torch.nn.Parameter(torch.zeros(60, device=DEV)) for _ in range(2)]
    ps[0].grad, ps[1].grad = flat[:60], flat[40:]
    with pytest.raises(ValueError):
        clip_grad_norm_(ps, 1.0)
    one = torch.nn.Parameter(torch.zeros(8, device=DEV))
    one.grad = torch.ones(1, device=DEV).expand(8)
    with pytest.raises(RuntimeError):
        clip_grad_norm_([one], 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("name", ["SGD", "Adam", "AdamW", "LAMB"])
def test_clipped_step(name, dtype):
    """step() with max_grad_norm against the formulas in 64 bits; p.grad
    itself stays as it was."""
    import axon.optim

    shapes = [(33, 65), (5,), (20000,), (3, 1000)]
    ps = _params(shapes, [dtype] * 4, std=0.3)
    g = torch.Generator(device=DEV).manual_seed(9)
    for p in ps:
        p.data.copy_(torch.randn(p.shape, generator=g, device=DEV))
    lr, wd = 0.01, 0.1
    kw = dict(momentum=0.9) if name == "SGD" else {}
    opt = getattr(axon.optim, "Fused" + name)(
        ps, lr=lr, weight_decay=wd, max_grad_norm=1.5, **kw)
    grads = [p.grad.clone() for p in ps]
    norm, clipped = _clip_wanted(grads, 1.5, 2)
    before = [p.detach().double().clone() for p in ps]
    opt.step()
    _close(opt.grad_norm, norm, norm * 1.01 * U)
    assert all(torch.equal(p.grad, h) for p, h in zip(ps, grads))
    assert "max_grad_norm" not in opt.state_dict()["param_groups"][0]
    b1, b2, eps = 0.9, 0.999, 1e-6 if name == "LAMB" else 1e-8
    for p, c, w in zip(ps, clipped, before):
        if name == "SGD":
            d = c + wd * w
            want = w - lr * d
            tol = 10 * U * lr * (c.abs() + wd * w.abs())
        else:
            h = c + wd * w if name == "Adam" else c
            m, v = (1 - b1) * h, (1 - b2) * h * h
            # The fp32 corrections 1 - b^t of the first step: b2's is 1e-3,
            # off by 2 u absolute, so its root by 6e-5 relative; the others
            # add less.
            u = (m / (1 - b1)) / (v.sqrt() / math.sqrt(1 - b2) + eps)
            step = u
            if name == "AdamW":
                w = w * (1 - lr * wd)
            ratio = 1.0
            if name == "LAMB":
                step = u + wd * w
                ratio = w.norm() / step.norm()
            want = w - lr * ratio * step
            tol = 2e-4 * lr * ratio * (u.abs() + 1)
            if name == "Adam":
                # h may be near 0, where u's sign and size depend on the
                # roundings of the sum h.
                tol = tol + lr * (8 * U * (c.abs() + wd * w.abs())) / (
                    h.abs() + eps)
        _close(p.detach(), want, tol + _rounded(want, dtype, 4), name)


# ------------------------------------------- together, graphs and streams

def test_training_step_together():
    """Lookup, a layer, loss, gradients at both ends of the vocabulary,
    clipping: against 64 bits, twice with the same bits."""
    from axon.ops import cross_entropy, embedding
    from axon.optim import clip_grad_norm_

    g = torch.Generator(device=DEV).manual_seed(0)
    ids = torch.randint(500, (4, 33), generator=g, device=DEV)
    table = torch.nn.Parameter(torch.randn(500, 48, generator=g, device=DEV))
    head = torch.nn.Parameter(
        torch.randn(500, 48, generator=g, device=DEV) * 0.1)
    target = torch.nn.functional.pad(ids[:, 1:], (0, 1), value=-100)

    def step():
        table.grad = head.grad = None
        x = embedding(ids, table, scale=48 ** 0.5)
        loss = cross_entropy(x @ head.t(), target)
        loss.backward()
        norm = clip_grad_norm_([table, head], 0.1)
        return [t.clone() for t in (loss.detach(), norm, table.grad,
                                    head.grad)]

    a, b = step(), step()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    t64 = table.detach().double().requires_grad_()
    h64 = head.detach().double().requires_grad_()
    loss = torch.nn.functional.cross_entropy(
        (t64[ids] * 48 ** 0.5 @ h64.t()).flatten(0, 1), target.flatten())
    loss.backward()
    norm = torch.stack([t64.grad.norm(), h64.grad.norm()]).norm()
    want = [loss.detach(), norm, t64.grad * 0.1 / norm, h64.grad * 0.1 / norm]
    # The layer's products of 48 values (and 500 in its gradient) in fp32:
    # each within 500 u of its sum of magnitudes, here 100 times its size at
    # most; compared by norms.
    for got, w in zip(a, want):
        assert (got.double() - w).norm() <= 500 * 100 * U * w.norm()


def test_graph_replays():
    """One captured pass through all three, replayed with new inputs and
    eager work between: every replay equals the eager result."""
    from axon.ops import cross_entropy, embedding
    from axon.optim import clip_grad_norm_

    vocab, dim, n = 700, 40, 2500
    ids = torch.zeros(n, dtype=torch.long, device=DEV)
    out_grad = torch.zeros(n, dim, device=DEV, dtype=torch.bfloat16)
    logits_in = torch.zeros(96, vocab, device=DEV, dtype=torch.bfloat16)
    labels = torch.zeros(96, dtype=torch.long, device=DEV)
    raw = torch.zeros(30000, device=DEV)

    def work(table, logits, param):
        out = embedding(ids, table, scale=2.0, padding_idx=1)
        (dt,) = torch.autograd.grad(out, table, out_grad)
        loss = cross_entropy(logits, labels)
        (dx,) = torch.autograd.grad(loss, logits)
        param.grad.copy_(raw)
        norm = clip_grad_norm_([param], 1.0)
        return out.detach(), dt, loss.detach(), dx, norm, param.grad

    def leaves():
        table = torch.ones(vocab, dim, device=DEV,
                           dtype=torch.bfloat16).requires_grad_()
        param = torch.nn.Parameter(torch.zeros(30000, device=DEV))
        param.grad = torch.zeros(30000, device=DEV)
        return table, logits_in.detach().requires_grad_(), param

    def new_inputs(seed):
        g = torch.Generator(device=DEV).manual_seed(seed)
        ids.copy_(torch.randint(vocab, (n,), generator=g, device=DEV))
        out_grad.normal_(generator=g)
        logits_in.normal_(generator=g)
        labels.copy_(torch.randint(vocab, (96,), generator=g, device=DEV))
        raw.normal_(generator=g)

    new_inputs(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(*leaves())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    captured = leaves()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = work(*captured)
        graphs.append((graph, got))
    for seed in range(1, 6):
        new_inputs(seed)
        graph, got = graphs[seed % 2]
        graph.replay()
        torch.cuda.synchronize()
        replayed = [t.clone() for t in got]
        want = work(*leaves())
        torch.cuda.synchronize()
        for a, b in zip(replayed, want):
            assert torch.equal(a, b)


def test_other_stream():
    """The calls run on the current stream, behind what made their inputs
    there."""
    from axon.ops import cross_entropy, embedding
    from axon.optim import grad_norm

    g = torch.Generator(device=DEV).manual_seed(2)
    base = torch.randn(64, 5000, generator=g, device=DEV)
    t = torch.randint(5000, (64,), generator=g, device=DEV)
    ids = torch.randint(64, (3000,), generator=g, device=DEV)
    torch.cuda.synchronize()

    def work():
        x = base * 1.0
        for _ in range(20):
            x = x * 1.0
        return (cross_entropy(x, t), embedding(ids, x, scale=3.0),
                grad_norm([x]))

    want = work()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = work()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals_gpu():
    from axon.ops import cross_entropy, embedding

    w = torch.zeros(4, 8, device=DEV)
    with pytest.raises(ValueError):
        embedding(torch.zeros(3, dtype=torch.long), w)
    with pytest.raises(ValueError):
        cross_entropy(w, torch.zeros(4, dtype=torch.long))
    many = torch.zeros(1, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError):
        embedding(many.expand(1 << 26), w)
    with pytest.raises(ValueError):
        cross_entropy(w[:1, :1].expand(1 << 24, 5000), many.expand(1 << 24))
    with pytest.raises(ValueError):
        cross_entropy(w[0, 0].expand(1, 1 << 30), many)
    for bad in (dict(padding_idx=4), dict(padding_idx=-5)):
        with pytest.raises(ValueError):
            embedding(many, w, **bad)
    with pytest.raises(TypeError):
        embedding(many.float(), w)
    with pytest.raises(TypeError):
        embedding(many, w, scale=torch.ones((), device=DEV))
    with pytest.raises(ValueError):
        embedding(many, w[0])
    for bad in (dict(reduction="max"), dict(label_smoothing=1.5)):
        with pytest.raises(ValueError):
            cross_entropy(w, many.expand(4), **bad)
    with pytest.raises(ValueError):
        cross_entropy(w, many)
    with pytest.raises(TypeError):
        cross_entropy(w, many.expand(4).float())
    double = torch.nn.Parameter(torch.ones(3, device=DEV,
                                           dtype=torch.float64))
    double.grad = torch.ones_like(double)
    from axon.optim import FusedAdamW
    with pytest.raises(RuntimeError):
        FusedAdamW([double]).step()
    x = torch.randn(4, 8, device=DEV, requires_grad=True)
    loss = cross_entropy(x, torch.zeros(4, dtype=torch.long, device=DEV))
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_large_logits():
    """Logits of more than the caches' share (both kinds of rows in one
    call), and rows that do not start on lines."""
    for n, vocab, dtype in [(3500, 30522, torch.bfloat16),
                            (900, 60001, torch.float32)]:
        x, t, g = _logits(n, vocab, dtype)
        t[torch.rand(n, generator=g, device=DEV) < 0.5] = -100
        _loss_check(x, t)
        del x
        torch.cuda.empty_cache()


def test_many_rows():
    """More rows than one block sums."""
    for n, vocab in [(16384, 5), (16385, 40), (200001, 3)]:
        x, t, g = _logits(n, vocab, torch.float32)
        t[torch.rand(n, generator=g, device=DEV) < 0.2] = -100
        _loss_check(x, t)


def test_clip_many_blocks():
    """More partial sums than the scaling blocks join themselves, more
    chunks than blocks, two types."""
    _clip_check(_params([(12_000_001,), (7,), (36_000_000,)],
                        [torch.float32, torch.float32, torch.bfloat16]), 1.0)
    _clip_check(_params([(20_000_000,)], [torch.float16], std=0.01), 2.0, 1.0)


def test_no_gradient_modes():
    from axon.ops import cross_entropy, embedding

    w = torch.randn(20, 16, device=DEV, requires_grad=True)
    ids = torch.arange(12, device=DEV)
    with torch.no_grad():
        assert not embedding(ids, w).requires_grad
        assert not cross_entropy(w, torch.arange(20, device=DEV) % 16
                                 ).requires_grad
    with torch.inference_mode():
        x = torch.randn(12, 16, device=DEV)
        assert torch.isfinite(cross_entropy(x, ids))
        assert torch.equal(embedding(ids, x), x)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss = cross_entropy(w @ w.t(), torch.arange(20, device=DEV))
    assert loss.dtype == torch.float32
    loss.backward()
    assert torch.isfinite(w.grad).all()


def test_graph_is_freed_and_guarded():
    """Twice backward, an input changed in between, forward-mode."""
    import torch.autograd.forward_ad as fwad

    from axon.ops import cross_entropy, embedding

    x = torch.randn(6, 9, device=DEV, requires_grad=True)
    t = torch.arange(6, device=DEV)
    loss = cross_entropy(x, t)
    loss.backward()
    with pytest.raises(RuntimeError, match="second time"):
        loss.backward()
    y = embedding(t, x)
    y.sum().backward()
    with pytest.raises(RuntimeError, match="second time"):
        y.sum().backward()
    z = x.detach() * 2.0
    z.requires_grad_()
    mid = z * 1.0
    loss = cross_entropy(mid, t)
    with torch.no_grad():
        mid.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with fwad.dual_level():
        dual = fwad.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(NotImplementedError):
            cross_entropy(dual, t)
        with pytest.raises(NotImplementedError):
            embedding(t, dual)


def test_threads():
    """Calls from two threads, each on a stream of its own."""
    import threading

    from axon.ops import cross_entropy, embedding
    from axon.optim import grad_norm

    g = torch.Generator(device=DEV).manual_seed(4)
    x = torch.randn(300, 3000, generator=g, device=DEV)
    t = torch.randint(3000, (300,), generator=g, device=DEV)
    ids = torch.randint(300, (4000,), generator=g, device=DEV)
    dy = torch.randn(4000, 3000, generator=g, device=DEV)

    def work():
        leaf = x.clone().requires_grad_()
        loss = cross_entropy(leaf, t)
        (a,) = torch.autograd.grad(loss, leaf)
        (b,) = torch.autograd.grad(embedding(ids, leaf), leaf, dy)
        return [loss.detach(), a, b, grad_norm([a, b])]

    want = work()
    torch.cuda.synchronize()
    got, errors = {}, []

    def run(name):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(5):
                    got[name] = work()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for r in got.values():
        assert all(torch.equal(a, b) for a, b in zip(r, want))


@pytest.mark.parametrize("name", ["Adam", "AdamW", "LAMB"])
@pytest.mark.parametrize("clip", [None, 0.5])
def test_group_path_is_the_general_path(name, clip, monkeypatch):
    """The step that reads a whole group in one call against the one that
    goes by each parameter: other layouts, types, step counts, parameters
    without a gradient, state that does not exist yet."""
    import axon.optim
    from axon import _core

    def make():
        ps = _params([(33, 7), (5,), (4, 6, 5, 3), (2000,), (64,)],
                     [torch.float32, torch.bfloat16, torch.float32,
                      torch.bfloat16, torch.float32], seed=3)
        ps[2].data = ps[2].data.to(memory_format=torch.channels_last)
        g = torch.Generator(device=DEV).manual_seed(8)
        for p in ps:
            p.data.normal_(generator=g)
        return ps, getattr(axon.optim, "Fused" + name)(
            [{"params": ps[:3]}, {"params": ps[3:], "lr": 0.02}], lr=0.01,
            weight_decay=0.1, max_grad_norm=clip)

    def steps(ps, opt):
        g = torch.Generator(device=DEV).manual_seed(1)
        for i in range(4):
            for k, p in enumerate(ps):
                p.grad = torch.randn(p.shape, generator=g,
                                     device=DEV).to(p.dtype)
                if k == 2 and i != 1:  # once of another layout than p
                    p.grad = p.grad.to(memory_format=torch.channels_last)
            if i < 2:
                ps[1].grad = None
            opt.step()
        return [p.detach() for p in ps] + [
            v for p in ps for k, v in sorted(opt.state[p].items())]

    calls = []
    whole = _core.fused_adam_group
    monkeypatch.setattr(_core, "fused_adam_group",
                        lambda *a: calls.append(whole(*a)) or calls[-1])
    got = steps(*make())
    assert True in calls and False in calls
    monkeypatch.setattr(_core, "fused_adam_group", lambda *a: False)
    want = steps(*make())
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and a.stride() == b.stride()
        if name == "LAMB":
            # Its norms are added with atomics, in any order: 2000 values'
            # fp32 sum, then half a step of the type.
            eps = torch.finfo(a.dtype).eps
            assert torch.allclose(a.double(), b.double(),
                                  rtol=max(2000 * U, eps),
                                  atol=max(1e-6, eps / 100))
        else:
            assert torch.equal(a, b)


def test_clipping_under_distributed_optimizer():
    import axon as hvd
    from axon.optim import FusedAdamW

    hvd.init()
    try:
        p = torch.nn.Parameter(torch.zeros(3, device=DEV))
        opt = hvd.DistributedOptimizer(
            FusedAdamW([p], lr=0.1, max_grad_norm=1.0),
            named_parameters=[("p", p)])
        (p * torch.tensor([6.0, 8.0, 0.0], device=DEV)).sum().backward()
        opt.step()
        assert abs(float(opt.grad_norm) - 10.0) <= 10.0 * U
    finally:
        hvd.shutdown()


def test_models_use_the_kernels():
    """Both language models' losses and gradients on the GPU against the
    same weights through torch's own functions."""
    import torch.nn.functional as F

    from axon.models.bert import BertForPreTraining, bert_tiny_config
    from axon.models.llama import LlamaForCausalLM, llama_tiny_config
    from axon.ops import FusedEmbedding

    def compare(model, got, want):
        # Losses over some 100 classes: a few tens of roundings. Gradients of
        # the vocabulary's table: products of at most 128 values and sums of
        # 64 rows on both sides, compared by norms.
        assert abs(got.item() - want.item()) <= 100 * U * want.item()
        table = (model.embed if hasattr(model, "embed") else model.tok).weight
        (a,) = torch.autograd.grad(got, table)
        (b,) = torch.autograd.grad(want, table)
        assert (a - b).norm() <= 1000 * U * b.norm()

    torch.manual_seed(0)
    llama = LlamaForCausalLM(llama_tiny_config()).to(DEV)
    assert isinstance(llama.embed, FusedEmbedding)
    ids = torch.randint(256, (2, 32), device=DEV)
    compare(llama, llama.lm_loss(ids),
            F.cross_entropy(llama(ids)[:, :-1].double().flatten(0, 1),
                            ids[:, 1:].flatten()))
    bert = BertForPreTraining(bert_tiny_config()).to(DEV)
    assert isinstance(bert.tok, FusedEmbedding)
    ids = torch.randint(128, (2, 32), device=DEV)
    labels = torch.where(torch.rand(2, 32, device=DEV) < 0.3, ids, -100)
    compare(bert, bert.mlm_loss(ids, labels),
            F.cross_entropy(bert(ids).double().view(-1, 128),
                            labels.view(-1)))
