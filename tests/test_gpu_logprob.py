"""loss.token_logprobs on the GPU against its definition in 64 bits: sizes around every border of the kernels, types, strides, masks,
refused targets, gradients, streams and graphs.

Tolerances, derived.  u = 2^-24 is half a step of fp32, L = ln C.  A weight exp(x - m) carries |x - m| u from the difference's
rounding, as much again from the product with log2 e, and 2 u from the exponential; a thread adds at most max(64, C / 256) of them one
after another and a tree of at most 12 levels joins the threads.  S is therefore off by (n + 14 + 2 (|x - m| averaged over p)) u, the
average being at most L + 1, so log S, a log-probability l and the entropy are off by at most
    E(v) = u (n + 64 + 4 |v|) (1 + L),   n = max(64, C / 256)
(the factor 1 + L only the entropy needs, whose W / S is at most L in size).  p is off by a factor of 1 + E(l) + |l| u + 2 u, and a
gradient by that on its smooth part, u on every sum, and half a step of its own type (half a subnormal step of fp16, 2^-25, at least).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _score(*a, **k):
    from curvecloudnet_amd.loss import token_logprobs
    return token_logprobs(*a, **k)


def _definition(x, target, top, ignore=-100):
    """64 bits, on the CPU: logprob, entropy, top_logprob, top_index, all log-probabilities."""
    x = x.detach().cpu().double()
    target = target.cpu().long()
    best = x.amax(1, keepdim=True)                      # (subtracted first: log C is lost beside the lowest values even in 64 bits)
    off = x - best
    empty = torch.isneginf(x).all(1, keepdim=True)
    logp = torch.where(empty, -math.inf, off - off.exp().sum(1, keepdim=True).log())
    odd = torch.isnan(x).any(1, keepdim=True) | torch.isposinf(x).any(1, keepdim=True)
    logp = torch.where(odd, math.nan, logp)
    p = logp.exp()
    entropy = -torch.where(p == 0, 0.0, p * logp).sum(1)
    inside = (target >= 0) & (target < x.size(1))
    given = logp.gather(1, torch.where(inside, target, 0)[:, None]).squeeze(1)
    logprob = torch.where(target == ignore, 0.0, torch.where(inside, given, math.nan))
    order = torch.sort(torch.where(torch.isnan(x), math.inf, x + 0.0), dim=1, descending=True, stable=True).indices
    # (a NaN comes before an infinity)
    order = order.gather(1, torch.sort(torch.isnan(x).gather(1, order).int(), dim=1, descending=True, stable=True).indices)[:, :top]
    return logprob, entropy, logp.gather(1, order), order, logp


def _gradient(logp, entropy, target, order, g_lp, g_h, g_top, ignore=-100):
    target = target.cpu().long()
    scored = target != ignore
    inside = (target >= 0) & (target < logp.size(1))
    g = torch.where(scored, g_lp.cpu().double(), 0.0)
    g = torch.where(scored & ~inside, math.nan, g)
    total = g.clone()
    onehot = torch.zeros_like(logp)
    onehot.scatter_add_(1, torch.where(inside, target, 0)[:, None], torch.where(inside, g, 0.0)[:, None])
    if g_top is not None:
        total = total + g_top.cpu().double().sum(1)
        onehot.scatter_add_(1, order, g_top.cpu().double())
    p = logp.exp()
    smooth = torch.where(p == 0, 0.0, -p * (total[:, None] + g_h.cpu().double()[:, None] * (logp + entropy[:, None])))
    return smooth, onehot, total


def _e(v, c):
    return U * (max(64, c / 256) + 64 + 4 * v.abs()) * (1 + math.log(c))


def _near(a, ref, tol, what):
    a, ref = a.detach().cpu().double(), ref.double()
    ref = torch.where(ref < -3.5e38, -math.inf, ref)                    # (below the range of the outputs' type)
    assert a.shape == ref.shape, what
    same = (a == ref) | (torch.isnan(a) & torch.isnan(ref))
    off = (a - ref).abs()
    bad = ~(same | (off <= tol))
    assert not bool(bad.any()), "%s: %d values off, worst %.3g, first at %s: %r for %r" % (
        what, int(bad.sum()), float(off[bad].max()), bad.nonzero()[0].tolist(), float(a[bad][0]), float(ref[bad][0]))


def _check(x, target, top, ignore=-100, r=None):
    r = _score(x, target, top=top, ignore_index=ignore) if r is None else r
    lp, h, best, order, logp = _definition(x, target, top, ignore)
    c = x.size(1)
    assert r.logprob.dtype == r.entropy.dtype == torch.float32
    _near(r.logprob, lp, _e(lp, c), "logprob")
    _near(r.entropy, h, _e(h, c), "entropy")
    if top:
        assert r.top_index.dtype == torch.int64
        assert torch.equal(r.top_index.cpu(), order), "alternatives"
        _near(r.top_logprob, best, _e(best, c), "alternatives' log-probabilities")
    else:
        assert r.top_logprob is None and r.top_index is None
    return lp, h, best, order, logp


def _check_gradient(x, target, top, ignore=-100, seed=1, use=(True, True, True)):
    gen = torch.Generator().manual_seed(seed)
    rows, c = x.shape
    g_lp, g_h = torch.randn(rows, generator=gen) * use[0], torch.randn(rows, generator=gen) * use[1]
    g_top = torch.randn(rows, top, generator=gen) if top and use[2] else None
    leaf = x.detach().requires_grad_(True)
    r = _score(leaf, target, top=top, ignore_index=ignore)
    _, h, _, order, logp = _check(x, target, top, ignore, r)
    outs, gs = [], []
    for on, out, g in zip(use, (r.logprob, r.entropy, r.top_logprob), (g_lp, g_h, g_top)):
        if on and out is not None:
            outs.append(out)
            gs.append(g.to(DEV))
    (d,) = torch.autograd.grad(outs, leaf, gs)
    assert d.dtype == x.dtype and d.shape == x.shape
    smooth, onehot, total = _gradient(logp, h, target, order, g_lp, g_h, g_top, ignore)
    ref = smooth + onehot
    lsafe = torch.where(torch.isinf(logp), 0.0, logp)
    p = logp.exp()
    factor = _e(lsafe, c) + U * (lsafe.abs() + 4)
    gh = g_h.double()[:, None].abs()
    sums = total[:, None].abs() + (g_lp.abs().double()[:, None] + (0 if g_top is None else g_top.abs().double().sum(1, keepdim=True)))
    tol = p * (sums + gh * (lsafe.abs() + h[:, None].abs())) * (factor + 70 * U)            # (up to 64 gradients in one sum)
    tol = tol + p * gh * (_e(lsafe, c) + _e(h, c)[:, None])
    tol = tol + U * (onehot.abs() + ref.abs()) * 66
    tol = tol + ref.abs() * torch.finfo(x.dtype).eps / 2 + (2.0 ** -25 if x.dtype == torch.float16 else 0.0)
    # (weights below the smallest normal number are zero)
    tol = tol + (sums + gh * 200) * 2.0 ** -126
    _near(d, ref, torch.nan_to_num(tol, nan=0.0), "gradient")
    return d


def _logits(rows, c, dtype, seed=0, spread=3.0, pad=0, shift=0):
    gen = torch.Generator().manual_seed(seed + 7 * rows + c)
    wide = (torch.randn(rows, c + pad + shift, generator=gen) * spread).to(dtype).to(DEV)
    return wide[:, shift: shift + c]


def _target(rows, c, seed=0):
    return torch.randint(0, c, (rows,), generator=torch.Generator().manual_seed(seed + rows + c)).to(DEV)


SIZES = [(1, 1), (1, 2), (2, 1), (3, 5), (257, 20), (1000, 20), (129, 23), (130, 24), (131, 25), (70, 26), (65, 33), (64, 55), (513, 55),
         (5, 63), (5, 64), (5, 65), (70, 66), (7, 127), (33, 128), (33, 129), (9, 255), (9, 256), (17, 257), (33, 300), (5, 511), (9, 512),
         (5, 513), (4, 1000), (4, 1023), (4, 1025), (3, 2047), (3, 2048), (3, 2049),
         (2, 4095), (2, 4097), (2, 8191), (2, 8193), (3, 16385), (1, 32769), (1, 50021), (2, 65535), (2, 65537), (300, 4099), (1, 262144),
         (1, 300007)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,c", SIZES)
def test_scores_and_gradient_over_sizes(rows, c, dtype):
    x, t = _logits(rows, c, dtype), _target(rows, c)
    for top in sorted({0, min(c, 1), min(c, 5), min(c, 20)}):
        _check(x, t, top)
    _check_gradient(x, t, 0)
    _check_gradient(x, t, min(c, 5))


@pytest.mark.parametrize("rows,c", [(3, 64), (40, 64), (3, 65), (3, 100), (40, 128), (17, 200), (18, 256), (9, 257), (10, 500), (9, 512),
                                    (5, 513), (2, 2048), (3, 9000), (1, 70000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["fp32", "bf16"])
def test_many_alternatives(rows, c, dtype):
    x, t = _logits(rows, c, dtype), _target(rows, c)
    for top in (2, 3, 4, 6, 8, 9, 12, 15, 16, 17, 18, 21, 31, 32, 33, 63, 64):
        _check(x, t, top)
    _check_gradient(x, t, 17)
    _check_gradient(x, t, 64)


@pytest.mark.parametrize("top", [1, 2, 3, 4, 5, 6, 9, 15, 16, 17, 20, 33])
def test_a_row_that_is_taken_in_many_pieces(top):
    """Random, rising and falling rows of a dozen pieces, in one part and in several, and rows whose first piece is the least."""
    for rows, c in ((2, 100003), (800, 40001)):
        x = _logits(rows, c, torch.float32)
        x[0] = torch.arange(c, device=DEV) * (40.0 / c)
        x[1] = x[0].flip(0)
        if rows > 2:
            x[2:200] += torch.arange(c, device=DEV) * (4.0 / c)
            x[200:400, :9000] -= 30.0
            x[400:500] = (x[400:500] * 2).round()
        _check(x, _target(rows, c), top)


def test_every_class_is_an_alternative():
    for rows, c in ((1, 1), (5, 2), (300, 20), (7, 33), (3, 64)):
        x, t = _logits(rows, c, torch.float32), _target(rows, c)
        lp, _, _, order, _ = _check(x, t, c)
        assert torch.equal(order.sort(1).values, torch.arange(c).expand(rows, c))
        _check_gradient(x, t, c)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("c", [20, 64, 65, 1500, 5000, 40000])
def test_strides_and_alignments(c, dtype):
    rows, top = 5, 4
    t = _target(rows, c)
    for pad, shift in ((1, 0), (0, 1), (3, 5), (8, 0), (7, 3)):
        x = _logits(rows, c, dtype, pad=pad, shift=shift)
        assert x.stride(0) == c + pad + shift
        _check_gradient(x, t, top)
    flat = _logits(1, rows * c + 3, dtype)[0]
    for k in range(4):
        _check_gradient(flat[k: k + rows * c].view(rows, c), t, top)
    x = _logits(c, rows, dtype).t()                                     # columns that are not adjacent
    assert x.stride() == (1, rows)
    _check_gradient(x, t, top)
    _check(_logits(1, c, dtype).expand(rows, c), t, top)               # one row for all
    _check(_logits(2 * rows, c, dtype)[::2], t, top)
    _check(_logits(2 * rows, c, dtype).flip(0)[1::2], t, top)


def test_shapes_and_target_types():
    x, t = _logits(24, 30, torch.float32), _target(24, 30)
    lp, h, best, order, _ = _definition(x, t, 3)
    r = _score(x.view(2, 3, 4, 30), t.view(2, 3, 4).to(torch.int32), top=3)
    assert r.logprob.shape == r.entropy.shape == (2, 3, 4) and r.top_logprob.shape == r.top_index.shape == (2, 3, 4, 3)
    _check(x, t, 3, r=type(r)(r.logprob.view(-1), r.entropy.view(-1), r.top_logprob.view(-1, 3), r.top_index.view(-1, 3)))
    one = _score(x[5], t[5], top=3)
    assert one.logprob.shape == () and one.top_index.shape == (3,)
    assert torch.equal(one.top_index.cpu(), order[5]) and float(one.logprob) == float(r.logprob.view(-1)[5])
    # a slice of a larger batch, an axis moved: no copy of the caller's is needed
    y = _logits(6 * 9, 30, torch.float32).view(6, 9, 30)[1:5, 2:8].requires_grad_(True)
    k = _target(24, 30).view(4, 6)
    s = _score(y, k)
    (d,) = torch.autograd.grad(s.logprob.sum(), y)
    ref = torch.softmax(y.detach().double(), -1)
    ref = torch.nn.functional.one_hot(k, 30).double() - ref
    _near(d, ref.cpu(), 300 * U, "gradient of a slice")
    for shape in ((0, 30), (2, 0, 30)):
        e = torch.empty(shape, device=DEV, requires_grad=True)
        s = _score(e, torch.empty(shape[:-1], dtype=torch.int64, device=DEV), top=2)
        assert s.logprob.shape == shape[:-1] and s.top_index.shape == shape[:-1] + (2,)
        (d,) = torch.autograd.grad(s.logprob.sum() + s.top_logprob.sum(), e)
        assert d.shape == shape


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("c", [7, 64, 65, 700, 3000, 20000, 70001])
def test_equal_logits_come_by_class(c, dtype):
    rows, top = 6, min(c, 33)
    t = _target(rows, c)
    x = torch.zeros(rows, c, dtype=dtype, device=DEV)
    x[1] = -5.0
    x[2, ::2] = -0.0                                                    # -0 and 0 are equal
    x[3] = torch.arange(c, device=DEV).div(max(1, c // 4), rounding_mode="floor").to(dtype)
    x[4] = torch.arange(c, device=DEV).div(max(1, c // 4), rounding_mode="floor").flip(0).to(dtype)
    x[5] = (torch.arange(c, device=DEV) % 3).to(dtype)
    _check_gradient(x, t, top)
    _check(x, t, min(c, 64))


@pytest.mark.parametrize("c", [64, 65, 2048, 5000, 40000])
def test_ordered_rows(c):
    """Rising, falling and one-lane-heavy rows: the alternatives lie next to one another, at the end, at the start, or a stride apart."""
    x = torch.empty(5, c, device=DEV)
    x[0] = torch.arange(c, device=DEV) * (30.0 / c)
    x[1] = x[0].flip(0)
    x[2] = torch.where(torch.arange(c, device=DEV) % 64 == 13, 20.0, 0.0) + x[0] * 0.01
    x[3] = torch.where(torch.arange(c, device=DEV) % 256 == 7, 20.0, 0.0) - x[0] * 0.01
    x[4] = torch.where((torch.arange(c, device=DEV) >= c // 2) & (torch.arange(c, device=DEV) < c // 2 + 64), 25.0, 0.0) + x[0] * 0.1
    for top in (1, 20, 64):
        _check(x, _target(5, c), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("c", [5, 20, 64, 65, 1000, 5001, 40000])
def test_masked_rows(c, dtype):
    rows, top, low = 12, 5, torch.finfo(dtype).min
    x = _logits(rows, c, dtype).clone()
    t = _target(rows, c)
    x[0] = -math.inf                                                    # nothing left
    x[1] = low                                                          # the type's lowest value throughout: uniform
    x[2] = -math.inf
    x[2, c - 1] = 1.5                                                   # one class left
    x[3] = low
    x[3, 0] = torch.finfo(dtype).max                                    # the widest difference
    x[4, : c // 2] = -math.inf
    x[5, c // 2:] = low
    x[6] = -math.inf
    x[6, 0], x[6, c - 1] = low, low
    x[7, 1::2] = -math.inf
    t[2], t[3], t[8] = c - 1, 0, -100
    t[9] = c - 1
    x[9, c - 1] = -math.inf                                             # the given class has no probability
    x[10] = -math.inf
    t[10] = -100
    r = _score(x, t, top=top)
    assert float(r.logprob[0]) == -math.inf and float(r.entropy[0]) == 0.0 and float(r.logprob[8]) == 0.0
    assert r.top_index[0].tolist() == list(range(top)) and float(r.logprob[9]) == -math.inf
    _check(x, t, top)
    d = _check_gradient(x, t, top)
    assert bool(torch.isfinite(d).all())
    d = _check_gradient(x, t, 0)
    assert float(d[10].abs().max()) == 0.0


@pytest.mark.parametrize("c", [5, 64, 65, 1000, 5001, 40000])
def test_nan_and_infinity_stay_in_their_rows(c):
    rows = 6
    x, t = _logits(rows, c, torch.float32).clone(), _target(rows, c)
    x[1, c // 2] = math.nan
    x[2, c - 1] = math.inf
    x[3] = math.nan
    x[4, 0], x[4, c - 1], x[4, c // 2] = math.inf, math.inf, -math.inf
    r = _score(x, t, top=4)
    assert torch.isnan(r.logprob[1:5]).all() and torch.isnan(r.entropy[1:5]).all() and torch.isnan(r.top_logprob[1:5]).all()
    _check(x, t, 4)
    leaf = x.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(_score(leaf, t).logprob.sum(), leaf)
    assert torch.isfinite(d[[0, 5]]).all() and torch.isnan(d[1:5]).any(1).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["fp32", "fp16"])
@pytest.mark.parametrize("c", [20, 100, 1500, 5000, 40000])
def test_rows_of_many_nan(c, dtype):
    """More of them than alternatives: everywhere, on odd classes, behind the first piece, in the last class and few before it."""
    x, t = _logits(5, c, dtype), _target(5, c)
    x[0] = math.nan
    x[1, 1::2] = math.nan
    x[2, c // 2:] = math.nan
    x[3, -1] = x[3, c // 3] = math.nan
    x[4, 0] = math.inf
    x[4, 3::5] = math.nan
    for top in (1, 3, min(c, 20)):
        _check(x, t, top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("c", [1, 2, 20, 24, 25, 55, 64, 65, 128, 129, 300, 512, 513, 1000, 2048, 2049, 5000, 40000, 200003])
def test_the_best_class_alone(c, dtype):
    x, t = _logits(12, c, dtype), _target(12, c)
    x[0] = 1.5                                                          # equal ones: the lowest class
    x[1] = -math.inf
    x[2, : c - 1] = -math.inf
    x[3, c // 2:] = 40.0
    x[4, -1] = x[4, c // 3] = math.nan
    x[5, -1] = math.inf
    x[6] = torch.linspace(-20, 20, c, device=DEV).to(dtype)
    x[7] = torch.linspace(20, -20, c, device=DEV).to(dtype)
    x[8] = 0.0
    x[8, 1::2] = -0.0
    x[9] = -0.0
    x[9, c // 2] = 0.0
    _check(x, t, 1)
    some = x[torch.tensor([0, 3, 6, 7, 8, 9, 10, 11], device=DEV)]
    _check_gradient(some, _target(8, c), 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("c", [4, 8, 20, 64, 300, 1000, 5000, 20000])
def test_subnormal_logits_and_zeros_of_both_signs(c, dtype):
    """Told apart by the alternatives, though they weigh the same."""
    step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    x = torch.zeros(4, c, dtype=dtype, device=DEV)
    x[0] = (torch.arange(c, device=DEV) % 7 * step).to(dtype)
    x[1] = (-(torch.arange(c, device=DEV) % 5) * step).to(dtype)
    x[2, 1::2] = -0.0
    x[3] = -0.0
    x[3, c // 2] = step
    assert float(x[0, 1]) == step > 0
    for top in (1, 2, 3, min(c, 5), min(c, 9)):
        _check(x, _target(4, c), top)


def test_targets_that_are_not_scored():
    for c in (20, 65, 3000):
        rows = 9
        x, t = _logits(rows, c, torch.float32), _target(rows, c)
        t[1], t[2], t[3], t[4], t[5] = -100, c, -1, 2 ** 40, -2 ** 62
        r = _score(x, t, top=2)
        assert float(r.logprob[1]) == 0.0 and torch.isnan(r.logprob[2:6]).all() and torch.isfinite(r.entropy).all()
        _check(x, t, 2)
        leaf = x.detach().requires_grad_(True)
        (d,) = torch.autograd.grad(_score(leaf, t).logprob.sum(), leaf)
        assert float(d[1].abs().max()) == 0.0 and torch.isnan(d[2:6]).any(1).all() and torch.isfinite(d[[0, 6, 7, 8]]).all()
        (d,) = torch.autograd.grad(_score(leaf, t).entropy.sum(), leaf)                 # (a bad target is no part of the entropy)
        assert torch.isfinite(d).all()
        # a class of the range that is not scored
        t = _target(rows, c) % 3
        _check_gradient(x, t, 2, ignore=0)


@pytest.mark.parametrize("use", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
@pytest.mark.parametrize("c", [20, 500, 9001])
def test_gradient_of_each_output_alone(c, use):
    _check_gradient(_logits(11, c, torch.float32), _target(11, c), 6, use=use)


def test_the_given_class_among_the_alternatives_and_gradients_broadcast():
    for c in (20, 700, 5000):
        x = _logits(8, c, torch.bfloat16)
        t = x.float().argmax(1)
        _check_gradient(x, t, 3)
        leaf = x.detach().requires_grad_(True)
        r = _score(leaf, t, top=3)
        loss = -r.logprob.mean() + 0.5 * r.entropy.mean() + r.top_logprob.mean()        # (gradients of stride 0)
        (a,) = torch.autograd.grad(loss, leaf)
        r = _score(leaf, t, top=3)
        n = float(x.size(0))
        (b,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], leaf,
                                   [torch.full_like(r.logprob, -1 / n), torch.full_like(r.entropy, 0.5 / n),
                                    torch.full_like(r.top_logprob, 1 / (3 * n))])
        assert torch.equal(a, b)


def test_gradient_against_differences():
    """Central differences of the definition in 64 bits: their own error, h^2 / 6 times the third derivative, is below 1e-8; the
    kernel's is at most p (n + 64 + 4 |l| + ...) u times gradients of up to 4, in all less than 4e-5."""
    x, t = _logits(2, 9, torch.float32, spread=1.0), _target(2, 9)
    gen = torch.Generator().manual_seed(5)
    g = [torch.randn(2, generator=gen), torch.randn(2, generator=gen), torch.randn(2, 3, generator=gen)]

    def value(y):
        lp, h, best, _, _ = _definition(y, t, 3)
        return float((lp * g[0]).sum() + (h * g[1]).sum() + (best * g[2]).sum())

    leaf = x.detach().requires_grad_(True)
    r = _score(leaf, t, top=3)
    (d,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], leaf, [v.to(DEV) for v in g])
    step, base = 1e-4, x.cpu().double()
    for i in range(2):
        for j in range(9):
            up, down = base.clone(), base.clone()
            up[i, j] += step
            down[i, j] -= step
            assert abs((value(up) - value(down)) / (2 * step) - float(d[i, j])) < 4e-5, (i, j)


def test_rows_behind_a_long_way():
    """Rows that start more than 2^31 values behind the first."""
    ld, c = (1 << 30) + 24, 100
    base = torch.empty(2 * ld + 5000, dtype=torch.bfloat16, device=DEV)
    for classes in (c, 5000):
        x = base.as_strided((3, classes), (ld, 1))
        x.copy_(_logits(3, classes, torch.bfloat16))
        assert 2 * ld > 2 ** 31
        _check_gradient(x, _target(3, classes), 5)


def test_many_rows():
    """More rows than workgroups fit at once, checked against torch on the device."""
    for rows, c, dtype in ((400070, 20, torch.float32), (70001, 130, torch.bfloat16), (9001, 2500, torch.float16)):
        gen = torch.Generator(device=DEV).manual_seed(c)
        x = (torch.randn(rows, c, generator=gen, device=DEV) * 3).to(dtype).requires_grad_(True)
        t = torch.randint(0, c, (rows,), generator=gen, device=DEV)
        r = _score(x, t, top=2)
        logp = torch.log_softmax(x.detach().double(), 1)
        lp = logp.gather(1, t[:, None]).squeeze(1)
        _near(r.logprob, lp.cpu(), _e(lp, c).cpu(), "logprob")
        (d,) = torch.autograd.grad(r.logprob.sum(), x)
        ref = torch.nn.functional.one_hot(t, c).double() - logp.exp()
        tol = 400 * U + ref.abs() * (torch.finfo(dtype).eps / 2) + 2.0 ** -25
        assert bool(((d.double() - ref).abs() <= tol).all())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("rows,c,tops", [(65541, 3, (3,)), (65541, 11, (3, 5, 11)), (65541, 12, (3, 5, 12)), (65541, 20, (4, 5, 7, 8, 20)),
                                         (65541, 24, (3, 7, 8, 24)), (2050, 2049, (0, 1, 2, 20, 64)), (2050, 2999, (0, 1, 5)),
                                         (2050, 4095, (0, 1, 5, 33)), (4100, 4097, (0, 1, 5)), (4100, 6001, (0, 1, 3)), (4100, 8192, (2, 20, 64))])
def test_many_rows_of_every_kind(rows, c, tops, dtype):
    """Kernels that are taken where rows are many: odd rows among ordinary ones, at the start, in the middle and at the end."""
    gen = torch.Generator(device=DEV).manual_seed(c)
    x = (torch.randn(rows, c, generator=gen, device=DEV) * 3).to(dtype)
    t = torch.randint(0, c, (rows,), generator=gen, device=DEV)
    parts = [slice(0, 13), slice(rows // 2, rows // 2 + 13), slice(rows - 13, rows)]
    for p in parts:
        y = x[p]
        y[0] = 1.5
        y[1] = -math.inf
        y[2, : c - 1] = -math.inf
        y[3, c // 2:] = 40.0
        y[4, -1] = y[4, c // 3] = math.nan
        y[5, -1] = math.inf
        y[6] = torch.linspace(-20, 20, c, device=DEV).to(dtype)
        y[7] = torch.linspace(20, -20, c, device=DEV).to(dtype)
        y[8] = math.nan
        y[9, torch.arange(c, device=DEV) % 50 != 7 % c] = -math.inf
        y[10, c - c // 3:] += 20.0
    for top in tops:
        r = _score(x, t, top=top)
        for p in parts:
            _check(x[p], t[p], top, r=type(r)(*(None if v is None else v[p] for v in r)))


def test_same_bits_every_time_and_two_streams_at_once():
    x, t = _logits(37, 40001, torch.bfloat16), _target(37, 40001)
    y, k = _logits(5000, 20, torch.float32), _target(5000, 20)
    first = [_score(x, t, top=9), _score(y, k, top=3)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = _score(x, t, top=9)
        b = _score(y, k, top=3)
        torch.cuda.current_stream().wait_stream(side)
        for got, want in zip((a, b), first):
            assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_captured_forward_and_backward():
    """Two graphs captured from the same code, replayed in turn with eager work and new logits between the replays."""
    cases = []
    for rows, c, dtype in ((50, 20, torch.float32), (3, 50021, torch.bfloat16), (40, 3000, torch.float16)):
        x = _logits(rows, c, dtype).clone().requires_grad_(True)
        t = _target(rows, c)
        g = torch.randn(rows, device=DEV)

        def step(x=x, t=t, g=g):
            r = _score(x, t, top=4)
            (d,) = torch.autograd.grad([r.logprob, r.entropy], x, [g, g])
            return [v.detach() for v in (*r, d)]                        # (no autograd graph outlives a step)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        cases.append((graph, out, step, x))
    for turn in range(4):
        for graph, out, step, x in cases:
            with torch.no_grad():
                x.copy_(torch.randn(x.shape, device=DEV) * (turn + 1))
            want = step()
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_rows_beside_the_outputs_stay():
    """The gradient's padding columns and the rows of the outputs' neighbours are not written."""
    from curvecloudnet_amd._lib import call, ptr
    for rows, c, dtype, code in ((5, 7, torch.float32, 0), (5, 65, torch.float16, 2), (2, 5001, torch.bfloat16, 1)):
        x, t = _logits(rows, c, dtype), _target(rows, c)
        f = [torch.full((rows + 2,), 7.0, device=DEV) for _ in range(2)]
        stats, best = torch.full((rows + 2, 2), 7.0, device=DEV), torch.full((rows + 2, 3), 7.0, device=DEV)
        index = torch.full((rows + 2, 3), 7, dtype=torch.int64, device=DEV)
        from curvecloudnet_amd._lib import lib, workspace
        n = lib().ccn_logprob_workspace_bytes(rows, c, 3)
        call("logprob_fwd", ptr(x), code, x.stride(0), ptr(t), rows, c, -100, 3, ptr(f[0][1:]), ptr(f[1][1:]), ptr(stats[1:]),
             ptr(best[1:]), ptr(index[1:]), ptr(workspace(n, DEV)), n)
        for v in f + [stats, best, index]:
            assert bool((v[0] == 7).all()) and bool((v[-1] == 7).all())
        _check(x, t, 3, r=type(_score(x, t))(f[0][1:-1], f[1][1:-1], best[1:-1], index[1:-1]))
        d = torch.full((rows + 2, c + 5), 7.0, dtype=dtype, device=DEV)
        g = torch.ones(rows, device=DEV)
        call("logprob_bwd", ptr(x), code, x.stride(0), ptr(t), rows, c, -100, 0, None, ptr(stats[1:]), ptr(f[1][1:]), ptr(g), 1,
             None, 0, None, ptr(d[1:]), d.stride(0))
        assert bool((d[0] == 7).all()) and bool((d[-1] == 7).all()) and bool((d[:, c:] == 7).all())
        assert bool((d[1:-1, :c] != 7).all())


def test_launches_are_observed(monkeypatch):
    """The timing of launches (bench.py's) sees these operators, the backward pass on autograd's thread among them; results stay."""
    from curvecloudnet_amd import _lib, costs
    from curvecloudnet_amd.parallel import grad_norm
    x, t = _logits(40, 5000, torch.float32).requires_grad_(True), _target(40, 5000)

    def step():
        r = _score(x, t, top=3)
        (d,) = torch.autograd.grad([r.logprob, r.top_logprob], x, [torch.ones_like(r.logprob), torch.ones_like(r.top_logprob)])
        return [v.detach() for v in (*r, d, grad_norm([d]))]

    want = step()
    monkeypatch.setattr(_lib, "PROFILE", [])
    got = step()
    torch.cuda.synchronize()
    records = _lib.PROFILE
    monkeypatch.setattr(_lib, "PROFILE", None)
    assert [r[0] for r in records] == ["logprob_fwd", "logprob_bwd", "grad_norm"]
    assert all(r[2].elapsed_time(r[3]) > 0 for r in records)
    for name, ints, _, _, _, work in records:
        family, _, nbytes, modelled = costs.entry_cost(name, ints, work)
        assert family == "loss_optim" and modelled and nbytes >= 40 * 5000 * 4
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


def test_gradient_is_not_differentiated_again():
    x, t = _logits(4, 30, torch.float32).requires_grad_(True), _target(4, 30)
    w = torch.ones((), device=DEV, requires_grad=True)
    (d,) = torch.autograd.grad((_score(x, t).logprob * w).sum(), x, create_graph=True)
    (ref,) = torch.autograd.grad(_score(x, t).logprob.sum(), x)
    assert torch.equal(d.detach(), ref)
    with pytest.raises(RuntimeError):                                  # (no way from the gradient back to the logits)
        torch.autograd.grad(d.sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        d.sum().backward()


def test_other_kinds_of_tensors():
    x, t = _logits(6, 40, torch.float32), _target(6, 40)
    want = _score(x, t, top=2)
    with torch.inference_mode():
        assert all(torch.equal(a, b) for a, b in zip(_score(x.clone(), t.clone(), top=2), want))
    z = torch.complex(torch.zeros_like(x), -x)
    assert z.conj().imag.is_neg() and all(torch.equal(a, b) for a, b in zip(_score(z.conj().imag, t, top=2), want))
    leaf = x.clone().requires_grad_(True)
    r = _score(leaf, t)
    r.entropy.sum().backward()
    a = leaf.grad.clone()
    r = _score(leaf, t)
    r.entropy.sum().backward()
    assert torch.equal(leaf.grad, 2 * a)                                # (accumulated as any gradient is)
    r = _score(leaf, t)
    with torch.no_grad():
        leaf.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprob.sum().backward()


def test_tangents_are_refused():
    import torch.autograd.forward_ad as forward
    x, t = _logits(4, 30, torch.float32), _target(4, 30)
    with forward.dual_level(), pytest.raises(RuntimeError, match="jvp"):
        _score(forward.make_dual(x, torch.ones_like(x)), t)


@pytest.mark.parametrize("c,top", [(3, 2), (33, 2), (600, 0), (4097, 0)])
def test_more_rows_than_a_launch_holds(c, top):
    rows, border = (1 << 22) + 5, 1 << 22
    x = torch.zeros(rows, c, dtype=torch.float16, device=DEV)
    t = torch.zeros(rows, dtype=torch.int64, device=DEV)
    for at in (0, border - 4):                                          # (the first rows, and those on both sides of the border)
        x[at: at + 9] = _logits(9, c, torch.float16, seed=at)
        t[at: at + 9] = _target(9, c, seed=at)
    x.requires_grad_(True)
    r = _score(x, t, top=top)
    (d,) = torch.autograd.grad(r.logprob.sum() + 2 * r.entropy.sum(), x)
    for at in (0, border - 4):
        part = slice(at, at + 9)
        # (as many rows as take the same kernels)
        small, given = torch.zeros(5000, c, dtype=x.dtype, device=DEV), torch.zeros(5000, dtype=torch.int64, device=DEV)
        small[:9], given[:9] = x.detach()[part], t[part]
        small.requires_grad_(True)
        q = _score(small, given, top=top)
        _check(small[:9].detach(), given[:9], top, r=type(q)(*(None if a is None else a[:9] for a in q)))
        (e,) = torch.autograd.grad(q.logprob.sum() + 2 * q.entropy.sum(), small)
        assert torch.equal(d[part], e[:9])
        assert all(torch.equal(a[part], b[:9]) for a, b in zip(r, q) if a is not None)
    rest = r.logprob.detach()[9: border - 4]
    _near(rest[:: 1 << 18], torch.full((rest[:: 1 << 18].numel(),), -math.log(c)), _e(torch.tensor(math.log(c)), c), "rows of zeros")
    assert bool((rest == rest[0]).all())


@pytest.mark.parametrize("c", [20, 300, 5000])
def test_gradients_whose_sign_is_still_to_be_turned(c):
    """Gradients with torch's negative bit, contiguous and strided, give the bits of the negated ones; so does the engine's own: the
    imaginary part of a conjugated complex number hands its gradient down that way."""
    x, t = _logits(33, c, torch.float32).requires_grad_(True), _target(33, c)
    gen = torch.Generator().manual_seed(c)
    for k, shape in enumerate(((33,), (33,), (33, 7))):
        g = torch.randn(shape, generator=gen).to(DEV)
        far = torch.stack([g, g + 1], -1)[..., 0]
        for lazy in (torch._neg_view(g), torch._neg_view(far)):
            assert lazy.is_neg()
            r = _score(x, t, top=7)
            (want,) = torch.autograd.grad(r[k], x, -g, retain_graph=True)
            (got,) = torch.autograd.grad(r[k], x, lazy)
            assert float(want.abs().max()) > 0 and torch.equal(got, want)
    seen = []
    r = _score(x, t)
    r.entropy.register_hook(lambda g: seen.append(g.is_neg()))
    both = torch.view_as_real(torch.complex(r.logprob, r.entropy).conj().resolve_conj())
    (got,) = torch.autograd.grad(both.sum(), x, retain_graph=True)
    assert seen == [True]
    (want,) = torch.autograd.grad([r.logprob, r.entropy], x, [torch.ones_like(r.logprob), -torch.ones_like(r.entropy)])
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16], ids=["fp32", "fp16"])
@pytest.mark.parametrize("c", list(range(1, 25)))
def test_every_number_of_alternatives_of_short_rows(c, dtype):
    """Rows that a thread walks in shared memory, where results and keys take the place of the logits: waves of ordinary rows and waves with
    rows of NaN, infinities, equal logits and zeros of both signs, for every number of alternatives."""
    x, t = _logits(300, c, dtype), _target(300, c)
    for at in (0, 130, 140, 299 - 9):
        x[at], x[at + 1], x[at + 2, c // 2] = math.nan, -math.inf, math.nan
        x[at + 3], x[at + 4, -1], x[at + 5, 0] = 0.25, math.inf, -math.inf
        x[at + 6, ::2], x[at + 6, 1::2], x[at + 7, 1:] = -0.0, 0.0, -math.inf
        x[at + 8, ::3] = math.nan
    for top in range(c + 1):
        _check(x, t, top)
    many = x.repeat(220, 1)                                             # (as many rows as keep to that form)
    given = t.repeat(220)
    for top in sorted({c // 2, c}):
        r = _score(many, given, top=top)
        for part in (slice(0, 300), slice(300 * 219, 300 * 220)):
            _check(x, t, top, r=type(r)(*(None if v is None else v[part] for v in r)))


def _gradient_under_hooks(x, t, g, pack, unpack):
    from torch.autograd.graph import saved_tensors_hooks
    with saved_tensors_hooks(pack, unpack):
        r = _score(x, t, top=3)
    return torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], x, g)[0]


@pytest.mark.parametrize("c", [20, 300, 5000])
def test_saved_tensors_that_come_back_in_another_layout(c):
    """Hooks on saved tensors: copies, on the host meanwhile, spread out, transposed, with their sign still to be turned; checkpointing."""
    x, t = _logits(33, c, torch.float32).requires_grad_(True), _target(33, c)
    gen = torch.Generator().manual_seed(c)
    g = [torch.randn(s, generator=gen).to(DEV) for s in ((33,), (33,), (33, 3))]
    r = _score(x, t, top=3)
    (want,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], x, g)
    same = lambda v: v                                                  # noqa: E731
    for pack, unpack in ((torch.clone, same), (lambda v: v.cpu(), lambda v: v.to(DEV)), (torch.clone, lambda v: torch.stack([v, v], -1)[..., 0]),
                         (torch.clone, lambda v: v.t().contiguous().t()), (torch.neg, torch._neg_view)):
        assert torch.equal(_gradient_under_hooks(x, t, g, pack, unpack), want)
    from torch.utils.checkpoint import checkpoint
    r = checkpoint(lambda y: _score(y, t, top=3), x, use_reentrant=False)
    (got,) = torch.autograd.grad([r.logprob, r.entropy, r.top_logprob], x, g)
    assert torch.equal(got, want)


@pytest.mark.parametrize("unpack", [lambda v: v[:5], lambda v: v[..., None], lambda v: v.double() if v.is_floating_point() else v.int(),
                                    lambda v: v.cpu(), lambda v: v.cpu() if v.dim() == 1 else v, lambda v: v[:, :1] if v.dim() == 2 else v],
                         ids=["rows", "axes", "types", "host", "host-in-part", "columns"])
def test_saved_tensors_that_come_back_as_others_are_refused(unpack):
    x, t = _logits(33, 300, torch.float32).requires_grad_(True), _target(33, 300)
    g = [torch.ones(s, device=DEV) for s in ((33,), (33,), (33, 3))]
    with pytest.raises(RuntimeError, match="hook"):
        _gradient_under_hooks(x, t, g, torch.clone, unpack)


class _Nothing(torch.autograd.Function):
    @staticmethod
    def forward(ctx, v):
        return v.clone()

    @staticmethod
    def backward(ctx, g):
        return None


@pytest.mark.parametrize("c", [20, 300, 5000])
def test_outputs_that_get_no_gradient_at_all(c):
    """What follows gives none to any output: zeros come out."""
    x, t = _logits(7, c, torch.float32).requires_grad_(True), _target(7, c)
    r = _score(x, t, top=3)
    (d,) = torch.autograd.grad(sum(_Nothing.apply(v).sum() for v in r[:3]), x)
    assert d.shape == x.shape and not bool(d.any())


def test_saved_rows_that_come_back_expanded():
    """Every value of a row is the same, and comes back as one."""
    x, t = torch.full((1, 300), 0.5, device=DEV).requires_grad_(True), _target(1, 300)
    r = _score(x, t, top=3)
    g = [torch.ones_like(v) for v in r[:3]]
    (want,) = torch.autograd.grad(r[:3], x, g)
    got = _gradient_under_hooks(x, t, g, torch.clone, lambda v: v[:, :1].clone().expand(1, 300) if v.shape == (1, 300) else v)
    assert torch.equal(got, want)
