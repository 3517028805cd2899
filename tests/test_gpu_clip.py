"""parallel.grad_norm, clip_grad_norm_, adam_step_ and FlatAdam(max_norm=) on the GPU against their formulas in 64 bits.

Tolerances, derived.  u = 2^-24.  Norms are summed in 64 bits (their error there, 2^-53 times the number of values, is nothing) and
rounded once: u |norm|.  The factor is rounded to 32 bits and to the gradient's type (as torch's product with a scalar tensor does), the
product to 32 bits and to the type: (1 + u)^2 (1 + eps / 2)^2 - 1, a clipped value is off by (2 u + eps) of itself (2 u for fp32, whose type
rounds nothing more) and eps^2 / 4 + 2 u eps, less than a hundredth of that; and by half a subnormal step of fp16 (2^-25; the factor's own
may be subnormal too: 2^-25 of |g|) or bf16 / fp32 (2^-134 / 2^-150).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["fp32", "bf16", "fp16"]


def _params(sizes, dtypes, seed=0, spread=1.0, flat=False, shift=0):
    """Leaves with gradients; ``flat``: all of a type in one buffer, ``shift`` values behind its start, with no gap between them."""
    gen = torch.Generator().manual_seed(seed + len(sizes))
    out, used = [], {}
    total = {d: sum(torch.Size(s).numel() for s, e in zip(sizes, dtypes) if e == d) for d in set(dtypes)}
    bufs = {d: torch.zeros(n + shift, dtype=d, device=DEV) for d, n in total.items()} if flat else {}
    for size, d in zip(sizes, dtypes):
        p = torch.nn.Parameter(torch.zeros(size, dtype=d, device=DEV))
        g = (torch.randn(size, generator=gen) * spread).to(d)
        if flat:
            at = used.get(d, shift)
            used[d] = at + p.numel()
            p.grad = bufs[d][at: at + p.numel()].view(size)
            p.grad.copy_(g)
        else:
            p.grad = g.to(DEV)
        out.append(p)
    return out


def _norm64(grads, kind):
    every = torch.cat([g.detach().cpu().double().reshape(-1) for g in grads])
    if not every.numel():
        return 0.0
    if kind == 2:
        big = float(every.abs().max())
        return big * float((every / big).square().sum().sqrt()) if big > 0 and math.isfinite(big) else float(every.square().sum().sqrt())
    return float(every.abs().sum()) if kind == 1 else float(every.abs().max())


def _check_clip(params, max_norm, kind=2.0):
    from curvecloudnet_amd.parallel import clip_grad_norm_, grad_norm
    grads = [p.grad for p in params]
    before = [g.clone() for g in grads]
    at = [g.data_ptr() for g in grads]
    want = _norm64(before, kind)
    alone = grad_norm(grads, norm_type=kind)
    norm = clip_grad_norm_(params, max_norm, norm_type=kind)
    assert norm.dtype == torch.float32 and norm.shape == () and norm.is_cuda and torch.equal(alone, norm)
    if want > torch.finfo(torch.float32).max:           # (3e38 sqrt 3 = 5.2e38 leaves the result's type; the factor is right all the same)
        assert float(norm) == math.inf
    else:
        assert abs(float(norm) - want) <= U * want, (float(norm), want)
    scale = min(1.0, max_norm / (want + 1e-6))
    for p, g, b, a in zip(params, grads, before, at):
        assert p.grad is g and g.data_ptr() == a
        ref = b.cpu().double() * scale
        eps = 0.0 if g.dtype == torch.float32 else torch.finfo(g.dtype).eps
        tiny = 2.0 ** -25 * (1 + b.cpu().double().abs()) if g.dtype == torch.float16 else 2.0 ** -134
        if scale == 1.0:
            assert torch.equal(g, b)
            continue
        off = (g.cpu().double() - ref).abs()
        assert bool((off <= ref.abs() * (2 * U + eps) * 1.01 + tiny).all())
    return norm


@pytest.mark.parametrize("kind", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("dtype", DTYPES, ids=IDS)
@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 9, 255, 256, 257, 4095, 16383, 16384, 16385, 40001, 1000003])
def test_one_tensor(n, dtype, kind):
    for max_norm in (0.25, 1e9):
        _check_clip(_params([(n,)], [dtype]), max_norm, kind)


@pytest.mark.parametrize("kind", [1.0, 2.0, math.inf])
@pytest.mark.parametrize("flat,shift", [(False, 0), (True, 0), (True, 1), (True, 3)])
def test_many_tensors_of_mixed_types(flat, shift, kind):
    gen = torch.Generator().manual_seed(3)
    sizes = [(int(k),) for k in torch.randint(1, 3000, (77,), generator=gen)] + [(0,), (64, 3, 5), (1,), (0, 4), (20000,), (), (33, 1)]
    dtypes = [DTYPES[i % 3] for i in range(len(sizes))]
    _check_clip(_params(sizes, dtypes, flat=flat, shift=shift), 1.0, kind)
    for d in DTYPES:
        _check_clip(_params(sizes, [d] * len(sizes), flat=flat, shift=shift), 1.0, kind)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 159, 160, 161, 319, 320, 321, 640, 641, 1000])
def test_more_tensors_than_a_launch_holds(n):
    _check_clip(_params([(1 + i % 37,) for i in range(n)], [DTYPES[i % 3] for i in range(n)]), 0.5)


def test_a_long_tensor_and_short_ones():
    for d in DTYPES:
        _check_clip(_params([(5,), (30000001,), (7,)], [d] * 3, flat=True), 3.0)


def test_the_bound_itself():
    for bound in (0.0, 1e-30, math.inf):
        _check_clip(_params([(1000,), (7,)], [torch.float32, torch.bfloat16]), bound)
    p = _params([(4,)], [torch.float32])
    p[0].grad.copy_(torch.tensor([3.0, 0.0, 4.0, 0.0]))
    from curvecloudnet_amd.parallel import clip_grad_norm_
    norm = clip_grad_norm_(p[0], 5.1)                                   # (one tensor in place of a list; nothing to scale)
    assert float(norm) == 5.0 and p[0].grad.tolist() == [3.0, 0.0, 4.0, 0.0]
    norm = clip_grad_norm_(iter(p), 2.5)
    assert float(norm) == 5.0
    assert all(abs(a - b) <= b * (2e-7 + 2 * U) for a, b in zip(p[0].grad.tolist(), [1.5, 0.0, 2.0, 0.0]))
    z = _params([(100,), (3,)], [torch.float16, torch.float32], spread=0.0)
    assert float(clip_grad_norm_(z, 1.0)) == 0.0 and not any(bool(q.grad.any()) for q in z)


def test_values_whose_squares_leave_fp32():
    for value, n in ((1e30, 5000), (1e-30, 5000), (3e38, 3)):
        p = _params([(n,)], [torch.float32])
        p[0].grad.fill_(value)
        _check_clip(p, value, 2.0)
        p[0].grad.fill_(value)
        _check_clip(p, value, math.inf)


@pytest.mark.parametrize("kind", [1.0, 2.0, math.inf])
def test_norms_that_are_not_finite(kind):
    from curvecloudnet_amd.parallel import clip_grad_norm_, grad_norm
    for bad in (math.nan, math.inf, -math.inf):
        for where in (0, 500, 40000):
            p = _params([(700,), (50000,), (3,)], [torch.float32, torch.bfloat16, torch.float16])
            p[1].grad[where] = bad
            before = [q.grad.clone() for q in p]
            norm = grad_norm([q.grad for q in p], kind)
            assert math.isnan(float(norm)) if math.isnan(bad) else float(norm) == math.inf
            with pytest.raises(RuntimeError, match="norm of the gradients"):
                clip_grad_norm_(p, 1.0, norm_type=kind, error_if_nonfinite=True)
            assert all(torch.equal(q.grad.nan_to_num(7.0), b.nan_to_num(7.0)) for q, b in zip(p, before))
            clip_grad_norm_(p, 1.0, norm_type=kind)
            if math.isnan(bad):
                assert all(bool(torch.isnan(q.grad).all()) for q in p)
            else:
                assert bool(torch.isnan(p[1].grad[where])) and float(p[0].grad.abs().max()) == 0.0


def test_gradients_that_are_missing_or_of_another_layout():
    from curvecloudnet_amd.parallel import clip_grad_norm_, grad_norm
    p = _params([(8, 4, 6, 5), (9,), (40, 30)], [torch.float32] * 3)
    p[0].grad = p[0].grad.contiguous(memory_format=torch.channels_last)
    p[2] = torch.nn.Parameter(torch.zeros(30, 40, device=DEV).t())
    p[2].grad = torch.randn(30, 40, device=DEV).t()
    p[1].grad = None
    want = _norm64([p[0].grad, p[2].grad], 2)
    before = [p[0].grad.clone(), p[2].grad.clone()]
    assert abs(float(clip_grad_norm_(p, 1.0)) - want) <= U * want
    for q, b in zip((p[0], p[2]), before):
        ref = b.cpu().double() / (want + 1e-6)
        assert q.grad.stride() == b.stride()
        assert bool(((q.grad.cpu().double() - ref).abs() <= ref.abs() * 3.1 * U).all())
    assert float(clip_grad_norm_([p[1]], 1.0)) == 0.0 and float(grad_norm([])) == 0.0 and float(clip_grad_norm_([], 1.0)) == 0.0
    with pytest.raises(ValueError, match="does not fill its memory"):
        grad_norm([torch.zeros(6, 8, device=DEV)[:, :4]])
    with pytest.raises(ValueError, match="does not fill its memory"):
        grad_norm([torch.zeros(1, device=DEV).expand(5)])


def test_shared_memory_is_refused():
    from curvecloudnet_amd.parallel import clip_grad_norm_, grad_norm
    p = _params([(100,), (50,)], [torch.float32] * 2)
    before = [q.grad.clone() for q in p]
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([p[0], p[1], p[0]], 0.1)
    q = torch.nn.Parameter(torch.zeros(30, device=DEV))
    q.grad = p[0].grad[90:].new_zeros(0).set_(p[0].grad.untyped_storage(), 70, (30,))
    with pytest.raises(RuntimeError, match="share memory"):
        clip_grad_norm_([q, p[1], p[0]], 0.1)
    torch.cuda.synchronize()
    assert all(torch.equal(a.grad, b) for a, b in zip(p, before))
    twice = float(grad_norm([p[1].grad, p[1].grad]))                    # (a norm only reads: counted as often as it is given)
    want = math.sqrt(2.0) * _norm64([p[1].grad], 2)
    assert abs(twice - want) <= 2 * U * want


def test_same_bits_as_torch():
    """torch.nn.utils.clip_grad_norm_ on the same gradients: for 16-bit types its factor is taken from the norm here, torch rounds its own
    norm to the type."""
    from curvecloudnet_amd.parallel import clip_grad_norm_
    for d in DTYPES:
        p = _params([(1000,), (77, 3), (5,)], [d] * 3)
        q = _params([(1000,), (77, 3), (5,)], [d] * 3)
        norm = clip_grad_norm_(p, 1.5)
        torch._foreach_mul_([x.grad for x in q], (1.5 / (norm.double() + 1e-6)).float())
        assert all(torch.equal(a.grad, b.grad) for a, b in zip(p, q))


def test_small_factors_of_fp16():
    """A factor below 2^-14 is no normal fp16 number: rounded to one it would be off by up to all of itself.  In 32 bits a value is off by
    the norm's and the factor's roundings (2 u), the product's (u) and half a step of its type, 2^-25 at least."""
    from curvecloudnet_amd.parallel import clip_grad_norm_
    for bound in (1e-4, 2e-3, 0.03, 0.9):
        (p,) = _params([(100000,)], [torch.float16])
        before = p.grad.mul_(300).double()
        norm = clip_grad_norm_([p], bound)
        ref = before * (bound / (float(before.square().sum().sqrt()) + 1e-6))
        assert float(norm) > 5e4 and bound / float(norm) < 2.0 ** -14
        off = (p.grad.double() - ref).abs()
        assert bool((off <= ref.abs() * (2.0 ** -11 + 4 * U) + 2.0 ** -25).all())
    assert float(p.grad.abs().max()) > 0


def test_gradients_whose_memory_is_not_their_own_yet():
    from curvecloudnet_amd.parallel import clip_grad_norm_
    (p,) = _params([(1000,)], [torch.float32])
    origin = p.grad
    before = origin.clone()
    p.grad = torch._lazy_clone(origin)                                  # (copied when it is first written)
    clip_grad_norm_([p], 0.5)
    assert torch.equal(origin, before) and not torch.equal(p.grad, before)


def test_versions_move_and_neighbours_stay():
    from curvecloudnet_amd.parallel import clip_grad_norm_
    buf = torch.ones(3000, device=DEV)
    p = torch.nn.Parameter(torch.zeros(2001, device=DEV))
    p.grad = buf[501:2502]
    v = p.grad._version
    clip_grad_norm_(p, 1.0)
    assert p.grad._version > v
    assert bool((buf[:501] == 1).all()) and bool((buf[2502:] == 1).all()) and bool((buf[501:2502] < 1).all())


def test_same_bits_every_time_and_on_another_stream():
    from curvecloudnet_amd.parallel import grad_norm
    g = [p.grad for p in _params([(3000001,), (77,), (40000,)], [torch.float32, torch.bfloat16, torch.float16])]
    want = [grad_norm(g, k) for k in (1.0, 2.0, math.inf)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            a = [grad_norm(g, k) for k in (1.0, 2.0, math.inf)]
        b = [grad_norm(g, k) for k in (1.0, 2.0, math.inf)]
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(x, y) for x, y in zip(a, want)) and all(torch.equal(x, y) for x, y in zip(b, want))


def test_captured_clipping():
    from curvecloudnet_amd.parallel import clip_grad_norm_
    graphs = []
    for sizes, dtypes in (([(300001,), (7,)], [torch.float32, torch.bfloat16]), ([(50,)] * 200, [torch.float32] * 200)):
        p = _params(sizes, dtypes)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            clip_grad_norm_(p, 1.0)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = clip_grad_norm_(p, 1.0)
        graphs.append((graph, p, norm))
    for turn in range(4):
        for graph, p, norm in graphs:
            fresh = [torch.randn(q.shape, device=DEV).to(q.dtype) * (turn + 1) for q in p]
            for q, f in zip(p, fresh):
                q.grad.copy_(f)
            graph.replay()
            torch.cuda.synchronize()
            got = [q.grad.clone() for q in p]
            for q, f in zip(p, fresh):
                q.grad.copy_(f)
            assert torch.equal(clip_grad_norm_(p, 1.0), norm)
            assert all(torch.equal(q.grad, b) for q, b in zip(p, got)), turn


# ---- the update that clips


def _adam64(p, g, m, v, step, lr, betas, eps, decay, max_norm):
    norm = math.sqrt(sum(float(x.square().sum()) for x in g))
    scale = 1.0 if max_norm is None else min(1.0, max_norm / (norm + 1e-6))
    out = []
    for a, b, c, d in zip(p, g, m, v):
        b = b * scale + decay * a
        c = c + (b - c) * (1 - betas[0])
        d = d * betas[1] + (1 - betas[1]) * b * b
        e = (d / (1 - betas[1] ** step)).sqrt() + eps
        out.append((a - lr * (c / (1 - betas[0] ** step)) / e, c, d, b, e))
    return norm, out


@pytest.mark.parametrize("sizes", [(1,), (4,), (5, 1, 3), (1000, 7, 16385, 4096), (16384,) * 5, (300001, 20), (37,) * 70])
@pytest.mark.parametrize("max_norm", [0.01, 1e9])
def test_adam_step_that_clips(sizes, max_norm):
    """A first update and a later one.  In 32 bits the scaled gradient with decay is off by 4 u (|g'| + |decay p|), m by 8 u (|m| + |g'|
    + |decay p|), v by 12 u of itself and 8 u |g'| (|g'| + |decay p|), the update by lr times 16 u of (|m| + |g'|) / denominator and the
    share that v's error has in the denominator (half of its relative error), p by u |p| more."""
    from curvecloudnet_amd.parallel import adam_step_
    lr, betas, eps, decay = 1e-2, (0.9, 0.999), 1e-8, 0.02
    gen = torch.Generator().manual_seed(sum(sizes))
    draw = lambda s: [(torch.randn(n, generator=gen) * s) for n in sizes]      # noqa: E731
    for step, spread in ((1, 0.0), (50, 0.3)):
        p, g, m = draw(1.0), draw(0.5), draw(spread)
        v = [x.square() * spread for x in draw(0.5)]
        norm, want = _adam64(*[[x.double() for x in k] for k in (p, g, m, v)], step, lr, betas, eps, decay, max_norm)
        dev = [[x.to(DEV) for x in k] for k in (p, g, m, v)]
        got = adam_step_(*dev, step, lr=lr, betas=betas, eps=eps, weight_decay=decay, max_norm=max_norm)
        assert abs(float(got) - norm) <= U * norm
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev[1], g))            # (the gradients keep their values)
        for k, (wp, wm, wv, wg, den) in enumerate(want):
            g0 = wg.abs() + (decay * p[k].double()).abs() * 2
            em = 8 * U * (m[k].double().abs() + g0)
            ev = 12 * U * wv + 8 * U * g0 * g0
            assert bool(((dev[2][k].cpu().double() - wm).abs() <= em).all())
            assert bool(((dev[3][k].cpu().double() - wv).abs() <= ev).all())
            bc1 = 1 - betas[0] ** step
            up = lr / bc1 * ((em + 16 * U * wm.abs()) / den + wm.abs() / den * ev / (wv + 1e-300))
            assert bool(((dev[0][k].cpu().double() - wp).abs() <= up + 2 * U * wp.abs()).all())


def test_adam_step_without_a_bound_is_the_optimisers_own():
    from curvecloudnet_amd.parallel import adam_step_
    p = torch.randn(5000, device=DEV)
    a, b = [[p.clone()], [p * 0.1], [torch.zeros_like(p)], [torch.zeros_like(p)]], torch.nn.Parameter(p.clone())
    ref = torch.optim.Adam([b], lr=1e-2)
    for step in range(1, 4):
        b.grad = p * 0.1
        ref.step()
        assert adam_step_(*a, step, lr=1e-2) is None
        assert float((a[0][0] - b.detach()).abs().max()) < 1e-6 * step


def test_captured_adam_step():
    from curvecloudnet_amd.parallel import adam_step_
    make = lambda: [[torch.randn(n, device=DEV) for n in (30000, 12)] for _ in range(3)] + [[torch.rand(n, device=DEV) for n in (30000, 12)]]  # noqa: E731,E501
    x = make()
    y = [[t.clone() for t in k] for k in x]
    adam_step_(*make(), 3, max_norm=0.5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = adam_step_(*x, 3, max_norm=0.5)
    for turn in range(4):
        for a, b in zip(x[1], y[1]):
            a.copy_(torch.randn_like(a) * (turn + 1))
            b.copy_(a)
        want = adam_step_(*y, 3, max_norm=0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(norm, want)
        assert all(torch.equal(a, b) for k, q in zip(x, y) for a, b in zip(k, q)), turn


def test_adam_step_refuses_shared_and_unaligned_memory():
    from curvecloudnet_amd.parallel import adam_step_
    make = lambda n=64: [torch.zeros(n, device=DEV)]       # noqa: E731
    p = make()
    with pytest.raises(RuntimeError, match="share memory"):
        adam_step_(p, make(), p, make(), 1, max_norm=1.0)
    with pytest.raises(RuntimeError, match="share memory"):
        adam_step_(p + p, make() + make(), make() + make(), make() + make(), 1, max_norm=1.0)
    with pytest.raises(ValueError, match="multiple of 16"):
        adam_step_([make(65)[0][1:]], make(), make(), make(), 1, max_norm=1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        adam_step_([torch.zeros(64)], make(), make(), make(), 1, max_norm=1.0)


def test_flat_adam_with_a_bound_follows_torch():
    """FlatAdam(max_norm) against clip_grad_norm_ of torch and torch.optim.Adam in 64 bits: two updates of a parameter of size <= 4, each
    off by a few u of lr and of the parameter."""
    from curvecloudnet_amd.parallel import FlatAdam, GradientAllReduce
    torch.manual_seed(2)
    shapes = [(64, 37), (64,), (128, 64), (3, 5, 7), (1,), (1000, 33)]
    ref = [torch.nn.Parameter(torch.randn(s).double()) for s in shapes]
    holder = torch.nn.ParameterList([torch.nn.Parameter(p.detach().float().to(DEV)) for p in ref])
    for q, p in zip(holder, ref):
        p.data.copy_(q.detach().cpu())
    sync = GradientAllReduce(holder, bucket_bytes=40_000)
    mine, theirs = FlatAdam(sync, lr=1e-2, max_norm=1.5), torch.optim.Adam(ref, lr=1e-2)
    assert len(sync.buckets) > 1 and set(mine.state_dict()["param_groups"][0]) == set(FlatAdam(sync).state_dict()["param_groups"][0])
    mine = FlatAdam(sync, lr=1e-2, max_norm=1.5)
    for it in range(3):
        mine.zero_grad()
        for p, q in zip(ref, holder):
            g = torch.randn(p.shape)
            p.grad = g.double()
            q.grad.copy_(g)
        norm = torch.nn.utils.clip_grad_norm_(ref, 1.5)
        theirs.step()
        mine.step()
        assert abs(float(mine.grad_norm) - float(norm)) <= U * float(norm)
        for p, q in zip(ref, holder):
            assert float((p.detach() - q.detach().cpu().double()).abs().max()) <= (it + 1) * (2 * 4 * U + 1e-2 * 64 * U)


def test_a_run_of_all_of_them():
    """Points through the package's MLP, log-probabilities with their entropy as the loss, the gradients into the flat buckets, the
    update that clips; against the same in 64 bits from the same parameters, step by step: products in fp32 (K <= 48) put about
    100 u on the logits, which the gradients and one Adam step of at most lr carry on."""
    from curvecloudnet_amd.loss import token_logprobs
    from curvecloudnet_amd.nn import MLP
    from curvecloudnet_amd.parallel import FlatAdam, GradientAllReduce, clip_grad_norm_, grad_norm
    torch.manual_seed(0)
    mlp = MLP([12, 48, 20]).to(DEV)
    sync = GradientAllReduce(mlp)
    opt = FlatAdam(sync, lr=1e-2, max_norm=0.05)
    x = torch.randn(3000, 12, device=DEV)
    y = torch.randint(0, 20, (3000,), device=DEV)
    y[::7] = 0
    losses = []
    for it in range(4):
        opt.zero_grad()
        r = token_logprobs(mlp(x), y, top=3, ignore_index=0)
        loss = -r.logprob.sum() / (y != 0).sum() - 0.01 * r.entropy.mean() + 0.001 * r.top_logprob.mean()
        loss.backward()
        sync.finish()
        assert torch.isfinite(loss) and bool((r.top_logprob[:, 0] >= r.top_logprob[:, 2]).all())
        flat = torch.cat([p.grad.reshape(-1) for p in mlp.parameters()]).double()
        want = float(flat.norm())
        assert abs(float(grad_norm([p.grad for p in mlp.parameters()])) - want) <= 2 * U * want
        # the gradient of the last layer's bias: the mean over rows of the loss's gradient in the logits
        logits = mlp(x).detach().double()
        z = logits.requires_grad_(True)
        logp = torch.log_softmax(z, 1)
        ref = (-(logp.gather(1, y[:, None]).squeeze(1) * (y != 0)).sum() / (y != 0).sum() + 0.01 * (logp.exp() * logp).sum(1).mean()
               + 0.001 * logp.gather(1, r.top_index).mean())
        (d,) = torch.autograd.grad(ref, z)
        assert abs(float(ref.detach()) - float(loss.detach())) <= 400 * U * 4
        bias = mlp.lins[-1].bias.grad.double()
        assert float((bias - d.sum(0)).abs().max()) <= 3000 * U * float(d.abs().sum(0).max())
        opt.step()
        assert abs(float(opt.grad_norm) - want) <= 2 * U * want
        losses.append(float(loss.detach()))
    assert all(math.isfinite(v) for v in losses)
    sync.zero_grad()
    token_logprobs(mlp(x), y).logprob.mean().backward()
    before = float(grad_norm([p.grad for p in mlp.parameters()]))
    assert abs(float(clip_grad_norm_(mlp.parameters(), before / 2)) - before) <= U * before
    assert abs(float(grad_norm([p.grad for p in mlp.parameters()])) - before / 2) <= before * (4 * U) + 1e-6


@pytest.mark.parametrize("sizes", [(1,), (5, 1, 3), (1000, 7, 16385, 4096), (300001, 20), (37,) * 70, (0, 9, 0)])
def test_adam_step_without_a_bound(sizes):
    """Parameters and both moments, the bits of an infinite bound, another stream, and a captured update.  The errors are those of the update
    that clips, but for v's: the gradient with decay is off by 4 u (|g| + |decay p|), its square by 8 u of their square, which
    1 - beta2 takes along."""
    from curvecloudnet_amd.parallel import adam_step_
    how = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)
    gen = torch.Generator().manual_seed(sum(sizes))
    draw = lambda s: [(torch.randn(n, generator=gen) * s) for n in sizes]      # noqa: E731
    for step, spread in ((1, 0.0), (50, 0.3)):
        p, g, m = draw(1.0), draw(0.5), draw(spread)
        v = [x.square() * spread for x in draw(0.5)]
        _, want = _adam64(*[[x.double() for x in k] for k in (p, g, m, v)], step, 1e-2, (0.9, 0.999), 1e-8, 0.02, None)
        dev, other, away, kept = ([[x.to(DEV) for x in k] for k in (p, g, m, v)] for _ in range(4))
        assert adam_step_(*dev, step, **how) is None
        assert all(torch.equal(a.cpu(), b) for a, b in zip(dev[1], g))
        for k, (wp, wm, wv, wg, den) in enumerate(want):
            g0 = wg.abs() + (0.02 * p[k].double()).abs() * 2
            em = 8 * U * (m[k].double().abs() + g0)
            ev = 12 * U * wv + 8 * U * 0.001 * g0 * g0
            assert bool(((dev[2][k].cpu().double() - wm).abs() <= em).all())
            assert bool(((dev[3][k].cpu().double() - wv).abs() <= ev).all())
            up = 1e-2 / (1 - 0.9 ** step) * ((em + 16 * U * wm.abs()) / den + wm.abs() / den * ev / (wv + 1e-300))
            assert bool(((dev[0][k].cpu().double() - wp).abs() <= up + 2 * U * wp.abs()).all())
        adam_step_(*other, step, max_norm=math.inf, **how)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            adam_step_(*away, step, **how)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            adam_step_(*kept, step, **how)
        for turn in range(3):
            for a, b in zip(kept, (p, g, m, v)):
                for x, y in zip(a, b):
                    x.copy_(y)
            graph.replay()
            torch.cuda.synchronize()
            for also in (other, away, kept):
                assert all(torch.equal(a, b) for x, y in zip(also, dev) for a, b in zip(x, y)), turn


def test_adam_step_without_a_bound_refuses_shared_memory():
    from curvecloudnet_amd.parallel import adam_step_
    make = lambda n=64: [torch.ones(n, device=DEV)]        # noqa: E731
    p, wide = make(), torch.ones(100, device=DEV)
    for lists in ((p, make(), p, make()), (p, p, make(), make()), (p, make(), make(), p), (p + p, make() + make(), make() + make(), make() + make()),
                  ([wide[:64]], make(), [wide[36:]], make())):
        with pytest.raises(RuntimeError, match="share memory"):
            adam_step_(*lists, 1)
    torch.cuda.synchronize()
    assert bool((p[0] == 1).all()) and bool((wide == 1).all())
    with pytest.raises(ValueError, match="multiple of 16"):
        adam_step_([torch.ones(65, device=DEV)[1:]], make(), make(), make(), 1)
