"""CPU: what loss.token_logprobs, parallel.grad_norm / clip_grad_norm_ / adam_step_ and their C entry points refuse, before anything
is launched."""
import ctypes
import math

import pytest
import torch


def test_token_logprobs_refuses():
    from curvecloudnet_amd.loss import token_logprobs
    x, t = torch.zeros(4, 6), torch.zeros(4, dtype=torch.int64)
    with pytest.raises(TypeError, match="logits are torch.float64"):
        token_logprobs(x.double(), t)
    with pytest.raises(TypeError, match="logits are torch.int64"):
        token_logprobs(x.long(), t)
    for bad in (t.float(), t.bool(), t.to(torch.uint8)):
        with pytest.raises(TypeError, match="target is"):
            token_logprobs(x, bad)
    for shape in ((5,), (4, 1), (), (4, 6)):
        with pytest.raises(ValueError, match="want a target of shape"):
            token_logprobs(x, torch.zeros(shape, dtype=torch.int64))
    for bad in (torch.zeros(4, 0), torch.zeros(())):
        with pytest.raises(ValueError, match="no classes"):
            token_logprobs(bad, t)
    for top in (-1, 7, 65):
        with pytest.raises(ValueError, match="top="):
            token_logprobs(x, t, top=top)
    with pytest.raises(ValueError, match="0 to 64"):
        token_logprobs(torch.zeros(4, 100), t, top=65)
    with pytest.raises(RuntimeError, match="GPU only"):
        token_logprobs(x, t)


def test_the_norm_and_clipping_refuse():
    from curvecloudnet_amd.parallel import FlatAdam, GradientAllReduce, clip_grad_norm_, grad_norm
    p = torch.nn.Parameter(torch.zeros(5))
    p.grad = torch.zeros(5)
    for kind in (0, 3.0, -1, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            grad_norm([p.grad], kind)
        with pytest.raises(ValueError, match="norm_type"):
            clip_grad_norm_(p, 1.0, norm_type=kind)
    for bound in (-1.0, math.nan):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_(p, bound)
        with pytest.raises(ValueError, match="max_norm"):
            FlatAdam(GradientAllReduce(torch.nn.Linear(2, 2)), max_norm=bound)
    with pytest.raises(TypeError, match="float64"):
        grad_norm([p.grad.double()])
    with pytest.raises(TypeError, match="int64"):
        grad_norm([p.grad.long()])
    with pytest.raises(TypeError, match="sparse"):
        grad_norm([p.grad.to_sparse()])
    with pytest.raises(ValueError, match="does not fill its memory"):
        grad_norm([torch.zeros(4, 6)[:, :3]])
    with pytest.raises(RuntimeError, match="GPU only"):
        grad_norm([p.grad])
    with pytest.raises(RuntimeError, match="GPU only"):
        clip_grad_norm_(p, 1.0)


def test_adam_step_refuses():
    from curvecloudnet_amd.parallel import adam_step_
    t = lambda n=8, **k: [torch.zeros(n, **k)]          # noqa: E731
    with pytest.raises(ValueError, match="step 0"):
        adam_step_(t(), t(), t(), t(), 0)
    with pytest.raises(ValueError, match="1 parameters, 2 gradients"):
        adam_step_(t(), t() + t(), t(), t(), 1)
    with pytest.raises(TypeError, match="fp32"):
        adam_step_(t(), t(dtype=torch.bfloat16), t(), t(), 1)
    with pytest.raises(ValueError, match="of one size"):
        adam_step_(t(), t(), t(9), t(), 1)
    with pytest.raises(ValueError, match="contiguous"):
        adam_step_(t(), [torch.zeros(16)[::2]], t(), t(), 1)
    with pytest.raises(ValueError, match="max_norm"):
        adam_step_(t(), t(), t(), t(), 1, max_norm=-2.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        adam_step_(t(), t(), t(), t(), 1, max_norm=1.0)
    assert adam_step_([], [], [], [], 1) is None


def test_c_entries_of_the_scores_refuse():
    from curvecloudnet_amd import _lib
    lib = _lib.lib()
    null, fake = ctypes.c_void_p(None), ctypes.c_void_p(0x1000)     # (never read: the checks come first)
    err = lambda: lib.ccn_last_error().decode()                      # noqa: E731

    def fwd(x=fake, dtype=0, ld=8, t=fake, rows=4, c=8, top=0, lp=fake, h=fake, best=fake, index=fake, ws=fake, n=1 << 40):
        return lib.ccn_logprob_fwd(x, dtype, ld, t, rows, c, -100, top, lp, h, null, best, index, ws, n, null)

    def bwd(x=fake, dtype=0, ld=8, t=fake, rows=4, c=8, top=0, index=fake, stats=fake, h=fake, s1=1, s2=1, gt=fake, d=fake, ldd=8):
        return lib.ccn_logprob_bwd(x, dtype, ld, t, rows, c, -100, top, index, stats, h, fake, s1, fake, s2, gt, d, ldd, null)

    for call, word in ((lambda: fwd(x=null), "null"), (lambda: fwd(t=null), "null"), (lambda: fwd(lp=null), "null"),
                       (lambda: fwd(h=null), "null"), (lambda: fwd(dtype=3), "dtype"), (lambda: fwd(dtype=-1), "dtype"),
                       (lambda: fwd(rows=0), "rows"), (lambda: fwd(rows=1 << 31), "rows"), (lambda: fwd(c=0), "rows"),
                       (lambda: fwd(c=1 << 30, ld=1 << 30), "rows"), (lambda: fwd(ld=7), "ld"), (lambda: fwd(ld=-8), "ld"),
                       (lambda: fwd(top=-1), "top"), (lambda: fwd(top=9), "top"), (lambda: fwd(top=65, c=100, ld=100), "top"),
                       (lambda: fwd(top=2, best=null), "top"), (lambda: fwd(top=2, index=null), "top"),
                       (lambda: bwd(x=null), "null"), (lambda: bwd(stats=null), "null"), (lambda: bwd(d=null), "null"),
                       (lambda: bwd(dtype=7), "dtype"), (lambda: bwd(ldd=7), "ldd"), (lambda: bwd(ld=7), "ld"), (lambda: bwd(rows=-1), "rows"),
                       (lambda: bwd(top=2, gt=null), "top"), (lambda: bwd(top=2, index=null), "top"), (lambda: bwd(top=9), "top"),
                       (lambda: bwd(s1=-1), "stride"), (lambda: bwd(s2=-1), "stride"),
                       (lambda: bwd(stats=ctypes.c_void_p(0x1004)), "stats")):
        assert call() < 0 and word in err(), (word, err())
    sizes = [(r, c, k) for r in (1, 96, 1 << 20) for c in (1, 64, 65, 50021, 262144, (1 << 30) - 1) for k in (0, 64)]
    assert all(0 <= lib.ccn_logprob_workspace_bytes(*s) < 1 << 42 for s in sizes)
    assert lib.ccn_logprob_workspace_bytes(-1, 5, 0) == lib.ccn_logprob_workspace_bytes(5, -1, 0) == 0
    # where a workspace is needed, one that is missing or too small is refused
    for rows, c, k in sizes:
        n = lib.ccn_logprob_workspace_bytes(rows, c, k)
        if n and k <= c:
            assert fwd(rows=rows, c=c, ld=c, top=k, ws=null) < 0 and "workspace" in err()
            assert fwd(rows=rows, c=c, ld=c, top=k, n=n - 1) < 0 and "workspace" in err()


def test_c_entries_of_the_norm_refuse():
    from curvecloudnet_amd import _lib
    lib = _lib.lib()
    null, fake = ctypes.c_void_p(None), ctypes.c_void_p(0x1000)
    err = lambda: lib.ccn_last_error().decode()                      # noqa: E731
    table = lambda *v: (ctypes.c_int64 * len(v))(*v)                 # noqa: E731
    codes = lambda *v: (ctypes.c_int32 * len(v))(*v)                 # noqa: E731
    big = 1 << 40

    def norm(p=(0x1000, 0x8000), s=(4, 4), d=(0, 0), n=2, kind=2, ws=fake, wn=big, out=fake):
        return lib.ccn_grad_norm(p and table(*p), s and table(*s), d and codes(*d), n, kind, ws, wn, out, null)

    def clip(p=(0x1000, 0x8000), s=(4, 4), d=(0, 0), n=2, kind=2, bound=1.0, ws=fake, wn=big, out=fake):
        return lib.ccn_grad_clip(p and table(*p), s and table(*s), d and codes(*d), n, kind, bound, ws, wn, out, null)

    def adam(p=(0x1000,), g=(0x2000,), m=(0x3000,), v=(0x4000,), s=(4,), n=1, step=1, bound=1.0, ws=fake, wn=big, out=fake):
        return lib.ccn_adam_clip(table(*p), table(*g), table(*m), table(*v), s and table(*s), n, 1e-3, 0.9, 0.999, 1e-8, 0.0, step,
                                 bound, ws, wn, out, null)

    for call, word in ((lambda: norm(n=-1), "n=-1"), (lambda: norm(p=None), "null"), (lambda: norm(s=None), "null"),
                       (lambda: norm(d=(0, 3)), "dtype"), (lambda: norm(s=(4, -1)), "values"), (lambda: norm(s=(4, 1 << 36)), "values"),
                       (lambda: norm(p=(0x1000, 0)), "null"), (lambda: norm(p=(0x1000, 0x8002)), "aligned"),
                       (lambda: norm(p=(0x1000, 0x8001), d=(0, 1)), "aligned"), (lambda: norm(kind=0), "kind"),
                       (lambda: norm(kind=4), "kind"), (lambda: norm(out=null), "null"), (lambda: norm(ws=null), "null"),
                       (lambda: norm(wn=8), "workspace"), (lambda: clip(kind=5), "kind"), (lambda: clip(bound=-1.0), "max_norm"),
                       (lambda: clip(bound=math.nan), "max_norm"), (lambda: clip(wn=8), "workspace"), (lambda: clip(out=null), "null"),
                       (lambda: clip(p=(0x1000, 0x1000)), "share"), (lambda: clip(p=(0x100c, 0x1000)), "share"),
                       (lambda: clip(p=(0x1000, 0x100c)), "share"), (lambda: clip(p=(0x1006, 0x1000), d=(1, 1)), "share"),
                       (lambda: adam(step=0), "step"), (lambda: adam(n=-2), "n=-2"), (lambda: adam(s=None), "null"),
                       (lambda: adam(bound=-0.5), "max_norm"), (lambda: adam(p=(0x1008,)), "16-byte"),
                       (lambda: adam(m=(0x1000,)), "share"), (lambda: adam(v=(0x2000,)), "share"), (lambda: adam(g=(0x1000,)), "share"),
                       (lambda: adam(p=(0,)), "null"), (lambda: adam(wn=8), "workspace"), (lambda: adam(out=null), "null")):
        assert call() < 0 and word in err(), (word, err())
    sizes = [lib.ccn_grad_norm_workspace_bytes(n) for n in (0, 1, 160, 161, 320, 321, 1000, 1 << 20)]
    assert sizes == sorted(sizes) and 0 < sizes[0] and sizes[-1] < 1 << 30 and lib.ccn_grad_norm_workspace_bytes(-1) == 0


def test_lists_of_other_things_are_refused():
    from curvecloudnet_amd.parallel import clip_grad_norm_, grad_norm
    for bad in (1.0, None, "weight", [torch.zeros(3)]):
        with pytest.raises(TypeError, match="is no tensor"):
            grad_norm([bad])
        with pytest.raises(TypeError, match="is no tensor"):
            clip_grad_norm_([torch.nn.Parameter(torch.zeros(3)), bad], 1.0)


def test_the_update_without_a_bound_refuses_from_c():
    """Neither norm nor workspace, and an infinite bound: everything else is looked at all the same.  One of the two alone is refused."""
    from curvecloudnet_amd import _lib
    lib = _lib.lib()
    null, fake = ctypes.c_void_p(None), ctypes.c_void_p(0x10000)
    err = lambda: lib.ccn_last_error().decode()                      # noqa: E731
    table = lambda *v: (ctypes.c_int64 * len(v))(*v)                 # noqa: E731

    def adam(p=(0x1000,), g=(0x2000,), m=(0x3000,), v=(0x4000,), s=(4,), step=1, bound=math.inf, ws=null, wn=0, out=null):
        return lib.ccn_adam_clip(table(*p), table(*g), table(*m), table(*v), table(*s), len(s), 1e-3, 0.9, 0.999, 1e-8, 0.0, step, bound,
                                 ws, wn, out, null)

    for call, word in ((lambda: adam(m=(0x1000,)), "share"), (lambda: adam(p=(0x2000,)), "share"), (lambda: adam(v=(0x3000,)), "share"),
                       (lambda: adam(p=(0x1000, 0x1010), g=(0x2000, 0x2100), m=(0x3000, 0x3100), v=(0x4000, 0x4100), s=(8, 4)), "share"),
                       (lambda: adam(p=(0x1008,)), "16-byte"), (lambda: adam(p=(0,)), "null"), (lambda: adam(s=(-1,)), "values"),
                       (lambda: adam(step=0), "step"), (lambda: adam(bound=1.0), "null"), (lambda: adam(bound=math.nan), "max_norm"),
                       (lambda: adam(out=fake), "null"), (lambda: adam(ws=fake, wn=1 << 20), "null"),
                       (lambda: adam(out=fake, ws=fake, wn=8), "workspace")):
        assert call() < 0 and word in err(), (word, err())
