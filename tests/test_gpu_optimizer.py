"""Gradient norm, clipping and the AdamW step on the HIP kernels against the formulas in 64 bits.

Tolerances count roundings; u = 2^-24 is half a step of fp32, h that of the tensor's type (bf16 2^-8, fp16 2^-11).

norm        summed in 64 bits and rounded once: u, and 2^-40 for the sum itself.
clip        coefficient u, product u, rounding to the type h; below the type's normal range half its smallest step.
m           b1, 1 - b1, the coefficient and its product with g, two products and the sum: less than 5 u (b1 |m| + r1 |g'|).
v           the same with g' twice: less than 9 u (b2 v + r2 g'^2).
w           the ratio m / c1 / (sqrt(v) / sqrt(c2) + eps): 5 u from m, 4.5 u from sqrt(v), c1 and sqrt(c2) with the
            functions' own errors of two steps 5 u and 4 u, four more operations 4 u: below 24 u of lr U with
            U = (b1 |m| + r1 |g'|) / c1 / denominator; the decay term 4 u lr wd |w|; the last subtraction u |w|.
"""
import ctypes
import gc
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -150, torch.bfloat16: 2.0 ** -134, torch.float16: 2.0 ** -25}
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
NORMS = [1.0, 2.0, math.inf]
SIZES = {
    'one': [1],
    'zero': [0],
    'empty': [],
    'short': [3, 0, 1, 5, 2],
    'chunk': [1023, 1024, 1025, 255, 256, 257],
    'network': [256 * 60, 256, 65536, 256, 256 * 316, 256, 256, 1, 128 * 283, 128, 3 * 128, 3],
    'many': [(7 * i) % 61 for i in range(300)],
    'tables': [4097] * 129 + [2] * 64,
    'long': [3_000_017, 5, 70_001, 2_097_152 + 1],
}


def gen(seed=0):
    return torch.Generator(device='cuda').manual_seed(seed)


def make(sizes, dtype, offset=0, seed=0, scale=0.01):
    """Tensors of these sizes, each `offset` elements into an allocation of its own (`dtype` a list: in turn)."""
    g = gen(seed)
    dts = dtype if isinstance(dtype, list) else [dtype]
    out = []
    for i, n in enumerate(sizes):
        buf = torch.full((n + offset + 8,), 77.0, device='cuda', dtype=dts[i % len(dts)])
        buf[offset:offset + n] = (scale * (1 + i % 5)) * torch.randn(n, device='cuda', generator=g)
        out.append(buf[offset:offset + n])
    return out


def norm64(ts, p):
    if not sum(t.numel() for t in ts):
        return 0.0
    x = torch.cat([t.detach().reshape(-1).double() for t in ts])
    return float(x.abs().max() if p == math.inf else x.abs().sum() if p == 1.0 else (x * x).sum().sqrt())


def near_norm(got, want):
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    assert abs(float(got) - want) <= want * (U + 2.0 ** -40), (float(got), want)


def edges_kept(ts, offset):
    """The elements around each view, as they were made."""
    for t in ts:
        base = t._base
        assert bool((base[:offset] == 77).all()) and bool((base[offset + t.numel():] == 77).all())


@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', SIZES)
def test_norm(sizes, dtype, norm_type):
    from nerf_amd import ops
    ts = make(SIZES[sizes], dtype)
    near_norm(ops.grad_norm(ts, norm_type), norm64(ts, norm_type))


@pytest.mark.parametrize('offset', [1, 2, 3, 5, 7])
@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_and_clip_at_any_offset(dtype, offset):
    from nerf_amd import ops
    ts = make(SIZES['chunk'] + [30_011], dtype, offset)
    was = [t.double() for t in ts]
    near_norm(ops.grad_norm(ts), norm64(ts, 2.0))
    n = ops.clip_grad_norm_(ts, 0.25)
    check_clipped(ts, was, 0.25, 2.0, n)
    edges_kept(ts, offset)


def check_clipped(ts, was, max_norm, norm_type, got):
    want = norm64(was, norm_type)
    near_norm(got, want)
    c = min(1.0, max_norm / (want + 1e-6))
    for t, w in zip(ts, was):
        w = w * c
        tol = w.abs() * (2 * U + HALF_STEP[t.dtype]) * (1 + U) + TINY[t.dtype]
        assert bool(((t.double() - w).abs() <= tol).all())


@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES + [DTYPES])
@pytest.mark.parametrize('sizes', SIZES)
def test_clip(sizes, dtype, norm_type):
    from nerf_amd import ops
    ts = make(SIZES[sizes], dtype, seed=1)
    was = [t.double() for t in ts]
    half = 0.5 * norm64(ts, norm_type)
    check_clipped(ts, was, half, norm_type, ops.clip_grad_norm_(ts, half, norm_type))


@pytest.mark.parametrize('dtype', DTYPES)
def test_clip_above_the_norm_keeps_the_bits(dtype):
    from nerf_amd import ops
    ts = make(SIZES['network'], dtype)
    was = [t.clone() for t in ts]
    for most in (2 * norm64(ts, 2.0), math.inf):
        ops.clip_grad_norm_(ts, most)
        assert all(torch.equal(a, b) for a, b in zip(ts, was))
    ops.clip_grad_norm_(ts, 0.0)
    assert all(not t.any() for t in ts)


@pytest.mark.parametrize('scale', [1e-30, 1e-20, 1e18, 1e25, 3e36])
def test_norm_without_overflow_of_the_squares(scale):
    from nerf_amd import ops
    t = make([5001], torch.float32, scale=1.0)[0] * scale
    near_norm(ops.grad_norm(t), norm64([t], 2.0))
    n = ops.clip_grad_norm_(t, 1.0)
    assert float(n) > 0 and norm64([t], 2.0) <= 1.0 + 1e-6


def test_norm_beyond_the_largest_float():
    from nerf_amd import ops
    t = torch.full((100,), 3e38, device='cuda')
    assert float(ops.grad_norm(t)) == math.inf
    assert float(ops.grad_norm(t, math.inf)) == float(torch.tensor(3e38))


@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('bad', [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize('at', [0, 2500, 5000])
def test_values_that_are_not_finite(bad, at, dtype, norm_type):
    from nerf_amd import ops, optim
    ts = make([700, 5001, 3], dtype)
    ts[1][at] = bad
    same = lambda x: math.isnan(x) if math.isnan(bad) else x == math.inf       # noqa: E731
    assert same(float(ops.grad_norm(ts, norm_type)))
    ps = [torch.nn.Parameter(torch.zeros_like(t)) for t in ts]
    for p, t in zip(ps, ts):
        p.grad = t.clone()
    with pytest.raises(RuntimeError, match='not finite'):
        optim.clip_grad_norm_(ps, 1.0, norm_type, error_if_nonfinite=True)
    assert all(torch.equal(p.grad, t) or math.isnan(bad) for p, t in zip(ps, ts))
    assert same(float(ops.clip_grad_norm_(ts, 1.0, norm_type)))
    if math.isnan(bad):
        assert all(bool(t.isnan().all()) for t in ts)
    else:
        keep = torch.arange(5001, device='cuda') != at
        assert not ts[0].any() and not ts[1][keep].any() and bool(ts[1][at].isnan())


def test_a_nan_wins_over_what_comes_after():
    from nerf_amd import ops
    t = torch.rand(9000, device='cuda')
    t[3], t[4000], t[8999] = math.nan, math.inf, 1e30
    for p in NORMS:
        assert math.isnan(float(ops.grad_norm(t, p)))


def test_orders_of_dimensions():
    from nerf_amd import ops
    x = torch.randn(40, 30, 20, device='cuda', generator=gen())
    for t in (x.transpose(0, 2), x[:, 3:9], x[::3], x[0, 0].expand(7, 20), x[5].t()):
        near_norm(ops.grad_norm([t, x]), norm64([t, x], 2.0))
    t = x.clone().permute(2, 0, 1)
    was = t.double()
    n = ops.clip_grad_norm_([t], 0.5)
    check_clipped([t], [was], 0.5, 2.0, n)
    near_norm(ops.grad_norm([x, x]), norm64([x, x], 2.0))        # a tensor may be listed twice where it is only read
    for call in (lambda: ops.clip_grad_norm_([x, x], 1.0), lambda: ops.clip_grad_norm_([x[0], x], 1.0)):
        with pytest.raises(RuntimeError, match='invalid argument'):
            call()


def test_refusals_on_the_device():
    from nerf_amd import ops, optim
    x = torch.ones(4, device='cuda')
    for bad in (torch.ones(4, device='cuda', dtype=torch.float64), torch.ones(4, device='cuda', dtype=torch.int32)):
        with pytest.raises(RuntimeError, match='float32, bfloat16 or float16'):
            ops.grad_norm([x, bad])
    with pytest.raises(RuntimeError, match='one HIP device'):
        ops.grad_norm([x, torch.ones(4)])
    p = torch.nn.Parameter(x.clone())
    p.grad = torch.ones(4, device='cuda')
    opt = optim.AdamW([p], lr=torch.tensor([1.0, 2.0], device='cuda'))
    with pytest.raises(ValueError, match='one element'):
        opt.step()
    opt = optim.AdamW([p], lr=torch.tensor(1.0, device='cuda', dtype=torch.float64))
    with pytest.raises(ValueError, match='fp32'):
        opt.step()
    opt = optim.AdamW([p])
    opt.state[p] = dict(step=torch.zeros(()), exp_avg=torch.zeros_like(p), exp_avg_sq=torch.zeros_like(p))
    with pytest.raises(RuntimeError, match='step'):
        opt.step()
    opt.state[p] = dict(step=torch.zeros((), device='cuda'), exp_avg=torch.zeros(4), exp_avg_sq=torch.zeros_like(p))
    with pytest.raises(RuntimeError, match='shape, order and device'):
        opt.step()
    opt.state[p] = dict(step=torch.zeros((), device='cuda'), exp_avg=torch.zeros_like(p))
    with pytest.raises(RuntimeError, match='exp_avg_sq'):
        opt.step()
    opt.state[p] = dict(step=torch.zeros((), device='cuda', dtype=torch.bfloat16), exp_avg=torch.zeros_like(p),
                        exp_avg_sq=torch.zeros_like(p))
    with pytest.raises(RuntimeError, match='step'):
        opt.step()
    for t in (torch.zeros(4, 6, device='cuda')[:, :3], torch.zeros(1, 3, device='cuda').expand(4, 3)):
        with pytest.raises(RuntimeError, match='dense'):
            ops.clip_grad_norm_([x, t], 1.0)
    q = torch.nn.Parameter(torch.zeros(4, 6, device='cuda')[:, :3])
    q.grad = torch.zeros_like(q)
    with pytest.raises(RuntimeError, match='dense'):
        optim.AdamW([q]).step()
    assert torch.equal(p.detach(), x)


def test_writes_are_seen_by_autograd():
    from nerf_amd import ops, optim
    g = torch.ones(8, device='cuda')
    before = g._version
    ops.clip_grad_norm_(g, 1.0)
    assert g._version > before
    p = torch.nn.Parameter(torch.ones(8, device='cuda'))
    y = (p * p).sum()
    p.grad = torch.ones(8, device='cuda')
    optim.AdamW([p]).step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        y.backward()


# ---- AdamW ------------------------------------------------------------------------------------------------------

B1, B2, EPS, WD, LR = 0.9, 0.999, 1e-8, 0.02, 3e-3


def make_state(ps, t, seed=5):
    g = gen(seed)
    out = []
    for i, p in enumerate(ps):
        m = 0.01 * torch.randn(p.shape, device='cuda', generator=g)
        v = 1e-4 * torch.rand(p.shape, device='cuda', generator=g) ** 2
        if t == 0:
            m.zero_(), v.zero_()
        out.append(dict(step=torch.tensor(float(t), device='cuda'), exp_avg=m, exp_avg_sq=v))
    return out


def params_of(sizes, dtype, offset=0, seed=0):
    ps = [torch.nn.Parameter(x) for x in make(sizes, dtype, offset, seed, scale=0.3)]
    for p, g in zip(ps, make(sizes, dtype, offset, seed + 1)):
        p.grad = g
    return ps


def one_step64(w, g, m, v, t, c, lr=LR, b1=B1, b2=B2, eps=EPS, wd=WD):
    """New (w, m, v) and their tolerances, in 64 bits."""
    w, g, m, v = (x.double() for x in (w, g, m, v))
    g = g * c
    size = b1 * m.abs() + (1 - b1) * g.abs()
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    denom = (v1 / (1 - b2 ** t)).sqrt() + eps
    w1 = w - lr * (m1 / (1 - b1 ** t) / denom + wd * w)
    tol_w = U * (w1.abs() + lr * (24 * size / (1 - b1 ** t) / denom + 4 * wd * w.abs())) + 2.0 ** -149
    return (w1, m1, v1), (tol_w, 5 * U * size + 2.0 ** -149, 9 * U * v1 + 2.0 ** -148)


def check_step(ps, was, states, t, c, **kw):
    """`was`: (weight the step starts from, gradient, m, v) of each parameter ahead of the step."""
    for p, (w, g, m, v), st in zip(ps, was, states):
        want, tol = one_step64(w, g, m, v, t, c, **kw)
        got = (st['master'] if p.dtype != torch.float32 else p, st['exp_avg'], st['exp_avg_sq'])
        for x, y, e in zip(got, want, tol):
            assert x.dtype == torch.float32
            off = (x.detach().double() - y).abs() - e
            assert bool((off <= 0).all()), float(off.max())
        if p.dtype != torch.float32:
            assert torch.equal(p.detach(), st['master'].to(p.dtype))
        assert float(st['step']) == t


def snapshot(ps, states):
    return [(st['master'].clone() if 'master' in st else p.detach().clone(), p.grad.clone(), st['exp_avg'].clone(),
             st['exp_avg_sq'].clone()) for p, st in zip(ps, states)]


def optimizer(ps, states, **kw):
    from nerf_amd import optim
    kw = dict(dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD), **kw)
    opt = optim.AdamW(ps, **kw)
    for p, st in zip(ps, states):
        opt.state[p] = st
    return opt


@pytest.mark.parametrize('clip', [None, 1.0, 2.0, math.inf])
@pytest.mark.parametrize('dtype', DTYPES + [DTYPES])
@pytest.mark.parametrize('sizes', [k for k in SIZES if k != 'empty'])
def test_adamw_step(sizes, dtype, clip):
    ps = params_of(SIZES[sizes], dtype)
    states = make_state(ps, 10)
    was = snapshot(ps, states)
    grads = [p.grad for p in ps]
    n = norm64(grads, clip) if clip else None
    max_norm = 0.4 * n if clip else None
    opt = optimizer(ps, states, max_norm=max_norm, norm_type=clip or 2.0)
    opt.step()
    if clip:
        near_norm(opt.grad_norm, n)
    else:
        assert opt.grad_norm is None
    check_step(ps, was, states, 11, min(1.0, max_norm / (n + 1e-6)) if clip else 1.0)
    assert all(torch.equal(p.grad, w[1]) for p, w in zip(ps, was))      # gradients are only read


@pytest.mark.parametrize('offset', [1, 2, 3, 6])
@pytest.mark.parametrize('dtype', DTYPES)
def test_adamw_at_any_offset(dtype, offset):
    ps = params_of(SIZES['chunk'] + [20_003], dtype, offset)
    states = make_state(ps, 3)
    was = snapshot(ps, states)
    views = [p.data for p in ps]
    optimizer(ps, states).step()
    check_step(ps, was, states, 4, 1.0)
    for v, n in zip(views, SIZES['chunk'] + [20_003]):
        whole = torch.as_strided(v, (n + offset + 8,), (1,), 0)
        assert bool((whole[:offset] == 77).all()) and bool((whole[offset + n:] == 77).all())


@pytest.mark.parametrize('t', [0, 1, 999, 100_000, 5_000_000])
@pytest.mark.parametrize('betas', [(0.9, 0.999), (0.0, 0.0), (0.99, 0.9999), (0.5, 0.0)])
def test_adamw_bias_corrections(betas, t):
    ps = params_of([3000, 17], torch.float32)
    states = make_state(ps, t)
    was = snapshot(ps, states)
    optimizer(ps, states, betas=betas).step()
    check_step(ps, was, states, t + 1, 1.0, b1=betas[0], b2=betas[1])


def test_adamw_moments_from_zero():
    """Entries whose gradient and moments are zero move by the decay alone."""
    ps = params_of([5000], torch.float32)
    ps[0].grad[::2] = 0
    states = make_state(ps, 0)
    was = snapshot(ps, states)
    optimizer(ps, states).step()
    check_step(ps, was, states, 1, 1.0)
    assert not states[0]['exp_avg'][::2].any()


@pytest.mark.parametrize('bad', [math.nan, math.inf])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('max_norm', [None, 1.0])
def test_skipped_steps(dtype, bad, max_norm):
    ps = params_of(SIZES['network'], dtype)
    states = make_state(ps, 7)
    opt = optimizer(ps, states, skip_nonfinite=True, max_norm=max_norm)
    opt.step()                                  # (finite: taken; masters exist from here on)
    was = snapshot(ps, states) + [[p.detach().clone() for p in ps]]
    keep = ps[4].grad[99].clone()
    ps[4].grad[99] = bad
    opt.step()
    assert not math.isfinite(float(opt.grad_norm))
    now = snapshot(ps, states) + [[p.detach().clone() for p in ps]]
    for i, (a, b) in enumerate(zip(was, now)):
        assert all(torch.equal(x, y) for k, (x, y) in enumerate(zip(a, b)) if not (i == 4 and k == 1))
    assert all(float(st['step']) == 8 for st in states)
    ps[4].grad[99] = keep
    opt.step()
    assert math.isfinite(float(opt.grad_norm)) and all(float(st['step']) == 9 for st in states)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_masters_keep_small_updates_and_follow_writes(dtype):
    from nerf_amd import optim
    p = torch.nn.Parameter(torch.ones(4000, device='cuda', dtype=dtype))
    opt = optim.AdamW([p], lr=2.0 ** -14, weight_decay=0.0)
    for _ in range(40):             # each update is far below a step of the type at 1
        p.grad = torch.ones_like(p)
        opt.step()
    master = opt.state[p]['master']
    assert torch.allclose(master, torch.full_like(master, 1 - 40 * 2.0 ** -14), rtol=0, atol=1e-5)
    assert torch.equal(p.detach(), master.to(dtype)) and float(p.detach()[0]) < 1
    with torch.no_grad():
        p[::2] = 3.0                # written from outside: these start over from the parameter
    kept = master.clone()
    p.grad = torch.zeros_like(p)
    opt.state[p]['exp_avg'].zero_()
    opt.step()
    assert bool((master[::2] == 3.0).all()) and torch.equal(master[1::2], kept[1::2])


def test_groups_and_missing_gradients():
    ps = params_of([1000, 2000, 3000, 40, 500], torch.float32)
    states = make_state(ps, 4)
    ps[1].grad = None
    lr = torch.tensor(0.02, device='cuda')
    groups = [dict(params=ps[:2]), dict(params=[ps[2]], lr=lr, betas=(0.8, 0.95), eps=1e-3, weight_decay=0.3),
              dict(params=ps[3:], lr=torch.tensor(0.5))]
    was = [x if p.grad is not None else None for p, x in
           zip(ps, [None if p.grad is None else snapshot([p], [st])[0] for p, st in zip(ps, states)])]
    n = norm64([p.grad for p in ps if p.grad is not None], 2.0)
    second = ps[1].detach().clone()
    opt = optimizer(groups, [], max_norm=0.5 * n)
    for p, st in zip(ps, states):
        opt.state[p] = st
    opt.step()
    c = 0.5 * n / (n + 1e-6)
    check_step(ps[:1], was[:1], states[:1], 5, c)
    check_step(ps[2:3], was[2:3], states[2:3], 5, c, lr=float(lr), b1=0.8, b2=0.95, eps=1e-3, wd=0.3)
    check_step(ps[3:], was[3:], states[3:], 5, c, lr=0.5)
    assert torch.equal(ps[1].detach(), second) and float(states[1]['step']) == 4
    for p in ps:
        p.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0 and float(states[0]['step']) == 5


def test_orders_of_parameters_and_gradients():
    """Transposed parameters, gradients in the other order, and one-row shapes whose strides differ."""
    g = gen(3)
    base = torch.randn(30, 50, device='cuda', generator=g)
    a = torch.nn.Parameter(base.t())
    a.grad = torch.randn(50, 30, device='cuda', generator=g)                # contiguous; the parameter is not
    b = torch.nn.Parameter(torch.randn(50, 30, device='cuda', generator=g))
    b.grad = torch.randn(30, 50, device='cuda', generator=g).t()
    c = torch.nn.Parameter(torch.randn(1, 64, device='cuda', generator=g))
    c.grad = torch.randn(64, 1, device='cuda', generator=g).t()
    d = torch.nn.Parameter(torch.randn(40, device='cuda', generator=g).as_strided((3, 1, 4), (1, 7, 3)))
    d.grad = torch.randn(3, 1, 4, device='cuda', generator=g)
    ps = [a, b, c, d]
    from nerf_amd import optim
    opt = optim.AdamW(ps, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)
    was = [(p.detach().clone(), p.grad.clone(), torch.zeros_like(p), torch.zeros_like(p)) for p in ps]
    opt.step()
    check_step(ps, was, [opt.state[p] for p in ps], 1, 1.0)


def test_steps_against_the_other_optimizer_in_64_bits():
    """Ten steps with changing gradients, saved and loaded half way, against torch's AdamW and clipping in 64 bits.
    Each step adds at most the one-step bounds above; ten of them with moments of like size stay below ten times
    that, and 1e-6 of lr per step (the moments' own errors, 9 u, seen through later steps) is above it."""
    from nerf_amd import optim
    g = gen(11)
    shapes = [(64, 33), (64,), (1, 64), (7, 5, 3)]
    ps = [torch.nn.Parameter(torch.randn(s, device='cuda', generator=g)) for s in shapes]
    qs = [torch.nn.Parameter(p.detach().double().cpu()) for p in ps]
    kw = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
    mine, other = optim.AdamW(ps, max_norm=1.0, **kw), torch.optim.AdamW(qs, **kw)
    for k in range(10):
        for p, q in zip(ps, qs):
            p.grad = torch.randn(p.shape, device='cuda', generator=g) * (1 + k % 3)
            q.grad = p.grad.double().cpu()
        if k == 5:
            saved = mine.state_dict()
            mine = optim.AdamW(ps, lr=7.0, max_norm=1.0)
            mine.load_state_dict(saved)
        want = torch.nn.utils.clip_grad_norm_(qs, 1.0)
        other.step()
        mine.step()
        near_norm(mine.grad_norm, float(want))
    for p, q in zip(ps, qs):
        assert float((p.detach().double().cpu() - q.detach()).abs().max()) <= 10 * (U * 5.0 + 1e-6 * 1e-2)


# ---- streams, graphs, memory -------------------------------------------------------------------------------------

def test_another_stream_and_the_same_bits():
    from nerf_amd import ops
    ts = make(SIZES['long'], torch.bfloat16)
    want = ops.grad_norm(ts)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [ops.grad_norm(ts) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, want) for x in got)


def test_two_threads_at_once():
    """Two threads on streams of their own, each clipping its gradients and stepping its optimizer, against the same calls
    one after another."""
    import threading

    from nerf_amd import ops, optim

    def calls(seed, out):
        ps = params_of(SIZES['network'], torch.float32, seed=seed)
        opt = optim.AdamW(ps, lr=LR, max_norm=0.3)
        norms = []
        for _ in range(40):
            norms.append(ops.clip_grad_norm_([p.grad for p in ps], 2.0 - 0.02 * len(norms)))
            opt.step()
            norms.append(opt.grad_norm)
        out[seed] = ([float(n) for n in norms], [p.detach().clone() for p in ps])

    def on_stream(seed, out):
        with torch.cuda.stream(torch.cuda.Stream()):
            calls(seed, out)
            torch.cuda.current_stream().synchronize()
    want, got = {}, {}
    for seed in (20, 30):
        calls(seed, want)
    torch.cuda.synchronize()
    threads = [threading.Thread(target=on_stream, args=(seed, got)) for seed in (20, 30)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for seed in (20, 30):
        assert got[seed][0] == want[seed][0]
        assert all(torch.equal(a, b) for a, b in zip(got[seed][1], want[seed][1]))


def test_captured_steps_count_on():
    """Two graphs of one optimizer, replayed in turn with eager work between, against the same steps taken eagerly."""
    from nerf_amd import optim

    def build():
        ps = params_of(SIZES['network'], torch.float32)
        lr = torch.tensor(LR, device='cuda')
        return ps, lr, optim.AdamW(ps, lr=lr, weight_decay=WD, max_norm=0.5)
    ps, lr, opt = build()
    qs, lq, eager = build()
    fresh = build()
    with pytest.raises(RuntimeError, match='ahead of a graph capture'):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            fresh[2].step()
    opt.step()
    eager.step()
    graphs, norms = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        graphs.append(graph)
        norms.append(opt.grad_norm)
    for k in range(8):
        for p, q in zip(ps, qs):
            p.grad.copy_(torch.randn(p.shape, device='cuda', generator=gen(100 + k)) * 0.1)
            q.grad.copy_(p.grad)
        lr.fill_(LR / (k + 1))
        lq.fill_(LR / (k + 1))
        graphs[k % 2].replay()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(norms[k % 2], eager.grad_norm)
        for p, q in zip(ps, qs):
            assert torch.equal(p.detach(), q.detach())
            assert torch.equal(opt.state[p]['exp_avg_sq'], eager.state[q]['exp_avg_sq'])
    assert float(opt.state[ps[0]]['step']) == 9


def test_captured_clip():
    from nerf_amd import ops
    ts = make(SIZES['network'], [torch.float32, torch.bfloat16])
    raw = [t.clone() for t in ts]
    ops.clip_grad_norm_([t.clone() for t in ts], 0.5)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = ops.clip_grad_norm_(ts, 0.5)
    for k in range(4):
        for t, r in zip(ts, raw):
            t.copy_(r * (k + 1))
        was = [t.double() for t in ts]
        graph.replay()
        torch.cuda.synchronize()
        check_clipped(ts, was, 0.5, 2.0, norm)


def test_the_c_entries_allocate_nothing_and_need_no_stream():
    from nerf_amd import _lib
    t = make([100_001], torch.float32)[0]
    L = _lib.lib()
    args = _lib.lists().describe([t])[1:4]
    n = L.nerf_grad_workspace_bytes(1)
    ws, norm = torch.empty(n, dtype=torch.uint8, device='cuda'), torch.empty((), device='cuda')
    torch.cuda.synchronize()
    assert L.nerf_grad_norm(*args, 1, 2, ws.data_ptr(), n, norm.data_ptr(), ctypes.c_void_p(None)) == 0
    torch.cuda.synchronize()
    near_norm(norm, norm64([t], 2.0))


def test_more_than_2_to_the_31_elements():
    from nerf_amd import ops, optim
    n = 2 ** 31 + 5
    g = torch.zeros(n, device='cuda', dtype=torch.bfloat16)
    g[0], g[2 ** 31 - 1], g[2 ** 31], g[n - 1] = 4.0, 12.0, -84.0, 3.0      # squares: 16 + 144 + 7056 + 9 = 85^2
    near_norm(ops.grad_norm(g), 85.0)
    p = torch.nn.Parameter(torch.zeros(n, device='cuda', dtype=torch.bfloat16))
    p.grad = g
    opt = optim.AdamW([p], lr=0.5, weight_decay=0.0, max_norm=17.0)
    opt.step()
    near_norm(opt.grad_norm, 85.0)
    at = torch.tensor([0, 2 ** 31 - 1, 2 ** 31, n - 1], device='cuda')
    # the first step moves an entry by lr against the sign of its gradient; eps is 1e-8 of the gradient
    assert torch.equal(p.detach()[at], torch.tensor([-0.5, -0.5, 0.5, -0.5], device='cuda', dtype=torch.bfloat16))
    assert int((p.detach() != 0).sum()) == 4
    del p, opt
    ops.clip_grad_norm_(g, 17.0)
    # 17 / 85.000001 of 4, 12, -84, 3, to 8 bits
    want = torch.tensor([0.8, 2.4, -16.8, 0.6], dtype=torch.float64, device='cuda')
    assert bool(((g[at].double() - want).abs() <= want.abs() * (2.0 ** -8 + 2.0 ** -22)).all())
    assert int((g != 0).sum()) == 4
    del g
    gc.collect()
    torch.cuda.empty_cache()


def test_custom_ops():
    import nerf_amd.torch_ops  # noqa: F401
    K = torch.ops.nerf_amd
    for sizes in ('network', 'short'):
        ts = make(SIZES[sizes], torch.float32)
        near_norm(K.grad_norm(ts, 1.0), norm64(ts, 1.0))
        was = [t.double() for t in ts]
        check_clipped(ts, was, 0.1, 2.0, K.clip_grad_norm_(ts, 0.1, 2.0))
    ts = make([33, 1000], torch.bfloat16)
    torch.library.opcheck(K.grad_norm.default, (ts, 2.0), test_utils=('test_schema', 'test_faketensor'))
    torch.library.opcheck(K.clip_grad_norm_.default, (ts, 1.0, 2.0), test_utils=('test_schema', 'test_faketensor'))

    def scaled(ts):
        n = K.clip_grad_norm_(ts, 0.5, 2.0)
        return [t * 2 for t in ts], n + K.grad_norm(ts, math.inf)
    a = make(SIZES['network'], torch.float32)
    b = [t.clone() for t in a]
    ys, n = torch.compile(scaled, fullgraph=True, backend='aot_eager')(a)
    zs, m = scaled(b)
    assert torch.equal(n, m) and all(torch.equal(y, z) for y, z in zip(ys, zs))
    assert all(torch.equal(x, y) for x, y in zip(a, b))
