"""Corners of the gradient norm, clipping and the AdamW step that need a device: coefficients below fp32's normal range,
the norm that an optimizer shows, empty lists at the C entry, inference mode, refused gradients, state at odd places,
lists past the caches, long lists, layouts under capture, the way to torch's optimizer and back.  Tolerances as counted in
test_gpu_optimizer."""
import ctypes
import math

import pytest
import torch

from tests.test_gpu_optimizer import (B1, B2, DTYPES, EPS, HALF_STEP, LR, NORMS, SIZES, TINY, U, WD, check_clipped, check_step,
                                      gen, make, make_state, near_norm, norm64, one_step64, optimizer, params_of, snapshot)

pytestmark = pytest.mark.gpu


# ---- coefficients below the normal range of fp32 ------------------------------------------------------------------

def huge(dtype, n=4099):
    """Entries of the size of the type's largest; their norm is beyond fp32 (but for fp16)."""
    x = torch.rand(n, device='cuda', generator=gen(9)) * 0.5 + 0.5
    x[::3] *= -1
    return (x.double() * 0.99 * torch.finfo(dtype).max).to(dtype)


# the coefficient itself: normal, on both sides of 2^-126, subnormal, below the smallest subnormal, and far below
COEFFICIENTS = [2.0 ** -100, 2.0 ** -126 * (1 + 2.0 ** -10), 2.0 ** -126 * (1 - 2.0 ** -10), 2.0 ** -133, 1.1e-43, 2.0 ** -151,
                3e-48, 1e-60, 1e-200]


@pytest.mark.parametrize('coefficient', COEFFICIENTS)
@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_clip_by_a_coefficient_below_the_normal_range(dtype, norm_type, coefficient):
    from nerf_amd import ops
    t = huge(dtype)
    was, norm = t.double(), norm64([t], norm_type)
    got = ops.clip_grad_norm_(t, coefficient * norm, norm_type)
    assert float(got) == float(torch.tensor(norm, dtype=torch.float64).float())
    want = was * (coefficient * norm / (norm + 1e-6))
    # the coefficient, the product, the rounding to the type; below the normal ranges half a smallest step of both types
    tol = want.abs() * (2 * U + HALF_STEP[dtype]) * (1 + U) + TINY[dtype] + 2.0 ** -150
    off = (t.double() - want).abs() - tol
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize('coefficient', COEFFICIENTS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_adamw_with_a_coefficient_below_the_normal_range(dtype, coefficient):
    p = torch.nn.Parameter(make([4099], dtype, scale=0.3)[0].clone())
    p.grad = huge(dtype)
    norm = norm64([p.grad], 2.0)
    states = make_state([p], 0)             # (moments of zero: what the gradient adds is all there is)
    was = snapshot([p], states)
    opt = optimizer([p], states, max_norm=coefficient * norm)
    opt.step()
    check_step([p], was, states, 1, coefficient * norm / (norm + 1e-6))


# ---- the norm that an optimizer shows -----------------------------------------------------------------------------

def test_grad_norm_after_eager_and_captured_steps():
    """Whatever ran last, an eager step or a replay of either graph: grad_norm is its norm."""
    from nerf_amd import optim
    ps = params_of(SIZES['network'], torch.float32)
    opt = optim.AdamW(ps, lr=1e-4, max_norm=0.5)
    kept = []
    for k in range(2):
        ps[0].grad.mul_(1.5)
        opt.step()
        kept.append((opt.grad_norm, norm64([p.grad for p in ps], 2.0)))
    graphs = []
    for _ in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            opt.step()
    for k, run in enumerate((graphs[0].replay, opt.step, graphs[0].replay, graphs[1].replay, graphs[0].replay, opt.step, opt.step,
                             graphs[1].replay)):
        for p in ps:
            p.grad.copy_(torch.randn(p.shape, device='cuda', generator=gen(50 + k)) * (0.1 + 0.05 * k))
        run()
        torch.cuda.synchronize()
        near_norm(opt.grad_norm, norm64([p.grad for p in ps], 2.0))
    for got, want in kept:          # eager steps ahead of a capture: a tensor each, which nothing writes again
        near_norm(got, want)
    for p in ps:
        p.grad = None
    opt.step()
    assert float(opt.grad_norm) == 0


# ---- the C entry with nothing to update ---------------------------------------------------------------------------

@pytest.mark.parametrize('kind', [1, 2, 3])
def test_c_adamw_of_an_empty_list_writes_the_norm(kind):
    from nerf_amd import _lib
    L = _lib.lib()
    norm = torch.full((3,), 5.0, device='cuda')
    torch.cuda.synchronize()
    t = _lib.AdamwTensors(0, *([None] * 8))
    assert L.nerf_adamw_step(ctypes.byref(t), None, 0, kind, 1.0, 0, None, 0, norm[1:].data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert norm.tolist() == [5.0, 0.0, 5.0]


# ---- inference mode -----------------------------------------------------------------------------------------------

def test_tensors_of_inference_mode():
    from nerf_amd import ops, optim
    plain = make([300, 40], torch.float32)
    version = plain[1]._version
    was = [t.double() for t in plain]
    with torch.inference_mode():
        ts = [t.clone() for t in plain]
        check_clipped(ts, was, 0.01, 2.0, ops.clip_grad_norm_(ts, 0.01))
        mixed = [ts[0].copy_(plain[0]), plain[1]]
        check_clipped(mixed, was, 0.01, 2.0, ops.clip_grad_norm_(mixed, 0.01))
        near_norm(ops.grad_norm(ts), norm64(ts, 2.0))
        p = torch.nn.Parameter(torch.ones(500, device='cuda'))
        p.grad = torch.ones(500, device='cuda')
        opt = optim.AdamW([p], lr=0.25, weight_decay=0.0)
        opt.step()
        assert torch.allclose(p, torch.full_like(p, 0.75), rtol=0, atol=1e-6)
    assert plain[1]._version > version


# ---- gradients that are refused stay as they were -----------------------------------------------------------------

@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('bad', [math.nan, -math.nan, math.inf, -math.inf])
def test_refused_gradients_keep_their_bits(dtype, bad):
    from nerf_amd import optim
    ps = params_of([700, 5001, 3], dtype)
    ps[1].grad[2500] = bad
    bits = lambda t: t.detach().clone().view(torch.int32 if dtype == torch.float32 else torch.int16)     # noqa: E731
    was = [bits(p.grad) for p in ps]
    with pytest.raises(RuntimeError, match='not finite'):
        optim.clip_grad_norm_(ps, 1e-3, error_if_nonfinite=True)
    assert all(torch.equal(bits(p.grad), w) for p, w in zip(ps, was))


# ---- state at odd places ------------------------------------------------------------------------------------------

def guarded(values, offset):
    """A copy of `values` that starts `offset` elements into a buffer of 77s."""
    n = values.numel()
    buf = torch.full((offset + n + 40,), 77.0, device='cuda', dtype=values.dtype)
    buf[offset:offset + n] = values
    return buf[offset:offset + n]


def guards_kept(view, offset):
    whole = torch.as_strided(view, (offset + view.numel() + 40,), (1,), 0)
    assert bool((whole[:offset] == 77).all()) and bool((whole[offset + view.numel():] == 77).all())


# elements ahead of exp_avg, exp_avg_sq, master, parameter and gradient in their buffers (a line of memory holds 32 fp32)
PLACES = [(1, 0, 0, 0, 0), (3, 3, 3, 3, 3), (31, 1, 2, 3, 5), (5, 33, 30, 1, 7), (32, 31, 6, 9, 2), (30, 17, 13, 63, 1)]


@pytest.mark.parametrize('clip', [None, 2.0])
@pytest.mark.parametrize('places', PLACES)
@pytest.mark.parametrize('dtype', DTYPES)
def test_adamw_with_state_at_odd_places(dtype, places, clip):
    sizes = [1, 2, 3, 4, 5, 30, 31, 33, 0, 1023, 1024, 1025, 2048 - places[0], 2049 - places[0], 70_001]
    ps, states = [], []
    for p, st in zip(params_of(sizes, dtype), make_state(params_of(sizes, dtype), 10)):
        q = torch.nn.Parameter(guarded(p.detach(), places[3]))
        q.grad = guarded(p.grad, places[4])
        st.update(exp_avg=guarded(st['exp_avg'], places[0]), exp_avg_sq=guarded(st['exp_avg_sq'], places[1]))
        if dtype != torch.float32:
            st['master'] = guarded(p.detach().float(), places[2])
        ps.append(q)
        states.append(st)
    was = snapshot(ps, states)
    n = norm64([p.grad for p in ps], 2.0)
    opt = optimizer(ps, states, max_norm=0.4 * n if clip else None)
    opt.step()
    check_step(ps, was, states, 11, 0.4 * n / (n + 1e-6) if clip else 1.0)
    for p, st in zip(ps, states):
        for view, offset in zip((st['exp_avg'], st['exp_avg_sq'], st.get('master'), p.data, p.grad), places):
            if view is not None:
                guards_kept(view, offset)


@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_the_same_bits_at_the_same_places_within_a_line(dtype, norm_type):
    """Ranks hold their gradients at other addresses, but at the same places of their 128-byte lines: one norm, bit for bit."""
    from nerf_amd import ops
    values = make(SIZES['chunk'] + [70_001], dtype)
    line = 128 // values[0].element_size()
    for place in (0, 1, 5, line - 1):
        got = []
        for lines in (0, 1, 4, 33):
            got.append(ops.grad_norm([guarded(v, place + lines * line) for v in values], norm_type))
        near_norm(got[0], norm64(values, norm_type))
        assert all(torch.equal(x, got[0]) for x in got)


# ---- lists past the caches ----------------------------------------------------------------------------------------

def packed(total, dtype, seed, first=1):
    """Seven ragged tensors of `total` elements, behind one another from an odd place of one buffer on."""
    parts = [total // 3 + 1, 5, total // 4 + 3, 1, 0, total // 5]
    sizes = parts + [total - sum(parts)]
    flat = torch.full((first + total + 40,), 77.0, device='cuda', dtype=dtype)
    flat[first:first + total] = 0.01 * torch.randn(total, device='cuda', generator=gen(seed))
    out, at = [], first
    for k, n in enumerate(sizes):
        out.append(flat[at:at + n])
        out[-1].mul_(1 + k)
        at += n
    return flat, out


def ends_kept(flat, total, first=1):
    assert bool((flat[:first] == 77).all()) and bool((flat[first + total:] == 77).all())


@pytest.mark.parametrize('norm_type', NORMS)
@pytest.mark.parametrize('dtype', DTYPES)
def test_norm_and_clip_of_lists_past_the_caches(dtype, norm_type):
    from nerf_amd import ops
    total = (30_000_001 if dtype == torch.float32 else 60_000_001)      # 120 MB to read, 240 MB to read and write
    flat, ts = packed(total, dtype, seed=4)
    near_norm(ops.grad_norm(ts, norm_type), norm64(ts, norm_type))
    was = [t.double() for t in ts]
    most = 0.3 * norm64(ts, norm_type)
    check_clipped(ts, was, most, norm_type, ops.clip_grad_norm_(ts, most, norm_type))
    ends_kept(flat, total)


@pytest.mark.parametrize('dtype', DTYPES)
def test_adamw_of_lists_past_the_caches(dtype):
    total = 9_000_001               # 252 MB and more
    flats, lists = zip(*[packed(total, d, seed=k, first=f) for k, (d, f) in
                         enumerate([(dtype, 1), (dtype, 3), (torch.float32, 5), (torch.float32, 2), (torch.float32, 7)])])
    ps, states = [], []
    for p, g, m, v, w in zip(*lists):
        v.abs_().mul_(1e-2)
        ps.append(torch.nn.Parameter(p))
        ps[-1].grad = g
        states.append(dict(step=torch.tensor(10.0, device='cuda'), exp_avg=m, exp_avg_sq=v))
        if dtype != torch.float32:
            states[-1]['master'] = w.copy_(p)
    was = snapshot(ps, states)
    n = norm64([p.grad for p in ps], 2.0)
    opt = optimizer(ps, states, max_norm=0.4 * n)
    opt.step()
    near_norm(opt.grad_norm, n)
    check_step(ps, was, states, 11, 0.4 * n / (n + 1e-6))
    for flat, first in zip(flats, (1, 3, 5, 2, 7)):
        ends_kept(flat, total, first)


# ---- long lists, scalars, layouts under capture, the other optimizer --------------------------------------------------

@pytest.mark.parametrize('dtype', DTYPES + [DTYPES])
def test_thousands_of_small_parameters(dtype):
    """Forty launches of the norm and a hundred of the update; parameters without dimensions among them."""
    from nerf_amd import ops
    sizes = [(i * 37) % 71 for i in range(5000)]
    ps = params_of(sizes, dtype)
    for i in range(0, 5000, 100):           # (these become scalars)
        old = ps[i]
        ps[i] = torch.nn.Parameter(torch.full((), 0.25, device='cuda', dtype=old.dtype))
        ps[i].grad = torch.full((), -0.01 * (i + 1) / 5000, device='cuda', dtype=old.dtype)
    states = make_state(ps, 2)
    was = snapshot(ps, states)
    grads = [p.grad for p in ps]
    n = norm64(grads, 2.0)
    near_norm(ops.grad_norm(grads), n)
    opt = optimizer(ps, states, max_norm=0.4 * n)
    opt.step()
    near_norm(opt.grad_norm, n)
    check_step(ps, was, states, 3, 0.4 * n / (n + 1e-6))
    before = [g.double() for g in grads]
    check_clipped(grads, before, 0.1 * n, 2.0, ops.clip_grad_norm_(grads, 0.1 * n))


def test_gradients_of_another_order_in_a_captured_step():
    """Gradients that are laid out as their parameters inside the captured step, and one that is a broadcast number: each
    replay reads what they hold then."""
    from nerf_amd import optim

    def build():
        a = torch.nn.Parameter(torch.randn(30, 50, device='cuda', generator=gen(1)).t())
        a.grad = torch.zeros(50, 30, device='cuda')
        b = torch.nn.Parameter(torch.randn(77, device='cuda', generator=gen(2)))
        b.grad = torch.zeros(1, device='cuda').expand(77)
        c = torch.nn.Parameter(torch.randn(64, 3, device='cuda', generator=gen(3)))
        c.grad = torch.zeros(3, 64, device='cuda').t()
        return [a, b, c], optim.AdamW([a, b, c], lr=1e-2, max_norm=0.5)
    ps, opt = build()
    qs, eager = build()
    for o in (opt, eager):
        o.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(4):
        for p, q in zip(ps, qs):
            x = torch.randn(p.shape, device='cuda', generator=gen(60 + k))
            for r in (p, q):
                if r.grad.stride() == (0,):
                    r.grad[:1].copy_(x[:1])
                else:
                    r.grad.copy_(x)
        graph.replay()
        eager.step()
        torch.cuda.synchronize()
        assert torch.equal(opt.grad_norm, eager.grad_norm)
        assert all(torch.equal(p.detach(), q.detach()) for p, q in zip(ps, qs))


def test_state_to_the_other_optimizer_and_back():
    """torch's AdamW goes on from a saved state, and this one from torch's: one step from the same state is one step."""
    from nerf_amd import optim
    kw = dict(lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD)

    def fill(ps, seed):
        for p in ps:
            p.grad = torch.randn(p.shape, device='cuda', generator=gen(seed))
    ps = params_of(SIZES['network'], torch.float32)
    mine = optim.AdamW(ps, **kw)
    for k in range(3):
        fill(ps, k)
        mine.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    other = torch.optim.AdamW(qs, fused=True)
    other.load_state_dict(mine.state_dict())
    fill(qs, 7)
    was = [(q.detach().clone(), q.grad.clone(), other.state[q]['exp_avg'].clone(), other.state[q]['exp_avg_sq'].clone()) for q in qs]
    saved = other.state_dict()
    back = [torch.nn.Parameter(q.detach().clone()) for q in qs]
    third = optim.AdamW(back)
    third.load_state_dict(saved)
    for p, q in zip(back, qs):
        p.grad = q.grad.clone()
    third.step()
    check_step(back, was, [third.state[p] for p in back], 4, 1.0)
    other.step()
    # What torch keeps in fp32 is not ours to say: with beta and its power held in fp32, beta^4 is off by 4 u from beta, 2 u
    # from the function and u from the difference, so 1 - beta^4 by 7 u / (1 - beta^4): 1750 u for beta2, half of it under
    # the root, and 20 u for beta1; with the 24 u counted above below 920 u of the ratio.  The weight: three roundings.
    for q, (w, g, m, v) in zip(qs, was):
        (want, m1, v1), _ = one_step64(w, g, m, v, 4, 1.0)
        size = (B1 * m.abs() + (1 - B1) * g.abs()).double() / (1 - B1 ** 4) / ((v1 / (1 - B2 ** 4)).sqrt() + EPS)
        off = (q.detach().double() - want).abs() - U * (3 * want.abs() + LR * (920 * size + 4 * WD * w.double().abs()))
        assert bool((off <= 0).all()), float(off.max())
