"""Clipping and the fused AdamW step inside the training paths: the batch step of both precisions, the models' own
training_step, the SAR pulse step eager and captured.

With plain gradient descent at lr 1 the weights move by the clipped gradient itself, whose norm is known whatever the
order of the atomic sums behind it: max_norm N / (N + 1e-6), up to the rounding of the weights (2^-24 |w| an entry)."""
import math
from types import SimpleNamespace

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def config(**kw):
    base = dict(use_viewdirs=True, randomized=False, ray_shape='cone', white_bkgd=False, num_levels=2, num_samples=32,
                level_samples=[16, 32], min_deg=0, max_deg=4, viewdirs_min_deg=0, viewdirs_max_deg=4, density_noise=0.0,
                rgb_padding=0.001, resample_padding=0.01, density_bias=-1.0, hidden=64, coarse_weight_decay=0.1, lr_init=1e-3,
                lr_final=5e-5, max_steps=1000, lr_delay_steps=0, lr_delay_mult=1, weight_decay=1e-5, mlp_precision='bf16')
    return SimpleNamespace(**dict(base, **kw))


def model_and_batch(n=96, **kw):
    from nerf_amd.model import MipNeRF
    from nerf_amd.train import synthetic_rays
    torch.manual_seed(0)
    m = MipNeRF(config(**kw)).cuda().train()
    return m, synthetic_rays(n, 'cuda')


def weights(m):
    return [p.detach().clone() for k, p in m.named_parameters() if not k.endswith('scales')]


def norm64(ts):
    return math.sqrt(sum(float((t.double() ** 2).sum()) for t in ts))


def moved(m, was):
    now = weights(m)
    slack = math.sqrt(sum(float(((U * (a.abs() + b.abs())).double() ** 2).sum()) for a, b in zip(was, now)))
    return norm64([a.double() - b.double() for a, b in zip(was, now)]), slack


@pytest.mark.parametrize('precision', ['bf16', 'fp32'])
@pytest.mark.parametrize('chunk', [96, 40])
def test_batch_step_is_clipped(precision, chunk):
    from nerf_amd.train import grad_bucket, nerf_train_step
    m, (rays, pixels) = model_and_batch(mlp_precision=precision)
    sgd = torch.optim.SGD([p for p in m.parameters() if p.requires_grad], lr=1.0)
    nerf_train_step(m, rays, pixels, torch.optim.SGD([p for p in m.parameters() if p.requires_grad], lr=0.0), chunk=chunk)
    free = norm64([grad_bucket(m).flat])
    for most, source in ((free / 3, 'argument'), (free / 5, 'config')):
        was = weights(m)
        if source == 'config':
            m.config.max_grad_norm = most
        nerf_train_step(m, rays, pixels, sgd, chunk=chunk, max_grad_norm=most if source == 'argument' else None)
        got, slack = moved(m, was)
        after = norm64([grad_bucket(m).flat])
        assert after <= most * (1 + 4 * U) and after >= most * (1 - 1e-3)       # N is at least 1e-3: 1e-6 of it in the ratio
        assert abs(got - after) <= slack


def test_batch_step_with_the_fused_optimizer():
    """The optimizer clips as it reads: its norm is that of the bucket, which stays as the backward pass left it, and the
    weights are those of the step in 64 bits from the same gradients."""
    from nerf_amd import optim
    from nerf_amd.train import grad_bucket, nerf_train_step
    m, (rays, pixels) = model_and_batch()
    params = [p for p in m.parameters() if p.requires_grad]
    opt = optim.AdamW(m.parameters(), lr=1e-3, weight_decay=0.1, max_norm=0.01)
    refs = [p.detach().double().cpu() for p in params]
    moments = [(torch.zeros_like(r), torch.zeros_like(r)) for r in refs]
    for t in range(1, 4):
        refs = [p.detach().double().cpu() for p in params]
        version = params[0]._version
        nerf_train_step(m, rays, pixels, opt, chunk=96)
        assert params[0]._version > version                     # (the packed weight streams go by this)
        n = norm64([grad_bucket(m).flat])
        assert abs(float(opt.grad_norm) - n) <= n * 2 * U
        c = min(1.0, 0.01 / (n + 1e-6))
        for p, r, (a, b) in zip(params, refs, moments):
            g = p.grad.double().cpu() * c
            a.mul_(0.9).add_(0.1 * g)
            b.mul_(0.999).add_(0.001 * g * g)
            want = r - 1e-3 * (a / (1 - 0.9 ** t) / ((b / (1 - 0.999 ** t)).sqrt() + 1e-8) + 0.1 * r)
            # the ratio is at most sqrt(1 / 0.001) after equal steps and near 1 here; 100 u of a step of lr is above what
            # three steps' moments can be off, and u |w| is the last rounding
            assert bool(((p.detach().double().cpu() - want).abs() <= U * want.abs() + 1e-3 * 100 * U).all())
    with pytest.raises(ValueError, match='clips at'):
        nerf_train_step(m, rays, pixels, opt, chunk=96, max_grad_norm=0.5)


def test_training_step_of_the_model():
    from nerf_amd import optim
    for fused in (False, True):
        m, (rays, pixels) = model_and_batch(mlp_precision='fp32', max_grad_norm=0.02, fused_adamw=fused)
        assert isinstance(m.optimizers(), optim.AdamW) is fused
        before = weights(m)
        for _ in range(2):
            m.training_step((rays, pixels), 0)
        n = norm64([p.grad for p in m.parameters() if p.grad is not None])
        if fused:
            assert abs(float(m.optimizers().grad_norm) - n) <= n * 2 * U
        else:
            assert abs(n - 0.02) <= 0.02 * 1e-3
        assert all(torch.isfinite(w).all() and not torch.equal(w, b) for w, b in zip(weights(m), before))
        plain, _ = model_and_batch(mlp_precision='fp32')
        assert type(plain.optimizers()) is torch.optim.AdamW


@pytest.mark.parametrize('fused_step', [True, False])
@pytest.mark.parametrize('own', [True, False])
def test_sar_pulse_step(fused_step, own):
    from bench import make_sar_cfg, sar_batch
    from nerf_amd import optim
    from nerf_amd.model import SARNeRF
    from nerf_amd.train import grad_bucket, sar_train_step
    cfg = make_sar_cfg('bf16')
    cfg.rays_per_chunk = cfg.total_num_rays = 512
    cfg.wavelength = 40.0
    torch.manual_seed(3)
    m = SARNeRF(cfg).cuda().train()
    batch = sar_batch(torch.device('cuda'), seed=7)
    cfg.max_grad_norm = 1e-4
    opt = (optim.AdamW(m.parameters(), lr=1e-4, max_norm=1e-4) if own else
           torch.optim.SGD([p for p in m.parameters() if p.requires_grad], lr=1.0))
    was = weights(m)
    sar_train_step(m, batch, opt, fused=fused_step)
    n = norm64([grad_bucket(m).flat])
    if own:
        assert abs(float(opt.grad_norm) - n) <= n * 2 * U
    else:
        got, slack = moved(m, was)
        assert n <= 1e-4 * (1 + 4 * U) and abs(got - n) <= slack
    assert all(torch.isfinite(w).all() for w in weights(m))


@pytest.mark.parametrize('own', [True, False])
def test_captured_sar_pulse_step(own):
    """Replays with the fused optimizer, and with torch's behind a captured clip: after each the bucket's norm is what the
    step says, the counters count on, and a learning rate of zero stops the weights."""
    from bench import make_sar_cfg, sar_batch
    from nerf_amd import optim
    from nerf_amd.model import SARNeRF
    from nerf_amd.train import GraphedSarStep, grad_bucket
    cfg = make_sar_cfg('bf16')
    cfg.rays_per_chunk = cfg.total_num_rays = 512
    cfg.wavelength = 40.0
    torch.manual_seed(3)
    m = SARNeRF(cfg).cuda().train()
    batch = sar_batch(torch.device('cuda'), seed=7)
    opt = (optim.AdamW(m.parameters(), lr=1e-4, weight_decay=0.0, max_norm=1e-4) if own else
           torch.optim.AdamW(m.parameters(), lr=1e-4, weight_decay=0.0, fused=True, capturable=True))
    g = GraphedSarStep(m, batch, opt, warmup=2, max_grad_norm=1e-4)
    first = next(p for p in m.parameters() if p.requires_grad)
    for k in range(4):
        was = weights(m)
        g.step(lr=0.0 if k == 2 else 1e-4)
        torch.cuda.synchronize()
        n = norm64([grad_bucket(m).flat])
        if own:
            assert abs(float(opt.grad_norm) - n) <= n * 2 * U
        else:
            assert n <= 1e-4 * (1 + 4 * U)
        assert float(opt.state[first]['step']) == 3 + k
        same = all(torch.equal(a, b) for a, b in zip(was, weights(m)))
        assert same is (k == 2) and all(torch.isfinite(w).all() for w in weights(m))


def _rank(rank, port, own, q):
    import os

    import torch.distributed as dist

    from nerf_amd import optim
    from nerf_amd.train import grad_bucket, nerf_train_step, shard_range
    from nerf_amd.utils import namedtuple_map
    os.environ.update(MASTER_ADDR='127.0.0.1', MASTER_PORT=str(port))
    dist.init_process_group('gloo', rank=rank, world_size=2)
    m, (rays, pixels) = model_and_batch(n=97)
    lo, hi = shard_range(97, rank, 2)
    shard = namedtuple_map(lambda t: t[lo:hi], rays)
    opt = (optim.AdamW(m.parameters(), lr=1e-3, max_norm=0.01) if own else
           torch.optim.SGD([p for p in m.parameters() if p.requires_grad], lr=0.1))
    for _ in range(3):
        nerf_train_step(m, shard, pixels[lo:hi], opt, chunk=97, world_size=2, max_grad_norm=0.01)
    torch.cuda.synchronize()
    norm = float(opt.grad_norm) if own else 0.0
    q.put((rank, norm, norm64([grad_bucket(m).flat]), torch.cat([w.reshape(-1) for w in weights(m)]).cpu().numpy()))
    dist.barrier()
    dist.destroy_process_group()


@pytest.mark.parametrize('own', [True, False])
def test_two_ranks_clip_alike(own):
    """Two ranks (sharing the GPU, gloo between them) clip the all-reduced gradients by the same norm bit for bit: after
    three steps on shards of different sizes their weights are still the same."""
    import socket

    import numpy as np
    import torch.multiprocessing as mp
    s = socket.socket()
    s.bind(('127.0.0.1', 0))
    port = s.getsockname()[1]
    s.close()
    ctx = mp.get_context('spawn')
    q = ctx.Queue()
    procs = [ctx.Process(target=_rank, args=(r, port, own, q)) for r in range(2)]
    for pr in procs:
        pr.start()
    try:
        got = [q.get(timeout=100) for _ in range(2)]
    finally:
        for pr in procs:
            pr.join(20)
            if pr.is_alive():
                pr.kill()
    assert all(pr.exitcode == 0 for pr in procs)
    assert got[0][1:3] == got[1][1:3] and np.array_equal(got[0][3], got[1][3]) and np.isfinite(got[0][3]).all()
    if own:
        assert abs(got[0][1] - got[0][2]) <= got[0][2] * 2 * U
    else:
        assert got[0][2] <= 0.01 * (1 + 4 * U)
