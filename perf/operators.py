"""Cases that time the operators between a backward pass and the next forward pass: the global norm of a list of
gradients, clipping by it, and the AdamW step that clips while it reads the gradients.

A case holds a parameter list: the tensors of one of the networks (`net`), or `tensors` tensors of ragged sizes that
hold `elements` values together.  The tensors are views of one flat buffer, as a gradient bucket lays them out: `align`
= 64 starts each on a multiple of 64 elements (the bucket's own layout), `align` = 1 packs them without gaps, so that
most start at odd places.  The gaps are zero and stay zero, which is why the plain forms may go over the flat buffer as
a whole.
"""
import math
import random

import torch

own = False

DTYPES = {'float32': torch.float32, 'bfloat16': torch.bfloat16, 'float16': torch.float16}
BETA1, BETA2, EPS, DECAY, LR = 0.9, 0.999, 1e-8, 0.01, 1e-3
STEPS_BEFORE = 200          # steps that the moments have seen before the measured one
LARGEST = 1 << 30


def listed():
    return [
        # the gradients of the 8 x 256 network, 24 tensors: the norm that a training loop logs every step
        dict(name='norm, 8x256 network', op='norm', net='nerf', dtype='float32', norm_type=2.0, align=64),
        # 16-bit gradients of many tensors, packed: half of them start at odd places
        dict(name='norm, 389 ragged bf16', op='norm', net='', tensors=389, elements=301_234_567, dtype='bfloat16',
             norm_type=2.0, align=1),
        # the largest entry (a check for overflow ahead of a step in half precision)
        dict(name='max norm, 61 ragged fp16', op='norm', net='', tensors=61, elements=5_300_021, dtype='float16',
             norm_type=math.inf, align=64),
        # one flat bucket of 4 GB
        dict(name='norm, one buffer of 1.07e9', op='norm', net='', tensors=1, elements=LARGEST - 17, dtype='float32',
             norm_type=2.0, align=64),
        # the SAR network's gradients, clipped ahead of an optimizer of the caller's own
        dict(name='clip, 156-wide SAR network', op='clip', net='sar', dtype='float32', norm_type=2.0, align=64),
        # 16-bit gradients clipped in place, ordinary size
        dict(name='clip, 150 ragged bf16', op='clip', net='', tensors=150, elements=40_000_003, dtype='bfloat16',
             norm_type=2.0, align=1),
        # clipped in place, far beyond the caches
        dict(name='clip, 97 ragged, 5e8', op='clip', net='', tensors=97, elements=500_000_009, dtype='float32',
             norm_type=1.0, align=64),
        # the optimizer step of the two networks: latency counts
        dict(name='adamw, 8x256 network', op='adamw', net='nerf', dtype='float32', norm_type=2.0, align=64, clip=True),
        dict(name='adamw, 156-wide, no clip', op='adamw', net='sar', dtype='float32', norm_type=2.0, align=64, clip=False),
        # half-precision parameters of odd sizes with 32-bit masters
        dict(name='adamw, 40 ragged fp16', op='adamw', net='', tensors=40, elements=3_141_593, dtype='float16',
             norm_type=2.0, align=1, clip=True),
        # ordinary and largest models: the step is a stream through memory
        dict(name='adamw, 128 ragged, 1e8', op='adamw', net='', tensors=128, elements=100_000_007, dtype='float32',
             norm_type=2.0, align=64, clip=True),
        dict(name='adamw, 300 ragged bf16', op='adamw', net='', tensors=300, elements=250_000_013, dtype='bfloat16',
             norm_type=2.0, align=64, clip=True),
    ]


def draw(rng):
    op = rng.choice(('norm', 'clip', 'adamw'))
    most = {'norm': 9e8, 'clip': 4e8, 'adamw': 2e8}[op]
    elements = int(math.exp(rng.uniform(math.log(2e3), math.log(most)))) | 1
    tensors = max(1, min(int(math.exp(rng.uniform(0.0, math.log(400.0)))), elements // 8))
    case = dict(op=op, net='', tensors=tensors, elements=elements, dtype=rng.choice(sorted(DTYPES)),
                norm_type=rng.choice((2.0, 2.0, 1.0, math.inf)), align=rng.choice((1, 64)))
    if op == 'adamw':
        case['clip'] = rng.random() < 0.7
    return case


def _shapes(case):
    """The shapes of a case's parameter list."""
    if case['net']:
        sar = case['net'] == 'sar'
        hidden, enc, view, width = (156, 24, 27, 180) if sar else (256, 60, 27, 128)
        layers = []
        for first in (enc, enc + hidden):
            layers += [(hidden, first)] + [(hidden, hidden)] * 3
        heads = [(1, hidden), (hidden, hidden), (width, hidden + view), (3, width)] + ([(2, width)] if sar else [])
        shapes = [(hidden,), (hidden,)] if sar else []          # (the LayerNorm pair of the density head)
        for n, k in layers + heads:
            shapes += [(n, k), (n,)]
        return shapes
    n, total = case['tensors'], case['elements']
    rng = random.Random(n * 1_000_003 + total)
    parts = [math.exp(rng.uniform(0.0, 7.0)) for _ in range(n)]
    sizes = [max(1, int(total * x / sum(parts))) for x in parts]
    sizes[-1] = max(1, sizes[-1] + total - sum(sizes))
    return [(s,) for s in sizes]


def _layout(case):
    """Shapes, first elements, and the flat length of a case's tensors."""
    shapes, first, at = _shapes(case), [], 0
    for s in shapes:
        first.append(at)
        at += -(-math.prod(s) // case['align']) * case['align']
    return shapes, first, at


def _views(flat, shapes, first):
    return [flat[a:a + math.prod(s)].view(s) for s, a in zip(shapes, first)]


def prepare(case, seed):
    shapes, first, length = _layout(case)
    dtype = DTYPES[case['dtype']]
    g = torch.Generator(device='cuda').manual_seed(seed)
    rng = random.Random(seed)
    scales = [10.0 ** rng.uniform(-3.5, -1.0) for _ in shapes]         # layers differ in the size of their gradients
    zeros = lambda d: torch.zeros(length, dtype=d, device='cuda')      # noqa: E731
    s = dict(op=case['op'], norm_type=case['norm_type'], grads=zeros(dtype))
    s['grad_views'] = _views(s['grads'], shapes, first)
    for v, a in zip(s['grad_views'], scales):
        v.normal_(generator=g).mul_(a)
    if case['op'] == 'norm':
        return s
    # about a third of the norm that entries of these sizes have
    p, parts = case['norm_type'], [(a, math.prod(x)) for a, x in zip(scales, shapes)]
    s['max_norm'] = (0.3 + 0.1 * rng.random()) * (3.0 * max(scales) if p == math.inf else
                                                  sum(0.8 ** (2.0 - p) * n * a ** p for a, n in parts) ** (1.0 / p))
    if case['op'] == 'clip':
        return s
    if not case['clip']:
        s['max_norm'] = None
    master = dtype != torch.float32
    s['p'], s['m'], s['v'] = zeros(dtype), zeros(torch.float32), zeros(torch.float32)
    s['master'] = zeros(torch.float32) if master else None
    s['steps'] = torch.full((len(shapes),), float(STEPS_BEFORE), device='cuda')
    w, m, v = (_views(x, shapes, first) for x in (s['master'] if master else s['p'], s['m'], s['v']))
    for wi, mi, vi, a in zip(w, m, v, scales):
        wi.normal_(generator=g).mul_(0.05)
        mi.normal_(generator=g).mul_(0.3 * a)
        vi.normal_(generator=g).square_().add_(0.05).mul_(a * a)
    if master:
        s['p'].copy_(s['master'])
    if own:
        # the optimizer that a training program holds; its state is what earlier steps left
        from nerf_amd.optim import AdamW
        params = [torch.nn.Parameter(x) for x in _views(s['p'], shapes, first)]
        for p, gr in zip(params, s['grad_views']):
            p.grad = gr
        opt = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, max_norm=s['max_norm'],
                    norm_type=case['norm_type'])
        masters = _views(s['master'], shapes, first) if master else [None] * len(shapes)
        for i, p in enumerate(params):
            opt.state[p] = dict(step=s['steps'][i], exp_avg=m[i], exp_avg_sq=v[i])
            if master:
                opt.state[p]['master'] = masters[i]
        s['optimizer'] = opt
    return s


def _norm64(g, norm_type):
    """The norm of a flat buffer: entries in 32 bits, their sum in 64."""
    x = g.float()
    if norm_type == math.inf:
        return x.abs().max().double()
    if norm_type == 1.0:
        return x.abs().sum(dtype=torch.float64)
    return (x * x).sum(dtype=torch.float64).sqrt()


def _coefficient(norm, max_norm):
    return (max_norm / (norm + 1e-6)).clamp(max=1.0).float()


def _adamw_plain(s):
    out = {}
    g = s['grads'].float()
    if s['max_norm'] is not None:
        norm = _norm64(s['grads'], s['norm_type'])
        out['norm'] = norm.float()
        g = g * _coefficient(norm, s['max_norm'])
    s['steps'].add_(1.0)
    t = s['steps'][0].double()
    c1, c2 = (1.0 - BETA1 ** t).float(), (1.0 - BETA2 ** t).float()
    m, v = s['m'], s['v']
    m.mul_(BETA1).add_(g * (1.0 - BETA1))
    v.mul_(BETA2).add_(g * g * (1.0 - BETA2))
    w = s['p'] if s['master'] is None else s['master']
    w.sub_(((m / c1) / ((v / c2).sqrt() + EPS) + DECAY * w) * LR)
    if s['master'] is not None:
        s['p'].copy_(w)
    return _adamw_outputs(s, out)


def _adamw_outputs(s, out):
    out.update(p=s['p'], m=s['m'], v=s['v'], steps=s['steps'])
    if s['master'] is not None:
        out['master'] = s['master']
    return out


def run(s):
    if own:
        from nerf_amd import ops
        if s['op'] == 'norm':
            return {'norm': ops.grad_norm(s['grad_views'], s['norm_type'])}
        if s['op'] == 'clip':
            return {'norm': ops.clip_grad_norm_(s['grad_views'], s['max_norm'], s['norm_type']), 'grads': s['grads']}
        s['optimizer'].step()
        return _adamw_outputs(s, {} if s['max_norm'] is None else {'norm': s['optimizer'].grad_norm})
    if s['op'] == 'norm':
        return {'norm': _norm64(s['grads'], s['norm_type']).float()}
    if s['op'] == 'clip':
        norm = _norm64(s['grads'], s['norm_type'])
        c = _coefficient(norm, s['max_norm'])
        if s['grads'].dtype == torch.float32:
            s['grads'].mul_(c)
        else:
            s['grads'].copy_(s['grads'].float() * c)
        return {'norm': norm.float(), 'grads': s['grads']}
    return _adamw_plain(s)


def work(case):
    """Each input read once, each output written once."""
    n = sum(math.prod(s) for s in _shapes(case))
    size = 4 if case['dtype'] == 'float32' else 2
    if case['op'] == 'norm':
        return dict(bytes=n * size + 4, flops=2 * n)
    if case['op'] == 'clip':
        return dict(bytes=2 * n * size + 4, flops=3 * n)
    # gradient in; weights (in 32 bits) and two moments in and out; 16-bit parameters are a fourth output
    return dict(bytes=n * (size + 24 + (0 if size == 4 else 2)), flops=(17 if case['clip'] else 14) * n)


def exact(case, seed):
    """From the definition, in 64 bits, on the same inputs."""
    global own
    kept, own = own, False          # (the inputs alone)
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    g = s['grads'].double()
    if case['norm_type'] == math.inf:
        norm = torch.linalg.vector_norm(g, ord=math.inf)
    elif case['norm_type'] == 1.0:
        norm = torch.linalg.vector_norm(g, ord=1)
    else:
        norm = torch.linalg.vector_norm(g)
    if case['op'] == 'norm':
        return {'norm': norm}
    scale = 1.0 if s['max_norm'] is None else min(1.0, s['max_norm'] / (float(norm) + 1e-6))
    g = g * scale
    if case['op'] == 'clip':
        return {'norm': norm, 'grads': g}
    t = STEPS_BEFORE + 1
    m = BETA1 * s['m'].double() + (1.0 - BETA1) * g
    v = BETA2 * s['v'].double() + (1.0 - BETA2) * g ** 2
    w = (s['p'] if s['master'] is None else s['master']).double()
    ratio = m / (1.0 - BETA1 ** t) / (torch.sqrt(v / (1.0 - BETA2 ** t)) + EPS)
    w = (1.0 - LR * DECAY) * w - LR * ratio
    out = {} if s['max_norm'] is None else {'norm': norm}
    out.update(p=w, m=m, v=v, steps=torch.full((len(_shapes(case)),), float(t), device='cuda'))
    if s['master'] is not None:
        out['master'] = w
    return out
