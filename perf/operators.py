"""Timed cases of the operators that train and serve an MoE layer's experts in BF16: the
grouped matrix products over ragged row segments (forward, gradient of the input,
gradient of the weights) and SwiGLU with an 8-bit checkpoint of its input, forward and
backward. `listed()` names the cases and `draw(rng)` gives more of the same ranges;
`prepare` makes a case's inputs on the GPU, `run` is one pass through an operator (in
plain torch operations, or through the public entry points where `own` is true) and
`exact` the same outputs in 64 bits."""
import os
import random
import sys

import torch

own = False
DEV = 'cuda'
GROUPED_NK = ((4096, 7168), (7168, 2048), (4096, 4096), (4096, 2048), (2048, 7168), (7168, 4096))


def _deep_gemm():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepgemm-amd_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    import deep_gemm
    return deep_gemm


def listed():
    return [
        # Decode: one token routed to 8 of 32 experts, the gate/up product.
        dict(name='nt_token', kind='nt', groups=32, rows=8, n=4096, k=2048, spare=0, alignment=1, out='bf16'),
        # A small chunk over 16 experts, an odd number of columns, segments aligned to 16 rows.
        dict(name='nt_chunk', kind='nt', groups=16, rows=1001, n=1413, k=2048, spare=37, alignment=16, out='bf16'),
        # Training or prefill: 8 experts, 16384 rows split unevenly.
        dict(name='nt_prefill', kind='nt', groups=8, rows=16384, n=4096, k=7168, spare=0, alignment=1, out='bf16'),
        # Gradient of the input of a small chunk, FP32 result.
        dict(name='nn_chunk', kind='nn', groups=16, rows=777, n=2050, k=4096, spare=5, alignment=1, out='f32'),
        # Gradient of the input at the size of a training step.
        dict(name='nn_dgrad', kind='nn', groups=8, rows=8192, n=7168, k=4096, spare=0, alignment=1, out='bf16'),
        # Gradients of many small experts.
        dict(name='tn_small', kind='tn', groups=32, rows=1503, m=577, n=2048, spare=0, alignment=1, add=False,
             eight=False, out='f32'),
        # Gradients of large experts, added to the FP32 sums of earlier micro-batches.
        dict(name='tn_wgrad', kind='tn', groups=8, rows=16384, m=4096, n=7168, spare=0, alignment=1, add=True,
             eight=False, out='f32'),
        # The same with the activations read from an 8-bit checkpoint in the dispatched layout.
        dict(name='tn_checkpoint', kind='tn', groups=8, rows=8192, m=4096, n=2048, spare=100, alignment=128, add=True,
             eight=True, out='f32'),
        # A few tokens' activations.
        dict(name='swiglu_small', kind='swiglu', rows=33, inter=1024, weights=True, clamp=0.0),
        # A training step's.
        dict(name='swiglu_large', kind='swiglu', rows=16384, inter=2048, weights=True, clamp=0.0),
        # Their backward passes; the small one with the clamp of some models' activation.
        dict(name='swiglu_grad_small', kind='swiglu_grad', rows=33, inter=1024, weights=True, clamp=7.0),
        dict(name='swiglu_grad_large', kind='swiglu_grad', rows=16384, inter=2048, weights=True, clamp=0.0),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


MOST_FLOPS = 2 * 16384 * 4096 * 7168
MOST_WEIGHT = 1 << 30   # elements of all groups' weights (or weight gradients)


def draw(rng):
    kind = rng.choice(('nt', 'nt', 'nt', 'nn', 'nn', 'tn', 'tn', 'tn', 'swiglu', 'swiglu_grad'))
    if kind in ('swiglu', 'swiglu_grad'):
        return dict(kind=kind, rows=_log(rng, 1, 16384), inter=8 * _log(rng, 8, 512) if rng.random() < 0.5 else
                    rng.choice((512, 768, 1024, 2048, 4096)), weights=rng.random() < 0.7, clamp=rng.choice((0.0, 0.0, 7.0)))
    while True:
        groups = rng.choice((1, 2, 4, 8, 16, 32, 64, 128))
        rows = _log(rng, 1, 32768)
        if rng.random() < 0.5:
            n, k = rng.choice(GROUPED_NK)
        else:   # any layer: the reduced dimension in whole 16-byte pieces, the other one free
            n, k = _log(rng, 64, 8192), 8 * _log(rng, 8, 1024)
        if 2 * rows * n * k <= MOST_FLOPS and groups * n * k <= MOST_WEIGHT:
            break
    case = dict(kind=kind, groups=groups, rows=rows, n=n, k=k, spare=rng.choice((0, 0, 1, 77)),
                alignment=rng.choice((1, 1, 16, 128)), out=rng.choice(('bf16', 'bf16', 'f32')))
    if kind != 'tn':
        return case
    eight = rng.random() < 0.4
    del case['k']
    return dict(case, m=n, n=k, add=rng.random() < 0.5, eight=eight, out=rng.choice(('f32', 'f32', 'bf16')))


# ---------------------------------------------------------------- inputs

def sizes(case):
    """Rows of each group: uneven, some groups empty; at most one row each where there are
    fewer rows than groups. The same for every seed."""
    g, rows = case['groups'], case['rows']
    rng = random.Random('%d %d %d' % (g, rows, case['n']))
    if rows <= g:
        hit = set(rng.sample(range(g), rows))
        return [int(i in hit) for i in range(g)]
    share = [rng.gammavariate(3.0, 1.0) if g <= 2 or rng.random() > 0.08 else 0.0 for _ in range(g)]
    total = sum(share)
    if total == 0.0:
        share[0] = total = 1.0
    ends = [int(round(rows * sum(share[:i + 1]) / total)) for i in range(g)]
    ends[-1] = rows
    return [e - s for s, e in zip([0] + ends[:-1], ends)]


def segments(case):
    """(first row, end) of each group, and the rows of the whole buffer."""
    a, at, out = case['alignment'], 0, []
    for s in sizes(case):
        start = -(-at // a) * a
        at = start + s
        out.append((start, at))
    return out, at + case['spare']


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _empty(shape, dtype):
    """Rows that begin at whole 16-byte pieces, as a user pads an odd number of columns."""
    return torch.empty((*shape[:-1], -(-shape[-1] // 8) * 8), dtype=dtype, device=DEV)[..., :shape[-1]]


def _randn(shape, gen, scale=1.0):
    x = _empty(shape, torch.bfloat16)
    return x.copy_(torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale)


def _pieces(x):
    """[rows, cols] -> [rows, pieces, 128], zeros past cols."""
    x = torch.nn.functional.pad(x, (0, -x.shape[1] % 128))
    return x.view(x.shape[0], -1, 128)


def _cast(x):
    """e4m3 values of a BF16 matrix with one power-of-two scale per row and 128 columns:
    the scale is the largest magnitude (1e-4 at least) over 448, up to a power of two."""
    p = _pieces(x.float())
    sf = p.abs().amax(2).clamp(min=1e-4) * (1.0 / 448.0)
    bits = sf.view(torch.int32)
    sf = (((bits >> 23) + ((bits & 0x7FFFFF) != 0).int()) << 23).view(torch.float32)
    q = (p / sf[:, :, None]).reshape(x.shape[0], -1)[:, :x.shape[1]].contiguous().to(torch.float8_e4m3fn)
    return q, sf


def _value(q, sf):
    """The values that an 8-bit checkpoint stands for."""
    return (_pieces(q.float()) * sf[:, :, None]).reshape(q.shape[0], -1)[:, :q.shape[1]]


def _cast_halves(x):
    """_cast of the gate half and the up half, side by side."""
    half = x.shape[1] // 2
    (qg, sg), (qu, su) = _cast(x[:, :half]), _cast(x[:, half:])
    q = torch.cat((qg.view(torch.uint8), qu.view(torch.uint8)), 1).view(torch.float8_e4m3fn)
    return q, torch.cat((sg, su), 1)


def prepare(case, seed):
    gen = _gen(seed)
    kind, out = case['kind'], {'bf16': torch.bfloat16, 'f32': torch.float32}.get(case.get('out'))
    if kind in ('swiglu', 'swiglu_grad'):
        rows, inter = case['rows'], case['inter']
        x = _randn((rows, 2 * inter), gen, 2.0)
        w = torch.rand(rows, generator=gen, device=DEV) if case['weights'] else None
        s = dict(kind=kind, x=x, w=w, clamp=case['clamp'])
        if kind == 'swiglu_grad':   # what the forward pass left, and the gradient that comes back
            q, sf = _cast_halves(x)
            s = dict(kind=kind, q=q, sf=sf, w=w, clamp=case['clamp'], dh=_randn((rows, inter), gen, 0.1))
        return s
    seg, total = segments(case)
    g, n = case['groups'], case['n']
    ends = torch.tensor([e for _, e in seg], dtype=torch.int32, device=DEV)
    # the plan of the plain form: the rows of each group, padded to the longest one's
    most = max(1, max(e - s for s, e in seg))
    first = torch.tensor([s for s, _ in seg], device=DEV)
    idx = first[:, None] + torch.arange(most, device=DEV)[None]
    live = idx < ends[:, None]
    s = dict(kind=kind, ends=ends, alignment=case['alignment'], idx=torch.where(live, idx, total), live=live)
    if kind == 'tn':
        m = case['m']
        s['a'], b = _randn((total, m), gen, 0.1), _randn((total, n), gen)
        s['b'] = _cast(b) if case['eight'] else b
        s['c'] = torch.randn((g, m, n), generator=gen, device=DEV).to(out) if case['add'] else None
        s['d'] = torch.full((g, m, n), 0.5, dtype=out, device=DEV)
    else:
        k = case['k']
        s['a'] = _randn((total, k), gen)
        s['b'] = _empty((g, n, k) if kind == 'nt' else (g, k, n), torch.bfloat16)
        for i in range(g):   # one group at a time: the 32-bit values need not fit beside each other
            s['b'][i].copy_(_randn(s['b'].shape[1:], gen, k ** -0.5))
        s['d'] = torch.full((total, n), 0.5, dtype=out, device=DEV)
    return s


# ---------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    dg, kind = _deep_gemm(), s['kind']
    if kind == 'nt':
        dg.m_grouped_bf16_gemm_nt_ragged(s['a'], s['b'], s['d'], s['ends'], alignment=s['alignment'])
        return s['d']
    if kind == 'nn':
        dg.m_grouped_bf16_gemm_nn_ragged(s['a'], s['b'], s['d'], s['ends'], alignment=s['alignment'])
        return s['d']
    if kind == 'tn':
        dg.k_grouped_bf16_gemm_tn_ragged(s['a'], s['b'], s['d'], s['ends'], c=s['c'], alignment=s['alignment'])
        return s['d']
    if kind == 'swiglu':
        h, (q, sf) = dg.moe_swiglu_checkpoint(s['x'], s['w'], clamp_value=s['clamp'])
        return dict(h=h, q=q, sf=sf)
    dx, h, dw = dg.moe_swiglu_backward(s['dh'], (s['q'], s['sf']), s['w'], clamp_value=s['clamp'])
    return dict(dx=dx, h=h, dw=dw)


def _padded(x, idx):
    """The rows x[idx], zeros where idx is past the last row."""
    return torch.nn.functional.pad(x, (0, 0, 0, 1))[idx]


def _run_plain(s):
    kind = s['kind']
    if kind in ('nt', 'nn'):
        w = s['b'].float()
        y = torch.bmm(_padded(s['a'].float(), s['idx']), w.transpose(1, 2) if kind == 'nt' else w)
        s['d'][s['idx'][s['live']]] = y[s['live']].to(s['d'].dtype)
        return s['d']
    if kind == 'tn':
        b = _value(*s['b']) if isinstance(s['b'], tuple) else s['b'].float()
        y = torch.bmm(_padded(s['a'].float(), s['idx']).transpose(1, 2), _padded(b, s['idx']))
        if s['c'] is not None:
            y += s['c'].float()
        s['d'].copy_(y)
        return s['d']
    c, w = s['clamp'], s['w']
    wide = None if w is None else w[:, None]
    if kind == 'swiglu':
        inter = s['x'].shape[1] // 2
        gate, up = s['x'][:, :inter].float(), s['x'][:, inter:].float()
        if c > 0:
            gate, up = gate.clamp(max=c), up.clamp(-c, c)
        h = gate / (1 + torch.exp(-gate)) * up
        q, sf = _cast_halves(s['x'])
        return dict(h=(h if w is None else h * wide).bfloat16(), q=q, sf=sf)
    inter = s['dh'].shape[1]
    parts = s['sf'].shape[1] // 2
    gate, up = _value(s['q'][:, :inter], s['sf'][:, :parts]), _value(s['q'][:, inter:], s['sf'][:, parts:])
    dh = s['dh'].float()
    in_g = in_u = None
    if c > 0:
        in_g, in_u = gate <= c, up.abs() <= c
        gate, up = gate.clamp(max=c), up.clamp(-c, c)
    sig = 1 / (1 + torch.exp(-gate))
    act = gate * sig
    dw = None if w is None else (dh * act * up).sum(1)
    dy = dh if w is None else dh * wide
    dgate, dup = dy * up * sig * (1 + gate * (1 - sig)), dy * act
    if c > 0:
        dgate, dup = dgate * in_g, dup * in_u
    h = act * up if w is None else act * up * wide
    return dict(dx=torch.cat((dgate, dup), 1).bfloat16(), h=h.bfloat16(), dw=dw)


# ---------------------------------------------------------------- what it costs, and what is right

def work(case):
    kind = case['kind']
    if kind in ('swiglu', 'swiglu_grad'):
        r, i = case['rows'], case['inter']
        scales = r * 2 * -(-i // 128) * 4
        weights = r * 4 if case['weights'] else 0
        if kind == 'swiglu':   # gate and up in; h and the codes out
            return dict(bytes=r * i * (4 + 2 + 2) + scales + weights, flops=10 * r * i)
        return dict(bytes=r * i * (2 + 2 + 4 + 2) + scales + 2 * weights, flops=25 * r * i)   # dh and codes in; dx, h out
    r, n, g = case['rows'], case['n'], case['groups']
    size = 2 if case['out'] == 'bf16' else 4
    if kind == 'tn':
        m = case['m']
        b = r * n + r * -(-n // 128) * 4 if case['eight'] else r * n * 2
        return dict(bytes=r * m * 2 + b + g * m * n * size * (2 if case['add'] else 1) + 4 * g, flops=2 * r * m * n)
    k, used = case['k'], sum(s > 0 for s in sizes(case))
    return dict(bytes=r * k * 2 + used * n * k * 2 + r * n * size + 4 * g, flops=2 * r * n * k)


def _pow2(e):
    """2 ** e in 64 bits, to the bit."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _e4m3(v):
    """Nearest e4m3 value in 64 bits, ties to the even code (|v| <= 464)."""
    part, e = torch.frexp(v)   # |part| in [1/2, 1)
    step = _pow2((e - 1).clamp(min=-6) - 3)
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind = s['kind']
    if kind in ('nt', 'nn', 'tn'):
        seg, _ = segments(case)
        if kind == 'tn':
            b = s['b']
            if isinstance(b, tuple):
                q, sf = b
                b = q.float().double() * sf.double().repeat_interleave(128, 1)[:, :q.shape[1]]
            d = torch.zeros(s['d'].shape, dtype=torch.float64, device=DEV) if s['c'] is None else s['c'].double()
            for i, (lo, hi) in enumerate(seg):
                if hi > lo:
                    d[i] += s['a'][lo:hi].double().T.contiguous() @ b[lo:hi].double()
            return d
        d = s['d'].double()
        for i, (lo, hi) in enumerate(seg):
            if hi > lo:
                w = s['b'][i].double()
                d[lo:hi] = s['a'][lo:hi].double() @ (w.T.contiguous() if kind == 'nt' else w)
        return d
    c = s['clamp'] if s['clamp'] > 0 else float('inf')
    w = 1.0 if s['w'] is None else s['w'].double()[:, None]
    if kind == 'swiglu':
        x = s['x'].double()
        rows, inter = x.shape[0], x.shape[1] // 2
        gate, up = x[:, :inter].clamp(max=c), x[:, inter:].clamp(-c, c)
        h = gate * torch.sigmoid(gate) * up * w
        codes, scales = [], []
        for half in (x[:, :inter], x[:, inter:]):
            wide = torch.zeros((rows, -(-inter // 128) * 128), dtype=torch.float64, device=DEV)
            wide[:, :inter] = half
            wide = wide.view(rows, -1, 128)
            ratio = wide.abs().amax(2).clamp(min=float(torch.tensor(1e-4, dtype=torch.float32)))
            ratio = (ratio * float(torch.tensor(1 / 448, dtype=torch.float32))).float().double()   # a 32-bit product
            part, e = torch.frexp(ratio)   # part in [1/2, 1)
            sf = _pow2(torch.where(part == 0.5, e - 1, e))
            codes.append(_e4m3(wide / sf[:, :, None]).reshape(rows, -1)[:, :inter])
            scales.append(sf)
        return dict(h=h, q=torch.cat(codes, 1), sf=torch.cat(scales, 1))
    q, sf = s['q'].float().double(), s['sf'].double()
    inter, parts = s['dh'].shape[1], sf.shape[1] // 2
    gate = q[:, :inter] * sf[:, :parts].repeat_interleave(128, 1)[:, :inter]
    up = q[:, inter:] * sf[:, parts:].repeat_interleave(128, 1)[:, :inter]
    free_g, free_u = (gate <= c).double(), (up.abs() <= c).double()
    gate, up = gate.clamp(max=c), up.clamp(-c, c)
    sig, dh = torch.sigmoid(gate), s['dh'].double()
    act = gate * sig
    dgate = dh * w * up * (sig + act * (1 - sig)) * free_g
    dup = dh * w * act * free_u
    dw = None if s['w'] is None else (dh * act * up).sum(1)
    return dict(dx=torch.cat((dgate, dup), 1), h=act * up * w, dw=dw)
