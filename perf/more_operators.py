"""Timed cases of the operators that bring tokens to an MoE layer's experts and back in BF16,
with their gradients, and of the 4-bit forms of the experts' products: dispatch, its gradient, the
gradient of the combination, quantisation to 4 bits (32 elements a scale) and back, and the
product of 4-bit operands over ragged row segments. `listed()` names the cases and `draw(rng)`
gives more of the same ranges; `prepare` makes a case's inputs on the GPU, `run` is one pass
through an operator (in plain torch operations, or through the public entry points where
`own` is true) and `exact` the same outputs in 64 bits."""
import os
import random
import sys

import torch

own = False
DEV = 'cuda'
GROUPED_NK = ((4096, 7168), (7168, 2048), (4096, 4096), (4096, 2048), (2048, 7168), (7168, 4096))
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _deep_gemm():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'deepgemm-amd_amd')
    if path not in sys.path:
        sys.path.insert(0, path)
    import deep_gemm
    return deep_gemm


def listed():
    return [
        # Decode: a few tokens on their way to 32 experts.
        dict(name='dispatch_tokens', kind='dispatch', tokens=4, topk=8, experts=32, hidden=2048, alignment=16, lost=0.0,
             weights=True),
        # A chunk of a prompt whose batch is padded (some tokens are not routed), segments back to back.
        dict(name='dispatch_chunk', kind='dispatch', tokens=777, topk=6, experts=64, hidden=2056, alignment=1, lost=0.1,
             weights=True),
        # A training step's tokens.
        dict(name='dispatch_large', kind='dispatch', tokens=8192, topk=8, experts=256, hidden=7168, alignment=16, lost=0.0,
             weights=True),
        # The gradients that come back from the experts, of a small batch and of a training step.
        dict(name='dispatch_grad_small', kind='dispatch_grad', tokens=33, topk=8, experts=32, hidden=1024, alignment=16,
             lost=0.1, weights=True),
        dict(name='dispatch_grad_large', kind='dispatch_grad', tokens=8192, topk=8, experts=256, hidden=7168, alignment=16,
             lost=0.0, weights=True),
        # The gradients that go to them, and those of the routing weights.
        dict(name='combine_grad_small', kind='combine_grad', tokens=33, topk=8, experts=32, hidden=1024, alignment=16,
             lost=0.1, weights=True),
        dict(name='combine_grad_large', kind='combine_grad', tokens=8192, topk=8, experts=256, hidden=7168, alignment=16,
             lost=0.0, weights=True),
        # Activations of a few tokens, and of a training step (or a layer's weights), as 4 bits keep them.
        dict(name='quantise_small', kind='quantise', rows=33, cols=2048),
        dict(name='quantise_large', kind='quantise', rows=16384, cols=7168),
        # Decode in 4 bits: one token routed to 8 of 32 experts, the gate/up product.
        dict(name='product_token', kind='product', groups=32, rows=8, n=4096, k=2048, spare=0, alignment=1, out='bf16'),
        # A small chunk over 16 experts, odd numbers of columns and of scales, segments aligned to 16 rows.
        dict(name='product_chunk', kind='product', groups=16, rows=1001, n=1413, k=2080, spare=37, alignment=16, out='f32'),
        # Prefill: 8 experts, 16384 rows split unevenly.
        dict(name='product_prefill', kind='product', groups=8, rows=16384, n=4096, k=7168, spare=0, alignment=1, out='bf16'),
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


MOST_ROUTED = 8192 * 8 * 7168   # elements of the routed rows
MOST_CAST = 16384 * 7168
MOST_FLOPS = 2 * 16384 * 4096 * 7168
MOST_WEIGHT = 1 << 29           # elements of all groups' weights


def draw(rng):
    kind = rng.choice(('dispatch', 'dispatch', 'dispatch_grad', 'combine_grad', 'quantise', 'product', 'product', 'product'))
    if kind == 'quantise':
        while True:
            rows = _log(rng, 1, 65536)
            cols = rng.choice((512, 2048, 4096, 7168)) if rng.random() < 0.4 else rng.choice((2, 16, 32)) * _log(rng, 4, 512)
            if rows * cols <= MOST_CAST:
                return dict(kind=kind, rows=rows, cols=cols)
    if kind == 'product':
        while True:
            groups = rng.choice((1, 2, 4, 8, 16, 32, 64))
            rows = _log(rng, 1, 32768)
            if rng.random() < 0.5:
                n, k = rng.choice(GROUPED_NK)
            else:   # any layer: the reduced dimension in whole scales, the other one free
                n, k = _log(rng, 64, 8192), 32 * _log(rng, 2, 256)
            if 2 * rows * n * k <= MOST_FLOPS and groups * n * k <= MOST_WEIGHT:
                break
        return dict(kind=kind, groups=groups, rows=rows, n=n, k=k, spare=rng.choice((0, 0, 1, 77)),
                    alignment=rng.choice((1, 1, 16, 128)), out=rng.choice(('bf16', 'bf16', 'f32')))
    while True:
        tokens, topk = _log(rng, 1, 16384), rng.choice((1, 2, 4, 6, 8))
        hidden = rng.choice((512, 2048, 4096, 7168)) if rng.random() < 0.4 else 8 * _log(rng, 8, 1024)
        if tokens * topk * hidden <= MOST_ROUTED:
            break
    return dict(kind=kind, tokens=tokens, topk=topk, experts=rng.choice((8, 16, 32, 64, 128, 256)), hidden=hidden,
                alignment=rng.choice((1, 1, 16, 128)), lost=rng.choice((0.0, 0.0, 0.1)), weights=rng.random() < 0.8)


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


def buffer_rows(case):
    """Rows that any routing of the tokens fits: what the dispatch asks for."""
    a = case['alignment']
    return -(-(case['tokens'] * case['topk'] + case['experts'] * (a - 1)) // a) * a


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(shape, gen, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV, dtype=torch.float32) * scale).bfloat16()


def _routing(case, gen):
    """Experts of each token, some of them wanted more than others, each at most once in a row;
    a share `lost` of the entries is not routed."""
    t, k, e = case['tokens'], min(case['topk'], case['experts']), case['experts']
    liking = torch.randn((1, e), generator=gen, device=DEV) * 0.5
    idx = torch.topk(torch.randn((t, e), generator=gen, device=DEV) + liking, k, dim=1).indices.int()
    return torch.where(torch.rand((t, k), generator=gen, device=DEV) < case['lost'], -1, idx)


def _places(topk, experts, alignment):
    """Rows of the entries in the order of expert, token and slot (-1: not routed), the
    ends of the segments and the rows that they take, padding included."""
    flat = topk.reshape(-1).long()
    key = torch.where(flat >= 0, flat, experts)
    order = torch.argsort(key, stable=True)
    at = key[order]
    counts = (key[None] == torch.arange(experts + 1, device=DEV)[:, None]).sum(1)
    counts[experts] = 0
    room = (counts + alignment - 1) // alignment * alignment
    starts = torch.cumsum(room, 0) - room
    first = torch.cumsum(counts, 0) - counts
    row = torch.where(at < experts, starts[at] + torch.arange(at.numel(), device=DEV) - first[at], -1)
    pos = torch.empty_like(row)
    pos[order] = row
    return pos.view(topk.shape).int(), (starts + counts)[:experts].int(), starts[experts]


def _pad32(x):
    """[rows, cols] -> [rows, scales, 32], zeros past cols."""
    x = torch.nn.functional.pad(x, (0, -x.shape[-1] % 32))
    return x.view(*x.shape[:-1], -1, 32)


def _cast4(x):
    """4-bit codes of a matrix, two a byte (the even column's low), and its scales, four a word:
    for 32 columns, the largest magnitude (1e-4 at least) over 6, up to a power of two. Ties
    go to the even code, there is no negative zero, and what is past the last scale is one."""
    cols = x.shape[-1]
    p = _pad32(x.float())
    sf = p.abs().amax(-1).clamp(min=1e-4) * (1.0 / 6.0)
    bits = sf.view(torch.int32)
    e = ((bits >> 23) + ((bits & 0x7FFFFF) != 0).int()).clamp(1, 254)
    v = (p / (e << 23).view(torch.float32)[..., None]).flatten(-2)[..., :cols]
    m = v.abs()
    code = (m > 0.25).to(torch.uint8)
    for edge, even in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        code += (m >= edge) if even else (m > edge)
    code |= ((v < 0) & (code > 0)).to(torch.uint8) << 3
    q = (code[..., 0::2] | code[..., 1::2] << 4).view(torch.int8)
    e = torch.nn.functional.pad(e, (0, -e.shape[-1] % 4), value=127).to(torch.uint8)
    return q, e.view(torch.int32)


def _value4(q, sf):
    """The values that 4-bit codes and packed scales stand for."""
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=DEV)
    u = q.view(torch.uint8)
    code = torch.stack((u & 15, u >> 4), -1).flatten(-2)
    scale = (sf.view(torch.uint8).int() << 23).view(torch.float32)
    v = torch.nn.functional.pad(table[code.int()], (0, -code.shape[-1] % 32))
    v = v.view(*v.shape[:-1], -1, 32) * scale[..., :v.shape[-1] // 32, None]
    return v.flatten(-2)[..., :code.shape[-1]]


def prepare(case, seed):
    gen, kind = _gen(seed), case['kind']
    if kind == 'quantise':   # rows of different magnitudes, some scales of zeros only
        x = torch.randn((case['rows'], case['cols']), generator=gen, device=DEV)
        x *= torch.exp(torch.randn((case['rows'], 1), generator=gen, device=DEV))
        _pad = (torch.rand((case['rows'], -(-case['cols'] // 32)), generator=gen, device=DEV) > 0.02).float()
        return dict(kind=kind, x=(x * _pad.repeat_interleave(32, 1)[:, :case['cols']]).bfloat16())
    if kind == 'product':
        out = {'bf16': torch.bfloat16, 'f32': torch.float32}[case['out']]
        seg, total = segments(case)
        g, n, k = case['groups'], case['n'], case['k']
        ends = torch.tensor([e for _, e in seg], dtype=torch.int32, device=DEV)
        # the plan of the plain form: the rows of each group, padded to the longest one's
        most = max(1, max(e - s for s, e in seg))
        first = torch.tensor([s for s, _ in seg], device=DEV)
        idx = first[:, None] + torch.arange(most, device=DEV)[None]
        live = idx < ends[:, None]
        b, b_sf = torch.empty((g, n, k // 2), dtype=torch.int8, device=DEV), torch.empty((g, n, -(-k // 128)), dtype=torch.int32, device=DEV)
        for i in range(g):   # one group at a time: the 32-bit values need not fit beside each other
            b[i], b_sf[i] = _cast4(_randn((n, k), gen, k ** -0.5))
        return dict(kind=kind, ends=ends, alignment=case['alignment'], idx=torch.where(live, idx, total), live=live,
                    a=_cast4(_randn((total, k), gen)), b=(b, b_sf),
                    d=torch.full((total, n), 0.5, dtype=out, device=DEV))
    topk = _routing(case, gen)
    w = torch.rand(topk.shape, generator=gen, device=DEV) if case['weights'] else None
    t, h, rows = case['tokens'], case['hidden'], buffer_rows(case)
    s = dict(kind=kind, w=w)
    if kind == 'dispatch':
        return dict(s, x=_randn((t, h), gen), topk=topk, experts=case['experts'], alignment=case['alignment'],
                    a=torch.full((rows, h), 0.5, dtype=torch.bfloat16, device=DEV))
    s['pos'] = _places(topk, case['experts'], case['alignment'])[0]   # what the dispatch left
    if kind == 'dispatch_grad':
        return dict(s, da=_randn((rows, h), gen, 0.1), da_w=torch.randn(rows, generator=gen, device=DEV) if case['weights'] else None)
    return dict(s, dout=_randn((t, h), gen, 0.1), y=_randn((rows, h), gen),
                dy=torch.full((rows, h), 0.5, dtype=torch.bfloat16, device=DEV))


# ---------------------------------------------------------------- one pass

def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    dg, kind = _deep_gemm(), s['kind']
    if kind == 'dispatch':
        a, _, ends, pos, w = dg.moe_dispatch(s['x'], s['topk'], s['experts'], layout='psum', alignment=s['alignment'],
                                             topk_weights=s['w'], out=s['a'])
        return dict(a=a, ends=ends, pos=pos, w=w)
    if kind == 'dispatch_grad':
        dx, dw = dg.moe_dispatch_backward(s['da'], s['pos'], s['da_w'])
        return dict(dx=dx, dw=dw)
    if kind == 'combine_grad':
        dy, dw = dg.moe_combine_backward(s['dout'], s['y'], s['pos'], s['w'], out=s['dy'])
        return dict(dy=dy, dw=dw)
    if kind == 'quantise':
        q, sf = dg.per_token_cast_to_fp4(s['x'], use_ue8m0=True, gran_k=32, use_packed_ue8m0=True)
        v = dg.cast_back_from_fp4(q, sf, gran_k=32, use_packed_ue8m0=True, dtype=torch.bfloat16)
        return dict(sf=sf, values=v)
    dg.m_grouped_fp4_gemm_nt_ragged(s['a'], s['b'], s['d'], s['ends'], alignment=s['alignment'])
    return s['d']


def _padded(x, idx):
    """The rows x[idx], zeros where idx is past the last row."""
    return torch.nn.functional.pad(x, (0, 0, 0, 1))[idx]


def _run_plain(s):
    kind = s['kind']
    if kind == 'dispatch':
        x, topk, a = s['x'], s['topk'], s['a']
        pos, ends, used = _places(topk, s['experts'], s['alignment'])
        rows = a.shape[0]
        at = torch.where(pos < 0, rows, pos).long().view(-1)   # (one row more takes what is not routed)
        src = torch.full((rows + 1,), -1, device=DEV)
        src[at] = torch.arange(x.shape[0], device=DEV).repeat_interleave(topk.shape[1])
        src = src[:rows, None]
        old = torch.where(torch.arange(rows, device=DEV)[:, None] < used, 0, a)
        a.copy_(torch.where(src >= 0, x[src[:, 0].clamp(min=0)], old))
        w = s['w']
        if w is not None:
            w = torch.zeros(rows + 1, device=DEV).index_put((at,), w.reshape(-1))[:rows]
        return dict(a=a, ends=ends, pos=pos, w=w)
    if kind in ('dispatch_grad', 'combine_grad'):
        pos, routed = s['pos'].long(), s['pos'] >= 0
        at = pos.clamp(min=0)
    if kind == 'dispatch_grad':
        dx = (s['da'][at].float() * routed[..., None]).sum(1).bfloat16()
        return dict(dx=dx, dw=None if s['da_w'] is None else torch.where(routed, s['da_w'][at], 0.0))
    if kind == 'combine_grad':
        dout, dy, w = s['dout'].float()[:, None], s['dy'], s['w']
        each = dout.expand(-1, pos.shape[1], -1) if w is None else dout * w[..., None]
        dy[pos[routed]] = each[routed].bfloat16()
        return dict(dy=dy, dw=None if w is None else torch.where(routed, (dout * s['y'][at].float()).sum(2), 0.0))
    if kind == 'quantise':
        q, sf = _cast4(s['x'])
        return dict(sf=sf, values=_value4(q, sf).bfloat16())
    y = torch.bmm(_padded(_value4(*s['a']), s['idx']), _value4(*s['b']).transpose(1, 2))
    s['d'][s['idx'][s['live']]] = y[s['live']].to(s['d'].dtype)
    return s['d']


# ---------------------------------------------------------------- what it costs, and what is right

def work(case):
    kind = case['kind']
    if kind == 'quantise':   # x in, codes and scales out; codes and scales in, values out
        r, c = case['rows'], case['cols']
        return dict(bytes=r * c * (2 + 2) + 2 * (r * c / 2 + r * -(-c // 128) * 4), flops=4 * r * c)
    if kind == 'product':
        r, n, k, used = case['rows'], case['n'], case['k'], sum(s > 0 for s in sizes(case))
        row = k / 2 + -(-k // 128) * 4
        return dict(bytes=(r + used * n) * row + r * n * (2 if case['out'] == 'bf16' else 4) + 4 * case['groups'],
                    flops=2 * r * n * k)
    t, h, e, a = case['tokens'], case['hidden'], case['experts'], case['alignment']
    k = min(case['topk'], e)
    live = t * k * (1 - case['lost'])
    entries = t * k * (4 + (4 if case['weights'] else 0))
    if kind == 'dispatch':   # (padding: half a piece of the alignment for each expert that has rows)
        padding = min(e, live) * (a - 1) / 2
        return dict(bytes=(t + live + padding) * h * 2 + entries + t * k * 4 + 4 * e + (4 * live if case['weights'] else 0), flops=0)
    if kind == 'dispatch_grad':
        return dict(bytes=(live + t) * h * 2 + entries + (4 * live if case['weights'] else 0), flops=live * h)
    y = live * h * 2 if case['weights'] else 0
    return dict(bytes=(t + live) * h * 2 + y + entries + (t * k * 4 if case['weights'] else 0), flops=3 * live * h)


def _pow2(e):
    """2 ** e in 64 bits, to the bit."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _values64(q, sf):
    """4-bit codes and packed scales in 64 bits, from the formats' definition."""
    cols = q.shape[-1] * 2
    code = torch.empty((*q.shape[:-1], cols), dtype=torch.int16, device=DEV)
    code[..., 0::2], code[..., 1::2] = q.short() & 15, (q.short() >> 4) & 15
    expo, man = (code >> 1) & 3, (code & 1).double()
    mag = torch.where(expo == 0, man * 0.5, (1 + man * 0.5) * _pow2(expo - 1))
    e = sf.contiguous().view(torch.uint8).long() - 127
    return torch.where(code >= 8, -mag, mag) * _pow2(e).repeat_interleave(32, -1)[..., :cols]


def _order(topk, experts, alignment):
    """The rows of the entries and the segments' ends, counted on the host."""
    ids = topk.cpu().tolist()
    count = [0] * experts
    rank = [[-1] * len(r) for r in ids]
    for t, r in enumerate(ids):
        for j, e in enumerate(r):
            if 0 <= e < experts:
                rank[t][j], count[e] = count[e], count[e] + 1
    starts, ends, at = [], [], 0
    for c in count:
        at = -(-at // alignment) * alignment
        starts.append(at)
        at += c
        ends.append(at)
    pos = [[starts[e] + k if k >= 0 else -1 for e, k in zip(r, q)] for r, q in zip(ids, rank)]
    used = -(-at // alignment) * alignment
    return torch.tensor(pos, device=DEV), torch.tensor(ends, dtype=torch.int32, device=DEV), used


def exact(case, seed):
    s = prepare(case, seed)
    kind = s['kind']
    if kind == 'product':
        seg, _ = segments(case)
        d, a = s['d'].double(), _values64(*s['a'])
        for i, (lo, hi) in enumerate(seg):
            if hi > lo:
                d[lo:hi] = a[lo:hi] @ _values64(s['b'][0][i], s['b'][1][i]).T.contiguous()
        return d
    if kind == 'quantise':
        x = s['x'].double()
        rows, cols = x.shape
        wide = torch.zeros((rows, -(-cols // 32) * 32), dtype=torch.float64, device=DEV)
        wide[:, :cols] = x
        wide = wide.view(rows, -1, 32)
        ratio = wide.abs().amax(2).clamp(min=float(torch.tensor(1e-4, dtype=torch.float32)))
        ratio = (ratio * float(torch.tensor(1 / 6, dtype=torch.float32))).float().double()   # a 32-bit product
        part, e = torch.frexp(ratio)   # part in [1/2, 1)
        e = torch.where(part == 0.5, e - 1, e)
        v = wide / _pow2(e)[:, :, None]
        _, top = torch.frexp(v)
        step = _pow2((top - 1).clamp(min=0) - 1)   # of e2m1 around v: 1/2 below 2, 1 below 4, 2 from there
        q = (torch.round(v / step) * step).clamp(-6, 6)
        words = torch.full((rows, -(-cols // 128) * 4), 127, dtype=torch.uint8, device=DEV)
        words[:, :e.shape[1]] = (e + 127).to(torch.uint8)
        return dict(sf=words.view(torch.int32), values=(q * _pow2(e)[:, :, None]).reshape(rows, -1)[:, :cols])
    if kind == 'dispatch':
        pos, ends, used = _order(s['topk'], s['experts'], s['alignment'])
        t, j = torch.nonzero(pos >= 0, as_tuple=True)
        a, rows = s['a'].double(), s['a'].shape[0]
        a[:used] = 0
        a[pos[t, j]] = s['x'].double()[t]
        w = None
        if s['w'] is not None:
            w = torch.zeros(rows, dtype=torch.float64, device=DEV)
            w[pos[t, j]] = s['w'].double()[t, j]
        return dict(a=a, ends=ends, pos=pos.int(), w=w)
    pos = s['pos'].long()
    t, j = torch.nonzero(pos >= 0, as_tuple=True)
    if kind == 'dispatch_grad':
        dx = torch.zeros((case['tokens'], case['hidden']), dtype=torch.float64, device=DEV)
        for slot in range(pos.shape[1]):
            live = pos[:, slot] >= 0
            dx[live] += s['da'][pos[live, slot]].double()
        dw = None
        if s['da_w'] is not None:
            dw = torch.zeros(pos.shape, dtype=torch.float64, device=DEV)
            dw[t, j] = s['da_w'].double()[pos[t, j]]
        return dict(dx=dx, dw=dw)
    dy, dw, w = s['dy'].double(), None, s['w']
    if w is not None:
        dw = torch.zeros(pos.shape, dtype=torch.float64, device=DEV)
    for slot in range(pos.shape[1]):
        live = pos[:, slot] >= 0
        g = s['dout'][live].double()
        dy[pos[live, slot]] = g if w is None else g * w[live, slot].double()[:, None]
        if w is not None:
            dw[live, slot] = (g * s['y'][pos[live, slot]].double()).sum(1)
    return dict(dy=dy, dw=dw)
