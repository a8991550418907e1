"""Dispatch of BF16 and 4-bit rows, its gradient and the gradient of the combination, against plain
counting on the host and sums in 64 bits.

Dispatch copies: bit for bit. Sums (ragged.py): half a step of the result's type, plus half a step
2^-24 of FP32 for each addition or product on a value's way, of the magnitudes' sum.
"""
import numpy as np
import pytest
import torch

import deep_gemm
from fp4_ragged import operand
from ragged import DEV, bits, check, rounding

pytestmark = pytest.mark.gpu


def routing(t, k, e, seed, lost=0.1, again=False):
    """Experts of each slot, some not routed; `again`: the same expert may come twice to a token."""
    rng = np.random.default_rng(seed)
    idx = rng.integers(0, e, (t, k)) if again or k > e else np.stack([rng.permutation(e)[:k] for _ in range(t)]).reshape(t, k)
    return torch.from_numpy(np.where(rng.random((t, k)) < lost, -1, idx).astype(np.int32))


def places(idx, e, alignment):
    """pos, segment starts and ends by counting, token after token."""
    count, rank = [0] * e, torch.full(idx.shape, -1, dtype=torch.int64)
    for t, row in enumerate(idx.tolist()):
        for j, x in enumerate(row):
            if 0 <= x < e:
                rank[t, j], count[x] = count[x], count[x] + 1
    starts, ends, at = [], [], 0
    for c in count:
        at = -(-at // alignment) * alignment
        starts.append(at)
        at += c
        ends.append(at)
    live = rank >= 0
    pos = torch.where(live, rank + torch.tensor(starts)[idx.clamp(0, e - 1).long()], -1)
    return pos, starts, ends, -(-at // alignment) * alignment


def tokens(t, h, seed, pad=0, scale=1.0):
    x = (torch.randn((t, h), generator=torch.Generator().manual_seed(seed)) * scale).bfloat16()
    wide = torch.full((t, h + pad), float('nan'), dtype=torch.bfloat16)
    wide[:, :h] = x
    return wide.to(DEV)[:, :h], x


SHAPES = [(1, 1, 1, 8, 1), (1, 8, 32, 2048, 16), (4, 8, 8, 520, 1), (3, 2, 4, 64, 3), (33, 6, 64, 1024, 16), (64, 4, 256, 136, 128),
          (65, 8, 16, 2056, 1), (300, 16, 20, 264, 1), (777, 6, 64, 128, 7), (1030, 2, 1024, 64, 16), (2000, 8, 256, 72, 16),
          (5000, 8, 128, 40, 1), (700, 3, 5, 8200, 48), (20000, 2, 1000, 16, 1)]


@pytest.mark.parametrize('t,k,e,h,alignment', SHAPES)
@pytest.mark.parametrize('ids', [torch.int32, torch.int64])
def test_dispatch_bf16_psum(t, k, e, h, alignment, ids):
    print(f't={t} k={k} e={e} h={h} alignment={alignment}', flush=True)
    idx = routing(t, k, e, t + k, again=t % 2 == 0)
    x, x0 = tokens(t, h, t, pad=8 * (t % 3))
    w = torch.rand((t, k), generator=torch.Generator().manual_seed(1))
    pos, starts, ends, used = places(idx, e, alignment)
    a, sf, gl, got, rw = deep_gemm.moe_dispatch(x, idx.to(ids).to(DEV), e, layout='psum', alignment=alignment, topk_weights=w.to(DEV))
    assert sf is None and a.dtype == torch.bfloat16
    assert torch.equal(got.cpu().long(), pos)
    assert gl.tolist() == ends
    rows = torch.zeros((used, h), dtype=torch.bfloat16)
    weights = torch.zeros(a.shape[0])
    live = pos >= 0
    rows[pos[live]] = x0[live.nonzero()[:, 0]]
    weights[pos[live]] = w[live]
    assert torch.equal(bits(a[:used].cpu()), bits(rows))
    assert torch.equal(rw.cpu(), weights)


@pytest.mark.parametrize('t,k,e,h', [(1, 1, 4, 8), (100, 2, 8, 512), (1000, 8, 32, 1024), (3000, 6, 256, 40)])
@pytest.mark.parametrize('layout', ['contiguous', 'masked'])
def test_dispatch_bf16_other_layouts(t, k, e, h, layout):
    idx = routing(t, k, e, 3)
    x, x0 = tokens(t, h, 4)
    w = torch.rand((t, k), generator=torch.Generator().manual_seed(1))
    if layout == 'contiguous':
        pos, starts, ends, used = places(idx, e, 32)
        a, _, gl, got, rw = deep_gemm.moe_dispatch(x, idx.to(DEV), e, layout=layout, alignment=32, topk_weights=w.to(DEV))
        want = torch.full((a.shape[0],), -1, dtype=torch.int32)
        for g, (s, n) in enumerate(zip(starts, ends)):
            want[s:n] = g
        assert torch.equal(gl.cpu(), want)
        flat = a
    else:
        max_m = max(1, t * k // e)
        a, _, gl, got, rw = deep_gemm.moe_dispatch(x, idx.to(DEV), e, layout=layout, max_m=max_m, topk_weights=w.to(DEV))
        first, starts, ends, _ = places(idx, e, 1)
        rank = first - torch.tensor(starts)[idx.clamp(min=0).long()]
        pos = torch.where((idx >= 0) & (rank < max_m), idx.long() * max_m + rank, -1)
        assert gl.tolist() == [min(n - s, max_m) for s, n in zip(starts, ends)]
        flat, rw = a.reshape(-1, h), rw.reshape(-1)
    assert torch.equal(got.cpu().long(), pos)
    live = pos >= 0
    assert torch.equal(bits(flat.cpu()[pos[live]]), bits(x0[live.nonzero()[:, 0]]))
    assert torch.equal(rw.cpu()[pos[live]], w[live])


@pytest.mark.parametrize('t,k,e,h,alignment', [(1, 1, 1, 32, 1), (4, 8, 32, 2048, 16), (65, 6, 16, 416, 1), (1500, 8, 64, 1056, 16)])
@pytest.mark.parametrize('layout', ['rows', 'columns'])
def test_dispatch_of_4_bit_rows(t, k, e, h, alignment, layout):
    idx = routing(t, k, e, 5)
    (q, sf), _ = operand((t, h), 6, layout=layout)
    pos, starts, ends, used = places(idx, e, alignment)
    a, a_sf, gl, got, rw = deep_gemm.moe_dispatch((q, sf), idx.to(DEV), e, layout='psum', alignment=alignment)
    assert rw is None and gl.tolist() == ends and torch.equal(got.cpu().long(), pos)
    live = pos >= 0
    for src, dst in ((q, a), (sf, a_sf)):
        want = torch.zeros((used, src.shape[1]), dtype=src.dtype)
        want[pos[live]] = src.cpu()[live.nonzero()[:, 0]]
        assert torch.equal(dst[:used].cpu(), want)


def test_dispatch_into_given_rows():
    """`out` keeps what lies past the segments, and may have more rows and longer ones."""
    idx = routing(70, 4, 8, 7, lost=0.3)
    x, x0 = tokens(70, 264, 8)
    pos, _, ends, used = places(idx, 8, 16)
    room = torch.full((500, 280), 7.0, dtype=torch.bfloat16, device=DEV)
    a, _, gl, got, _ = deep_gemm.moe_dispatch(x, idx.to(DEV), 8, layout='psum', alignment=16, out=room[:, :264])
    assert a.data_ptr() == room.data_ptr() and torch.equal(got.cpu().long(), pos)
    live = pos >= 0
    want = torch.full((500, 280), 7.0, dtype=torch.bfloat16)
    want[:used, :264] = 0
    want[pos[live], :264] = x0[live.nonzero()[:, 0]]
    assert torch.equal(bits(room.cpu()), bits(want))
    (q, sf), _ = operand((70, 256), 9)
    q8 = torch.randn((70, 256), device=DEV).to(torch.float8_e4m3fn)
    s8 = torch.rand((70, 2), device=DEV)
    for data, out in (((q, sf), (torch.zeros((500, 128), dtype=torch.int8, device=DEV), torch.zeros((500, 2), dtype=torch.int32, device=DEV))),
                      ((q8, s8), (torch.zeros((500, 256), device=DEV).to(torch.float8_e4m3fn), torch.zeros((500, 2), device=DEV)))):
        a, a_sf, *_ = deep_gemm.moe_dispatch(data, idx.to(DEV), 8, layout='psum', alignment=16, out=out)
        assert a.data_ptr() == out[0].data_ptr() and a_sf.data_ptr() == out[1].data_ptr()
        assert torch.equal(a.view(torch.int8).cpu()[pos[live]], data[0].view(torch.int8).cpu()[live.nonzero()[:, 0]])
        assert torch.equal(a_sf.cpu()[pos[live]], data[1].cpu()[live.nonzero()[:, 0]])


@pytest.mark.parametrize('kind', ['none', 'one', 'last'])
@pytest.mark.parametrize('t', [1, 50, 3000])
def test_dispatch_unusual_routings(kind, t):
    """No token routed, all to one expert, all to the last one from the second slot."""
    e, k = 16, 3
    idx = torch.full((t, k), -1, dtype=torch.int32)
    if kind == 'one':
        idx[:] = 5
    elif kind == 'last':
        idx[:, 1] = e - 1
        idx[:, 2] = 1 << 20   # (no expert)
    x, x0 = tokens(t, 64, 1)
    pos, _, ends, used = places(torch.where(idx < e, idx, -1), e, 16)
    a, _, gl, got, rw = deep_gemm.moe_dispatch(x, idx.to(DEV), e, layout='psum', alignment=16, topk_weights=torch.ones((t, k), device=DEV))
    assert torch.equal(got.cpu().long(), pos) and gl.tolist() == ends
    live = pos >= 0
    assert torch.equal(bits(a.cpu()[pos[live]]), bits(x0[live.nonzero()[:, 0]]))
    assert rw.sum().item() == live.sum().item()


def test_dispatch_no_tokens():
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV)
    a, _, gl, pos, rw = deep_gemm.moe_dispatch(x, torch.empty((0, 2), dtype=torch.int32, device=DEV), 4, layout='psum', alignment=1,
                                               topk_weights=torch.empty((0, 2), device=DEV))
    assert a.shape == (0, 64) and pos.shape == (0, 2) and gl.tolist() == [0] * 4


# ---------------------------------------------------------------- gradients

def rows_of(pos, rows, h, seed, masked=0, scale=1.0):
    """Expert rows (NaN where no entry of pos points), in NaN-padded memory, and their values."""
    v = (torch.randn((rows, h), generator=torch.Generator().manual_seed(seed)) * scale).bfloat16()
    hit = torch.zeros(rows, dtype=torch.bool)
    hit[pos[pos >= 0]] = True
    v[~hit] = float('nan')
    wide = torch.full((rows, h + 8), float('nan'), dtype=torch.bfloat16)
    wide[:, :h] = v
    dev = wide.to(DEV)[:, :h]
    return (dev.view(masked, -1, h) if masked else dev), v, hit


GRADS = [(1, 1, 1, 8), (1, 8, 32, 2048), (4, 8, 8, 520), (33, 6, 64, 1024), (65, 9, 16, 2056), (300, 16, 20, 264), (777, 6, 64, 128),
         (130, 2, 8, 512), (50, 8, 16, 7168), (3000, 8, 32, 16), (20, 3, 5, 1544)]


def setup(t, k, e, layout):
    idx = routing(t, k, e, t * k, again=True)
    if layout == 'masked':
        max_m = max(1, t * k // e)
        x, _ = tokens(t, 8, 0)
        pos = deep_gemm.moe_dispatch(x, idx.to(DEV), e, layout='masked', max_m=max_m)[3]
        return pos, pos.cpu().long(), e * max_m, e
    pos, *_, used = places(idx, e, 16)
    return pos.int().to(DEV), pos, used + 3, 0


@pytest.mark.parametrize('t,k,e,h', GRADS)
@pytest.mark.parametrize('layout', ['psum', 'masked'])
def test_dispatch_backward(t, k, e, h, layout):
    print(f't={t} k={k} e={e} h={h}', flush=True)
    pos, at, rows, masked = setup(t, k, e, layout)
    d, v, _ = rows_of(at, rows, h, 1, masked)
    dw_rows = torch.randn(rows, generator=torch.Generator().manual_seed(2))
    dx, dw = deep_gemm.moe_dispatch_backward(d, pos, dw_rows.to(DEV))
    live = at >= 0
    each = torch.where(live[..., None], v.double()[at.clamp(min=0)], 0.0)
    ref, mag = each.sum(1), each.abs().sum(1)
    check(dx, ref, rounding(torch.bfloat16, ref) + (k - 1) * 2.0 ** -24 * mag * (1 + 2.0 ** -8), 'dx')
    assert torch.equal(dw.cpu(), torch.where(live, dw_rows[at.clamp(min=0)], 0.0))
    again, none = deep_gemm.moe_dispatch_backward(d, pos)
    assert none is None and torch.equal(bits(again), bits(dx))


@pytest.mark.parametrize('t,k,e,h', GRADS)
@pytest.mark.parametrize('layout', ['psum', 'masked'])
def test_combine_backward(t, k, e, h, layout):
    print(f't={t} k={k} e={e} h={h}', flush=True)
    pos, at, rows, masked = setup(t, k, e, layout)
    y, v, hit = rows_of(at, rows, h, 1, masked)
    dout, g = tokens(t, h, 3, pad=16)
    w = torch.randn((t, k), generator=torch.Generator().manual_seed(4))
    live = at >= 0
    dy, dw = deep_gemm.moe_combine_backward(dout, y, pos, w.to(DEV))
    assert dy.shape == y.shape and dy.dtype == torch.bfloat16
    ref = torch.zeros((rows, h), dtype=torch.float64)
    ref[at[live]] = (g.double()[:, None] * w.double()[..., None])[live]
    check(dy.reshape(rows, h), ref, (1 + 2.0 ** -8) * 2.0 ** -24 * ref.abs() + rounding(torch.bfloat16, ref), 'dy')
    assert not dy.reshape(rows, h)[(~hit).to(DEV)].any()
    terms = torch.where(live[..., None], g.double()[:, None] * torch.nan_to_num(v.double()[at.clamp(min=0)]), 0.0)
    # a product passes its lane's additions (8 for each 512 to 2048 columns), six between lanes and three between waves
    length = 8 * -(-h // 512) + 10
    check(dw, terms.sum(2), length * 2.0 ** -24 * terms.abs().sum(2) + rounding(torch.float32, terms.sum(2)), 'dw')
    # without weights: copies, y is not read
    dy, none = deep_gemm.moe_combine_backward(dout, torch.full_like(y, float('nan')), pos)
    want = torch.zeros((rows, h), dtype=torch.bfloat16)
    want[at[live]] = g[live.nonzero()[:, 0]]
    assert none is None and torch.equal(bits(dy.reshape(rows, h).cpu()), bits(want))


def test_combine_backward_into_given_rows():
    """`out` keeps the rows that nothing names; y itself may be it."""
    pos, at, rows, _ = setup(90, 4, 8, 'psum')
    y, v, hit = rows_of(at, rows, 136, 1)
    dout, _ = tokens(90, 136, 2)
    w = torch.rand((90, 4), generator=torch.Generator().manual_seed(3)).to(DEV)
    want, dw = deep_gemm.moe_combine_backward(dout, y, pos, w)
    out = torch.full((rows, 160), 7.0, dtype=torch.bfloat16, device=DEV)
    got, dw2 = deep_gemm.moe_combine_backward(dout, y, pos, w, out=out[:, 8:144])
    assert got.data_ptr() == out[:, 8:144].data_ptr() and torch.equal(bits(dw), bits(dw2))
    kept = torch.full_like(out, 7.0)
    kept[:, 8:144][hit.to(DEV)] = want[hit.to(DEV)]
    assert torch.equal(bits(out), bits(kept))
    got, dw3 = deep_gemm.moe_combine_backward(dout, y, pos, w, out=y)
    assert torch.equal(bits(y[hit.to(DEV)]), bits(want[hit.to(DEV)])) and torch.equal(bits(dw), bits(dw3))
    assert torch.isnan(y[(~hit).to(DEV)]).all()


def test_gradients_against_differences():
    """Dispatch and combination are linear in x, y and w each: the change of sum(out * dout) along a
    direction is the gradient's product with it, up to the gradients' own rounding."""
    t, k, e, h = 37, 4, 8, 264
    idx = routing(t, k, e, 11)
    pos, _, _, used = places(idx, e, 16)
    gen = torch.Generator().manual_seed(12)
    normal = lambda *s: torch.randn(s, generator=gen).bfloat16()
    y, dout, dy_dir, x_dir, drows = normal(used, h), normal(t, h), normal(used, h), normal(t, h), normal(used, h)
    w, w_dir = torch.rand((t, k), generator=gen), torch.randn((t, k), generator=gen)
    live, at = pos >= 0, pos.clamp(min=0)

    def combined(y, w):   # sum(out * dout) in 64 bits
        out = (torch.where(live[..., None], y.double()[at], 0.0) * w.double()[..., None]).sum(1)
        return (out * dout.double()).sum()

    dy, dw = deep_gemm.moe_combine_backward(dout.to(DEV), y.to(DEV), pos.int().to(DEV), w.to(DEV))
    step = combined(y.double() + dy_dir.double(), w) - combined(y, w)
    got = dy.double().cpu() * dy_dir.double()
    assert abs(got.sum() - step) <= 2.0 ** -8 * got.abs().sum() * 1.01
    step = combined(y, w.double() + w_dir.double()) - combined(y, w)
    got = dw.double().cpu() * w_dir.double()
    mag = (torch.where(live[..., None], y.double()[at], 0.0) * dout.double()[:, None]).abs().sum(2) * w_dir.double().abs()
    assert abs(got.sum() - step) <= (8 * 1 + 12) * 2.0 ** -24 * mag.sum() * 1.01

    def dispatched(x):   # sum(rows * drows)
        rows = torch.zeros((used, h), dtype=torch.float64)
        rows[pos[live]] = x.double()[live.nonzero()[:, 0]]
        return (rows * drows.double()).sum()

    dx, _ = deep_gemm.moe_dispatch_backward(drows.to(DEV), pos.int().to(DEV))
    got = dx.double().cpu() * x_dir.double()
    step = dispatched(x_dir)
    slack = (torch.where(live[..., None], drows.double()[at], 0.0).abs().sum(1) * x_dir.double().abs()).sum() * 3 * 2.0 ** -24
    assert abs(got.sum() - step) <= 2.0 ** -8 * got.abs().sum() * 1.01 + slack


def test_rows_that_are_none_are_skipped():
    """Entries of pos past the rows, or far below zero, count as not routed."""
    pos = torch.tensor([[0, 5, -7], [1 << 30, 2, -(1 << 31)]], dtype=torch.int32, device=DEV)
    d = torch.arange(5 * 8, dtype=torch.float32, device=DEV).view(5, 8).bfloat16()
    dx, dw = deep_gemm.moe_dispatch_backward(d, pos, torch.arange(5.0, device=DEV) + 1)
    assert torch.equal(dx, d[[0, 2]]) and dw.tolist() == [[1, 0, 0], [0, 3, 0]]
    dy, dw = deep_gemm.moe_combine_backward(torch.ones((2, 8), dtype=torch.bfloat16, device=DEV), d, pos,
                                            torch.full((2, 3), 2.0, device=DEV))
    assert torch.equal(dy[[0, 2]], torch.full((2, 8), 2.0, dtype=torch.bfloat16, device=DEV)) and not dy[[1, 3, 4]].any()
    assert dw.tolist() == [[28, 0, 0], [0, 156, 0]]


def test_weights_of_any_strides():
    pos, at, rows, _ = setup(50, 4, 8, 'psum')
    y, _, _ = rows_of(at, rows, 72, 1)
    dout, _ = tokens(50, 72, 2)
    w = torch.rand((50, 4), generator=torch.Generator().manual_seed(3)).to(DEV)
    want = deep_gemm.moe_combine_backward(dout, y, pos, w)
    wide = torch.full((4, 60), float('nan'), device=DEV)
    wide[:, :50] = w.t()
    got = deep_gemm.moe_combine_backward(dout, y, pos, wide[:, :50].t())
    assert all(torch.equal(bits(a), bits(b)) for a, b in zip(want, got))


def test_non_finite_gradients_stay_with_their_tokens():
    pos, at, rows, _ = setup(40, 4, 8, 'psum')
    d, v, _ = rows_of(at, rows, 64, 1)
    clean, _ = deep_gemm.moe_dispatch_backward(d, pos)
    t, j = next((t, j) for t in range(40) for j in range(4) if at[t, j] >= 0)
    d[at[t, j], 5] = float('inf')
    dx, _ = deep_gemm.moe_dispatch_backward(d, pos)
    assert dx[t, 5] == float('inf')
    dx[t, 5] = clean[t, 5]
    assert torch.equal(bits(dx), bits(clean))


def test_offsets_past_32_bits():
    """Rows whose bytes lie past 2^32."""
    rows, h = 600000, 4096
    y = torch.zeros((rows, h), dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([[0, rows - 1], [rows - 2, 5]], dtype=torch.int32, device=DEV)
    y[at.long().view(-1)] = torch.randn((4, h), device=DEV).bfloat16()
    dx, _ = deep_gemm.moe_dispatch_backward(y, at)
    for t in range(2):
        ref = y[at[t].long()].double().sum(0).cpu()
        check(dx[t], ref, rounding(torch.bfloat16, ref) + 2.0 ** -24 * y[at[t].long()].double().abs().sum(0).cpu(), f'token {t}')
    dout = torch.randn((2, h), device=DEV).bfloat16()
    w = torch.tensor([[1.0, 2.0], [4.0, 0.5]], device=DEV)
    deep_gemm.moe_combine_backward(dout, y, at, w, out=y)
    for t in range(2):
        for j in range(2):
            assert torch.equal(y[at[t, j]], dout[t] * w[t, j].bfloat16())


def test_graphs_of_dispatch_and_gradients():
    """Captured calls follow their inputs; two graphs do not share anything."""
    t, k, e, h = 60, 4, 16, 264
    x = torch.zeros((t, h), dtype=torch.bfloat16, device=DEV)
    idx = torch.full((t, k), -1, dtype=torch.int32, device=DEV)
    w = torch.zeros((t, k), device=DEV)

    def step():
        a, _, ends, pos, rw = deep_gemm.moe_dispatch(x, idx, e, layout='psum', alignment=1, topk_weights=w)
        dx, dw = deep_gemm.moe_dispatch_backward(a, pos, rw)
        dy, dw2 = deep_gemm.moe_combine_backward(x, a, pos, w)
        return a, ends, pos, rw, dx, dw, dy, dw2

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    for seed in range(3):
        x.copy_(tokens(t, h, seed)[1])
        idx.copy_(routing(t, k, e, seed, lost=0.0))
        w.copy_(torch.rand((t, k), generator=torch.Generator().manual_seed(seed)))
        want = step()
        for graph, out in graphs:
            graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(out, want):
                assert torch.equal(bits(a), bits(b))


# Sizes at which the dispatch changes its form (one or four tokens a workgroup, one launch or three), around
# the workgroups' last token, and ids that lie apart.
@pytest.mark.parametrize('t', [3, 361, 362, 363, 365, 2045, 2048, 2049])
@pytest.mark.parametrize('layout,alignment', [('psum', 1), ('psum', 48), ('contiguous', 16), ('masked', 0)])
def test_dispatch_forms(t, layout, alignment):
    print(f't={t} {layout}', flush=True)
    k, e, h = 8, 1024 if t > 1000 else 40, 24
    idx = routing(t, k, e, t, again=True)
    x, x0 = tokens(t, h, t, pad=8)
    w = torch.rand((t, k), generator=torch.Generator().manual_seed(1))
    max_m = max(1, t * k // e)
    wide = torch.full((t, 3 * k), 1, dtype=torch.int64)
    wide[:, ::3] = idx
    wide_w = torch.full((k, t), float('nan'))
    wide_w[:] = w.t()
    more = dict(max_m=max_m) if layout == 'masked' else dict(alignment=alignment)
    a, _, gl, got, rw = deep_gemm.moe_dispatch(x, wide.to(DEV)[:, ::3], e, layout=layout, topk_weights=wide_w.to(DEV).t(), **more)
    if layout == 'masked':
        first, starts, ends, _ = places(idx, e, 1)
        rank = first - torch.tensor(starts)[idx.clamp(min=0).long()]
        pos = torch.where((idx >= 0) & (rank < max_m), idx.long() * max_m + rank, -1)
        assert gl.tolist() == [min(n - s, max_m) for s, n in zip(starts, ends)]
    else:
        pos, starts, ends, used = places(idx, e, alignment)
        if layout == 'psum':
            assert gl.tolist() == ends
        else:
            want = torch.full((a.shape[0],), -1, dtype=torch.int32)
            for g, (s, n) in enumerate(zip(starts, ends)):
                want[s:n] = g
            assert torch.equal(gl.cpu(), want)
    live = pos >= 0
    assert torch.equal(got.cpu().long(), pos)
    flat, rw = a.reshape(-1, h).cpu(), rw.reshape(-1).cpu()
    assert torch.equal(bits(flat[pos[live]]), bits(x0[live.nonzero()[:, 0]]))
    assert torch.equal(rw[pos[live]], w[live])
    if layout != 'masked':
        rest = torch.ones(flat.shape[0], dtype=torch.bool)
        rest[pos[live]] = False
        assert not rw[rest].any()
        rest[used:] = False
        assert not flat[rest].any()


@pytest.mark.parametrize('layout', ['psum', 'contiguous', 'masked'])
def test_dispatch_no_tokens_of_any_layout(layout):
    x = torch.empty((0, 64), dtype=torch.bfloat16, device=DEV)
    a, _, gl, pos, rw = deep_gemm.moe_dispatch(x, torch.empty((0, 2), dtype=torch.int32, device=DEV), 4, layout=layout, alignment=16, max_m=8,
                                               topk_weights=torch.empty((0, 2), device=DEV))
    assert pos.shape == (0, 2) and not (gl.cpu() > 0).any()
    if layout != 'masked':
        assert not rw.any()


def test_dispatches_beside_each_other():
    """Calls on two streams, and two graphs replayed on them, share nothing."""
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    t, k, e, h = 3000, 8, 64, 264
    sets = [(tokens(t, h, i)[0], routing(t, k, e, i).to(DEV)) for i in range(2)]
    run = lambda x, idx: deep_gemm.moe_dispatch(x, idx, e, layout='psum', alignment=1)
    want = [run(*s) for s in sets]
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = run(*s)
        graphs.append((graph, out))
    for _ in range(5):
        got = []
        for (graph, out), stream, s in zip(graphs, streams, sets):
            with torch.cuda.stream(stream):
                graph.replay()
                got.append(run(*s))
        torch.cuda.synchronize()
        for (_, out), eager, ref in zip(graphs, got, want):
            used = int(ref[2][-1])
            for res in (out, eager):
                assert torch.equal(res[3], ref[3]) and torch.equal(res[2], ref[2])
                assert torch.equal(bits(res[0][:used]), bits(ref[0][:used]))


@pytest.mark.parametrize('t,k,h', [(3200, 16, 1024), (6300, 1, 8192), (513, 2, 4104), (512, 2, 4104), (512, 3, 2056), (100, 2, 16392)])
def test_gradients_of_many_and_of_wide_rows(t, k, h):
    """The forms for more than 100 MB of rows, and for up to and above 512 tokens."""
    print(f't={t} k={k} h={h}', flush=True)
    gen = torch.Generator().manual_seed(t)
    pos = torch.randperm(t * k, generator=gen).view(t, k)
    pos[torch.rand((t, k), generator=gen) < 0.1] = -1
    rows = torch.randn((t * k, h), generator=gen).bfloat16()
    dout = torch.randn((t, h), generator=gen).bfloat16()
    w = torch.randn((t, k), generator=gen)
    at, y = pos.int().to(DEV), rows.to(DEV)
    dx, _ = deep_gemm.moe_dispatch_backward(y, at)
    dy, dw = deep_gemm.moe_combine_backward(dout.to(DEV), y, at, w.to(DEV))
    some = torch.randint(0, t, (150,), generator=gen)
    some[:3] = torch.tensor([0, t // 2, t - 1])
    live = pos[some] >= 0
    each = torch.where(live[..., None], rows[pos[some].clamp(min=0)].double(), 0.0)
    ref, mag = each.sum(1), each.abs().sum(1)
    check(dx[some.to(DEV)], ref, rounding(torch.bfloat16, ref) + (k - 1) * 2.0 ** -24 * mag * (1 + 2.0 ** -8), 'dx')
    terms = each * dout[some].double()[:, None]
    # a product passes its lane's additions, six between lanes and up to fifteen between waves
    length = 8 * -(-h // 512) + 22
    check(dw[some.to(DEV)], terms.sum(2), length * 2.0 ** -24 * terms.abs().sum(2) + rounding(torch.float32, terms.sum(2)), 'dw')
    ref = (dout[some].double()[:, None] * w[some].double()[..., None])[live]
    check(dy.cpu()[pos[some][live]], ref, (1 + 2.0 ** -8) * 2.0 ** -24 * ref.abs() + rounding(torch.bfloat16, ref), 'dy')
    none = torch.ones(t * k, dtype=torch.bool)
    none[pos[pos >= 0]] = False
    assert not dy[none.to(DEV)].any()


@pytest.mark.parametrize('h', [8, 256, 264])
@pytest.mark.parametrize('t', [4099, 8208])
@pytest.mark.parametrize('layout', ['psum', 'masked'])
def test_dispatch_of_many_short_rows(t, h, layout):
    """Several tokens of a wave, the last wave's and workgroup's fewer."""
    k, e = 16, 24
    idx = routing(t, k, e, t)
    x, x0 = tokens(t, h, t)
    w = torch.rand((t, k), generator=torch.Generator().manual_seed(1))
    kw = dict(alignment=16) if layout == 'psum' else dict(max_m=t // 2)
    a, _, gl, got, rw = deep_gemm.moe_dispatch(x, idx.to(DEV), e, layout=layout, topk_weights=w.to(DEV), **kw)
    pos, starts, ends, used = places(idx, e, 16 if layout == 'psum' else 1)
    if layout == 'masked':
        rank = pos - torch.tensor(starts)[idx.clamp(min=0).long()]
        pos = torch.where((idx >= 0) & (rank < t // 2), idx.long() * (t // 2) + rank, -1)
        assert gl.tolist() == [min(n - s, t // 2) for s, n in zip(starts, ends)]
    else:
        assert gl.tolist() == ends
    live = pos >= 0
    assert torch.equal(got.cpu().long(), pos)
    assert torch.equal(bits(a.reshape(-1, h).cpu()[pos[live]]), bits(x0[live.nonzero()[:, 0]]))
    assert torch.equal(rw.reshape(-1).cpu()[pos[live]], w[live])


def test_dispatch_of_8_bit_rows_far_apart():
    """Segments at multiples of 2^21 rows, and rows of more than 2^30 bytes."""
    idx = torch.tensor([[1, 0], [1, -1], [-1, 1]], dtype=torch.int32)
    x = torch.arange(3 * 16, dtype=torch.uint8).view(3, 16)
    sf = torch.tensor([[1.0], [2.0], [3.0]])
    a, a_sf, ends, got, _ = deep_gemm.moe_dispatch((x.view(torch.float8_e4m3fn).to(DEV), sf.to(DEV)), idx.to(DEV), 2, layout='psum',
                                                   alignment=1 << 21)
    pos, _, want, _ = places(idx, 2, 1 << 21)
    live = pos >= 0
    assert torch.equal(got.cpu().long(), pos) and ends.tolist() == want
    assert torch.equal(a.view(torch.uint8)[pos[live].to(DEV)].cpu(), x[live.nonzero()[:, 0]])
    assert torch.equal(a_sf[pos[live].to(DEV)].cpu(), sf[live.nonzero()[:, 0]])
    del a, a_sf
    k = (1 << 30) + 4096 + 16
    wide = torch.zeros((1, k), dtype=torch.uint8, device=DEV)
    at = torch.tensor([0, 1 << 30, k - 1], device=DEV)
    wide[0, at] = torch.tensor([5, 6, 7], dtype=torch.uint8, device=DEV)
    scales = torch.zeros((1, -(-k // 128)), device=DEV)
    scales[0, -1] = 9.0
    a, a_sf, count, got, _ = deep_gemm.moe_dispatch((wide.view(torch.float8_e4m3fn), scales), torch.tensor([[2]], dtype=torch.int32, device=DEV),
                                                    3, layout='masked', max_m=1)
    assert count.tolist() == [0, 0, 1] and got.tolist() == [[2]]
    assert torch.equal(a.view(torch.uint8)[2], wide) and torch.equal(a_sf[2], scales)
