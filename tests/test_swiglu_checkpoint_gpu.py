"""SwiGLU with an 8-bit checkpoint and its backward pass against the formulas in 64 bits,
and a whole MoE layer's training step made of the BF16 expert operators.

Bounds: exp(-g) is 2^(-g log2 e) from an FP32 product, off by |g| 2^-23 relative to itself,
and the steps after it (exp2, sum, reciprocal, products) by a few steps more: factors of s
are within (|g| + 8) 2^-23, and results rounded to BF16 within half its step more. s + g s
(1 - s) is a sum of terms of either sign: its bound goes by their magnitudes. Far below
zero (g < -87.3) s leaves FP32's normal range and may count as zero: h is then off by
2^-126 |g u w| (1.03e-36 at g = -88, u = w = 1, where s = 2^-126.9), beside 1e-37 for
results that are themselves below BF16's normal range.
"""
import numpy as np
import pytest
import torch

import deep_gemm
import generators as gen
from oracle import quant as oquant
from ragged import DEV, bits, check, ends_of, matrix, segments

pytestmark = pytest.mark.gpu
HALF = 2.0 ** -8     # half a step of BF16


def steps(g):
    return (g.abs() + 8) * 2.0 ** -23


def sigmoid(g):
    return 1 / (1 + torch.exp(-g))


def forward(gate, up, w, clamp):
    if clamp > 0:
        gate, up = gate.clamp(max=clamp), up.clamp(-clamp, clamp)
    return gate * sigmoid(gate) * up * w


def inputs(m, i, seed, weights=True, scale=3.0, pad=8):
    x, x64 = matrix((m, 2 * i), seed, scale, pad=pad)
    w = torch.rand(m, generator=torch.Generator().manual_seed(seed + 1)) + 0.25 if weights else None
    return x, x64, (w.to(DEV) if weights else None), (w.double()[:, None] if weights else torch.ones(m, 1, dtype=torch.float64))


def oracle_cast(half):
    return oquant.per_token_cast_to_fp8(half, use_ue8m0=True)


def value(q, sf, i):
    """(gate, up) in 64 bits as a checkpoint holds them."""
    q, sf = q.float().double().cpu(), sf.double().cpu()
    p = sf.shape[1] // 2
    wide = lambda s: s.repeat_interleave(128, 1)[:, :i]
    return q[:, :i] * wide(sf[:, :p]), q[:, i:] * wide(sf[:, p:])


SHAPES = [(1, 8), (1, 128), (3, 120), (5, 136), (33, 256), (64, 512), (7, 520), (130, 768), (9, 1032), (17, 2048), (3, 4104)]


@pytest.mark.parametrize('clamp', [0.0, 2.5])
@pytest.mark.parametrize('weights', [True, False])
@pytest.mark.parametrize('m,i', SHAPES)
def test_forward(m, i, weights, clamp):
    print(f'swiglu checkpoint m={m} i={i}', flush=True)
    x, x64, w, w64 = inputs(m, i, m + i, weights, pad=24)
    h, (q, sf) = deep_gemm.moe_swiglu_checkpoint(x, w, clamp_value=clamp)
    torch.cuda.synchronize()
    ref = forward(x64[:, :i], x64[:, i:], w64, clamp)
    check(h, ref, ref.abs() * (HALF + steps(x64[:, :i])) + 1e-37, 'h')
    for k, half in enumerate((x64[:, :i], x64[:, i:])):
        oq, osf = oracle_cast(half.float().numpy())
        assert np.array_equal(q[:, k * i:(k + 1) * i].contiguous().view(torch.uint8).cpu().numpy(), oq)
        parts = sf.shape[1] // 2
        assert np.array_equal(sf[:, k * parts:(k + 1) * parts].cpu().numpy(), osf)


def test_forward_is_the_cast_of_whole_halves():
    """Halves of whole 128-column groups: the checkpoint is per_token_cast_to_fp8(x)."""
    x, _, w, _ = inputs(40, 384, 3)
    x = x.contiguous()
    _, (q, sf) = deep_gemm.moe_swiglu_checkpoint(x, w)
    cq, csf = deep_gemm.per_token_cast_to_fp8(x, use_ue8m0=True)
    assert torch.equal(bits(q), bits(cq)) and torch.equal(sf, csf)


def test_forward_zeros_far_gates_and_non_finite():
    i = 256
    x = torch.zeros((6, 2 * i), dtype=torch.bfloat16)
    x[1, :i], x[1, i:] = -200.0, 1e30          # silu is zero there
    x[2, :i], x[2, i:] = 200.0, -2.0           # and g here
    x[3, 5], x[4, i + 9] = float('nan'), float('inf')
    x[5, :i], x[5, i:] = torch.linspace(-100, 100, i).bfloat16(), 1.0
    h, (q, sf) = deep_gemm.moe_swiglu_checkpoint(x.to(DEV))
    cq, csf = deep_gemm.per_token_cast_to_fp8(x.to(DEV), use_ue8m0=True)
    assert torch.equal(bits(q), bits(cq)) and torch.equal(bits(sf), bits(csf))     # Inf and NaN included
    h = h.float().cpu()
    assert (h[0] == 0).all() and (h[1] == 0).all() and (h[2] == -400.0).all()
    assert torch.isnan(h[3, 5]) and (torch.isnan(h[3]).sum() == 1)
    assert torch.isnan(h[4, 9])                                                    # 0 x Inf
    g = x[5, :i].double()
    ref = forward(g, torch.ones(i, dtype=torch.float64), 1.0, 0.0)
    check(h[5], ref, ref.abs() * (HALF + steps(g)) + 2.0 ** -126 * g.abs() + 1e-37, 'far gates')


def test_row_layout_gives_zero_rows():
    x, _, w, _ = inputs(20, 136, 5)
    layout = torch.tensor([-1 if r % 3 == 0 else r for r in range(20)], dtype=torch.int32, device=DEV)
    x[::3] = float('nan')
    h, (q, sf) = deep_gemm.moe_swiglu_checkpoint(x, w, layout)
    dh = torch.full((20, 136), float('nan'), dtype=torch.bfloat16, device=DEV)
    dh[layout >= 0] = 1.0
    dx, h2, dw = deep_gemm.moe_swiglu_backward(dh, (q, sf), w, layout)
    skipped = layout < 0
    for t in (h, q.float(), dx, h2, dw):
        assert (t[skipped] == 0).all() and torch.isfinite(t.float()).all()
    keep = ~skipped
    h1, (q1, sf1) = deep_gemm.moe_swiglu_checkpoint(x[keep].contiguous(), w[keep])
    assert torch.equal(h[keep], h1) and torch.equal(bits(q[keep]), bits(q1)) and torch.equal(sf[keep], sf1)
    dx1, h3, dw1 = deep_gemm.moe_swiglu_backward(dh[keep].contiguous(), (q1, sf1), w[keep])
    assert torch.equal(dx[keep], dx1) and torch.equal(h2[keep], h3) and torch.equal(dw[keep], dw1)


def backward(gate, up, dh, w64, clamp):
    """The formulas in 64 bits: (dgate, dup, h, dw) and the magnitudes their bounds go by."""
    free_g = free_u = torch.ones_like(gate)
    if clamp > 0:
        free_g, free_u = (gate <= clamp).double(), (up.abs() <= clamp).double()
        gate, up = gate.clamp(max=clamp), up.clamp(-clamp, clamp)
    s = sigmoid(gate)
    act, dy = gate * s, dh * w64
    return (dy * up * (s + act * (1 - s)) * free_g, dy * act * free_u, act * up * w64, (dh * act * up).sum(1),
            (dy * up).abs() * (s + act.abs()), (dh * act * up).abs().sum(1), gate)


@pytest.mark.parametrize('clamp', [0.0, 2.5])
@pytest.mark.parametrize('weights', [True, False])
@pytest.mark.parametrize('m,i', SHAPES)
def test_backward(m, i, weights, clamp):
    print(f'swiglu backward m={m} i={i}', flush=True)
    x, _, w, w64 = inputs(m, i, m + i, weights)
    h, ckpt = deep_gemm.moe_swiglu_checkpoint(x, w, clamp_value=clamp)
    dh, dh64 = matrix((m, i), 77, pad=16)
    dx, h2, dw = deep_gemm.moe_swiglu_backward(dh, ckpt, w, clamp_value=clamp)
    torch.cuda.synchronize()
    gate, up = value(*ckpt, i)
    dg, du, rh, rdw, mag_g, mag_w, g = backward(gate, up, dh64, w64, clamp)
    check(dx[:, :i], dg, dg.abs() * HALF + mag_g * 4 * steps(g) + 1e-37, 'dgate')
    check(dx[:, i:], du, du.abs() * (HALF + steps(g)) + 1e-37, 'dup')
    check(h2, rh, rh.abs() * (HALF + steps(g)) + 1e-37, 'h')
    if weights:    # a lane's i / 64 terms or fewer in order, then six exchanges and three more waves
        check(dw, rdw, mag_w * ((i / 64 + 16) * 2.0 ** -23 + float(steps(g).max())) + 1e-37, 'dw')
    else:
        assert dw is None


def test_backward_against_differences():
    """Difference quotients of L = <dh, h(gate, up, w)> in 64 bits at the checkpoint's values."""
    m, i, clamp = 4, 16, 2.5
    x, _, w, w64 = inputs(m, i, 9)
    _, ckpt = deep_gemm.moe_swiglu_checkpoint(x, w, clamp_value=clamp)
    dh, dh64 = matrix((m, i), 10)
    dx, _, dw = deep_gemm.moe_swiglu_backward(dh, ckpt, w, clamp_value=clamp)
    gate, up = value(*ckpt, i)
    loss = lambda g, u, ww: (dh64 * forward(g, u, ww, clamp))
    step = 2.0 ** -12
    edge = ((gate - clamp).abs() < 2 * step) | ((up.abs() - clamp).abs() < 2 * step)    # no derivative there
    qg = (loss(gate + step, up, w64) - loss(gate - step, up, w64)) / (2 * step)
    qu = (loss(gate, up + step, w64) - loss(gate, up - step, w64)) / (2 * step)
    qw = ((loss(gate, up, w64 + step) - loss(gate, up, w64 - step)) / (2 * step)).sum(1)
    # BF16's half step, and the quotient's step^2 / 6 times a third derivative below 1 of silu
    for got, q, other in ((dx[:, :i], qg, up), (dx[:, i:], qu, gate)):
        off = (got.double().cpu() - q).abs() - (q.abs() * HALF * 1.01 + 1e-6 * (1 + (dh64 * other * w64).abs()))
        assert (off[~edge] <= 0).all()
    assert ((dw.double().cpu() - qw).abs() < 1e-4).all()


def test_backward_recomputes_the_forward_of_what_the_checkpoint_holds():
    """Inputs that e4m3 holds exactly: h comes back to the bit."""
    i = 256
    x = torch.randint(-8, 9, (12, 2 * i), generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    w = torch.rand(12, generator=torch.Generator().manual_seed(2)).to(DEV)
    h, ckpt = deep_gemm.moe_swiglu_checkpoint(x, w)
    _, h2, _ = deep_gemm.moe_swiglu_backward(torch.zeros((12, i), dtype=torch.bfloat16, device=DEV), ckpt, w)
    assert torch.equal(h, h2)


def test_empty_calls():
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)
    h, (q, sf) = deep_gemm.moe_swiglu_checkpoint(z(0, 16))
    assert h.shape == (0, 8) and q.shape == (0, 16) and sf.shape == (0, 2)
    dx, h, dw = deep_gemm.moe_swiglu_backward(z(0, 8), (q, sf), torch.zeros(0, device=DEV))
    assert dx.shape == (0, 16) and dw.shape == (0,)


def test_graph_replays():
    x, _, w, _ = inputs(50, 640, 4)
    dh, _ = matrix((50, 640), 5)
    ref = (deep_gemm.moe_swiglu_checkpoint(x, w), )
    ref = (*ref, deep_gemm.moe_swiglu_backward(dh, ref[0][1], w))
    flat = lambda r: [r[0][0], r[0][1][0], r[0][1][1], *r[1]]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        f = deep_gemm.moe_swiglu_checkpoint(x, w)
        got = (f, deep_gemm.moe_swiglu_backward(dh, f[1], w))
    for _ in range(3):
        for t in flat(got):
            t.view(torch.uint8).fill_(0x55)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(flat(got), flat(ref)):
            assert torch.equal(bits(a), bits(b))


@pytest.mark.parametrize('t,e,topk,hidden,inter', [(1, 4, 2, 128, 128), (90, 6, 2, 256, 136), (300, 16, 4, 384, 256)])
def test_training_step_of_a_layer(t, e, topk, hidden, inter):
    """Dispatch of FP8 tokens, gate/up product, SwiGLU with its checkpoint, down product,
    combine, and back: gradients of both weights, the routing weights and the tokens,
    against the same steps in 64 bits with the checkpoints' values where the backward pass
    reads them. Five roundings to BF16 lie between the inputs and the last gradient, each
    of half a step: 5 x 2^-8 of a result's norm.
    """
    print(f'layer t={t} e={e} topk={topk} hidden={hidden} inter={inter}', flush=True)
    rng = np.random.default_rng(t)
    idx = torch.from_numpy(np.stack([rng.choice(e, size=topk, replace=False) for _ in range(t)]).astype(np.int32)).to(DEV)
    tw = torch.from_numpy(rng.random((t, topk)).astype(np.float32) + 0.1).to(DEV)
    x = gen.to_dev(gen.randn_bf16((t, hidden), 1)).bfloat16()
    w1, w1_64 = matrix((e, 2 * inter, hidden), 2, hidden ** -0.5)
    w2, w2_64 = matrix((e, hidden, inter), 3, inter ** -0.5)
    dout, dout64 = matrix((t, hidden), 4)
    xq = deep_gemm.per_token_cast_to_fp8(x, use_ue8m0=True)
    a, a_sf, ends, pos, rw = deep_gemm.moe_dispatch(xq, idx, e, layout='psum', alignment=16, topk_weights=tw)
    rows = a.shape[0]
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)
    # forward
    rows_in = (a.float() * a_sf.repeat_interleave(128, 1)[:, :hidden]).bfloat16()     # exact: powers of two
    gu, y = bf(rows, 2 * inter), bf(rows, hidden)
    deep_gemm.m_grouped_bf16_gemm_nt_ragged(rows_in, w1, gu, ends, alignment=16)
    h, ckpt = deep_gemm.moe_swiglu_checkpoint(gu, rw)
    deep_gemm.m_grouped_bf16_gemm_nt_ragged(h, w2, y, ends, alignment=16)
    out = deep_gemm.moe_combine(y, pos)
    # backward
    dy, dh, drows = bf(rows, hidden), bf(rows, inter), bf(rows, hidden)
    dy[pos.long().view(-1)] = dout.repeat_interleave(topk, 0)
    dw1, dw2 = torch.empty((e, 2 * inter, hidden), device=DEV), torch.empty((e, hidden, inter), device=DEV)
    deep_gemm.m_grouped_bf16_gemm_nn_ragged(dy, w2, dh, ends, alignment=16)
    dgu, h2, drw = deep_gemm.moe_swiglu_backward(dh, ckpt, rw)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(dy, h2, dw2, ends, alignment=16)
    deep_gemm.m_grouped_bf16_gemm_nn_ragged(dgu, w1, drows, ends, alignment=16)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(dgu, (a, a_sf), dw1, ends, alignment=16)
    dx = deep_gemm.moe_combine(drows, pos)
    torch.cuda.synchronize()

    # the same in 64 bits, expert by expert
    x64 = (xq[0].float() * xq[1].repeat_interleave(128, 1)[:, :hidden]).double().cpu()
    gate_c, up_c = value(*ckpt, inter)
    r_out, r_dx, r_dtw = torch.zeros(t, hidden).double(), torch.zeros(t, hidden).double(), torch.zeros(t, topk).double()
    r_dw1, r_dw2 = torch.zeros_like(w1_64), torch.zeros_like(w2_64)
    idx_c, pos_c, tw64 = idx.cpu(), pos.cpu().long(), tw.double().cpu()
    for ex in range(e):
        tok, slot = torch.nonzero(idx_c == ex, as_tuple=True)
        if len(tok) == 0:
            continue
        w, p = tw64[tok, slot][:, None], pos_c[tok, slot]
        z = x64[tok] @ w1_64[ex].T
        r_out.index_add_(0, tok, forward(z[:, :inter], z[:, inter:], w, 0.0) @ w2_64[ex].T)
        d2 = dout64[tok]
        rdh = d2 @ w2_64[ex]
        dg, du, rh, rdw, *_ = backward(gate_c[p], up_c[p], rdh, w, 0.0)
        dz = torch.cat((dg, du), 1)
        r_dw2[ex] = d2.T @ rh
        r_dw1[ex] = dz.T @ x64[tok]
        r_dx.index_add_(0, tok, dz @ w1_64[ex])
        r_dtw[tok, slot] = rdw
    drw_t = drw.cpu()[pos_c]
    for name, got, ref in (('out', out, r_out), ('dx', dx, r_dx), ('dw1', dw1, r_dw1), ('dw2', dw2, r_dw2), ('drw', drw_t, r_dtw)):
        rel = float((got.double().cpu() - ref).norm() / ref.norm())
        assert rel < 5 * HALF, f'{name}: {rel:.3e}'
