"""Whole MoE layers made of the dispatch, the expert operators, the combination and their gradients,
against the layer in 64 bits: a BF16 training step with the weights at the dispatch or at the
combination, eager and captured, and the documented 4-bit layer, stage by stage."""
import glob
import os
import re
import textwrap

import pytest
import torch

import deep_gemm
from conftest import ROOT
from fp4_ragged import operand, sum_error
from ragged import DEV, bits, check, matrix, rounding
from test_moe_rows_gpu import routing
from test_swiglu_checkpoint_gpu import HALF, backward, forward, steps, value

pytestmark = pytest.mark.gpu

LAYERS = [(90, 6, 2, 256, 136, 0.0), (1, 5, 3, 128, 128, 0.0), (70, 8, 4, 136, 256, 0.3), (5, 4, 2, 128, 64, 0.8), (513, 4, 3, 264, 200, 0.1),
          (20, 4, 2, 64, 64, 1.0)]


class Layer:
    def __init__(self, t, e, topk, hidden, inter, skipped, at_combine):
        self.__dict__.update(t=t, e=e, topk=topk, hidden=hidden, inter=inter, at_combine=at_combine)
        self.ids = routing(t, topk, e, t, lost=skipped)
        self.idx = self.ids.to(DEV)
        self.x, self.x64 = matrix((t, hidden), 1)
        self.w1, self.w1_64 = matrix((e, 2 * inter, hidden), 2, hidden ** -0.5)
        self.w2, self.w2_64 = matrix((e, hidden, inter), 3, inter ** -0.5)
        self.dout, self.dout64 = matrix((t, hidden), 4)
        self.tw = torch.rand((t, topk), generator=torch.Generator().manual_seed(5)) + 0.1
        self.tw_dev = self.tw.to(DEV)

    def step(self):
        e, hidden, inter = self.e, self.hidden, self.inter
        a, _, ends, pos, w = deep_gemm.moe_dispatch(self.x, self.idx, e, layout='psum', alignment=1,
                                                    topk_weights=None if self.at_combine else self.tw_dev)
        rows = a.shape[0]
        bf = lambda n: torch.full((rows, n), float('nan'), dtype=torch.bfloat16, device=DEV)
        gate_up, y, dh, drows = bf(2 * inter), bf(hidden), bf(inter), bf(hidden)
        deep_gemm.m_grouped_bf16_gemm_nt_ragged(a, self.w1, gate_up, ends)
        h, ckpt = deep_gemm.moe_swiglu_checkpoint(gate_up, w)
        deep_gemm.m_grouped_bf16_gemm_nt_ragged(h, self.w2, y, ends)
        tw = self.tw_dev if self.at_combine else None
        out = deep_gemm.moe_combine(y, pos, tw)
        dy, dtw = deep_gemm.moe_combine_backward(self.dout, y, pos, tw, out=y)
        deep_gemm.m_grouped_bf16_gemm_nn_ragged(dy, self.w2, dh, ends)
        dgate_up, h, dw = deep_gemm.moe_swiglu_backward(dh, ckpt, w)
        dw2 = torch.zeros((e, hidden, inter), device=DEV)
        dw1 = torch.zeros((e, 2 * inter, hidden), device=DEV)
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(dy, h, dw2, ends)
        deep_gemm.m_grouped_bf16_gemm_nn_ragged(dgate_up, self.w1, drows, ends)
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(dgate_up, a, dw1, ends)
        dx, from_rows = deep_gemm.moe_dispatch_backward(drows, pos, None if self.at_combine else dw)
        return dict(out=out, dx=dx, dw1=dw1, dw2=dw2, dtw=dtw if self.at_combine else from_rows), pos, ckpt

    def check(self, got, pos, ckpt):
        gate_c, up_c = value(*ckpt, self.inter)
        ref = dict(out=torch.zeros(self.t, self.hidden).double(), dx=torch.zeros(self.t, self.hidden).double(),
                   dw1=torch.zeros_like(self.w1_64), dw2=torch.zeros_like(self.w2_64), dtw=torch.zeros(self.t, self.topk).double())
        size = torch.zeros(self.t, self.topk).double()   # the magnitudes of dtw's sums
        pos, tw = pos.cpu().long(), self.tw.double()
        for ex in range(self.e):
            tok, slot = torch.nonzero(self.ids == ex, as_tuple=True)
            if len(tok) == 0:
                continue
            w, p, one = tw[tok, slot][:, None], pos[tok, slot], torch.ones(len(tok), 1).double()
            z = self.x64[tok] @ self.w1_64[ex].T
            plain = forward(z[:, :self.inter], z[:, self.inter:], one, 0.0)
            ref['out'].index_add_(0, tok, w * (plain @ self.w2_64[ex].T))
            inside, above = (one, w) if self.at_combine else (w, one)
            dy = above * self.dout64[tok]
            dg, du, h, dw, *_ = backward(gate_c[p], up_c[p], dy @ self.w2_64[ex], inside, 0.0)
            dz = torch.cat((dg, du), 1)
            ref['dw2'][ex], ref['dw1'][ex] = dy.T @ h, dz.T @ self.x64[tok]
            ref['dx'].index_add_(0, tok, dz @ self.w1_64[ex])
            y = plain @ self.w2_64[ex].T
            ref['dtw'][tok, slot] = (self.dout64[tok] * y).sum(1) if self.at_combine else dw
            size[tok, slot] = self.dout64[tok].abs().mul(plain.abs() @ self.w2_64[ex].T.abs()).sum(1) if self.at_combine else dw.abs()
        # at most five roundings to BF16 between the inputs and each result, each of half a step
        for name, want in ref.items():
            have = got[name].double().cpu()
            assert torch.isfinite(have).all(), name
            assert float((have - want).norm()) <= 5 * HALF * float((size if name == 'dtw' else want).norm()), name


@pytest.mark.parametrize('at_combine', [False, True])
@pytest.mark.parametrize('t,e,topk,hidden,inter,skipped', LAYERS)
def test_training_step(t, e, topk, hidden, inter, skipped, at_combine):
    print(f'layer t={t} e={e} topk={topk} hidden={hidden} inter={inter} skipped={skipped}', flush=True)
    layer = Layer(t, e, topk, hidden, inter, skipped, at_combine)
    layer.check(*layer.step())


@pytest.mark.parametrize('at_combine', [False, True])
def test_captured_training_step(at_combine):
    """A captured step, its eager twin alive, follows new tokens, ids and weights on every replay."""
    layer = Layer(60, 6, 2, 128, 136, 0.1, at_combine)
    eager = layer.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer.step()
    for seed in range(3):
        fresh = Layer(60, 6, 2, 128, 136, 0.0, at_combine)
        gen = torch.Generator().manual_seed(seed)
        layer.x64 = torch.randn((60, 128), generator=gen).bfloat16().double()
        layer.x.copy_(layer.x64)
        layer.ids = fresh.ids.roll(seed, 0)
        layer.idx.copy_(layer.ids)
        layer.tw = torch.rand((60, 2), generator=gen) + 0.1
        layer.tw_dev.copy_(layer.tw)
        graph.replay()
        torch.cuda.synchronize()
        layer.check(*captured)
        eager = layer.step()
        for name in eager[0]:
            assert torch.equal(bits(eager[0][name]), bits(captured[0][name])), name


def recipe():
    blocks = []
    for path in sorted(glob.glob(os.path.join(ROOT, '*.md'))):
        with open(path) as f:
            blocks += re.findall(r'^ *```python\n(.*?)^ *```', f.read(), flags=re.S | re.M)
    blocks = [textwrap.dedent(b) for b in blocks if 'm_grouped_fp4_gemm_nt_ragged' in b]
    assert len(blocks) == 1
    return blocks[0]


@pytest.mark.parametrize('t,e,topk,hidden,inter,skipped', [
    (90, 6, 2, 256, 160, 0.0), (1, 5, 3, 128, 128, 0.0), (70, 8, 4, 160, 256, 0.3), (300, 4, 2, 544, 96, 0.5), (4, 4, 2, 64, 64, 1.0)])
def test_documented_4_bit_layer(t, e, topk, hidden, inter, skipped):
    print(f'layer t={t} e={e} topk={topk} hidden={hidden} inter={inter} skipped={skipped}', flush=True)
    ids = routing(t, topk, e, t, lost=skipped)
    x, x64 = matrix((t, hidden), 1)
    tw = torch.rand((t, topk), generator=torch.Generator().manual_seed(5)) + 0.1
    # weights of the size of 1 / sqrt(hidden): codes of up to 6 under scales of 2^-9 to 2^-6
    (w1, w1_64), (w2, w2_64) = operand((e, 2 * inter, hidden), 2, 118, 121), operand((e, hidden, inter), 3, 118, 121)
    names = dict(torch=torch, deep_gemm=deep_gemm, x=x.contiguous(), topk_idx=ids.to(DEV), topk_weights=tw.to(DEV), E=e, hidden=hidden,
                 inter=inter, w1=w1, w2=w2)
    exec(recipe(), names)
    torch.cuda.synchronize()
    pos = names['pos'].cpu().long()
    back = lambda q: deep_gemm.cast_back_from_fp4(*q, 32, True).double().cpu()
    q64, h64 = back(names['xq']), back(names['hq'])
    # half a step of a code is at most 1/4 of the group's unit (1 between 4 and 6 at most), whose 6 is below twice the largest value
    assert ((q64 - x64).abs() <= 2 * x64.abs().amax(1, keepdim=True) / 6).all()
    gate_up, y, out = (names[n].double().cpu() for n in ('gate_up', 'y', 'out'))
    total = torch.zeros(t, hidden).double()
    size = torch.zeros(t, hidden).double()
    for ex in range(e):
        tok, slot = torch.nonzero(ids == ex, as_tuple=True)
        if len(tok) == 0:
            continue
        p = pos[tok, slot]
        for what, got, a, b in (('gate_up', gate_up, q64[tok], w1_64[ex]), ('y', y, h64[p], w2_64[ex])):
            ref, mag = a @ b.T, a.abs() @ b.T.abs()
            check(got[p], ref, rounding(torch.bfloat16, ref) + sum_error(a.shape[1], mag) * (1 + HALF), what)
        gate, up = gate_up[p][:, :inter], gate_up[p][:, inter:]
        ref = forward(gate, up, tw.double()[tok, slot][:, None], 0.0)
        check(names['h'].cpu()[p], ref, ref.abs() * (HALF + steps(gate)) + 1e-37, 'h')
        total.index_add_(0, tok, y[p])
        size.index_add_(0, tok, y[p].abs())
    check(out, total, rounding(torch.bfloat16, total) + topk * 2.0 ** -24 * size * (1 + HALF), 'out')
