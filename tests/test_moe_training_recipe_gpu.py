"""The documented training step of an MoE layer's experts runs as it is written: the code
block is taken out of the repository's documents and executed on small layers, among them
one with ids that are not routed, and its results are compared with the layer in 64 bits."""
import glob
import os
import re
import textwrap

import numpy as np
import pytest
import torch

import deep_gemm
from conftest import ROOT
from ragged import DEV, matrix
from test_swiglu_checkpoint_gpu import HALF, backward, forward, value

pytestmark = pytest.mark.gpu


def recipe():
    blocks = []
    for path in sorted(glob.glob(os.path.join(ROOT, '*.md'))):
        with open(path) as f:
            blocks += re.findall(r'^ *```python\n(.*?)^ *```', f.read(), flags=re.S | re.M)
    blocks = [textwrap.dedent(b) for b in blocks if 'moe_swiglu_backward' in b]
    assert len(blocks) == 1
    return blocks[0]


@pytest.mark.parametrize('t,e,topk,hidden,inter,skipped', [
    (90, 6, 2, 256, 136, 0.0), (3, 5, 3, 128, 128, 0.0), (70, 8, 4, 128, 256, 0.3), (5, 4, 2, 128, 64, 0.8), (16, 1, 1, 128, 64, 0.1)])
def test_documented_training_step(t, e, topk, hidden, inter, skipped):
    print(f'layer t={t} e={e} topk={topk} hidden={hidden} inter={inter} skipped={skipped}', flush=True)
    rng = np.random.default_rng(t)
    ids = np.stack([rng.choice(e, size=topk, replace=False) for _ in range(t)]).astype(np.int32)
    ids[rng.random((t, topk)) < skipped] = -1
    x, _ = matrix((t, hidden), 1)
    w1, w1_64 = matrix((e, 2 * inter, hidden), 2, hidden ** -0.5)
    w2, w2_64 = matrix((e, hidden, inter), 3, inter ** -0.5)
    dout, dout64 = matrix((t, hidden), 4)
    tw = torch.from_numpy(rng.random((t, topk)).astype(np.float32) + 0.1).to(DEV)
    rows = int(deep_gemm._ffi.lib.dg_moe_dispatch_max_rows(t, topk, e, 16))
    bf = lambda n: torch.full((rows, n), float('nan'), dtype=torch.bfloat16, device=DEV)
    names = dict(torch=torch, deep_gemm=deep_gemm, x=x, topk_idx=torch.from_numpy(ids).to(DEV), topk=topk, E=e, hidden=hidden,
                 topk_weights=tw, w1=w1, w2=w2, gate_up=bf(2 * inter), y=bf(hidden), dout=dout, dy=bf(hidden), dh=bf(inter),
                 drows=bf(hidden), dw1=torch.zeros((e, 2 * inter, hidden), device=DEV),
                 dw2=torch.zeros((e, hidden, inter), device=DEV))
    exec(recipe(), names)
    torch.cuda.synchronize()

    q, sf = deep_gemm.per_token_cast_to_fp8(x.contiguous(), use_ue8m0=True)
    x64 = (q.float() * sf.repeat_interleave(128, 1)[:, :hidden]).double().cpu()
    gate_c, up_c = value(*names['ckpt'], inter)
    out, dx, dtw = torch.zeros(t, hidden).double(), torch.zeros(t, hidden).double(), torch.zeros(t, topk).double()
    dw1, dw2 = torch.zeros_like(w1_64), torch.zeros_like(w2_64)
    pos, tw64 = names['pos'].cpu().long(), tw.double().cpu()
    for ex in range(e):
        tok, slot = torch.nonzero(torch.from_numpy(ids) == ex, as_tuple=True)
        if len(tok) == 0:
            continue
        w, p = tw64[tok, slot][:, None], pos[tok, slot]
        z = x64[tok] @ w1_64[ex].T
        out.index_add_(0, tok, forward(z[:, :inter], z[:, inter:], w, 0.0) @ w2_64[ex].T)
        dg, du, h, dw, *_ = backward(gate_c[p], up_c[p], dout64[tok] @ w2_64[ex], w, 0.0)
        dz = torch.cat((dg, du), 1)
        dw2[ex], dw1[ex] = dout64[tok].T @ h, dz.T @ x64[tok]
        dx.index_add_(0, tok, dz @ w1_64[ex])
        dtw[tok, slot] = dw
    # five roundings to BF16 between the inputs and the last gradient, each of half a step
    for name, ref in (('out', out), ('dx', dx), ('dw1', dw1), ('dw2', dw2), ('dtopk_weights', dtw)):
        got = names[name].double().cpu()
        assert torch.isfinite(got).all(), name
        assert float((got - ref).norm()) <= 5 * HALF * float(ref.norm()), name
