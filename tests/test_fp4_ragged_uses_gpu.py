"""Uses of the 4-bit operands beside the ragged product's own cases: ends outside the rows and out of order,
workspaces through the C entry, gradients through the operands' values, and rows dispatched into the
masked layout for the masked product.

Bounds: half a step of a result's type plus the FP32 sums' (fp4_ragged.py, ragged.py).
"""
import ctypes
import glob
import os
import re
import textwrap

import pytest
import torch

import deep_gemm
import ragged
from conftest import ROOT
from deep_gemm import _ffi
from fp4_ragged import operand, sum_error
from ragged import DEV, bits, check, rounding
from test_moe_rows_gpu import routing

pytestmark = pytest.mark.gpu


def bound(a, b, dtype=torch.float32):
    ref, mag = a @ b.T, a.abs() @ b.T.abs()
    return ref, rounding(dtype, ref) + sum_error(a.shape[1], mag) * (1 + torch.finfo(dtype).eps)


@pytest.mark.parametrize('block', [256, 128, 64, 32])
def test_ends_outside_the_rows_hold_the_products(block):
    """An end below zero leaves its group empty and the next ones their rows; a group that ends before the last one did
    is empty, and the next begins there: its rows are then those of two groups."""
    deep_gemm.set_tile_override(block, 0, variant=14)
    (a, a64), (b, b64) = operand((9, 64), 1), operand((3, 16, 64), 2)
    run = lambda ends, d: deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d[1:10], torch.tensor(ends, dtype=torch.int32, device=DEV))
    new = lambda: torch.full((11, 16), 7.0, dtype=torch.float32, device=DEV)
    d = new()
    run([-5, 2, 9], d)
    check(d[1:3], *bound(a64[:2], b64[1]), 'group 1')
    check(d[3:10], *bound(a64[2:], b64[2]), 'group 2')
    assert (d[[0, 10]] == 7.0).all()
    d = new()
    run([5, 2, 5], d)
    check(d[1:3], *bound(a64[:2], b64[0]), 'group 0')
    got = d[3:6].double().cpu()
    fits = [(got - ref).abs() <= off for ref, off in (bound(a64[2:5], b64[0]), bound(a64[2:5], b64[2]))]
    assert (fits[0] | fits[1]).all()
    assert (d[0] == 7.0).all() and (d[6:] == 7.0).all()


@pytest.mark.parametrize('block,pieces', [(32, 4), (64, 3), (128, 2)])
def test_workspaces_of_the_c_entry(block, pieces):
    """No workspace, one byte too few, as many as asked for, and more: the axis stays whole in the first two."""
    m, n, k, g = 45, 70, 2080, 2
    (a, a64), (b, b64) = operand((m, k), 1), operand((g, n, k), 2)
    ends = torch.tensor([20, 45], dtype=torch.int32, device=DEV)
    deep_gemm.set_tile_override(block, pieces, variant=14)
    size = _ffi.lib.dg_fp4_gemm_ragged_workspace_size(m, n, k, g)
    assert size == m * 72 * 4 * pieces
    whole = None
    for room, splits in ((None, 1), (size - 1, 1), (size, pieces), (size + 4096, pieces)):
        print(f'workspace of {room} bytes', flush=True)
        d = torch.full((m, n), 7.0, dtype=torch.float32, device=DEV)
        ws = None if room is None else torch.full((room + 512,), 0x7F, dtype=torch.uint8, device=DEV)[:room]
        args = [_ffi.describe(t) for t in (*a, *b, d, ends)]
        args = [ctypes.byref(t) for t in args] + [1, None if ws is None else ctypes.byref(_ffi.describe(ws)), _ffi.stream_of(d)]
        _ffi.check(_ffi.lib.dg_m_grouped_fp4_gemm_nt_ragged(*args))
        assert f' splits={splits} ' in deep_gemm.get_last_config()
        torch.cuda.synchronize()
        check(d[:20], *bound(a64[:20], b64[0]), 'group 0')
        check(d[20:], *bound(a64[20:], b64[1]), 'group 1')
        if splits == 1:
            assert whole is None or torch.equal(bits(d), bits(whole))
            whole = d
        if ws is not None:   # nothing past what was asked for
            assert (torch.as_strided(ws, (room + 512,), (1,))[(size if splits > 1 else 0):] == 0x7F).all()


@pytest.mark.parametrize('sizes,n,k', [([70, 0, 33], 96, 160), ([1, 1], 64, 64), ([300], 200, 288)])
def test_gradients_through_the_values(sizes, n, k):
    """dA = dD B and dB = dD^T A with A's and B's values, which BF16 holds exactly, by the BF16 products: against sums in
    64 bits, and against differences of the 4-bit product itself (it is linear in A and in B)."""
    g, rows = len(sizes), sum(sizes)
    seg = ragged.segments(sizes)
    ends = ragged.ends_of(seg)
    (a, a64), (b, b64) = operand((rows, k), 1), operand((g, n, k), 2)
    gen = torch.Generator().manual_seed(3)
    dd = torch.randn((rows, n), generator=gen).bfloat16()
    values = lambda q, sf: deep_gemm.cast_back_from_fp4(q, sf, 32, True, torch.bfloat16)
    a_bf = values(*a)
    b_bf = values(b[0].view(g * n, k // 2), b[1].view(g * n, -1)).view(g, n, k)
    assert torch.equal(a_bf.double().cpu(), a64) and torch.equal(b_bf.double().cpu(), b64)
    da = torch.empty((rows, k), dtype=torch.float32, device=DEV)
    db = torch.zeros((g, n, k), dtype=torch.float32, device=DEV)
    deep_gemm.m_grouped_bf16_gemm_nn_ragged(dd.to(DEV), b_bf, da, ends)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(dd.to(DEV), a_bf, db, ends)
    dd = dd.double()
    for i, (lo, hi) in enumerate(seg):
        if hi > lo:
            ref = dd[lo:hi] @ b64[i]
            check(da[lo:hi], ref, rounding(torch.float32, ref) + ragged.sum_error(n, dd[lo:hi].abs() @ b64[i].abs()), 'dA')
        ref = dd[lo:hi].T @ a64[lo:hi]
        check(db[i], ref, rounding(torch.float32, ref) + ragged.sum_error(hi - lo, dd[lo:hi].T.abs() @ a64[lo:hi].abs()), 'dB')
    # other codes and scales of A, then of B: the product's change along dD is the gradient's product with theirs
    (a2, a2_64), (b2, b2_64) = operand((rows, k), 4), operand((g, n, k), 5)
    out = []
    for x, y in ((a, b), (a2, b), (a, b2)):
        d = torch.empty((rows, n), dtype=torch.float32, device=DEV)
        deep_gemm.m_grouped_fp4_gemm_nt_ragged(x, y, d, ends)
        out.append(d.double().cpu())
    big = torch.cat([(a64[lo:hi].abs() + a2_64[lo:hi].abs()) @ (b64[i].abs() + b2_64[i].abs()).T for i, (lo, hi) in enumerate(seg)])
    # every sum is off by at most its FP32 bound, of terms whose magnitudes are below `big`
    off = 2 * (big * dd.abs()).sum() * ((-(-k // 64) + 65) + (-(-max(n, rows) // 16) + 17)) * 2.0 ** -23
    for new, got in ((out[1], (da.double().cpu() * (a2_64 - a64)).sum()), (out[2], (db.double().cpu() * (b2_64 - b64)).sum())):
        assert abs(((new - out[0]) * dd).sum() - got) <= off


@pytest.mark.parametrize('t,k,e,n,cols,max_m', [(50, 2, 4, 96, 256, 40), (300, 4, 8, 128, 512, 160), (3, 2, 4, 64, 128, 4)])
def test_masked_rows_for_the_masked_product(t, k, e, n, cols, max_m):
    """Scale words go where `out` has them: with those of consecutive rows side by side, as the masked product reads them.
    (Its matrix instructions may take 128 products each: 64 additions more than in the ragged one's bound.)"""
    print(f't={t} k={k} e={e} n={n} cols={cols} max_m={max_m}', flush=True)
    idx = routing(t, k, e, t)
    x, x64 = operand((t, cols), 1)
    (codes, words), w64 = operand((e, n, cols), 2)
    words = torch.empty((e, cols // 128, n), dtype=torch.int32, device=DEV).copy_(words.transpose(1, 2)).transpose(1, 2)
    room = -(-max_m // 4) * 4
    sf = torch.full((e, cols // 128, room), -1, dtype=torch.int32, device=DEV).transpose(1, 2)[:, :max_m]
    a = torch.zeros((e, max_m, cols // 2), dtype=torch.int8, device=DEV)
    got_a, got_sf, count, pos, _ = deep_gemm.moe_dispatch(x, idx.to(DEV), e, layout='masked', max_m=max_m, out=(a, sf))
    assert got_a.data_ptr() == a.data_ptr() and got_sf.data_ptr() == sf.data_ptr() and got_sf.stride() == sf.stride()
    d = torch.full((e, max_m, n), 7.0, dtype=torch.bfloat16, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_masked((a, sf), (codes, words), d, count, max_m, recipe_a=(1, 32), recipe_b=(1, 32))
    torch.cuda.synchronize()
    pos, d = pos.cpu().long(), d.cpu()
    written = torch.zeros((e * max_m,), dtype=torch.bool)
    for ex in range(e):
        tok, slot = torch.nonzero((idx == ex) & (pos >= 0), as_tuple=True)
        p = pos[tok, slot]
        written[p] = True
        if len(tok):
            ref, off = bound(x64[tok], w64[ex], torch.bfloat16)
            check(d.view(-1, n)[p], ref, off + 65 * 2.0 ** -23 * (x64[tok].abs() @ w64[ex].abs().T), f'expert {ex}')
    assert (d.view(-1, n)[~written] == 7.0).all()


def documented(word):
    """The one documented piece of code with `word` in it."""
    blocks = []
    for path in sorted(glob.glob(os.path.join(ROOT, '*.md'))):
        with open(path) as f:
            blocks += re.findall(r'^ *```python\n(.*?)^ *```', f.read(), flags=re.S | re.M)
    blocks = [textwrap.dedent(b) for b in blocks if word in b]
    assert len(blocks) == 1
    return blocks[0]


def test_documented_gradients():
    E, hidden, inter, rows = 3, 160, 96, 50
    ends = torch.tensor([20, 20, 50], dtype=torch.int32, device=DEV)
    hq, h64 = operand((rows, inter), 1)
    w2, w64 = operand((E, hidden, inter), 2)
    dy = torch.randn((rows, hidden), generator=torch.Generator().manual_seed(3)).bfloat16()
    names = dict(torch=torch, deep_gemm=deep_gemm, E=E, hidden=hidden, inter=inter, ends=ends, hq=hq, w2=w2, dy=dy.to(DEV),
                 dh=torch.empty((rows, inter), dtype=torch.float32, device=DEV), dw2=torch.zeros((E, hidden, inter), device=DEV))
    exec(documented('w2_bf16'), names)
    dy = dy.double()
    for g, lo, hi in ((0, 0, 20), (2, 20, 50)):
        ref = dy[lo:hi] @ w64[g]
        check(names['dh'][lo:hi], ref, rounding(torch.float32, ref) + ragged.sum_error(hidden, dy[lo:hi].abs() @ w64[g].abs()), 'dh')
        ref = dy[lo:hi].T @ h64[lo:hi]
        check(names['dw2'][g], ref, rounding(torch.float32, ref) + ragged.sum_error(hi - lo, dy[lo:hi].T.abs() @ h64[lo:hi].abs()), 'dw2')
    assert not names['dw2'][1].any()


def test_documented_masked_rows():
    t, E, hidden, max_m = 60, 4, 256, 40
    idx = routing(t, 2, E, 1)
    xq, _ = operand((t, hidden), 1)
    names = dict(torch=torch, deep_gemm=deep_gemm, E=E, hidden=hidden, max_m=max_m, xq=xq, topk_idx=idx.to(DEV),
                 topk_weights=torch.rand((t, 2), device=DEV))
    exec(documented("layout='masked', max_m=max_m, out=rows"), names)
    codes, sf = names['rows']
    assert sf.stride(1) == 1 and sf.stride(2) == max_m
    pos = names['pos'].cpu().long()
    at, token = pos[pos >= 0], (pos >= 0).nonzero()[:, 0]
    assert torch.equal(codes.reshape(-1, hidden // 2).cpu()[at], xq[0].cpu()[token])
    assert torch.equal(sf.reshape(-1, hidden // 128).cpu()[at], xq[1].cpu()[token])
