"""The fused 4-bit cast and its way back against the torch forms on the host, bit for bit:
granularities, scale forms, odd sizes, pitches, non-finite values, and every BF16 value."""
import pytest
import torch

import deep_gemm
from deep_gemm.utils import math as plain

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def both(x, gran, ue8m0, packed):
    q, sf = deep_gemm.per_token_cast_to_fp4(x, ue8m0, gran, packed)
    rq, rsf = plain.per_token_cast_to_fp4(x.cpu(), ue8m0, gran, packed)
    assert 'per_token_cast_to_fp4' in deep_gemm.get_last_config()
    assert q.dtype == rq.dtype and sf.dtype == rsf.dtype and sf.shape == rsf.shape
    assert torch.equal(sf.cpu().view(torch.int32), rsf.contiguous().view(torch.int32)), 'scales'
    assert torch.equal(q.cpu(), rq), 'codes'
    return q, sf


def back(q, sf, gran, packed):
    for dtype in (torch.float32, torch.bfloat16):
        v = deep_gemm.cast_back_from_fp4(q, sf, gran, packed, dtype)
        n = q.shape[1] * 2
        if n == 0 or q.shape[0] == 0:
            assert v.shape == (q.shape[0], n)
            continue
        ref = plain.cast_back_from_fp4(q.cpu(), sf.cpu(), gran, packed).to(dtype)
        view = torch.int32 if dtype == torch.float32 else torch.int16
        nan = torch.isnan(ref)
        assert torch.equal(torch.isnan(v.cpu()), nan)
        assert torch.equal(v.cpu()[~nan].view(view), ref[~nan].view(view)), f'{dtype}'


FORMS = [(True, True), (True, False), (False, False)]


@pytest.mark.parametrize('gran', [32, 64, 128])
@pytest.mark.parametrize('ue8m0,packed', FORMS)
@pytest.mark.parametrize('m,n', [(1, 2), (1, 30), (3, 32), (5, 34), (7, 130), (33, 2048), (2, 2056), (65, 1022), (130, 7168),
                                 (9, 1024), (1, 8192)])
def test_cast_and_back(m, n, gran, ue8m0, packed):
    gen = torch.Generator().manual_seed(m * n + gran)
    x = torch.randn((m, n), generator=gen) * torch.exp(3 * torch.randn((m, 1), generator=gen))
    x[:, : min(n, 40)] *= (torch.rand((m, min(n, 40)), generator=gen) > 0.5)
    q, sf = both(x.bfloat16().to(DEV), gran, ue8m0, packed)
    back(q, sf, gran, packed)


@pytest.mark.parametrize('ue8m0,packed', FORMS)
@pytest.mark.parametrize('top', [6.0, 5.0, 0.75, 1e-4, 1e-30, 1e30, 3.3e38])
def test_every_value_under_a_scale(top, ue8m0, packed):
    """All BF16 values up to `top`, in groups whose largest magnitude is `top`."""
    every = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    every = every[every.float().abs() <= top]
    pad = -every.numel() % 31
    every = torch.cat([every, torch.zeros(pad, dtype=torch.bfloat16)]).view(-1, 31)
    x = torch.cat([every, torch.full((every.shape[0], 1), top, dtype=torch.bfloat16)], 1)
    q, sf = both(x.to(DEV), 32, ue8m0, packed)
    back(q, sf, 32, packed)


@pytest.mark.parametrize('ue8m0,packed', FORMS)
def test_non_finite_values(ue8m0, packed):
    """An Inf or NaN sets its own group's scale and codes; other groups of the row do not see it."""
    x = torch.randn((6, 256), generator=torch.Generator().manual_seed(3)).bfloat16()
    for r, v in enumerate((float('inf'), float('-inf'), float('nan'), -float('nan'))):
        x[r, 70] = v
    x[4, 3], x[4, 9] = float('inf'), float('nan')
    q, sf = both(x.to(DEV), 32, ue8m0, packed)
    back(q, sf, 32, packed)


@pytest.mark.parametrize('pitch,offset', [(300, 0), (301, 0), (304, 1), (304, 8)])
def test_rows_that_begin_anywhere(pitch, offset):
    wide = torch.randn((9, pitch), generator=torch.Generator().manual_seed(4)).bfloat16().to(DEV)
    both(wide[:, offset:offset + 290], 32, True, True)


def test_rows_not_contiguous_within():
    """Columns apart: the torch operations take them, as the 8-bit cast's do."""
    x = torch.randn((64, 40), device=DEV).bfloat16().t()
    q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
    rq, rsf = plain.per_token_cast_to_fp4(x.cpu(), True, 32, True)
    assert torch.equal(q.cpu(), rq) and torch.equal(sf.cpu(), rsf)


def test_back_takes_scales_of_any_strides():
    x = torch.randn((70, 640), generator=torch.Generator().manual_seed(5)).bfloat16().to(DEV)
    q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
    want = deep_gemm.cast_back_from_fp4(q, sf, 32, True)
    columns = sf.t().contiguous().t()
    assert columns.stride() != sf.stride()
    assert torch.equal(deep_gemm.cast_back_from_fp4(q, columns, 32, True), want)
    wide = torch.zeros((70, 400), dtype=torch.int8, device=DEV)
    wide[:, 1:321] = q
    assert torch.equal(deep_gemm.cast_back_from_fp4(wide[:, 1:321], sf, 32, True), want)


def test_empty():
    for m, n in ((0, 64), (4, 0)):
        q, sf = deep_gemm.per_token_cast_to_fp4(torch.empty((m, n), dtype=torch.bfloat16, device=DEV), True, 32, True)
        assert q.shape == (m, n // 2) and sf.shape == (m, n // 128 if n == 0 else 1)
        back(q, sf, 32, True)


def test_offsets_past_32_bits():
    """More than 2^32 elements; the last rows are checked."""
    m, n = 70000, 65536
    x = torch.zeros((m, n), dtype=torch.bfloat16, device=DEV)
    x[-2:] = torch.randn((2, n), generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
    rq, rsf = plain.per_token_cast_to_fp4(x[-2:].cpu(), True, 32, True)
    assert torch.equal(q[-2:].cpu(), rq) and torch.equal(sf[-2:].cpu(), rsf)
    assert not q[:-2].any()
    del x
    v = deep_gemm.cast_back_from_fp4(q, sf, 32, True, torch.bfloat16)
    assert torch.equal(v[-2:].float().cpu(), plain.cast_back_from_fp4(rq, rsf, 32, True))
    assert not v[:1000].any() and not v[-1002:-2].any()


def test_graph():
    x = torch.randn((50, 512), device=DEV).bfloat16()
    deep_gemm.cast_back_from_fp4(*deep_gemm.per_token_cast_to_fp4(x, True, 32, True), 32, True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
        v = deep_gemm.cast_back_from_fp4(q, sf, 32, True)
    for seed in range(3):
        x.copy_(torch.randn((50, 512), generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        rq, rsf = plain.per_token_cast_to_fp4(x.cpu(), True, 32, True)
        assert torch.equal(q.cpu(), rq) and torch.equal(sf.cpu(), rsf)
        assert torch.equal(v.cpu(), plain.cast_back_from_fp4(rq, rsf, 32, True))
