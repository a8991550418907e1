"""Every form of the dispatch (one launch or several, one or four tokens of a wave, rows and scales in one
round or more) against counting on the host, bit for bit: rows, scales, weights, and what no token owns."""
import pytest
import torch

import deep_gemm
from ragged import DEV
from test_moe_rows_gpu import places, routing

pytestmark = pytest.mark.gpu


def rows_of(kind, t, cols, seed):
    """Token rows and scales on the host: bytes as they lie (any bits are allowed: rows are copied)."""
    gen = torch.Generator().manual_seed(seed)
    if kind == 'bf16':
        return torch.randn((t, cols), generator=gen).bfloat16(), None
    if kind == 'e4m3':
        return torch.randint(0, 127, (t, cols), generator=gen, dtype=torch.uint8).view(torch.float8_e4m3fn), \
            torch.rand((t, -(-cols // 128)), generator=gen)
    return torch.randint(-128, 128, (t, cols // 2), generator=gen, dtype=torch.int8), \
        torch.randint(-2 ** 31, 2 ** 31, (t, -(-cols // 128)), generator=gen).int()


def raw(x):
    return x.view(torch.int16) if x.dtype == torch.bfloat16 else x.view(torch.int8) if x.element_size() == 1 else x.view(torch.int32)


def dispatch(kind, t, k, e, cols, layout, alignment=16, launches=None, lost=0.1, idx=None):
    print(f'{kind} t={t} k={k} e={e} cols={cols} {layout} alignment={alignment}', flush=True)
    idx = routing(t, k, e, t + k, lost=lost, again=True) if idx is None else idx
    x, sf = rows_of(kind, t, cols, t)
    w = torch.rand((t, k), generator=torch.Generator().manual_seed(1)) + 0.1
    max_m = max(1, t * k // e)
    more = dict(max_m=max_m) if layout == 'masked' else dict(alignment=alignment)
    given = x.to(DEV) if sf is None else (x.to(DEV), sf.to(DEV))
    a, a_sf, gl, got, rw = deep_gemm.moe_dispatch(given, idx.to(DEV), e, layout=layout, topk_weights=w.to(DEV), **more)
    config = deep_gemm.get_last_config()
    assert launches is None or f' launches={launches}' in config, config
    pos, starts, ends, used = places(idx, e, 1 if layout == 'masked' else alignment)
    if layout == 'masked':
        rank = pos - torch.tensor(starts)[idx.clamp(0, e - 1).long()]
        pos = torch.where((pos >= 0) & (rank < max_m), idx.long() * max_m + rank, -1)
        assert gl.tolist() == [min(n - s, max_m) for s, n in zip(starts, ends)]
    elif layout == 'psum':
        assert gl.tolist() == ends
    else:
        want = torch.full((a.shape[0],), -1, dtype=torch.int32)
        for g, (s, n) in enumerate(zip(starts, ends)):
            want[s:n] = g
        assert torch.equal(gl.cpu(), want)
    live = pos >= 0
    assert torch.equal(got.cpu().long(), pos)
    at, token = pos[live], live.nonzero()[:, 0]
    weights = rw.reshape(-1).cpu()
    assert torch.equal(weights[at], w[live])
    for src, dst in ((x, a), (sf, a_sf)):
        if src is None:
            assert dst is None
            continue
        dst = raw(dst).reshape(-1, dst.shape[-1]).cpu()
        assert torch.equal(dst[at], raw(src)[token])
        if layout != 'masked':   # padding rows
            rest = torch.ones(used, dtype=torch.bool)
            rest[at] = False
            assert not dst[:used][rest].any()
    if layout != 'masked':
        weights[at] = 0
        assert not weights.any()


@pytest.mark.parametrize('kind,cols', [('bf16', 64), ('e4m3', 256), ('e2m1', 512)])
@pytest.mark.parametrize('t,k,layout', [(7168, 3, 'psum'), (7169, 3, 'psum'), (8191, 3, 'psum'), (8192, 3, 'psum'), (8197, 1, 'contiguous'), (11999, 3, 'masked'),
                                        (12000, 3, 'masked'), (12005, 1, 'masked'), (8192, 2, 'masked'), (9000, 16, 'psum')])
def test_one_and_four_tokens_of_a_wave(kind, cols, t, k, layout):
    dispatch(kind, t, k, 40, cols, layout)


@pytest.mark.parametrize('t,k,e,cols,layout,launches', [
    (7168, 1, 16, 1024, 'psum', 3), (7169, 1, 16, 1024, 'psum', 4), (8191, 2, 16, 2048, 'psum', 3), (8192, 2, 16, 2048, 'psum', 4), (8193, 2, 1000, 2304, 'contiguous', 4), (8200, 4, 300, 1152, 'psum', 4),
    (8192, 4, 256, 1152, 'psum', 3), (8192, 5, 300, 1152, 'contiguous', 3), (8195, 8, 24, 512, 'psum', 4), (8195, 1, 24, 1024, 'masked', 3)])
@pytest.mark.parametrize('kind', ['e4m3', 'bf16'])
def test_segment_starts_of_a_launch_of_their_own(kind, t, k, e, cols, layout, launches):
    """Many tokens with little to store; the same bytes a row in both types."""
    dispatch(kind, t, k, e, cols // (2 if kind == 'bf16' else 1), layout, launches=launches)


@pytest.mark.parametrize('layout', ['psum', 'contiguous'])
def test_no_token_routed_in_four_launches(layout):
    dispatch('e4m3', 8192, 1, 5, 1024, layout, launches=4, lost=1.0)


@pytest.mark.parametrize('layout', ['psum', 'contiguous'])
@pytest.mark.parametrize('t,k,e,alignment', [(8200, 1, 50, 2048), (2100, 8, 200, 512), (3, 1, 30, 4096), (8192, 3, 40, 1), (4100, 4, 1, 16)])
def test_many_rows_past_the_segments(t, k, e, alignment, layout):
    """Up to 16 workgroups, and one alone, for the rows that no segment has (and none of them: one expert, all routed)."""
    kind = 'bf16' if alignment % 16 else 'e4m3'   # (8-bit rows take alignments of 16 only)
    dispatch(kind, t, k, e, 128, layout, alignment=alignment, lost=0.0 if e == 1 else 0.2)


@pytest.mark.parametrize('t,k,e,size,layout,launches', [
    (724, 1, 1, 256, 'psum', 1), (725, 1, 1, 256, 'masked', 1), (1448, 1, 1, 256, 'contiguous', 1), (1448, 8, 8, 256, 'psum', 1),
    (1449, 1, 1, 256, 'psum', 3), (1449, 1, 2, 256, 'psum', 1), (1449, 8, 8, 4096, 'masked', 1), (2048, 2, 8, 256, 'psum', 1),
    (2900, 2, 8, 256, 'masked', 3), (1250, 16, 64, 256, 'psum', 1), (1251, 16, 64, 256, 'psum', 3), (1772, 8, 64, 256, 'contiguous', 1),
    (1773, 8, 64, 256, 'psum', 3), (1618, 8, 64, 256, 'masked', 1), (1619, 8, 64, 256, 'masked', 3), (2048, 8, 20, 4096, 'psum', 1),
    (2049, 8, 20, 4096, 'psum', 3), (4578, 1, 32, 256, 'masked', 1), (4579, 1, 32, 256, 'masked', 3), (2048, 2, 1024, 256, 'psum', 1),
    (2049, 2, 1024, 256, 'psum', 3), (4096, 1, 1024, 256, 'psum', 1), (4097, 1, 1024, 256, 'psum', 4), (1500, 8, 600, 256, 'psum', 3),
    (3000, 2, 1024, 256, 'contiguous', 4), (2999, 2, 1024, 256, 'psum', 3)])
def test_sizes_of_one_launch_and_of_several(t, k, e, size, layout, launches):
    """Around the sizes at which the number of launches changes; `size` bytes a row. (Entries x workgroups of four tokens:
    1772 x 8 x 443 is at most 6 x 2^20, 1773 x 8 x 444 more; masked 1618 x 8 x 405 and 4578 x 1145 at most 5 x 2^20, 1619 x 8 x
    405 and 4579 x 1145 more.)"""
    dispatch('bf16', t, k, e, size // 2, layout, launches=launches)
    if e > 1:   # all tokens to the same experts
        dispatch('e4m3', t, k, e, size, layout, launches=launches, idx=torch.arange(k, dtype=torch.int32).expand(t, k).contiguous() % e)


WIDE = [('e4m3', 8320), ('e4m3', 1024), ('e4m3', 7168), ('e2m1', 2080), ('e2m1', 16640), ('bf16', 7168), ('bf16', 4104), ('bf16', 520)]


@pytest.mark.parametrize('layout', ['psum', 'contiguous', 'masked'])
@pytest.mark.parametrize('kind,cols', WIDE)
def test_wide_rows_and_scales_of_many_tokens(kind, cols, layout):
    """Three launches, a token a wave: rows of one and of two rounds of 8 KB, scales of one and of two rounds of 64."""
    dispatch(kind, 2050, 8, 24, cols, layout, launches=3)


@pytest.mark.parametrize('layout', ['psum', 'contiguous'])
@pytest.mark.parametrize('kind,cols', WIDE)
def test_wide_rows_and_scales_with_starts_of_their_own(kind, cols, layout):
    dispatch(kind, 8195, 2, 24, cols, layout, launches=4)


@pytest.mark.parametrize('layout', ['psum', 'contiguous', 'masked'])
@pytest.mark.parametrize('kind,cols', WIDE)
@pytest.mark.parametrize('t,k', [(800, 4), (1449, 3)])
def test_wide_rows_and_scales_of_four_tokens_a_workgroup(kind, cols, t, k, layout):
    """One launch, a token a wave: rounds of 8 KB and 64 scales."""
    dispatch(kind, t, k, 20, cols, layout, launches=1)


@pytest.mark.parametrize('layout', ['psum', 'contiguous', 'masked'])
@pytest.mark.parametrize('kind,cols', [('e4m3', 33024), ('e4m3', 16384), ('e2m1', 33056), ('e2m1', 66048), ('bf16', 8200)])
def test_wide_rows_and_scales_of_a_token_a_workgroup(kind, cols, layout):
    """One launch, the four waves share a token: rounds of 16 KB and 256 scales."""
    dispatch(kind, 50, 3, 9, cols, layout, launches=1)
    dispatch(kind, 1, 1, 1, cols, layout, launches=1, lost=0.0)
