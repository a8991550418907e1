"""The 256 x 256 kernels of the ragged BF16 products themselves. Forced tiles alone do not run
them on small shapes: a last round that is at most 58% full goes to 128 x 128 quarters, and
a small shape is nothing but a last round. With one CU every round is full (no quarters),
with 16 or 24 some TN lists leave tiles for the quarters too.

Bounds as in test_bf16_ragged_gpu.py, whose helpers these tests share."""
import pytest
import torch

import deep_gemm
from ragged import DEV, cast8, check, ends_of, matrix, rounding, segments, sum_error
from test_bf16_ragged_gpu import MIXED, k_grouped, m_grouped

pytestmark = pytest.mark.gpu


def whole_tiles(tiles, slots):
    """256 x 256 tiles of a list that stay 256 x 256: the kernels' split."""
    rest = tiles % slots
    return tiles - (rest if rest * 128 <= slots * 75 else 0)


def tn_whole_tiles(m, n, groups, cus):
    per = -(-m // 256) * -(-n // 256)
    if per % 8 and per < 64:
        return whole_tiles(per * groups, cus)
    return sum(whole_tiles(((x + 1) * per // 8 - x * per // 8) * groups, max(cus // 8, 1)) for x in range(8))


@pytest.fixture(autouse=True)
def whole():
    assert whole_tiles(1, 1) == 1 and whole_tiles(5, 256) == 0
    deep_gemm.set_tile_override(256, 0, variant=13)
    deep_gemm.set_num_sms(1)
    yield
    assert 'block=256' in deep_gemm.get_last_config()


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('sizes,n,k,alignment', [
    ([1], 1, 8, 1), ([3], 65, 8, 1), ([7], 130, 72, 1), ([0, 1, 0, 1], 33, 120, 1), (MIXED, 129, 264, 1),
    (MIXED, 255, 128, 16), (MIXED, 256, 64, 128), ([300], 520, 1000, 1), ([1] * 70, 40, 136, 1),
    ([0] * 65 + [9, 0, 2], 96, 256, 16), ([513, 255, 256, 257, 1], 257, 192, 1), ([700, 0, 1300, 65], 776, 200, 1)])
def test_m_grouped(direction, out, sizes, n, k, alignment):
    m_grouped(direction, sizes, n, k, alignment, out)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('k', [8, 56, 64, 72, 120, 128, 136, 192, 248, 256, 264, 1000, 4096])
def test_reduced_lengths(direction, k):
    m_grouped(direction, [17, 140, 260], 300, k)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('pitch', [301, 302, 304, 330, 4000])
def test_output_pitch(direction, out, pitch):
    """D's rows start anywhere; what lies between them stays."""
    d = m_grouped(direction, [150, 9, 300], 301, 72, out=out, d_pitch=pitch)
    assert (d.as_strided((d.shape[0], pitch), (pitch, 1))[:, 301:] == 7.0).all()


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('out,add,in_place', [(torch.float32, False, False), (torch.float32, True, False),
                                              (torch.float32, True, True), (torch.bfloat16, False, False),
                                              (torch.bfloat16, True, False), (torch.bfloat16, True, True)])
@pytest.mark.parametrize('sizes,m,n,alignment', [
    ([1], 1, 1, 1), ([1], 8, 8, 1), ([0], 16, 16, 1), ([3], 65, 33, 1), (MIXED, 129, 264, 1), (MIXED, 72, 130, 16),
    (MIXED, 256, 128, 128), ([1, 0, 2] * 30, 40, 48, 1), ([300, 0, 131, 65], 390, 520, 1)])
def test_k_grouped(eight, out, add, in_place, sizes, m, n, alignment):
    assert tn_whole_tiles(m, n, len(sizes), 1) == -(-m // 256) * -(-n // 256) * len(sizes)
    k_grouped(sizes, m, n, alignment, out, add, eight, in_place)


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('rows', [1, 2, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 129, 191, 192, 193, 255, 256, 257, 1000])
def test_k_grouped_lengths(eight, rows):
    k_grouped([13, rows, 5], 300, 270, eight=eight, add=True)


@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
def test_k_grouped_output_pitch(out):
    """Rows that begin anywhere: no 16-byte accesses, with and without C."""
    for add in (False, True):
        d = k_grouped([300, 210], 290, 301, d_pitch=307, out=out, add=add)
        assert (d.as_strided((2, 290, 307), (290 * 307, 307, 1))[..., 301:] == 7.0).all()


@pytest.mark.parametrize('mixed', [False, True])
@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('m,n', [(1, 4), (31, 100), (33, 252), (95, 256), (129, 260), (160, 101), (161, 516), (255, 8), (257, 257),
                                 (390, 300), (2000, 260)])
def test_c_loaded_ahead(m, n, eight, mixed):
    """FP32 D with C is D without it plus C, to the bit, for groups of 0 to 11 steps of 64 rows
    (C is loaded under the last steps from 3 on, with codes from 2 on), tiles that end inside
    a 32-row slab, C with a pitch, NaN between its rows and groups, and C in place."""
    sizes = [0, 1, 64, 65, 128, 129, 192, 193, 257, 320, 700]
    seg, g = segments(sizes), len(sizes)
    cus = 1 if not mixed else 24 if m == 2000 else 16
    deep_gemm.set_num_sms(cus)
    left = tn_whole_tiles(m, n, g, cus)
    assert left == -(-m // 256) * -(-n // 256) * g if cus == 1 else left > 0
    print(f'm={m} n={n} eight={eight} cus={cus}: {left} whole tiles', flush=True)
    a, a64 = matrix((seg[-1][1], m), 21)
    b, b64 = matrix((seg[-1][1], n), 22)
    if eight:
        q, sf, b64 = cast8(b64)
        codes = torch.full((seg[-1][1], -(-n // 8) * 8), 0x7F, dtype=torch.uint8)
        codes[:, :n] = q.view(torch.uint8)
        b = (codes.to(DEV).view(torch.float8_e4m3fn)[:, :n], sf.to(DEV))
    plain = torch.full((g, m, n), 7.0, device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, plain, ends_of(seg))
    torch.cuda.synchronize()
    for i, (lo, hi) in enumerate(seg):
        ref = a64[lo:hi].T @ b64[lo:hi]
        check(plain[i], ref, rounding(plain.dtype, ref) + sum_error(hi - lo, a64[lo:hi].abs().T @ b64[lo:hi].abs()), f'group {i}')
    gen = torch.Generator(DEV).manual_seed(23)
    pitch = -(-n // 4) * 4
    for gap in (0, 8, 3):     # (3: rows that begin anywhere, C is not loaded ahead)
        wide = torch.full((g, m + 3, pitch + gap), float('nan'), device=DEV)
        c = wide[:, :m, :n]
        c.copy_(torch.randn((g, m, n), generator=gen, device=DEV))
        want = plain + c
        d = torch.full((g, m, pitch), 7.0, device=DEV)
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, d[..., :n], ends_of(seg), c=c)
        torch.cuda.synchronize()
        assert torch.equal(d[..., :n], want) and (d[..., n:] == 7.0).all(), f'gap {gap}'
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, c, ends_of(seg), c=c)
        torch.cuda.synchronize()
        assert torch.equal(c, want), f'in place, gap {gap}'
        inside = torch.zeros_like(wide, dtype=torch.bool)
        inside[:, :m, :n] = True
        assert torch.isnan(wide[~inside]).all(), f'in place, gap {gap}: written beside'


@pytest.mark.parametrize('direction', ['nt', 'nn'])
def test_weights_past_32_bits(direction):
    n, k = (36000, 32768) if direction == 'nt' else (32768, 36000)
    b = torch.empty((3, n, k) if direction == 'nt' else (3, k, n), dtype=torch.bfloat16, device=DEV)
    b[2].normal_(generator=torch.Generator(DEV).manual_seed(1))
    a, a64 = matrix((5, k), 2)
    d = torch.full((5, n), 7.0, device=DEV)
    fn = deep_gemm.m_grouped_bf16_gemm_nt_ragged if direction == 'nt' else deep_gemm.m_grouped_bf16_gemm_nn_ragged
    fn(a, b, d, torch.tensor([0, 0, 5], dtype=torch.int32, device=DEV))
    cols = [0, 1, 17999, n - 1]
    w = (b[2, cols].T if direction == 'nt' else b[2][:, cols]).double().cpu()
    ref = a64 @ w
    check(d[:, cols], ref, rounding(d.dtype, ref) + sum_error(k, a64.abs() @ w.abs()), 'weights past 2^31')


@pytest.mark.parametrize('eight', [False, True])
def test_c_and_result_past_32_bits(eight):
    """C in place, of 2.4e9 FP32 values: the last rows of the last group."""
    m, n, rows = 32768, 36864, 210
    a, a64 = matrix((rows, m), 5)
    b, b64 = matrix((rows, n), 6)
    if eight:
        q, sf, b64 = cast8(b64)
        b = (q.to(DEV), sf.to(DEV))
    d = torch.full((2, m, n), 3.0, device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, d, ends_of([(0, 4), (4, rows)]), c=d)
    for g, lo, hi in ((0, 0, 4), (1, 4, rows)):
        at, bt = a64[lo:hi, -70:], b64[lo:hi, -70:]
        ref, mag = at.T @ bt + 3.0, at.abs().T @ bt.abs()
        check(d[g, -70:, -70:], ref, rounding(d.dtype, ref) + sum_error(hi - lo, mag) + 2.0 ** -23 * (mag + 3.0), f'group {g}')
