"""The BF16 products over ragged row segments against plain sums in 64 bits: every
direction, output type and layout, segments of no rows, one row and many, rows outside the
groups, odd sizes, wide and unaligned pitches, and what lies beside the operands.

Bounds (ragged.py): half a step of D's type, plus the FP32 sum's.
"""
import pytest
import torch

import deep_gemm
from ragged import DEV, bits, cast8, check, ends_of, matrix, rounding, segments, sum_error

pytestmark = pytest.mark.gpu

MIXED = [5, 0, 1, 130, 0, 64, 257, 31, 0]


@pytest.fixture(autouse=True, params=['heuristic', '256', '128', '128 in 3 pieces', '32', '32 in 2 pieces'])
def tiles(request):
    """Every test with the tiles the sizes choose, and with each kind forced."""
    block, pieces = {'heuristic': (0, 0), '256': (256, 0), '128': (128, 1), '128 in 3 pieces': (128, 3), '32': (32, 1), '32 in 2 pieces': (32, 2)}[request.param]
    if block:
        deep_gemm.set_tile_override(block, pieces, variant=13)
    yield request.param
    deep_gemm.set_tile_override(0, 0)


def m_grouped(direction, sizes, n, k, alignment=1, out=torch.bfloat16, spare=3, seed=0, d_pitch=None):
    print(f'{direction} sizes={sizes} n={n} k={k} alignment={alignment} {out}', flush=True)
    seg = segments(sizes, alignment)
    rows, g = seg[-1][1] + spare, len(sizes)
    inside = torch.zeros(rows, dtype=torch.bool)
    for lo, hi in seg:
        inside[lo:hi] = True
    a, a64 = matrix((rows, k), seed)
    a[~inside.to(DEV)] = float('nan')          # rows of no group hold anything
    b, b64 = matrix((g, n, k) if direction == 'nt' else (g, k, n), seed + 1)
    for i, s in enumerate(sizes):
        if s == 0:
            b[i] = float('nan')                # and so do weights that no row uses
    d = torch.full((rows, d_pitch or n), 7.0, dtype=out, device=DEV)[:, :n]
    fn = deep_gemm.m_grouped_bf16_gemm_nt_ragged if direction == 'nt' else deep_gemm.m_grouped_bf16_gemm_nn_ragged
    fn(a, b, d, ends_of(seg), alignment=alignment)
    torch.cuda.synchronize()
    for i, (lo, hi) in enumerate(seg):
        if hi > lo:
            w = b64[i].T if direction == 'nt' else b64[i]
            ref, mag = a64[lo:hi] @ w, a64[lo:hi].abs() @ w.abs()
            s = sum_error(k, mag)
            check(d[lo:hi], ref, rounding(out, ref) + s * (1 + torch.finfo(out).eps), f'group {i}')
    assert (d[~inside.to(DEV)] == 7.0).all(), 'rows of no group were written'
    return d


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('sizes,n,k,alignment', [
    ([1], 1, 8, 1), ([1], 64, 64, 1), ([3], 65, 8, 1), ([7], 130, 72, 1), ([0, 1, 0, 1], 33, 120, 1),
    (MIXED, 129, 264, 1), (MIXED, 255, 128, 16), (MIXED, 256, 64, 128), ([300], 520, 1000, 1),
    ([1] * 70, 40, 136, 1), ([0] * 65 + [9, 0, 2], 96, 256, 16), ([513, 255, 256, 257, 1], 257, 192, 1)])
def test_m_grouped(direction, out, sizes, n, k, alignment):
    m_grouped(direction, sizes, n, k, alignment, out)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('k', [8, 16, 56, 64, 104, 120, 128, 136, 248, 256, 264, 4096])
def test_m_grouped_reduced_lengths(direction, k):
    m_grouped(direction, [17, 140], 72, k)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('n', [2, 7, 8, 31, 63, 127, 128, 191, 256, 383, 511])
def test_m_grouped_columns(direction, n):
    m_grouped(direction, [40, 3], n, 96, out=torch.float32)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('rows', [1, 2, 8, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128, 129, 1000])
def test_m_grouped_rows(direction, rows):
    """From a single token to many, over 1 and over 40 groups (fewer rows a group than any tile)."""
    m_grouped(direction, [rows], 320, 512)
    per = [rows // 40 + (i * 7 % 40 < rows % 40) for i in range(40)]
    assert sum(per) == rows
    m_grouped(direction, per, 320, 512)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
@pytest.mark.parametrize('pitch', [101, 102, 104, 130, 4000])
def test_m_grouped_output_pitch(direction, pitch):
    """D's rows start anywhere; what lies between them stays."""
    d = m_grouped(direction, [150, 9], 101, 64, d_pitch=pitch)
    assert (d.as_strided((d.shape[0], pitch), (pitch, 1))[:, 101:] == 7.0).all()


def test_m_grouped_more_groups_than_a_wave_and_wide_k():
    m_grouped('nt', [(i * 37) % 5 for i in range(300)], 64, 2048)
    m_grouped('nn', [(i * 37) % 5 for i in range(300)], 64, 2048)


@pytest.mark.parametrize('direction', ['nt', 'nn'])
def test_m_grouped_large(direction):
    """Tiles of every size inside one call, more tiles than compute units."""
    m_grouped(direction, [1400, 0, 700, 1, 333, 2048], 2304, 320, out=torch.bfloat16)


def test_m_grouped_empty_calls():
    """No rows, no columns, no groups: nothing happens. No reduced elements: zeros."""
    d = torch.full((4, 8), 7.0, dtype=torch.bfloat16, device=DEV)
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)
    ends = torch.tensor([3], dtype=torch.int32, device=DEV)
    deep_gemm.m_grouped_bf16_gemm_nt_ragged(z(0, 16), z(1, 8, 16), d[:0], ends)
    deep_gemm.m_grouped_bf16_gemm_nt_ragged(z(4, 16), z(1, 0, 16), d[:, :0], ends)
    deep_gemm.m_grouped_bf16_gemm_nn_ragged(z(4, 16), z(0, 16, 8), d, ends[:0])
    torch.cuda.synchronize()
    assert (d == 7.0).all()
    for fn, b in ((deep_gemm.m_grouped_bf16_gemm_nt_ragged, z(1, 8, 0)), (deep_gemm.m_grouped_bf16_gemm_nn_ragged, z(1, 0, 8))):
        d.fill_(7.0)
        fn(z(4, 0), b, d, ends)
        assert (d[:3] == 0).all() and (d[3:] == 7.0).all()


@pytest.mark.parametrize('ends', [[-5, 2, 9], [9, 9, 1 << 30], [5, 2, 5], [0, 0, 0]])
def test_m_grouped_ends_outside_the_rows(ends):
    """Ends below zero, past the rows and decreasing ones are cut off: nothing is written
    outside D, and groups in order hold their products."""
    a, a64 = matrix((9, 32), 1)
    b, b64 = matrix((3, 16, 32), 2)
    d = torch.full((11, 16), 7.0, dtype=torch.float32, device=DEV)
    deep_gemm.m_grouped_bf16_gemm_nt_ragged(a, b, d[1:10], torch.tensor(ends, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert (d[0] == 7.0).all() and (d[10] == 7.0).all()
    if ends == [9, 9, 1 << 30]:
        ref = a64 @ b64[0].T
        check(d[1:10], ref, rounding(d.dtype, ref) + sum_error(32, a64.abs() @ b64[0].T.abs()), 'group 0')
    if ends == [0, 0, 0]:
        assert (d == 7.0).all()


def test_m_grouped_non_finite_rows_stay_in_their_rows():
    """An Inf or NaN of one row or weight shows in its own outputs only."""
    for fn, shape in ((deep_gemm.m_grouped_bf16_gemm_nt_ragged, (2, 70, 72)),
                      (deep_gemm.m_grouped_bf16_gemm_nn_ragged, (2, 72, 70))):
        a, _ = matrix((20, 72), 3)
        b, _ = matrix(shape, 4)
        seg = segments([11, 9])
        ref = torch.zeros((20, 70), dtype=torch.float32, device=DEV)
        fn(a, b, ref, ends_of(seg))
        a[4, 71], a[12, 0] = float('inf'), float('nan')
        if shape[1] == 70:
            b[1, 69, 5] = float('nan')
        else:
            b[1, 5, 69] = float('nan')
        d = torch.zeros_like(ref)
        fn(a, b, d, ends_of(seg))
        torch.cuda.synchronize()
        bad = torch.zeros_like(d, dtype=torch.bool)
        bad[4], bad[12], bad[11:, 69] = True, True, True
        assert (~torch.isfinite(d) == bad).all()
        assert torch.equal(d[~bad], ref[~bad])


def k_grouped(sizes, m, n, alignment=1, out=torch.float32, add=False, eight=False, in_place=False, spare=2, seed=0,
              d_pitch=None):
    print(f'tn sizes={sizes} m={m} n={n} alignment={alignment} {out} add={add} eight={eight}', flush=True)
    seg = segments(sizes, alignment)
    rows, g = seg[-1][1] + spare, len(sizes)
    inside = torch.zeros(rows, dtype=torch.bool)
    for lo, hi in seg:
        inside[lo:hi] = True
    a, a64 = matrix((rows, m), seed)
    a[~inside.to(DEV)] = float('nan')
    if eight:
        _, b64 = matrix((rows, n), seed + 1)
        q, sf, b64 = cast8(b64)
        wide = torch.full((rows, -(-n // 8) * 8), 0x7F, dtype=torch.uint8)     # NaN codes between the rows
        wide[:, :n] = q.view(torch.uint8)
        wide[~inside] = 0x7F
        sf = sf.clone()
        sf[~inside] = float('nan')
        b = (wide.to(DEV).view(torch.float8_e4m3fn)[:, :n], sf.to(DEV))
    else:
        b, b64 = matrix((rows, n), seed + 1)
        b[~inside.to(DEV)] = float('inf')
    c = c64 = None
    d = torch.full((g, m, d_pitch or n), 7.0, dtype=out, device=DEV)[..., :n]
    if add:
        c = torch.randn((g, m, n), generator=torch.Generator().manual_seed(seed + 2)).to(out).to(DEV)
        c64 = c.double().cpu()
        if in_place:
            d.copy_(c)
            c = d
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, d, ends_of(seg), c=c, alignment=alignment)
    torch.cuda.synchronize()
    for i, (lo, hi) in enumerate(seg):
        ref, mag = a64[lo:hi].T @ b64[lo:hi], a64[lo:hi].abs().T @ b64[lo:hi].abs()
        s = sum_error(hi - lo, mag)
        if c64 is not None:     # one more FP32 addition
            ref = ref + c64[i]
            s = s + 2.0 ** -23 * (mag + c64[i].abs())
        check(d[i], ref, rounding(out, ref) + s * (1 + torch.finfo(out).eps), f'group {i}')
    return d


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('out,add,in_place', [(torch.float32, False, False), (torch.float32, True, False),
                                              (torch.float32, True, True), (torch.bfloat16, False, False),
                                              (torch.bfloat16, True, True)])
@pytest.mark.parametrize('sizes,m,n,alignment', [
    ([1], 1, 1, 1), ([1], 8, 8, 1), ([0], 16, 16, 1), ([3], 65, 33, 1), (MIXED, 129, 264, 1), (MIXED, 72, 130, 16),
    (MIXED, 256, 128, 128), ([1, 0, 2] * 30, 40, 48, 1)])
def test_k_grouped(eight, out, add, in_place, sizes, m, n, alignment):
    k_grouped(sizes, m, n, alignment, out, add, eight, in_place)


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('rows', [1, 2, 15, 16, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 191, 192, 1000])
def test_k_grouped_lengths(eight, rows):
    """Every length of the summed axis around the kernels' steps, after a group that shifts its start."""
    k_grouped([13, rows, 5], 96, 160, eight=eight)


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('m,n', [(2, 7), (7, 2), (63, 65), (127, 129), (255, 257), (257, 255), (384, 513), (640, 128)])
def test_k_grouped_shapes(eight, m, n):
    k_grouped([40, 0, 71], m, n, eight=eight, add=True)


@pytest.mark.parametrize('eight', [False, True])
def test_k_grouped_long_few_outputs(eight):
    """A long summed axis with few outputs, and groups of very different lengths."""
    k_grouped([6000], 136, 72, eight=eight)
    k_grouped([3, 5000, 0, 700, 64], 72, 200, eight=eight, add=True)


def test_k_grouped_output_pitch():
    d = k_grouped([30, 21], 40, 101, d_pitch=107, add=True)
    assert (d.as_strided((2, 40, 107), (40 * 107, 107, 1))[..., 101:] == 7.0).all()


def test_k_grouped_large():
    k_grouped([700, 0, 1300, 65], 1030, 1544)
    k_grouped([700, 0, 1300, 65], 1030, 1544, eight=True, add=True)


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('m,n', [(1, 4), (33, 100), (129, 260), (161, 516), (300, 101)])
def test_k_grouped_adds_c_to_the_sums(m, n, eight):
    """FP32 D with C is D without it plus C, to the bit, for groups of 0 to 11 steps, C's rows
    as they lie (in place with a pitch, and apart with another one)."""
    sizes = [128, 129, 64, 192, 193, 0, 257, 700]
    seg = segments(sizes)
    a, _ = matrix((seg[-1][1], m), 21)
    b, b64 = matrix((seg[-1][1], n), 22)
    if eight:
        q, sf, _ = cast8(b64)
        codes = torch.full((seg[-1][1], -(-n // 8) * 8), 0x7F, dtype=torch.uint8)
        codes[:, :n] = q.view(torch.uint8)
        b = (codes.to(DEV).view(torch.float8_e4m3fn)[:, :n], sf.to(DEV))
    gen = torch.Generator(DEV).manual_seed(23)
    wide = torch.randn((len(sizes), m + 3, -(-n // 4) * 4 + 8), generator=gen, device=DEV)
    c = wide[:, :m, :n]
    plain = torch.empty((len(sizes), m, n), device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, plain, ends_of(seg))
    d = torch.full((len(sizes), m, -(-n // 4) * 4), 7.0, device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, d[..., :n], ends_of(seg), c=c)
    torch.cuda.synchronize()
    assert torch.equal(d[..., :n], plain + c) and (d[..., n:] == 7.0).all()
    ref = wide.clone()
    ref[:, :m, :n] += plain
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, b, c, ends_of(seg), c=c)
    torch.cuda.synchronize()
    assert torch.equal(wide, ref)


def test_k_grouped_empty_calls():
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device=DEV)
    ends = torch.tensor([0, 0], dtype=torch.int32, device=DEV)
    d = torch.full((2, 8, 16), 7.0, device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(0, 8), z(0, 16), d, ends)       # no rows at all
    assert (d == 0).all()
    c = torch.randn(2, 8, 16, device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(5, 8), z(5, 16), d, ends, c=c)  # rows of no group
    assert torch.equal(d, c)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(5, 0), z(5, 16), d[:, :0], ends)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(5, 8), z(5, 16), d[:0], ends[:0])
    torch.cuda.synchronize()
    assert torch.equal(d, c)


def test_k_grouped_scales_of_any_value_and_layout():
    """FP32 scales that are no powers of two (values rounded to BF16 after their scale), in
    the MN-major layout."""
    rows, m, n = 77, 40, 200
    a, a64 = matrix((rows, m), 5)
    x = torch.randn((rows, n), generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    q, sf = deep_gemm.per_token_cast_to_fp8_mn_major(x, use_ue8m0=False)
    v = (q.float() * sf.repeat_interleave(128, 1)[:, :n]).bfloat16().double().cpu()
    d = torch.empty((1, m, n), device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, (q, sf), d, torch.tensor([rows], dtype=torch.int32, device=DEV))
    ref = a64.T @ v
    check(d[0], ref, rounding(d.dtype, ref) + sum_error(rows, a64.abs().T @ v.abs()), 'dequantised')


def test_gradients_against_differences():
    """L = <T, X W^T> over two groups: its difference quotients in 64 bits against the NN
    form (dL/dX) and the TN form (dL/dW)."""
    sizes, n, k = [9, 14], 24, 16
    seg = segments(sizes)
    x, x64 = matrix((23, k), 1)
    w, w64 = matrix((2, n, k), 2)
    t, t64 = matrix((23, n), 3)
    dx = torch.empty((23, k), device=DEV)
    dw = torch.empty((2, n, k), device=DEV)
    deep_gemm.m_grouped_bf16_gemm_nn_ragged(t, w, dx, ends_of(seg))
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(t, x, dw, ends_of(seg))

    def loss(xv, wv):
        return sum(float((t64[lo:hi] * (xv[lo:hi] @ wv[i].T)).sum()) for i, (lo, hi) in enumerate(seg))
    h = 2.0 ** -10
    for r, c in ((0, 0), (8, 15), (9, 3), (22, 7)):
        e = torch.zeros_like(x64)
        e[r, c] = h
        q = (loss(x64 + e, w64) - loss(x64 - e, w64)) / (2 * h)
        assert abs(q - float(dx[r, c])) < 1e-4     # 24 products of order 1: the FP32 sum's bound is 5e-5, the quotient's 1e-9
    for g, r, c in ((0, 0, 0), (0, 23, 15), (1, 11, 4)):
        e = torch.zeros_like(w64)
        e[g, r, c] = h
        q = (loss(x64, w64 + e) - loss(x64, w64 - e)) / (2 * h)
        assert abs(q - float(dw[g, r, c])) < 1e-4


# ---------------------------------------------------------------- graphs, streams

def _calls():
    seg = segments([40, 0, 3, 200], 16)
    rows, ends = seg[-1][1] + 4, ends_of(segments([40, 0, 3, 200], 16))
    a, _ = matrix((rows, 128), 1)
    w, _ = matrix((4, 136, 128), 2)
    t, _ = matrix((rows, 136), 3)
    q, sf = deep_gemm.per_token_cast_to_fp8(a.contiguous(), use_ue8m0=True)
    return [
        (lambda d: deep_gemm.m_grouped_bf16_gemm_nt_ragged(a, w, d, ends, alignment=16), torch.zeros((rows, 136), dtype=torch.bfloat16, device=DEV)),
        (lambda d: deep_gemm.m_grouped_bf16_gemm_nn_ragged(t, w, d, ends, alignment=16), torch.zeros((rows, 128), device=DEV)),
        (lambda d: deep_gemm.k_grouped_bf16_gemm_tn_ragged(t, a, d, ends, alignment=16), torch.zeros((4, 136, 128), device=DEV)),
        (lambda d: deep_gemm.k_grouped_bf16_gemm_tn_ragged(t, (q, sf), d, ends, alignment=16), torch.zeros((4, 136, 128), device=DEV)),
    ]


def test_graphs_replay_the_eager_results():
    """Two graphs, captured over the same calls, replayed in turn with eager calls between."""
    for run, out in _calls():
        run(out)
        torch.cuda.synchronize()
        ref, other = out.clone(), torch.zeros_like(out)
        graphs = []
        for d in (out, other):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                run(d)
            graphs.append(g)
        third = torch.zeros_like(out)
        for _ in range(3):
            out.zero_(), other.zero_(), third.zero_()
            for g in graphs:
                g.replay()
            run(third)
            torch.cuda.synchronize()
            assert torch.equal(bits(out), bits(ref)) and torch.equal(bits(other), bits(ref)) and torch.equal(bits(third), bits(ref))


def test_graphs_follow_the_group_ends():
    """A graph replayed with other ends in the same tensor: other segments, other counts."""
    a, _ = matrix((300, 64), 1)
    w, _ = matrix((5, 72, 64), 2)
    t, _ = matrix((300, 72), 3)
    ends = ends_of(segments([10, 0, 200, 30, 60]))
    d, e = torch.zeros((300, 72), device=DEV), torch.zeros((5, 72, 64), device=DEV)

    def run(d, e, ends):
        deep_gemm.m_grouped_bf16_gemm_nt_ragged(a, w, d, ends)
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(t, a, e, ends)
    run(d, e, ends)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(d, e, ends)
    for sizes in ([300, 0, 0, 0, 0], [60] * 5, [0, 0, 1, 0, 0], [1, 120, 1, 130, 48]):
        now = ends_of(segments(sizes))
        d.fill_(3.0), e.fill_(3.0)
        d2, e2 = torch.full_like(d, 3.0), torch.full_like(e, 3.0)
        ends.copy_(now)
        g.replay()
        run(d2, e2, now)
        torch.cuda.synchronize()
        assert torch.equal(bits(d), bits(d2)) and torch.equal(bits(e), bits(e2))


@pytest.mark.parametrize('sms', [7, 64])
def test_fewer_compute_units(sms):
    """Rounds, tails and plans of another number of CUs."""
    deep_gemm.set_num_sms(sms)
    try:
        m_grouped('nt', [700, 0, 1300, 65], 776, 192)
        m_grouped('nn', [700, 0, 1300, 65], 776, 192)
        k_grouped([300, 0, 130, 65], 776, 520, add=True)
        k_grouped([300, 0, 130, 65], 520, 776, eight=True)
    finally:
        deep_gemm.set_num_sms(256)


def test_offsets_past_32_bits(tiles):
    """Operands and results of more than 2^31 elements: their last group, row and column."""
    if tiles not in ('256', '128', '32'):
        pytest.skip('each kind of tile is enough')
    n, k = 36000, 32768
    print('nt, weights of 3.5e9 elements', flush=True)
    b = torch.empty((3, n, k), dtype=torch.bfloat16, device=DEV)
    b[2].normal_(generator=torch.Generator(DEV).manual_seed(1))
    a, a64 = matrix((5, k), 2)
    d = torch.full((5, n), 7.0, device=DEV)
    deep_gemm.m_grouped_bf16_gemm_nt_ragged(a, b, d, torch.tensor([0, 0, 5], dtype=torch.int32, device=DEV))
    cols = [0, 1, 17999, n - 1]
    w = b[2, cols].double().cpu()
    ref = a64 @ w.T
    check(d[:, cols], ref, rounding(d.dtype, ref) + sum_error(k, a64.abs() @ w.T.abs()), 'weights past 2^31')
    del b, d
    print('tn, rows past 2^31 elements', flush=True)
    rows, m = 70000, 32768
    t = torch.empty((rows, m), dtype=torch.bfloat16, device=DEV)
    t[-30:].normal_(generator=torch.Generator(DEV).manual_seed(3))
    x, x64 = matrix((rows, 40), 4)
    d = torch.empty((2, m, 40), device=DEV)
    seg = [(0, rows - 30), (rows - 30, rows)]
    t[:-30] = 0
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(t, x, d, ends_of(seg))
    ms = [0, 5, m - 1]
    tv = t[-30:, ms].double().cpu()
    ref = tv.T @ x64[-30:]
    check(d[1, ms], ref, rounding(d.dtype, ref) + sum_error(30, tv.abs().T @ x64[-30:].abs()), 'rows past 2^31')
    assert (d[0] == 0).all()
    del t, d
    print('tn, a result of 2.4e9 elements', flush=True)
    m, n = 32768, 36864
    t, t64 = matrix((9, m), 5)
    x, x64 = matrix((9, n), 6)
    d = torch.full((2, m, n), 7.0, dtype=torch.bfloat16, device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(t, x, d, ends_of([(0, 4), (4, 9)]))
    ref = t64[4:].T[-3:] @ x64[4:][:, -70:]
    mag = t64[4:].abs().T[-3:] @ x64[4:].abs()[:, -70:]
    check(d[1, -3:, -70:], ref, rounding(d.dtype, ref) + sum_error(5, mag) * 1.01, 'result past 2^31')


def test_two_streams_at_once():
    for run, out in _calls():
        run(out)
        torch.cuda.synchronize()
        ref = out.clone()
        streams, outs = [torch.cuda.Stream() for _ in range(2)], [torch.zeros_like(out) for _ in range(2)]
        torch.cuda.synchronize()
        for _ in range(4):
            for s, d in zip(streams, outs):
                with torch.cuda.stream(s):
                    run(d)
        torch.cuda.synchronize()
        for d in outs:
            assert torch.equal(bits(d), bits(ref))
