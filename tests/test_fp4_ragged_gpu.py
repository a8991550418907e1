"""The 4-bit product over ragged row segments against plain sums in 64 bits: output types and
layouts, segments of no rows, one row and many, rows outside the groups, reduced lengths that end
inside a word of scales, scale layouts, wide pitches, and what lies beside the operands.

Bounds: half a step of D's type, plus the FP32 sum's (fp4_ragged.py).
"""
import pytest
import torch

import deep_gemm
from fp4_ragged import operand, sum_error
from ragged import DEV, bits, check, ends_of, rounding, segments

pytestmark = pytest.mark.gpu

MIXED = [5, 0, 1, 130, 0, 64, 257, 31, 0]


@pytest.fixture(autouse=True, params=['heuristic', '256', '128', '128 in 3 pieces', '64', '32', '32 in 2 pieces'])
def tiles(request):
    """Every test with the tiles the sizes choose, and with each kind forced."""
    block, pieces = {'heuristic': (0, 0), '256': (256, 0), '128': (128, 1), '128 in 3 pieces': (128, 3), '64': (64, 1), '32': (32, 1),
                     '32 in 2 pieces': (32, 2)}[request.param]
    if block:
        deep_gemm.set_tile_override(block, pieces, variant=14)
    yield request.param
    deep_gemm.set_tile_override(0, 0)


def product(sizes, n, k, alignment=1, out=torch.bfloat16, spare=3, seed=0, d_pitch=None, layout='rows', pitch=0, low=120, high=130):
    print(f'sizes={sizes} n={n} k={k} alignment={alignment} {out} {layout}', flush=True)
    seg = segments(sizes, alignment)
    rows, g = seg[-1][1] + spare, len(sizes)
    inside = torch.zeros(rows, dtype=torch.bool)
    for lo, hi in seg:
        inside[lo:hi] = True
    a, a64 = operand((rows, k), seed, low, high, layout, pitch=pitch)
    a[1][~inside.to(DEV)] = -1                 # rows of no group have NaN scales
    b, b64 = operand((g, n, k), seed + 1, low, high, layout, pitch=pitch)
    for i, s in enumerate(sizes):
        if s == 0:
            b[1][i] = -1                       # and so do weights that no row uses
    d = torch.full((rows, d_pitch or n), 7.0, dtype=out, device=DEV)[:, :n]
    deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d, ends_of(seg), alignment=alignment)
    torch.cuda.synchronize()
    for i, (lo, hi) in enumerate(seg):
        if hi > lo:
            ref, mag = a64[lo:hi] @ b64[i].T, a64[lo:hi].abs() @ b64[i].T.abs()
            check(d[lo:hi], ref, rounding(out, ref) + sum_error(k, mag) * (1 + torch.finfo(out).eps), f'group {i}')
    assert (d[~inside.to(DEV)] == 7.0).all(), 'rows of no group were written'
    return d


@pytest.mark.parametrize('out', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('sizes,n,k,alignment', [
    ([1], 1, 32, 1), ([1], 64, 64, 1), ([3], 65, 32, 1), ([7], 130, 288, 1), ([0, 1, 0, 1], 33, 480, 1),
    (MIXED, 129, 1056, 1), (MIXED, 255, 512, 16), (MIXED, 256, 256, 128), ([300], 520, 4000, 1),
    ([1] * 70, 40, 544, 1), ([0] * 65 + [9, 0, 2], 96, 1024, 16), ([513, 255, 256, 257, 1], 257, 768, 1)])
def test_product(out, sizes, n, k, alignment):
    product(sizes, n, k, alignment, out)


@pytest.mark.parametrize('k', [32, 64, 96, 128, 160, 192, 224, 256, 288, 384, 416, 480, 512, 544, 1000 // 32 * 32, 1024, 1056, 8192])
def test_reduced_lengths(k):
    product([17, 140], 72, k)


@pytest.mark.parametrize('n', [2, 7, 8, 31, 63, 127, 128, 191, 256, 383, 511])
def test_columns(n):
    product([40, 3], n, 384, out=torch.float32)


@pytest.mark.parametrize('rows', [1, 2, 8, 15, 16, 17, 32, 33, 48, 64, 65, 100, 128, 129, 1000])
def test_rows(rows):
    """From a single token to many, over 1 and over 40 groups (fewer rows a group than any tile)."""
    product([rows], 320, 2048)
    per = [rows // 40 + (i * 7 % 40 < rows % 40) for i in range(40)]
    assert sum(per) == rows
    product(per, 320, 2048)


@pytest.mark.parametrize('layout', ['rows', 'columns', 'padded'])
@pytest.mark.parametrize('k', [96, 512, 640, 1056, 2048])
def test_scale_layouts(layout, k):
    """Words of a row side by side (also in rows that begin anywhere), or words of a column."""
    product([200, 0, 60], 160, k, layout=layout)
    product([3, 1], 160, k, layout=layout)


@pytest.mark.parametrize('pitch', [16, 48, 4096])
def test_operand_pitch(pitch):
    product([150, 9], 200, 352, pitch=pitch)


@pytest.mark.parametrize('pitch', [101, 102, 104, 130, 4000])
def test_output_pitch(pitch):
    """D's rows start anywhere; what lies between them stays."""
    d = product([150, 9], 101, 256, d_pitch=pitch)
    assert (d.as_strided((d.shape[0], pitch), (pitch, 1))[:, 101:] == 7.0).all()


def test_scales_far_apart():
    """Scales over the whole range that FP32 sums of the products hold."""
    product([40], 96, 320, out=torch.float32, low=70, high=180)


def test_more_groups_than_a_wave_and_a_long_axis():
    product([(i * 37) % 5 for i in range(300)], 64, 8192)


def test_large():
    """Tiles of every size inside one call, more tiles than compute units."""
    product([1400, 0, 700, 1, 333, 2048], 2304, 1280)


def test_every_code_and_scale_position():
    """One element of A at a time meets a row of B of ones: each code, each of the 8 scale
    positions of a step, shows alone in its output."""
    k = 512
    codes = torch.zeros((k, k), dtype=torch.uint8)
    codes[torch.arange(k), torch.arange(k)] = (torch.arange(k) % 16).to(torch.uint8)
    scales = (120 + torch.arange(k)[:, None] % 13 + torch.arange(16)[None]).to(torch.uint8)
    from fp4_ragged import values
    v = values(codes, scales)
    a = ((codes[:, 0::2] | codes[:, 1::2] << 4).view(torch.int8).to(DEV), scales.view(torch.int32).to(DEV))
    ones = torch.full((1, 40, k // 2), 0x22, dtype=torch.int8, device=DEV)
    b_scales = (119 + torch.arange(16)).to(torch.uint8).expand(1, 40, 16).contiguous()
    b = (ones, b_scales.view(torch.int32).to(DEV))
    ref = v @ torch.exp2(b_scales[0].double() - 127).repeat_interleave(32, 1).T
    d = torch.empty((k, 40), dtype=torch.float32, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d, torch.tensor([k], dtype=torch.int32, device=DEV))
    assert torch.equal(d.double().cpu(), ref)


def test_empty_calls():
    """No rows, no columns, no groups: nothing happens. No reduced elements: zeros."""
    d = torch.full((4, 8), 7.0, dtype=torch.bfloat16, device=DEV)
    q = lambda *s: torch.zeros(s, dtype=torch.int8, device=DEV)
    w = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)
    ends = torch.tensor([3], dtype=torch.int32, device=DEV)
    run = deep_gemm.m_grouped_fp4_gemm_nt_ragged
    run((q(0, 16), w(0, 1)), (q(1, 8, 16), w(1, 8, 1)), d[:0], ends)
    run((q(4, 16), w(4, 1)), (q(1, 0, 16), w(1, 0, 1)), d[:, :0], ends)
    run((q(4, 16), w(4, 1)), (q(0, 8, 16), w(0, 8, 1)), d, ends[:0])
    torch.cuda.synchronize()
    assert (d == 7.0).all()
    run((q(4, 0), w(4, 0)), (q(1, 8, 0), w(1, 8, 0)), d, ends)
    assert (d[:3] == 0).all() and (d[3:] == 7.0).all()


@pytest.mark.parametrize('ends', [[-5, 2, 9], [9, 9, 1 << 30], [5, 2, 5], [0, 0, 0]])
def test_ends_outside_the_rows(ends):
    """Ends below zero, past the rows and decreasing ones are cut off: nothing is written
    outside D, and groups in order hold their products."""
    a, a64 = operand((9, 64), 1)
    b, b64 = operand((3, 16, 64), 2)
    d = torch.full((11, 16), 7.0, dtype=torch.float32, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d[1:10], torch.tensor(ends, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    assert (d[0] == 7.0).all() and (d[10] == 7.0).all()
    if ends == [9, 9, 1 << 30]:
        ref = a64 @ b64[0].T
        check(d[1:10], ref, rounding(d.dtype, ref) + sum_error(64, a64.abs() @ b64[0].T.abs()), 'group 0')
    if ends == [0, 0, 0]:
        assert (d == 7.0).all()


def test_a_nan_scale_stays_in_its_row():
    a, _ = operand((200, 384), 1)
    b, _ = operand((1, 130, 384), 2)
    ends = torch.tensor([200], dtype=torch.int32, device=DEV)
    clean = torch.empty((200, 130), dtype=torch.float32, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, clean, ends)
    a[1].view(torch.uint8)[77, 9] = 255
    b[1].view(torch.uint8)[0, 5, 2] = 255
    d = torch.empty_like(clean)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d, ends)
    bad = torch.zeros((200, 130), dtype=torch.bool, device=DEV)
    bad[77], bad[:, 5] = True, True
    assert torch.equal(torch.isnan(d), bad)
    assert torch.equal(bits(d[~bad]), bits(clean[~bad]))


def test_runs_are_alike_and_on_another_stream():
    a, _ = operand((700, 2048), 1)
    b, _ = operand((4, 512, 2048), 2)
    ends = torch.tensor([100, 100, 650, 700], dtype=torch.int32, device=DEV)
    first = torch.zeros((700, 512), dtype=torch.bfloat16, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, first, ends)
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        outs = [torch.zeros_like(first) for _ in range(3)]
        for d in outs:
            deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d, ends)
    stream.synchronize()
    assert all(torch.equal(bits(d), bits(first)) for d in outs)


def test_graph_follows_its_ends():
    """A captured call reads group_ends when it is replayed."""
    a, a64 = operand((40, 1024), 1)
    b, b64 = operand((3, 96, 1024), 2)
    ends = torch.tensor([40, 40, 40], dtype=torch.int32, device=DEV)
    d = torch.empty((40, 96), dtype=torch.float32, device=DEV)
    run = lambda: deep_gemm.m_grouped_fp4_gemm_nt_ragged(a, b, d, ends)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for now in ([40, 40, 40], [0, 13, 40], [1, 1, 39], [13, 20, 40]):
        ends.copy_(torch.tensor(now, dtype=torch.int32))
        d.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        lo = 0
        for g, hi in enumerate(now):
            ref = a64[lo:hi] @ b64[g].T
            if hi > lo:
                check(d[lo:hi], ref, rounding(d.dtype, ref) + sum_error(1024, a64[lo:hi].abs() @ b64[g].T.abs()), f'{now} {g}')
            lo = hi
        assert (d[lo:] == 7.0).all()


def test_rows_past_32_bits():
    """A's codes, its scales' rows and D's rows of a group that begins past 2^32 bytes of A."""
    k, n, first, rows = 8192, 64, 1 << 20, 70
    total = first + rows
    codes = torch.zeros((total, k // 2), dtype=torch.int8, device=DEV)
    scales = torch.full((total, k // 128), -1, dtype=torch.int32, device=DEV)
    (q0, s0), head = operand((5, k), 1)
    (q1, s1), tail = operand((rows, k), 2)
    codes[:5], scales[:5], codes[first:], scales[first:] = q0, s0, q1, s1
    b, b64 = operand((2, n, k), 3)
    d = torch.full((total, n), 7.0, dtype=torch.bfloat16, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged((codes, scales), b, d, torch.tensor([5, total], dtype=torch.int32, device=DEV), alignment=first)
    torch.cuda.synchronize()
    for got, a, w in ((d[:5], head, b64[0]), (d[first:], tail, b64[1])):
        ref, mag = a @ w.T, a.abs() @ w.T.abs()
        check(got, ref, rounding(torch.bfloat16, ref) + sum_error(k, mag) * (1 + 2.0 ** -7), 'rows')
    assert (d[5:first] == 7.0).all()


def test_scales_words_far_apart():
    """Words of scales nearly 2^30 bytes apart, of A (a step has two of them, two steps four)."""
    k, n, rows = 544, 40, 33
    a, a64 = operand((rows, k), 1)
    b, b64 = operand((1, n, k), 2)
    pitch = (1 << 28) - 64
    far = torch.empty(4 * pitch + rows, dtype=torch.int32, device=DEV)
    words = far.as_strided((rows, 5), (1, pitch))
    words.copy_(a[1])
    d = torch.zeros((rows, n), dtype=torch.float32, device=DEV)
    deep_gemm.m_grouped_fp4_gemm_nt_ragged((a[0], words), b, d, torch.tensor([rows], dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    ref, mag = a64 @ b64[0].T, a64.abs() @ b64[0].T.abs()
    check(d, ref, rounding(torch.float32, ref) + sum_error(k, mag) * (1 + 2.0 ** -7), 'far words')


def test_workspace_sizes(tiles):
    size = deep_gemm._ffi.lib.dg_fp4_gemm_ragged_workspace_size
    pieces = {'32 in 2 pieces': 2, '128 in 3 pieces': 3}.get(tiles, 0)
    if tiles != 'heuristic':
        assert size(10, 30, 4096, 2) == 10 * 32 * 4 * pieces   # each piece's FP32 sums, rows of whole fours
    assert size(1 << 29, 1 << 20, 256, 1) == -1                # more threads than a launch counts
