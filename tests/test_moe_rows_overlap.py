"""Places of the combination's gradient beside the rows that it reads: y itself, or memory of its own.
Calls of no tokens, which launch nothing: without a GPU those that are right end at the device."""
import itertools

import pytest
import torch

import deep_gemm
from deep_gemm import _ffi
from test_moe_rows_cpu import BF16, F32, I32, call, dev

AT = 1 << 24   # bytes


def status(y, dy, n):
    args = dict(dout=dev(BF16, 0, n), y=y, pos=dev(I32, 0, 2), w=dev(F32, 0, 2), dy=dy, dw=dev(F32, 0, 2))
    return call('dg_moe_combine_backward', *args.values())


@pytest.mark.parametrize('shape,strides', [((16, 64), (64, 1)), ((16, 64), (160, 1)), ((1, 64), (64, 1)), ((5, 3, 64), (200, 64, 1)),
                                           ((5, 3, 64), (512, 160, 1)), ((1, 3, 64), (0, 72, 1)), ((4, 1, 64), (136, 0, 1))])
def test_rows_that_overlap_are_refused(shape, strides):
    """Every offset, against the elements themselves."""
    y = dev(BF16, *shape, strides=strides, data=AT)
    elements = {sum(i * s for i, s in zip(at, strides)) for at in itertools.product(*map(range, shape))}
    end = max(elements) + 1
    for off in range(-end - 16, end + 17, 8):
        got = status(y, dev(BF16, *shape, strides=strides, data=AT + 2 * off), 64)
        wrong = off != 0 and any(e + off in elements for e in elements)
        assert (got == _ffi.DG_ERR_INVALID) == wrong, (off, got, _ffi.lib.dg_last_error())


def test_rows_of_other_strides():
    y = dev(BF16, 16, 64, strides=(160, 1), data=AT)
    for off, wrong in ((-16 * 64, False), (-16 * 64 + 8, True), (8, True), (15 * 160 + 56, True), (15 * 160 + 64, False)):
        assert (status(y, dev(BF16, 16, 64, data=AT + 2 * off), 64) == _ffi.DG_ERR_INVALID) == wrong, off


def test_nothing_overlaps_no_rows():
    assert status(dev(BF16, 0, 64, data=AT), dev(BF16, 0, 64, data=AT + 16), 64) != _ffi.DG_ERR_INVALID
    assert status(dev(BF16, 16, 0, data=AT), dev(BF16, 16, 0, data=AT + 16), 0) != _ffi.DG_ERR_INVALID


@pytest.mark.gpu
def test_gradient_beside_its_rows():
    """dy in other columns of y's buffer; a row on it is refused."""
    buf = torch.randn((9, 160), generator=torch.Generator().manual_seed(1)).bfloat16().to('cuda:0')
    dout = torch.randn((3, 64), generator=torch.Generator().manual_seed(2)).bfloat16().to('cuda:0')
    pos = torch.tensor([[0, 5], [8, -1], [2, 3]], dtype=torch.int32, device='cuda:0')
    w = torch.tensor([[1.0, 2.0], [0.5, 4.0], [-1.0, 1.0]], device='cuda:0')
    y = buf[:, :64]
    want, dw = deep_gemm.moe_combine_backward(dout, y.clone(), pos, w)
    with pytest.raises(RuntimeError):
        deep_gemm.moe_combine_backward(dout, buf[:8, :64], pos.clamp(max=7), w, out=buf[1:, :64])
    got, dw2 = deep_gemm.moe_combine_backward(dout, y, pos, w, out=buf[:, 80:144])
    named = [0, 5, 8, 2, 3]
    assert torch.equal(got[named], want[named]) and torch.equal(dw, dw2)
