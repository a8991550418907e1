"""What the row dispatch, its gradients and the 4-bit operators refuse, before anything is launched
(no GPU: device tensors are described, not touched), and the binding's own behaviour."""
import ctypes
import threading

import pytest
import torch

import deep_gemm
from deep_gemm import _ffi
from test_bind_cpu import stub  # noqa: F401

lib = _ffi.lib
BF16, F32, E4M3, I32, I8, I64 = _ffi.DG_BF16, _ffi.DG_F32, _ffi.DG_E4M3, _ffi.DG_I32, _ffi.DG_I8, _ffi.DG_I64


def dev(dtype, *sizes, strides=None, data=1 << 20, device=0):
    """A device tensor that is only described."""
    t = _ffi.DgTensor()
    t.data, t.dtype, t.ndim, t.device = data, dtype, len(sizes), device
    if strides is None:
        strides, n = [0] * len(sizes), 1
        for i in reversed(range(len(sizes))):
            strides[i], n = n, n * sizes[i]
    for i, (s, p) in enumerate(zip(sizes, strides)):
        t.sizes[i], t.strides[i] = s, p
    return t


def call(entry, *args):
    args = [ctypes.byref(a) if isinstance(a, _ffi.DgTensor) else a for a in args]
    return getattr(lib, entry)(*args, None)


def refused(entry, args, changes, status=_ffi.DG_ERR_INVALID):
    """Every change of one argument of a call that is right is refused, with a message."""
    for name, value in changes:
        new = dict(args)
        assert name in new
        new[name] = value
        got = call(entry, *new.values())
        assert got == status, (name, got)
        assert b'error (' in lib.dg_last_error()


DISPATCH = dict(x=dev(BF16, 8, 64), x_sf=None, topk=dev(I32, 8, 2), topk_w=None, experts=4, layout=1, alignment=1,
                a=dev(BF16, 16, 64), sf=None, meta=dev(I32, 4), pos=dev(I32, 8, 2), w=None, ws=dev(I32, 64))


def test_dispatch_of_bf16_rows_refuses():
    refused('dg_moe_dispatch', DISPATCH, [
        ('x', dev(F32, 8, 64)), ('x', dev(BF16, 8, 60)), ('x', dev(BF16, 8, 64, strides=(1, 8))), ('x', dev(BF16, 8, 64, data=8)),
        ('x', dev(BF16, 8, 64, strides=(66, 1))), ('x', dev(BF16, 8, 64, device=-1)), ('x', dev(BF16, 7, 64)), ('x', None),
        ('x_sf', dev(F32, 8, 1)), ('sf', dev(F32, 16, 1)), ('a', dev(E4M3, 16, 64)), ('a', dev(BF16, 15, 64)),
        ('a', dev(BF16, 16, 72)), ('a', dev(BF16, 4, 16, 64)), ('a', dev(BF16, 16, 64, device=1)), ('alignment', 0), ('alignment', -1),
        ('alignment', (1 << 20) + 1), ('experts', 0), ('experts', 1025), ('layout', 3), ('meta', dev(I32, 5)), ('meta', dev(I64, 4)),
        ('pos', dev(I32, 8, 3)), ('topk', dev(I32, 8, 17)), ('topk', dev(F32, 8, 2)), ('topk_w', dev(F32, 8, 3)), ('w', dev(F32, 15)),
        ('ws', dev(I32, 5)), ('ws', None)])


def test_dispatch_of_4_bit_rows_refuses():
    args = dict(DISPATCH, x=dev(I8, 8, 64), x_sf=dev(I32, 8, 1), a=dev(I8, 16, 64), sf=dev(I32, 16, 1))
    refused('dg_moe_dispatch', args, [
        ('x', dev(I8, 8, 56)), ('x_sf', None), ('x_sf', dev(F32, 8, 1)), ('x_sf', dev(I32, 8, 2)), ('x_sf', dev(I32, 7, 1)), ('sf', None),
        ('sf', dev(F32, 16, 1)), ('sf', dev(I32, 15, 1)), ('sf', dev(I32, 16, 2)), ('a', dev(BF16, 16, 64)), ('a', dev(I8, 16, 80))])


def test_dispatch_of_8_bit_rows_still_takes_padded_alignments_only():
    args = dict(DISPATCH, x=dev(E4M3, 8, 64), x_sf=dev(F32, 8, 1), a=dev(E4M3, 76, 64), sf=dev(F32, 76, 1), alignment=16)
    refused('dg_moe_dispatch', args, [('alignment', 8), ('alignment', 1), ('x_sf', None), ('sf', None), ('x_sf', dev(I32, 8, 1))])


def test_dispatch_backward_refuses():
    args = dict(drows=dev(BF16, 16, 64), pos=dev(I32, 8, 2), drow_w=dev(F32, 16), dx=dev(BF16, 8, 64), dw=dev(F32, 8, 2))
    refused('dg_moe_dispatch_backward', args, [
        ('drows', dev(F32, 16, 64)), ('drows', dev(BF16, 16, 72)), ('drows', dev(BF16, 16, 64, strides=(64, 2))),
        ('drows', dev(BF16, 16, 64, strides=(60, 1))), ('drows', dev(BF16, 16, 64, data=2)), ('drows', dev(BF16, 16, 64, device=-1)),
        ('drows', dev(BF16, 64)), ('drows', None), ('pos', dev(I64, 8, 2)), ('pos', dev(I32, 7, 2)), ('pos', dev(I32, 8, 17)), ('pos', dev(I32, 8, 0)),
        ('pos', dev(I32, 8, 2, strides=(1, 8))), ('drow_w', None), ('drow_w', dev(F32, 15)), ('drow_w', dev(BF16, 16)), ('dw', None),
        ('dw', dev(F32, 8, 3)), ('dw', dev(F32, 8, 2, strides=(1, 8))), ('dx', dev(BF16, 8, 60)), ('dx', dev(F32, 8, 64)),
        ('dx', dev(BF16, 8, 64, strides=(32, 1))), ('dx', dev(BF16, 8, 64, device=1))])
    # more threads than a launch counts
    big = dict(drows=dev(BF16, 16, 8), pos=dev(I32, 1 << 27, 2), drow_w=None, dx=dev(BF16, 1 << 27, 8), dw=None)
    assert call('dg_moe_dispatch_backward', *big.values()) == _ffi.DG_ERR_INVALID


def test_combine_backward_refuses():
    args = dict(dout=dev(BF16, 8, 64), y=dev(BF16, 16, 64, data=1 << 24), pos=dev(I32, 8, 2), w=dev(F32, 8, 2), dy=dev(BF16, 16, 64),
                dw=dev(F32, 8, 2))
    refused('dg_moe_combine_backward', args, [
        ('dout', dev(BF16, 8, 60)), ('dout', dev(F32, 8, 64)), ('dout', dev(BF16, 8, 64, data=8)), ('y', None), ('y', dev(BF16, 15, 64)),
        ('y', dev(BF16, 2, 8, 64)), ('y', dev(F32, 16, 64)), ('y', dev(BF16, 16, 64, strides=(72, 1))),   # (at dy: in place with other rows)
        ('pos', dev(I32, 9, 2)), ('w', None), ('w', dev(BF16, 8, 2)), ('w', dev(F32, 8, 1)), ('dw', None), ('dw', dev(F32, 8, 1)),
        ('dy', dev(BF16, 16, 72)), ('dy', dev(BF16, 16, 64, strides=(0, 1))), ('dy', dev(BF16, 16, 64, device=-1)),
        ('dy', dev(BF16, 4, 4, 64, strides=(64, 64, 1)))])
    assert b'error (' in lib.dg_last_error()
    big = dict(dout=dev(BF16, 1 << 24, 1032), y=None, pos=dev(I32, 1 << 24, 1), w=None, dy=dev(BF16, 16, 1032), dw=None)
    assert call('dg_moe_combine_backward', *big.values()) == _ffi.DG_ERR_INVALID


def test_casts_refuse():
    args = dict(x=dev(BF16, 8, 64), q=dev(I8, 8, 32), sf=dev(F32, 8, 2), gran=32, ue8m0=0)
    refused('dg_per_token_cast_to_fp4', args, [
        ('x', dev(F32, 8, 64)), ('x', dev(BF16, 8, 63)), ('x', dev(BF16, 8, 64, strides=(1, 8))), ('x', dev(BF16, 64)), ('x', None),
        ('q', dev(I8, 8, 64)), ('q', dev(E4M3, 8, 32)), ('q', dev(I8, 8, 32, device=1)), ('sf', dev(F32, 8, 1)), ('sf', dev(I32, 8, 1)),
        ('sf', dev(BF16, 8, 2)), ('gran', 16), ('gran', 0), ('sf', dev(F32, 8, 2, device=-1))])
    args = dict(q=dev(I8, 8, 32), sf=dev(I32, 8, 1), y=dev(BF16, 8, 64), gran=32)
    refused('dg_cast_back_from_fp4', args, [
        ('q', dev(I8, 8, 31)), ('sf', dev(I32, 8, 2)), ('sf', dev(F32, 8, 1)), ('y', dev(I32, 8, 64)), ('y', dev(BF16, 7, 64)),
        ('y', dev(BF16, 8, 64, strides=(1, 8))), ('gran', 48)])
    big = dict(x=dev(BF16, 1 << 26, 2), q=dev(I8, 1 << 26, 1), sf=dev(I32, 1 << 26, 1), gran=32, ue8m0=1)
    assert call('dg_per_token_cast_to_fp4', *big.values()) == _ffi.DG_ERR_INVALID


PRODUCT = dict(a=dev(I8, 8, 64), a_sf=dev(I32, 8, 1), b=dev(I8, 3, 24, 64), b_sf=dev(I32, 3, 24, 1), d=dev(BF16, 8, 24), ends=dev(I32, 3),
               alignment=1, ws=None)


def test_product_refuses():
    refused('dg_m_grouped_fp4_gemm_nt_ragged', PRODUCT, [
        ('a', dev(BF16, 8, 64)), ('a', dev(I8, 8, 72)), ('a', dev(I8, 8, 64, strides=(72, 1))), ('a', dev(I8, 8, 64, data=8)),
        ('a', dev(I8, 8, 64, strides=(1, 8))), ('a', dev(I8, 8, 64, device=-1)), ('a', None), ('a', dev(I8, 7, 64)),
        ('a_sf', dev(F32, 8, 1)), ('a_sf', dev(I32, 8, 2)), ('a_sf', dev(I32, 7, 1)), ('a_sf', dev(I32, 8, 1, strides=((1 << 20) + 1, 1))),
        ('a_sf', dev(I32, 8, 1, strides=(-4, 1))), ('a_sf', dev(I32, 8, 1, data=2)), ('a_sf', dev(I32, 8)), ('a_sf', None),
        ('b', dev(E4M3, 3, 24, 64)), ('b', dev(I8, 24, 64)), ('b', dev(I8, 3, 24, 48)), ('b', dev(I8, 3, 24, 64, strides=(64, 64, 1))),
        ('b_sf', dev(I32, 3, 24, 2)), ('b_sf', dev(I32, 3, 25, 1)), ('b_sf', dev(I32, 2, 24, 1)), ('b_sf', dev(I32, 24, 1)),
        ('d', dev(I32, 8, 24)), ('d', dev(BF16, 8, 25)), ('d', dev(BF16, 9, 24)), ('d', dev(BF16, 8, 24, strides=(1, 8))),
        ('d', dev(BF16, 8, 24, device=1)), ('ends', dev(I64, 3)), ('ends', dev(I32, 4)), ('ends', dev(I32, 3, strides=(2,))),
        ('alignment', 0), ('alignment', (1 << 20) + 1)])
    wide = dict(PRODUCT, a=dev(I8, 8, 128), a_sf=dev(I32, 8, 2), b=dev(I8, 3, 24, 128), b_sf=dev(I32, 3, 24, 2))
    refused('dg_m_grouped_fp4_gemm_nt_ragged', wide, [('a_sf', dev(I32, 8, 2, strides=(2, 1 << 28))), ('a_sf', dev(I32, 8, 2, strides=(2, -1)))])


def test_workspace_sizes():
    size = lib.dg_fp4_gemm_ragged_workspace_size
    assert size(0, 64, 64, 1) == size(8, 0, 64, 1) == size(8, 64, 64, 0) == 0
    assert size(-1, 64, 64, 1) == size(8, 64, 33, 1) == size(8, 64, 1 << 30, 1) == -1


def test_python_arguments():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    idx = torch.zeros((4, 2), dtype=torch.int32)
    with pytest.raises(RuntimeError, match='on_device'):
        deep_gemm.moe_dispatch(x, idx, 4, layout='psum', alignment=1)
    with pytest.raises(ValueError):
        deep_gemm.moe_dispatch(x, idx, 4, layout='rows')
    with pytest.raises(ValueError):
        deep_gemm.moe_dispatch(x, idx, 4, layout='masked')
    with pytest.raises(RuntimeError):
        deep_gemm.moe_dispatch(x, idx, 0, layout='psum', alignment=1)
    with pytest.raises(RuntimeError):
        deep_gemm.moe_dispatch(x, idx[0], 4, layout='psum', alignment=1)
    with pytest.raises(TypeError):
        deep_gemm.moe_dispatch([1, 2], [3], 4, layout='psum')
    with pytest.raises(TypeError):
        deep_gemm.m_grouped_fp4_gemm_nt_ragged(x, (x, x), x, idx)
    with pytest.raises(RuntimeError):
        deep_gemm.moe_dispatch_backward(x, idx)
    with pytest.raises(RuntimeError):
        deep_gemm.moe_combine_backward(x, x, idx)
    with pytest.raises(TypeError):
        deep_gemm.cast_back_from_fp4(torch.zeros((2, 16), dtype=torch.int8), torch.ones((2, 1)), dtype=torch.float16)


def test_casts_on_the_host_take_the_torch_forms():
    x = torch.randn((5, 96), generator=torch.Generator().manual_seed(0)).bfloat16()
    q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
    rq, rsf = deep_gemm.utils.math.per_token_cast_to_fp4(x, True, 32, True)
    assert torch.equal(q, rq) and torch.equal(sf, rsf)
    v = deep_gemm.cast_back_from_fp4(q, sf, 32, True, torch.bfloat16)
    assert v.dtype == torch.bfloat16
    assert torch.equal(v.float(), deep_gemm.utils.math.cast_back_from_fp4(q, sf, 32, True))


def calls(mod):
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    w = lambda *s: torch.zeros(s, dtype=torch.int32)
    q = lambda *s: torch.zeros(s, dtype=torch.int8)
    return {
        'product': lambda: mod.ragged_fp4(q(4, 16), w(4, 1), q(2, 8, 16), w(2, 8, 1), z(4, 8), w(2), 1, 0),
        'cast': lambda: mod.cast4(z(4, 64), 32, 1, 1, 0),
        'cast back': lambda: mod.cast_back4(q(4, 32), w(4, 1), 32, 1, 0),
        'dispatch': lambda: mod.dispatch_rows(z(4, 64), None, w(4, 2), torch.zeros(4, 2), 3, 1, 1, 0, None, None, 0),
        'dispatch backward': lambda: mod.dispatch_backward(z(9, 64), w(4, 2), torch.zeros(9), 0),
        'combine backward': lambda: mod.combine_backward(z(4, 64), z(9, 64), w(4, 2), torch.zeros(4, 2), None, 0),
    }


@pytest.mark.parametrize('name', ['product', 'cast', 'cast back', 'dispatch', 'dispatch backward', 'combine backward'])
def test_other_threads_run_during_a_call(stub, name):  # noqa: F811
    lib, mod = stub
    blocked = ctypes.cast(lib.blocked, ctypes.c_void_p).value
    size = ctypes.cast(_ffi.lib.dg_moe_dispatch_max_rows, ctypes.c_void_p).value
    room = ctypes.cast(_ffi.lib.dg_moe_dispatch_workspace_size, ctypes.c_void_p).value
    ws = ctypes.cast(_ffi.lib.dg_fp4_gemm_ragged_workspace_size, ctypes.c_void_p).value
    mod.init_rows(size, room, *[blocked] * 5, ws)
    entered, go = (ctypes.c_int.in_dll(lib, v) for v in ('entered', 'go'))
    entered.value = go.value = 0
    got = []
    t = threading.Thread(target=lambda: got.append(calls(mod)[name]()))
    t.start()
    while not entered.value and t.is_alive():
        threading.Event().wait(0.001)
    go.value = 1        # only reached, within the call's five seconds, if it left the GIL
    t.join(20)
    out = got[0]
    shapes = {'cast': [(4, 32), (4, 1)], 'cast back': [(4, 64)], 'dispatch': [(8, 64), None, (3,), (4, 2), (8,)],
              'dispatch backward': [(4, 64), (4, 2)], 'combine backward': [(9, 64), (4, 2)]}
    if name == 'product':
        assert out == 7
    else:
        assert out[0] == 7
        assert [None if v is None else tuple(v.shape) for v in out[1:]] == shapes[name]


def test_dispatches_of_a_moe_dispatch_that_names_its_launches():
    from deep_gemm.testing import rocprof_summary
    for n in (1, 3):
        assert rocprof_summary.dispatches_per_call(f'moe_dispatch layout=psum experts=4 t=8 k=2 kdim=64 launches={n}') == n


def test_tiles_of_the_4_bit_product_that_are_not_there():
    try:
        for block, pieces in ((16, 0), (96, 1), (512, 0), (256, 1), (128, 33), (32, -1)):
            assert lib.dg_set_tile_override(14, block, pieces) != 0, (block, pieces)
        for block, pieces in ((256, 0), (128, 32), (64, 1), (32, 0)):
            assert lib.dg_set_tile_override(14, block, pieces) == 0, (block, pieces)
    finally:
        lib.dg_set_tile_override(0, 0, 0)


@pytest.mark.parametrize('few', [True, False])
def test_dispatch_refuses_a_workspace_of_another_device(few):
    t = 8 if few else 4096
    args = dict(DISPATCH, x=dev(BF16, t, 64), topk=dev(I32, t, 2), a=dev(BF16, 2 * t, 64), pos=dev(I32, t, 2), ws=dev(I32, 1 << 14, device=1))
    refused('dg_moe_dispatch', args, [('ws', args['ws']), ('ws', dev(I32, 1 << 14, device=-1))])
    assert call('dg_moe_dispatch', *dict(args, x=None).values()) == _ffi.DG_ERR_INVALID
