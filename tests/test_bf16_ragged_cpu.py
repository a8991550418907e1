"""Refusals of the BF16 expert operators, on the host: every call below must be rejected
before the library could touch device memory (device tensors with made-up addresses)."""
import ctypes

import pytest
import torch

import deep_gemm
from deep_gemm import _ffi
from test_abi_cpu import fake

BF, F32, E4, I32 = _ffi.DG_BF16, _ffi.DG_F32, _ffi.DG_E4M3, _ffi.DG_I32


def call(name, *args):
    st = getattr(_ffi.lib, name)(*[ctypes.byref(a) if isinstance(a, _ffi.DgTensor) else a for a in args], None)
    return st, _ffi.lib.dg_last_error().decode()


def rejected(name, *args, match=''):
    st, msg = call(name, *args)
    assert st == _ffi.DG_ERR_INVALID and msg.startswith('Assertion error (') and match in msg, (st, msg)


def nt(m=64, n=48, k=32, g=3):
    return dict(a=fake((m, k), BF), b=fake((g, n, k), BF), d=fake((m, n), BF), ends=fake((g,), I32), alignment=1, ws=None)


def nn(m=64, n=48, k=32, g=3):
    return dict(a=fake((m, k), BF), b=fake((g, k, n), BF), d=fake((m, n), BF), ends=fake((g,), I32), alignment=1, ws=None)


@pytest.mark.parametrize('name,make', [('dg_m_grouped_bf16_gemm_nt_ragged', nt), ('dg_m_grouped_bf16_gemm_nn_ragged', nn)])
@pytest.mark.parametrize('key,value', [
    ('a', fake((64, 32), BF, device=-1)), ('a', fake((64, 32), F32)), ('a', fake((64, 40), BF)), ('a', fake((1, 64, 32), BF)),
    ('a', fake((64, 32), BF, strides=(1, 64))), ('a', fake((64, 32), BF, addr=0x10000008)),
    ('a', fake((64, 32), BF, strides=(36, 1))), ('a', fake((64, 32), BF, strides=(16, 1))),
    ('a', fake((64, 32), BF, strides=((1 << 22) + 8, 1))), ('a', fake((64, 32), BF, device=1)),
    ('b', fake((3, 48, 32), E4)), ('b', fake((48, 32), BF)), ('b', fake((3, 32, 32), BF)), ('b', fake((2, 48, 32), BF)),
    ('b', fake((3, 48, 48), BF)),
    ('d', fake((64, 48), E4)), ('d', fake((63, 48), BF)), ('d', fake((64, 47), BF)), ('d', fake((64, 48), BF, strides=(47, 1))),
    ('d', fake((64, 48), BF, strides=(1, 64))), ('d', fake((64, 48), BF, device=-1)),
    ('ends', fake((4,), I32)), ('ends', fake((3,), _ffi.DG_I64)), ('ends', fake((3,), I32, strides=(2,))),
    ('ends', fake((3,), I32, device=-1)), ('ends', fake((3, 1), I32)),
    ('alignment', 0), ('alignment', -16), ('alignment', (1 << 20) + 1), ('ws', fake((64,), F32, device=1))])
def test_m_grouped_refusals(name, make, key, value):
    args = make()
    args[key] = value
    rejected(name, *args.values())


@pytest.mark.parametrize('name,make', [('dg_m_grouped_bf16_gemm_nt_ragged', nt), ('dg_m_grouped_bf16_gemm_nn_ragged', nn)])
def test_m_grouped_reduced_length_and_null(name, make):
    rejected(name, *make(k=36).values())
    rejected(name, *make(n=8, k=8, g=65537).values(), match='kRaggedMaxGroups')
    for key in ('a', 'b', 'd', 'ends'):
        args = make()
        args[key] = None
        rejected(name, *args.values(), match='nullptr')


def tn(r=64, m=40, n=48, g=3, eight=False):
    return dict(a=fake((r, m), BF), b=fake((r, n), E4 if eight else BF), sf=fake((r, -(-n // 128)), F32) if eight else None,
                d=fake((g, m, n), F32), ends=fake((g,), I32), c=None, alignment=1, ws=None)


@pytest.mark.parametrize('key,value', [
    ('a', fake((64, 40), E4)), ('a', fake((63, 40), BF)), ('a', fake((64, 32), BF)), ('a', fake((64, 40), BF, strides=(1, 64))),
    ('a', fake((64, 40), BF, strides=(44, 1))), ('b', fake((64, 48), E4)), ('b', fake((64, 48), BF, addr=0x10000008)),
    ('b', fake((64, 48), BF, strides=(52, 1))), ('b', fake((64, 47), BF)), ('sf', fake((64, 1), F32)),
    ('d', fake((3, 40, 48), _ffi.DG_F16)), ('d', fake((40, 48), F32)), ('d', fake((3, 40, 48), F32, strides=(1900, 48, 1))),
    ('c', fake((3, 40, 48), BF)), ('c', fake((3, 40, 40), F32)), ('c', fake((3, 40, 48), F32, device=-1)),
    ('c', fake((3, 40, 48), F32, device=1)), ('c', fake((3, 40, 48), F32, strides=(2080, 52, 1))),
    ('ends', fake((2,), I32)), ('alignment', 0)])
def test_k_grouped_refusals(key, value):
    args = tn()
    args[key] = value
    rejected('dg_k_grouped_bf16_gemm_tn_ragged', *args.values())


@pytest.mark.parametrize('key,value', [
    ('b', fake((64, 48), BF)), ('b', fake((64, 48), E4, addr=0x10000004)), ('b', fake((64, 48), E4, strides=(52, 1))),
    ('sf', fake((64, 2), F32)), ('sf', fake((63, 1), F32)), ('sf', fake((64, 1), I32)), ('sf', fake((64, 1), F32, device=-1)),
    ('sf', fake((64,), F32))])
def test_k_grouped_checkpoint_refusals(key, value):
    args = tn(eight=True)
    args[key] = value
    rejected('dg_k_grouped_bf16_gemm_tn_ragged', *args.values())


def fwd(m=8, i=64):
    return dict(x=fake((m, 2 * i), BF), w=fake((m,), F32), rl=fake((m,), I32), clamp=0.0, h=fake((m, i), BF),
                q=fake((m, 2 * i), E4), sf=fake((m, 2), F32))


@pytest.mark.parametrize('key,value', [
    ('x', fake((8, 120), BF)), ('x', fake((8, 128), F32)), ('x', fake((8, 128), BF, addr=0x10000008)),
    ('x', fake((8, 128), BF, strides=(1, 8))), ('x', fake((8, 128), BF, strides=(132, 1))), ('w', fake((7,), F32)),
    ('w', fake((8,), BF)), ('rl', fake((8,), _ffi.DG_I64)), ('rl', fake((9,), I32)), ('h', fake((8, 128), BF)),
    ('h', fake((8, 64), F32)), ('h', fake((8, 64), BF, strides=(68, 1))), ('q', fake((8, 64), E4)),
    ('q', fake((8, 128), E4, addr=0x10000004)), ('q', fake((8, 128), BF)), ('sf', fake((8, 1), F32)), ('sf', fake((8, 2), I32)),
    ('h', fake((8, 64), BF, device=1))])
def test_swiglu_checkpoint_refusals(key, value):
    args = fwd()
    args[key] = value
    rejected('dg_moe_swiglu_checkpoint', *args.values())


def bwd(m=8, i=64):
    return dict(dh=fake((m, i), BF), q=fake((m, 2 * i), E4), sf=fake((m, 2), F32), w=fake((m,), F32), rl=None, clamp=0.0,
                dx=fake((m, 2 * i), BF), h=fake((m, i), BF), dw=fake((m,), F32))


@pytest.mark.parametrize('key,value', [
    ('dh', fake((8, 60), BF)), ('dh', fake((8, 64), F32)), ('dh', fake((8, 64), BF, addr=0x10000002)), ('q', fake((8, 120), E4)),
    ('q', fake((7, 128), E4)), ('sf', fake((8, 1), F32)), ('dx', fake((8, 64), BF)), ('dx', fake((8, 128), F32)),
    ('h', fake((7, 64), BF)), ('dw', fake((7,), F32)), ('dw', fake((8,), BF)), ('w', None), ('w', fake((8, 1), F32))])
def test_swiglu_backward_refusals(key, value):
    args = bwd()
    args[key] = value
    rejected('dg_moe_swiglu_backward', *args.values())


def test_swiglu_refuses_more_rows_than_a_launch_holds():
    # a wave a row, four a workgroup of 256 threads: 2^26 rows are 2^32 threads
    rejected('dg_moe_swiglu_checkpoint', *fwd(m=1 << 26).values(), match='<< 32')
    rejected('dg_moe_swiglu_backward', *bwd(m=1 << 26).values(), match='<< 32')


def test_python_entry_points_refuse_host_tensors():
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    ends = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match='on_device'):
        deep_gemm.m_grouped_bf16_gemm_nt_ragged(z(4, 8), z(2, 8, 8), z(4, 8), ends)
    with pytest.raises(RuntimeError, match='on_device'):
        deep_gemm.m_grouped_bf16_gemm_nn_ragged(z(4, 8), z(2, 8, 8), z(4, 8), ends)
    with pytest.raises(RuntimeError, match='on_device'):
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(4, 8), z(4, 8), torch.zeros(2, 8, 8), ends)
    with pytest.raises(RuntimeError, match='on_device'):
        deep_gemm.moe_swiglu_checkpoint(z(4, 16))
    with pytest.raises(RuntimeError, match='on_device'):
        deep_gemm.moe_swiglu_backward(z(4, 8), (torch.zeros(4, 16, dtype=torch.float8_e4m3fn), torch.zeros(4, 2)))
    with pytest.raises(TypeError, match='pair'):
        deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(4, 8), (z(4, 8),), torch.zeros(2, 8, 8), ends)


@pytest.mark.parametrize('name,make', [('dg_m_grouped_bf16_gemm_nt_ragged', nt), ('dg_m_grouped_bf16_gemm_nn_ragged', nn)])
def test_calls_with_nothing_to_do_launch_nothing(name, make):
    for args in (make(m=0), make(n=0), make(g=0)):
        assert call(name, *args.values())[0] == _ffi.DG_OK


def test_workspace_sizes_and_plans():
    """Few tiles split a long reduced axis, with a workspace of the pieces' FP32 sums; large
    calls and short axes do not. A given number of pieces is taken as it is."""
    size = _ffi.lib.dg_bf16_gemm_ragged_workspace_size
    deep_gemm.set_num_sms(256)
    try:
        assert size(0, 8, 0, 4096, 7168, 1) % (8 * 4096 * 4) == 0 and size(0, 8, 0, 4096, 7168, 1) > 8 * 4096 * 4
        assert size(2, 20000, 104, 504, 0, 1) > 0 and size(3, 20000, 104, 504, 0, 1) > 0
        assert size(0, 16384, 0, 4096, 7168, 8) == 0 and size(1, 8, 0, 4096, 64, 1) == 0
        assert size(0, 0, 0, 4096, 7168, 1) == 0 and size(2, 64, 0, 512, 0, 1) == 0 and size(0, 64, 0, 512, 512, 0) == 0
        deep_gemm.set_tile_override(128, 5, variant=13)
        assert size(0, 10, 0, 30, 640, 2) == 5 * 10 * 32 * 4
        deep_gemm.set_tile_override(256, 0, variant=13)
        assert size(0, 10, 0, 30, 640, 2) == 0
        for args in ((4, 8, 8, 8, 8, 1), (0, -1, 8, 8, 8, 1), (0, 8, 8, 1 << 30, 8, 1)):
            assert size(*args) == -1 and 'Assertion error' in _ffi.lib.dg_last_error().decode()
        for bad in ((64, 0), (256, 2), (128, 33), (128, -1)):
            with pytest.raises(RuntimeError, match='Unsupported'):
                deep_gemm.set_tile_override(*bad, variant=13)
    finally:
        deep_gemm.init()
