"""Integer arguments that the C ABI's 32 bits do not hold are refused by the native binding, on
a copy of the module whose entry points return at once."""
import ctypes

import pytest
import torch

import deep_gemm
from test_bind_cpu import stub  # noqa: F401

TOO_LONG = [(1 << 31), (1 << 32) + 16, -(1 << 31) - 1, 1 << 63, 1 << 70]


@pytest.mark.parametrize('value', TOO_LONG)
def test_ragged_alignment(value):
    """2^32 + 16 is no alignment of 16."""
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    ends = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: deep_gemm.m_grouped_bf16_gemm_nt_ragged(z(4, 8), z(2, 8, 8), z(4, 8), ends, alignment=value),
                 lambda: deep_gemm.m_grouped_bf16_gemm_nn_ragged(z(4, 8), z(2, 8, 8), z(4, 8), ends, alignment=value),
                 lambda: deep_gemm.k_grouped_bf16_gemm_tn_ragged(z(4, 8), z(4, 8), z(2, 8, 8), ends, alignment=value)):
        with pytest.raises(OverflowError):
            call()


@pytest.mark.parametrize('value', TOO_LONG)
@pytest.mark.parametrize('name,tensors,optional,integers,nargs', [
    ('gemm_nt', (0, 1, 2, 3, 4), (5,), (7,), 10), ('contiguous', (0, 1, 2, 3, 4, 5), (), (7, 8, 9, 10), 13),
    ('masked', (0, 1, 2, 3, 4, 5), (), (6, 8), 11), ('cast', (0, 1, 2), (), (3, 4), 6),
    ('dispatch', (0, 1, 2, 7, 8, 9, 10, 12), (3, 11), (4, 5, 6), 14), ('swiglu', (0, 4, 5), (1, 2), (6,), 8),
    ('contiguous_swiglu', (0, 1, 2, 3, 4, 7, 8), (5,), (9, 10), 12),
    ('masked_swiglu', (0, 1, 2, 3, 4, 8, 9), (6,), (5,), 11)])
def test_every_integer(stub, name, tensors, optional, integers, nargs, value):  # noqa: F811
    lib, mod = stub
    ctypes.c_int.in_dll(lib, 'go').value = 1    # the entry points return 7
    t = torch.zeros((128, 8), dtype=torch.bfloat16)
    plain = [t if i in tensors else None if i in optional else 0 for i in range(nargs)]
    assert getattr(mod, name)(*plain) == 7
    for at in integers:
        args = list(plain)
        args[at] = value
        with pytest.raises(OverflowError):
            getattr(mod, name)(*args)
