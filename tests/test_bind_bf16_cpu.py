"""The native binding of the BF16 expert operators leaves the GIL while a library call runs,
and returns new outputs beside the status, on a copy of the module whose entry points
block until another Python thread lets them go."""
import ctypes
import threading

import pytest
import torch

import deep_gemm
from test_bind_cpu import stub  # noqa: F401


def calls(mod):
    z = lambda *s: torch.zeros(s, dtype=torch.bfloat16)
    ends = torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(4, 16, dtype=torch.float8_e4m3fn)
    return {
        'nt': lambda: mod.m_grouped_ragged(0, z(4, 8), z(2, 8, 8), z(4, 8), ends, 1, 0),
        'nn': lambda: mod.m_grouped_ragged(1, z(4, 8), z(2, 8, 8), z(4, 8), ends, 1, 0),
        'tn': lambda: mod.k_grouped_ragged(z(4, 8), z(4, 8), None, z(2, 8, 8), ends, None, 1, 0),
        'tn 8-bit': lambda: mod.k_grouped_ragged(z(4, 8), q, torch.zeros(4, 1), z(2, 8, 16), ends, z(2, 8, 16), 1, 0),
        'swiglu': lambda: mod.swiglu_checkpoint(z(4, 16), None, None, 0.0, 0),
        'swiglu backward': lambda: mod.swiglu_backward(z(4, 8), q, torch.zeros(4, 2), torch.zeros(4), None, 0.0, 0),
    }


@pytest.mark.parametrize('name', ['nt', 'nn', 'tn', 'tn 8-bit', 'swiglu', 'swiglu backward'])
def test_other_threads_run_during_a_call(stub, name):  # noqa: F811
    lib, mod = stub
    mod.init_bf16(*[ctypes.cast(lib.blocked, ctypes.c_void_p).value] * 6)
    entered, go = (ctypes.c_int.in_dll(lib, v) for v in ('entered', 'go'))
    entered.value = go.value = 0
    got = []
    t = threading.Thread(target=lambda: got.append(calls(mod)[name]()))
    t.start()
    while not entered.value and t.is_alive():
        threading.Event().wait(0.001)
    go.value = 1        # only reached, within the call's five seconds, if it left the GIL
    t.join(20)
    if name == 'swiglu':
        status, h, codes, sf = got[0]
        assert (h.shape, codes.shape, sf.shape) == ((4, 8), (4, 16), (4, 2))
        assert (h.dtype, codes.dtype, sf.dtype) == (torch.bfloat16, torch.float8_e4m3fn, torch.float32)
    elif name == 'swiglu backward':
        status, dx, h, dw = got[0]
        assert (dx.shape, h.shape, dw.shape, dw.dtype) == ((4, 16), (4, 8), (4,), torch.float32)
    else:
        status = got[0]
    assert status == 7


def test_bad_arguments_raise():
    z = torch.zeros(4, 16, dtype=torch.bfloat16)
    with pytest.raises(TypeError):
        deep_gemm.moe_swiglu_checkpoint([1, 2])
    with pytest.raises(TypeError):
        deep_gemm.moe_swiglu_checkpoint(z, row_weights=3)
    with pytest.raises(RuntimeError, match='dim'):
        deep_gemm.moe_swiglu_checkpoint(z[0])
    with pytest.raises(RuntimeError, match='unsupported dtype'):
        deep_gemm.moe_swiglu_checkpoint(z.double())
    with pytest.raises((ValueError, TypeError)):
        deep_gemm.moe_swiglu_checkpoint(z, clamp_value='x')
