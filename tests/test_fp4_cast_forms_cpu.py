"""4-bit casts where the torch operations stand for the kernels: results keep the scales' type, and tensors
without memory of their own (device tensors that are only traced) never reach a kernel."""
import pytest
import torch

import deep_gemm


@pytest.mark.parametrize('scales,result', [(torch.float64, torch.float64), (torch.float32, torch.float32), (torch.bfloat16, torch.float32),
                                           (torch.int32, torch.float32)])
def test_back_has_the_type_of_the_scales(scales, result):
    gen = torch.Generator().manual_seed(0)
    q = torch.randint(-128, 128, (5, 32), generator=gen, dtype=torch.int8)
    sf = torch.randint(1, 9, (5, 2), generator=gen).to(scales)
    want = deep_gemm.utils.math.cast_back_from_fp4(q, sf, 32)
    got = deep_gemm.cast_back_from_fp4(q, sf, 32)
    assert got.dtype == want.dtype == result and torch.equal(got, want)
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(deep_gemm.cast_back_from_fp4(q, sf, 32, dtype=dtype), want.to(dtype))
    wide = torch.randint(1, 9, (5, 2), generator=gen).double() + 2.0 ** -30   # (no float32 value)
    assert torch.equal(deep_gemm.cast_back_from_fp4(q, wide, 32), deep_gemm.utils.math.cast_back_from_fp4(q, wide, 32))


def test_traced_device_tensors():
    from torch._subclasses import FakeTensorMode
    with FakeTensorMode():
        q = torch.empty((6, 64), dtype=torch.int8, device='cuda')
        sf = torch.empty((6, 4), device='cuda')
        v = deep_gemm.cast_back_from_fp4(q, sf, 32)
        assert v.shape == (6, 128) and v.dtype == torch.float32 and v.is_cuda
        q, sf = deep_gemm.per_token_cast_to_fp4(torch.empty((6, 128), dtype=torch.bfloat16, device='cuda'), False, 32)
        assert q.shape == (6, 64) and q.dtype == torch.int8 and sf.shape == (6, 4) and sf.is_cuda


def test_odd_columns_are_refused_alike():
    with pytest.raises(AssertionError):
        deep_gemm.per_token_cast_to_fp4(torch.zeros((2, 33), dtype=torch.bfloat16), True, 32)
