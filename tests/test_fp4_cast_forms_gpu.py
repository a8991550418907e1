"""4-bit casts of device tensors that the kernels do not take: codes that lie apart, scales of other shapes
and types, gradients, tangents and batches go through torch operations, with the results
that those have on the host."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import deep_gemm
from deep_gemm.utils import math as plain

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


def codes(m, half, seed=0):
    return torch.randint(-128, 128, (m, half), generator=torch.Generator().manual_seed(seed), dtype=torch.int8)


def scales(*shape, seed=1):
    return torch.rand(shape, generator=torch.Generator().manual_seed(seed)) + 0.5


def test_codes_that_lie_apart():
    q, sf = codes(64, 24), scales(24, 4)
    want = plain.cast_back_from_fp4(q.t(), sf, 32)
    assert torch.equal(deep_gemm.cast_back_from_fp4(q.to(DEV).t(), sf.to(DEV), 32).cpu(), want)
    wide = codes(9, 96, 2)
    want = plain.cast_back_from_fp4(wide[:, ::3], sf[:9, :2], 32)
    assert torch.equal(deep_gemm.cast_back_from_fp4(wide.to(DEV)[:, ::3], sf[:9, :2].to(DEV), 32).cpu(), want)


@pytest.mark.parametrize('sf', [scales(7, 5), scales(1, 2), scales(1, 6), scales(7, 2).double(), scales(7, 2).bfloat16(),
                                (scales(7, 2) * 9).int()], ids=['more columns', 'one row', 'one wide row', 'fp64', 'bf16', 'whole numbers'])
def test_scales_of_other_shapes_and_types(sf):
    q = codes(7, 32)
    want = plain.cast_back_from_fp4(q, sf, 32)
    got = deep_gemm.cast_back_from_fp4(q.to(DEV), sf.to(DEV), 32)
    assert got.dtype == want.dtype and torch.equal(got.cpu(), want)
    got = deep_gemm.cast_back_from_fp4(q.to(DEV), sf.to(DEV), 32, dtype=torch.bfloat16)
    assert torch.equal(got.cpu(), want.bfloat16())


def test_more_words_than_scales():
    q, sf = plain.per_token_cast_to_fp4(torch.randn((6, 256), generator=torch.Generator().manual_seed(3)).bfloat16(), True, 32, True)
    wide = torch.full((6, 5), -1, dtype=torch.int32)
    wide[:, :2] = sf
    want = plain.cast_back_from_fp4(q, sf, 32, True)
    assert torch.equal(deep_gemm.cast_back_from_fp4(q.to(DEV), wide.to(DEV), 32, True).cpu(), want)


def test_gradient_of_the_scales():
    """d(sum of v * g) / d sf[r, j] = the sum over the group of value of the code * g: products of powers of
    two here, so that FP32 sums of them are exact."""
    q = codes(5, 48)
    g = torch.exp2(torch.randint(-3, 4, (5, 96), generator=torch.Generator().manual_seed(4)).float())
    sf = scales(5, 3).to(DEV).requires_grad_()
    v = deep_gemm.cast_back_from_fp4(q.to(DEV), sf, 32)
    v.backward(g.to(DEV))
    unit = plain.cast_back_from_fp4(q, torch.ones(5, 3), 32).double()
    assert torch.equal(sf.grad.double().cpu(), (unit * g.double()).view(5, 3, 32).sum(2))
    with torch.no_grad():
        assert torch.equal(deep_gemm.cast_back_from_fp4(q.to(DEV), sf, 32), v)
        assert deep_gemm.get_last_config().startswith('cast_back_from_fp4')


def test_gradient_of_the_float_scales_of_a_cast():
    """sf = largest magnitude / 6 carries its group's gradient to that element."""
    x = torch.randn((3, 64), generator=torch.Generator().manual_seed(5)).bfloat16()
    want = x.clone().requires_grad_()
    q0, sf0 = plain.per_token_cast_to_fp4(want, False, 32)
    sf0.sum().backward()
    got = x.to(DEV).requires_grad_()
    q, sf = deep_gemm.per_token_cast_to_fp4(got, False, 32)
    assert torch.equal(q.cpu(), q0) and torch.equal(sf.detach().cpu(), sf0.detach())
    sf.sum().backward()
    assert torch.equal(got.grad.cpu(), want.grad) and got.grad.count_nonzero() == 6
    # power-of-two scales carry none: the kernel
    q, sf = deep_gemm.per_token_cast_to_fp4(got, True, 32)
    assert not sf.requires_grad and deep_gemm.get_last_config().startswith('per_token_cast_to_fp4')


def test_tangent_of_the_scales():
    q, sf, d = codes(4, 32), scales(4, 2), scales(4, 2, seed=6)
    with forward_ad.dual_level():
        v = deep_gemm.cast_back_from_fp4(q.to(DEV), forward_ad.make_dual(sf.to(DEV), d.to(DEV)), 32)
        v, tangent = forward_ad.unpack_dual(v)
    assert torch.equal(v.cpu(), plain.cast_back_from_fp4(q, sf, 32)) and torch.equal(tangent.cpu(), plain.cast_back_from_fp4(q, d, 32))


def test_negative_views():
    """Views whose memory holds the negative of their values."""
    q, sf = codes(4, 32), scales(4, 2)
    got = deep_gemm.cast_back_from_fp4(q.to(DEV), torch._neg_view(sf.to(DEV)), 32)
    assert torch.equal(got.cpu(), plain.cast_back_from_fp4(q, -sf, 32))
    x = torch.randn((4, 64), generator=torch.Generator().manual_seed(7)).bfloat16()
    got = deep_gemm.per_token_cast_to_fp4(torch._neg_view(x.to(DEV)), True, 32, True)
    want = plain.per_token_cast_to_fp4(-x, True, 32, True)
    assert torch.equal(got[0].cpu(), want[0]) and torch.equal(got[1].cpu(), want[1])


def test_batches_of_vmap():
    q = torch.stack([codes(4, 32, i) for i in range(3)])
    sf = scales(3, 4, 2)
    got = torch.vmap(lambda a, b: deep_gemm.cast_back_from_fp4(a, b, 32))(q.to(DEV), sf.to(DEV))
    assert torch.equal(got.cpu(), torch.stack([plain.cast_back_from_fp4(a, b, 32) for a, b in zip(q, sf)]))


def test_more_rows_than_a_launch_has():
    """Past 2^26 rows of two values."""
    m = (1 << 26) + 3
    q = torch.zeros((m, 1), dtype=torch.int8, device=DEV)
    sf = torch.ones((m, 1), device=DEV)
    q[-2:, 0], sf[-2:, 0] = torch.tensor([0x75, -0x46], dtype=torch.int8, device=DEV), torch.tensor([3.0, 0.5], device=DEV)
    v = deep_gemm.cast_back_from_fp4(q, sf, 32)
    assert torch.equal(v[-2:].cpu(), plain.cast_back_from_fp4(q[-2:].cpu(), sf[-2:].cpu(), 32)) and not v[:-2].any()


def test_casts_of_more_rows_than_a_launch_has():
    """Past 2^26 rows of two values."""
    m = (1 << 26) + 3
    x = torch.zeros((m, 2), dtype=torch.bfloat16, device=DEV)
    x[-2:] = torch.tensor([[6.0, -3.0], [0.25, 1.0]], dtype=torch.bfloat16, device=DEV)
    q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
    rq, rsf = plain.per_token_cast_to_fp4(x[-2:].cpu(), True, 32, True)
    assert torch.equal(q[-2:].cpu(), rq) and torch.equal(sf[-2:].cpu(), rsf) and not q[:-2].any()
    v = deep_gemm.cast_back_from_fp4(q, sf, 32, True, torch.bfloat16)
    assert torch.equal(v[-2:].float().cpu(), plain.cast_back_from_fp4(rq, rsf, 32, True)) and not v[:-2].any()


def test_parameters_take_the_kernel():
    x = torch.nn.Parameter(torch.randn((8, 64), device=DEV).bfloat16())
    q, sf = deep_gemm.per_token_cast_to_fp4(x, True, 32, True)
    assert deep_gemm.get_last_config().startswith('per_token_cast_to_fp4')
    rq, rsf = plain.per_token_cast_to_fp4(x.detach().cpu(), True, 32, True)
    assert torch.equal(q.cpu(), rq) and torch.equal(sf.cpu(), rsf)
