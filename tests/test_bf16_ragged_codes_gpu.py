"""The TN product from e4m3 codes against its definition, D = A^T (codes x scales), in 64 bits:
with scales that are no powers of two the kernel rounds code x scale to BF16, half a step
of it (2^-8 of the value at most) on top of an FP32 product's (2^-24); with powers of two
that product is exact and only the sum's bound is left."""
import pytest
import torch

import deep_gemm
from ragged import DEV, check, ends_of, matrix, rounding, segments, sum_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize('block', [0, 128, 256])
@pytest.mark.parametrize('pow2', [True, False])
@pytest.mark.parametrize('sizes,m,n', [([77], 40, 200), ([300, 0, 131, 1], 261, 388), ([1500], 264, 136)])
def test_error_against_the_definition(sizes, m, n, pow2, block):
    if block:
        deep_gemm.set_tile_override(block, 0, variant=13)
        deep_gemm.set_num_sms(1)
    seg = segments(sizes)
    rows = seg[-1][1]
    a, a64 = matrix((rows, m), 5)
    x = torch.randn((rows, n), generator=torch.Generator().manual_seed(6)).bfloat16().to(DEV)
    q, sf = deep_gemm.per_token_cast_to_fp8(x, use_ue8m0=pow2)
    v = q.float().double().cpu() * sf.double().cpu().repeat_interleave(128, 1)[:, :n]
    codes = torch.zeros((rows, -(-n // 8) * 8), dtype=torch.uint8, device=DEV)
    codes[:, :n] = q.view(torch.uint8)
    d = torch.empty((len(sizes), m, n), device=DEV)
    deep_gemm.k_grouped_bf16_gemm_tn_ragged(a, (codes.view(torch.float8_e4m3fn)[:, :n], sf), d, ends_of(seg))
    torch.cuda.synchronize()
    values = 0.0 if pow2 else 2.0 ** -8 + 2.0 ** -24 + 2.0 ** -32    # (both roundings, and their product)
    worst = 0.0
    for i, (lo, hi) in enumerate(seg):
        ref, mag = a64[lo:hi].T @ v[lo:hi], a64[lo:hi].abs().T @ v[lo:hi].abs()
        bound = rounding(d.dtype, ref) + values * mag + sum_error(hi - lo, mag * (1 + values))
        check(d[i], ref, bound, f'group {i}')
        if hi > lo:
            worst = max(worst, float(((d[i].double().cpu() - ref).abs() / mag).max()))
    print(f'pow2={pow2} block={block}: off by at most {worst:.2e} of the products magnitudes', flush=True)
