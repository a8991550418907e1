"""Inputs, references in 64 bits and error bounds for the BF16 expert operators' tests."""
import numpy as np
import torch

DEV = 'cuda:0'


def segments(sizes, alignment=1):
    """(first row, end) of each group of `sizes` rows."""
    at, out = 0, []
    for s in sizes:
        start = -(-at // alignment) * alignment
        at = start + s
        out.append((start, at))
    return out


def ends_of(seg):
    return torch.tensor([e for _, e in seg], dtype=torch.int32, device=DEV)


def matrix(shape, seed, scale=1.0, pad=8, fill=float('nan')):
    """A BF16 device matrix whose rows start at multiples of `pad` elements, `fill` between
    them, and its values in 64 bits."""
    v = (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).bfloat16()
    width = -(-shape[-1] // pad) * pad
    wide = torch.full((*shape[:-1], width), fill, dtype=torch.bfloat16)
    wide[..., :shape[-1]] = v
    return wide.to(DEV)[..., :shape[-1]], v.double()


def sum_error(k, magnitude):
    """Bound on the error of an FP32 sum of k exact products of BF16 values whose
    magnitudes add up to `magnitude`: a product passes at most 16 additions inside a matrix
    instruction and one for each of the ceil(k / 16) instructions, each off by at most a
    whole step 2^-23 of a partial sum (rounding or truncation)."""
    return (-(-k // 16) + 16) * 2.0 ** -23 * magnitude


def rounding(dtype, ref):
    """Half a step of D's type at the result (twice the bound of the smallest normal covers zero)."""
    return torch.finfo(dtype).eps / 2 * ref.abs() + 1e-38


def check(got, ref, bound, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), f'{what}: not finite'
    off = (got - ref).abs() - bound
    assert (off <= 0).all(), f'{what}: off by {(got - ref).abs().max():.3e}, over the bound by {off.max():.3e}'


def cast8(x):
    """e4m3 codes and power-of-two scales per row and 128 columns of a 64-bit matrix of BF16
    values, by the oracle, and the values they stand for."""
    from oracle import quant as oquant
    q, sf = oquant.per_token_cast_to_fp8(x.float().numpy(), use_ue8m0=True)
    v = torch.from_numpy(q).view(torch.float8_e4m3fn).float().double()
    v = v * torch.from_numpy(np.repeat(sf, 128, 1)[:, :x.shape[1]].astype(np.float64))
    return torch.from_numpy(q).view(torch.float8_e4m3fn), torch.from_numpy(sf), v


def bits(t):
    return t.view(torch.int16) if t.element_size() == 2 else t.view(torch.int32) if t.element_size() == 4 \
        else t.view(torch.uint8)
