"""4-bit operands for the ragged products' tests: codes and scales made on the host, and the values
they stand for in 64 bits."""
import torch

from ragged import DEV

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
E2M1 = torch.cat([E2M1, -E2M1])


def values(codes, scales):
    """codes [.., n] of 0 to 15, scales [.., ceil(n / 32)] of 0 to 254: 64-bit values."""
    v = E2M1[codes.long()] * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)[..., :codes.shape[-1]]
    return v


def operand(shape, seed, low=120, high=130, layout='rows', spare_bytes=255, pitch=0):
    """A 4-bit device operand [.., n] with scales from 2^(low - 127) to 2^(high - 127) in words of four
    along the last dimension ('rows': words of a row side by side, 'columns': words of
    consecutive rows side by side, 'padded': rows of words 5 apart more). Bytes past the last scale are
    `spare_bytes` (255: NaN). pitch: bytes between rows of codes beside n / 2. Returns (codes, words) and the values."""
    gen = torch.Generator().manual_seed(seed)
    *lead, n = shape
    codes = torch.randint(0, 16, shape, generator=gen, dtype=torch.uint8)
    groups = -(-n // 32)
    words = -(-n // 128)
    scales = torch.full((*lead, words * 4), spare_bytes, dtype=torch.uint8)
    scales[..., :groups] = torch.randint(low, high + 1, (*lead, groups), generator=gen, dtype=torch.uint8)
    v = values(codes, scales[..., :groups])
    q = (codes[..., 0::2] | codes[..., 1::2] << 4).view(torch.int8)
    wide = torch.full((*lead, n // 2 + pitch), 0x77, dtype=torch.int8)
    wide[..., :n // 2] = q
    w = scales.view(torch.int32).to(DEV)
    if layout == 'columns':
        w = w.transpose(-1, -2).contiguous().transpose(-1, -2)
    elif layout == 'padded':
        room = torch.full((*lead, words + 5), -1, dtype=torch.int32, device=DEV)
        room[..., :words] = w
        w = room[..., :words]
    return (wide.to(DEV)[..., :n // 2], w), v


def sum_error(k, magnitude):
    """Bound on the error of an FP32 sum of k exact products whose magnitudes add up to
    `magnitude`: a product passes at most 64 additions inside a matrix instruction and one for
    each of the ceil(k / 64) instructions, each off by at most a whole step 2^-23 of a
    partial sum (rounding or truncation)."""
    return (-(-k // 64) + 64) * 2.0 ** -23 * magnitude
