"""The MXFP4 operators written plainly in 64 bits: what the tests of the kernels compare with."""
import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}


def quantize(x):
    """[rows, K] -> codes [rows, whole blocks of K] (0..15) and scale bytes [rows, blocks], both int64."""
    x = x.double()
    rows, K = x.shape
    wide = torch.zeros(rows, -(-K // 32) * 32, dtype=torch.float64, device=x.device)
    wide[:, :K] = x
    b = wide.reshape(rows, -1, 32)
    finite = torch.isfinite(b).all(-1)
    b = torch.where(finite.unsqueeze(-1), b, torch.zeros_like(b))
    top = b.abs().amax(-1)
    e = torch.where(top > 0, torch.frexp(top)[1].long() - 3, torch.full_like(top, -127).long()).clamp(-127, 127)
    y = b * torch.exp2(-e.unsqueeze(-1).double())
    mag = y.abs().clamp(max=6.0)
    dist = (mag.unsqueeze(-1) - GRID.to(x.device)).abs()
    # nearest element; of two equally near ones the one with the even code
    odd = torch.arange(8, device=x.device) % 2
    best = dist.amin(-1, keepdim=True)
    code = torch.where(dist == best, odd, 2).argmin(-1)
    code = code + 8 * torch.signbit(y).long()
    code = torch.where(finite.unsqueeze(-1), code, torch.zeros_like(code))
    return code.reshape(rows, -1), torch.where(finite, e + 127, torch.full_like(e, 255))


def pack(code, byte):
    """Codes and scale bytes in the library's layout."""
    rows, blocks = byte.shape
    q = (code[:, 0::2] | (code[:, 1::2] << 4)).to(torch.uint8).contiguous()
    bands, tiles = -(-rows // 128), -(-blocks // 4)
    s = torch.zeros(bands * tiles * 512, dtype=torch.uint8, device=byte.device)
    r = torch.arange(rows, device=byte.device).unsqueeze(1)
    b = torch.arange(blocks, device=byte.device).unsqueeze(0)
    s[((r // 128) * tiles + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4] = byte.to(torch.uint8)
    return q, s.reshape(bands, tiles, 32, 4, 4)


def unpack(q, s):
    """Codes and scale bytes (int64) of a packed matrix."""
    rows, width = q.shape
    code = torch.stack([q & 15, q >> 4], -1).reshape(rows, -1).long()
    r = torch.arange(rows, device=q.device).unsqueeze(1)
    b = torch.arange(width // 16, device=q.device).unsqueeze(0)
    byte = s.flatten()[((r // 128) * s.shape[1] + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4]
    return code, byte.long()


def values(code, byte):
    """[rows, whole blocks of K] in 64 bits."""
    mag = GRID.to(code.device)[code % 8]
    v = torch.where(code >= 8, -mag, mag)
    scale = torch.exp2(byte.double() - 127)
    scale = torch.where(byte == 255, torch.full_like(scale, float("nan")), scale)
    return (v.reshape(*byte.shape, 32) * scale.unsqueeze(-1)).reshape(code.shape)


def random_packed(rows, K, low, high, g):
    """A packed matrix of random codes whose block exponents are low..high; the elements beyond K are zero."""
    blocks = -(-K // 32)
    code = torch.randint(0, 16, (rows, blocks * 32), device=g.device, generator=g)
    code[:, K:] = 0
    byte = torch.randint(127 + low, 127 + high + 1, (rows, blocks), device=g.device, generator=g)
    return code, byte


def sum_bound(va, vb, dtype):
    """How far an output may be from the exact sum of products: K additions in fp32, each off by at most 2^-23 of
    the sum of magnitudes (a cut where it is not a rounding), and the one rounding to `dtype`."""
    c = va @ vb.t()
    return c, va.shape[1] * 2.0**-23 * (va.abs() @ vb.abs().t()) + HALF_STEP[dtype] * c.abs()
