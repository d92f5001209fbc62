"""The 8-bit block quantization and the layer on it in 64 bits, straight from the definition (test infrastructure)."""
import torch

MAX_TOP = {torch.float8_e4m3fn: (8, 3, -6), torch.float8_e5m2: (15, 2, -14)}  # exponent of MAX = 1.75 * 2^top, mantissa bits, least normal exponent


def two(e):
    e = torch.as_tensor(e)
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)  # the double's own bits


def pad128(n):
    return (n + 127) // 128 * 128


def quantize(x, dtype, square=False):
    """x [R, C] on the CPU -> (values of the codes float64 [R, pad128(C)], exponent of each row's blocks int [R, pad128(C) / 128])."""
    top, bits, low = MAX_TOP[dtype]
    R, C = x.shape
    v = torch.zeros(pad128(R) if square else R, pad128(C), dtype=torch.float64)
    v[:R, :C] = x.double()
    b = v.view(-1, 128 if square else 1, v.shape[1] // 128, 128)
    amax = b.abs().amax((1, 3))
    m, p = torch.frexp(amax)                       # amax = m 2^p, MAX 2^e = 0.875 * 2^(top + 1 + e)
    e = torch.where(m <= 0.875, p - top - 1, p - top)
    e = torch.where(amax == 0, torch.full_like(e, -127), e).clamp_min(-127)
    s = b / two(e)[:, None, :, None]
    _, q = torch.frexp(s)
    step = two((q - 1).clamp_min(low) - bits)
    codes = (torch.round(s / step) * step).reshape(v.shape)[:R]
    return codes, e.repeat_interleave(128, 0)[:R] if square else e


def values(x, dtype, square=False):
    c, e = quantize(x, dtype, square)
    return (c * two(e).repeat_interleave(128, 1))[:, :x.shape[1]]


def blocked(e, rows):
    """Exponents [rows, blocks] -> the scale bytes as the kernels lay them out."""
    out = torch.zeros(pad128(rows) // 128, e.shape[1], 32, 4, 4, dtype=torch.uint8)
    r = torch.arange(rows)
    out[r // 128, :, r % 32, r % 128 // 32, :] = (e + 127).to(torch.uint8)[:, :, None]
    return out.reshape(-1)


def layer(x, w, e, grad_dtype):
    f8 = torch.float8_e4m3fn
    wq = values(w, f8, True)
    return values(x, f8) @ wq.T, values(e, grad_dtype) @ wq, values(e.T, grad_dtype) @ values(x.T, f8).T
