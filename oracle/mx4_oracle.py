"""Microscaled 4-bit floating point in 64 bits on the CPU: the rounding and the
values of hi_rocm_mx4_quantize and the products that take them.  Test
infrastructure only."""
import numpy as np
import torch

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """x [rows][k] (torch, any float type) -> codes uint8 [rows][k] (one a
    byte), scales uint8 [rows][k / 32]."""
    b = x.detach().cpu().double().numpy().reshape(x.shape[0], -1, 32)
    a = np.abs(b).max(2)
    bad = ~np.isfinite(a)
    a = np.where(bad, 1.0, a)
    mant, exp = np.frexp(a)  # a = mant 2^exp, 0.5 <= mant < 1
    s = np.where(a > 0, np.clip(exp - 1 - 2 + 127, 0, 254), 0)
    v = np.ldexp(np.where(bad[:, :, None], 0.0, b), (127 - s)[:, :, None])
    m = np.abs(v)
    # the nearest of the eight; of two equally near, the one with an even code
    d = np.abs(m[..., None] - VALUES)
    near = d.min(-1, keepdims=True)
    ties = d == near
    even = np.where(ties, np.arange(8) % 2, 2)
    code = even.argmin(-1).astype(np.uint8)
    code = np.where(m >= 6.0, 7, code)
    code = code | (np.signbit(v).astype(np.uint8) << 3)
    code = np.where(bad[:, :, None], 0, code).astype(np.uint8)
    s = np.where(bad, 255, s).astype(np.uint8)
    return torch.from_numpy(code.reshape(x.shape)), torch.from_numpy(s)


def pack_nibbles(codes):
    return codes[..., 0::2] | codes[..., 1::2] << 4


def values(packed, scales):
    """The values (float64, CPU) of packed codes [..][k / 2] and scales [..][k / 32]."""
    p, s = packed.cpu(), scales.cpu().numpy()
    c = torch.stack((p & 15, p >> 4), -1).reshape(*p.shape[:-1], -1, 32).numpy()
    v = np.where(c & 8, -VALUES[c & 7], VALUES[c & 7])
    v = np.ldexp(v, s.astype(np.int64)[..., None] - 127)
    v = np.where((s == 255)[..., None], np.nan, v)
    return torch.from_numpy(v.reshape(*p.shape[:-1], -1))


def rounded(x):
    """Q(x) in float64."""
    codes, scales = quantize(x)
    return values(pack_nibbles(codes), scales)
