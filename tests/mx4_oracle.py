"""MXFP4 quantisation restated on the CPU in 64 bits with integer codes (numpy only): the checker of deepipr_amd.mx4."""
import numpy as np
import torch

VALUES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
KP = 128


def to64(x):
    return x.detach().cpu().to(torch.float64).numpy()


def code_of(a):
    """Nearest code of magnitudes a >= 0 (already divided by the scale); ties to the even code, above 6 saturates."""
    d = np.abs(a[..., None] - VALUES)
    best = d.min(-1, keepdims=True)
    near = d == best
    # at most two codes are equally near: take the even one
    even = near & (np.arange(8) % 2 == 0)
    return np.where(even.any(-1), even.argmax(-1), near.argmax(-1))


def quantise(x):
    """x [R, C] float64 (numpy) -> (codes [R, C] with sign in bit 3, scale bytes [R, ceil(C/32)], values [R, C])."""
    r, c = x.shape
    blocks = -(-c // 32)
    p = np.zeros((r, blocks * 32))
    p[:, :c] = x
    p = p.reshape(r, blocks, 32)
    bad = ~np.isfinite(p).all(-1)
    top = np.where(bad, 0.0, np.abs(np.where(np.isfinite(p), p, 0.0)).max(-1))
    _, e = np.frexp(top)                                        # top = m 2^e, m in [0.5, 1): floor(log2 top) = e - 1
    scale = np.where(top > 0, np.clip(e - 1 - 2, -127, 127), -127)
    v = np.where(np.isfinite(p), p, 0.0) / np.exp2(scale.astype(np.float64))[..., None]
    code = code_of(np.abs(v)) | np.where(np.signbit(v), 8, 0)
    val = VALUES[code & 7] * np.where(code & 8, -1.0, 1.0) * np.exp2(scale.astype(np.float64))[..., None]
    val = np.where(bad[..., None], np.nan, val)
    return code.reshape(r, -1)[:, :c], np.where(bad, 255, scale + 127).astype(np.int64), val.reshape(r, -1)[:, :c]


def values(x, dim):
    """The values of a torch matrix in 4 bits, blocks along `dim`, float64 numpy."""
    a = to64(x)
    return quantise(a)[2] if dim == 1 else quantise(np.ascontiguousarray(a.T))[2].T


def unpack(codes, scales, rows, cols):
    """The library's buffers -> (codes [rows, cols], scale bytes [rows, blocks], whether everything behind the columns is zero)."""
    kp = -(-cols // KP) * KP
    b = codes.cpu().numpy().reshape(kp // KP, rows, KP // 2).transpose(1, 0, 2).reshape(rows, kp // 2)
    full = np.stack([b & 15, b >> 4], -1).reshape(rows, kp)
    rg = -(-rows // 64)
    s = scales.cpu().numpy().reshape(kp // KP, rg, 2, 32, 2, 2)    # [k128][group][block % 2][row % 32][block / 2][row / 32]
    s = s.transpose(1, 5, 3, 0, 4, 2).reshape(rg * 64, kp // 32)[:rows]
    return full[:, :cols].astype(np.int64), s[:, :-(-cols // 32)].astype(np.int64), not full[:, cols:].any()


def pack(code, scale):
    """(codes [rows, cols], scale bytes [rows, blocks]) -> the library's two buffers."""
    rows, cols = code.shape
    kp, rg = -(-cols // KP) * KP, -(-rows // 64)
    full = np.zeros((rows, kp), dtype=np.uint8)
    full[:, :cols] = code
    b = (full[:, 0::2] | full[:, 1::2] << 4).reshape(rows, kp // KP, KP // 2).transpose(1, 0, 2)
    s = np.zeros((rg * 64, kp // 32), dtype=np.uint8)
    s[:rows, :scale.shape[1]] = scale
    s = s.reshape(rg, 2, 32, kp // KP, 2, 2).transpose(3, 0, 5, 2, 4, 1)      # [k128][group][block % 2][row % 32][block / 2][row / 32]
    return torch.from_numpy(np.ascontiguousarray(b).reshape(-1)), torch.from_numpy(np.ascontiguousarray(s).reshape(-1))
