"""A plain implementation of the 4-bit KV cache and its attention (numpy, 64 bits where values are summed)."""
import numpy as np


def quantize(x):
    """f32 [..., hd] -> codes uint8 [..., hd / 32, 32], scales f16 [..., hd / 32]; 32-bit arithmetic, each operation rounded."""
    x = np.asarray(x, np.float32).reshape(x.shape[:-1] + (-1, 32))
    big = np.finfo(np.float32).max
    x = np.clip(np.where(np.isnan(x), np.float32(0), x), -big, big).astype(np.float32)
    hi, lo = x.max(-1), x.min(-1)
    m = np.where(hi >= -lo, hi, lo)
    with np.errstate(over="ignore", divide="ignore", invalid="ignore"):
        d = np.clip(m * np.float32(-0.125), np.float32(-65504), np.float32(65504))
        d16 = d.astype(np.float16)
        inv = np.where(d16 == 0, np.float32(0), np.float32(1) / np.where(d == 0, np.float32(1), d)).astype(np.float32)
        c = np.floor((x * inv[..., None]).astype(np.float32) + np.float32(8.5))
    return np.clip(c, 0, 15).astype(np.uint8), d16


def values(codes, scales):
    return ((codes.astype(np.float64) - 8) * scales.astype(np.float64)[..., None]).reshape(codes.shape[:-2] + (-1,))


def turn(pos, hd):
    return (pos >> 1) & 3 if hd == 128 else (pos >> 2) & 1


def _slots(pos, nb):
    return np.arange(nb)[None] ^ turn(np.asarray(pos), 32 * nb)[:, None]


def pack(codes, pos):
    """codes [n, blocks, 32] of the rows at positions pos -> the bytes of the codes plane [n, blocks * 16]."""
    n, nb, _ = codes.shape
    out = np.zeros((n, nb, 16), np.uint8)
    out[np.arange(n)[:, None], _slots(pos, nb)] = codes[..., 0::2] | (codes[..., 1::2] << 4)
    return out.reshape(n, -1)


def unpack(data, pos):
    n, nb = data.shape[0], data.shape[1] // 16
    chunks = data.reshape(n, nb, 16)[np.arange(n)[:, None], _slots(pos, nb)]
    out = np.zeros((n, nb, 32), np.uint8)
    out[..., 0::2], out[..., 1::2] = chunks & 15, chunks >> 4
    return out


def attend(q, K, V, last, window, n_sink, scale):
    """One query [nh, hd] at position `last` over values K, V [n, nkv, hd] -> out f64 [nh, hd], the largest |score|,
    the largest sum |q||k| * scale, the largest |v|; zeros where nothing is seen."""
    nh, hd = q.shape
    G = nh // K.shape[1]
    p = np.arange(K.shape[0])
    keep = (p <= last) & ((window == 0) | (last - p < window) | (p < n_sink))
    out = np.zeros((nh, hd))
    smax = sabs = 0.0
    if not keep.any():
        return out, 0.0, 0.0, 0.0
    for h in range(nh):
        k, v = K[keep, h // G], V[keep, h // G]
        s = k @ q[h] * scale
        e = np.exp(s - s.max())
        out[h] = e @ v / e.sum()
        smax = max(smax, np.abs(s).max())
        sabs = max(sabs, (np.abs(k) @ np.abs(q[h])).max() * scale)
    return out, smax, sabs, np.abs(V[keep]).max()
