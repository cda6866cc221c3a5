"""The 4-bit cache in plain numpy, from the layout that the C header states,
and attention over it in 64 bits: what the kernels are held against."""

from __future__ import annotations

import numpy as np
import torch


def nibble_maps():
    """(token, dim) of every nibble of a block's K part and V part, [2048, 2]."""
    k = np.zeros((2048, 2), int)
    v = np.zeros((2048, 2), int)
    for kg in range(4):
        for n in range(16):
            for w in range(4):
                dword = (16 * (16 * kg + n) + 4 * w) // 4
                for i in range(4):
                    k[8 * dword + i] = n, 32 * w + 8 * kg + 2 * i
                    k[8 * dword + i + 4] = n, 32 * w + 8 * kg + 2 * i + 1
                for t, (a, b) in enumerate(zip((0, 4, 1, 5), (2, 6, 3, 7))):
                    v[8 * dword + a] = 4 * kg + t, 8 * n + 2 * w
                    v[8 * dword + b] = 4 * kg + t, 8 * n + 2 * w + 1
    return k, v


_K_MAP, _V_MAP = nibble_maps()


def unpack(codes: torch.Tensor, scales: torch.Tensor):
    """(codes, scales) of K and of V: int [pages, 16, H, 128], FP16 [pages, 16, H]."""
    raw = codes.cpu().numpy()                                        # [P, H, 2, 1024]
    pages, heads = raw.shape[:2]
    nibbles = np.stack((raw & 15, raw >> 4), axis=-1).reshape(pages, heads, 2, 2048)
    out = []
    for part, where in enumerate((_K_MAP, _V_MAP)):
        full = np.zeros((pages, heads, 16, 128), np.int64)
        full[:, :, where[:, 0], where[:, 1]] = nibbles[:, :, part].astype(np.int64) - 8
        s = scales.cpu().numpy()[:, :, :, part].reshape(pages, heads, 16)
        out.append((full.transpose(0, 2, 1, 3), s.transpose(0, 2, 1)))
    return out


def held(x: np.ndarray):
    """Codes and FP16 scales of centered float32 rows [..., 128]."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        amax = np.fmax.reduce(np.abs(x), axis=-1, initial=0.0)
        seventh = np.float32(1.0) / np.float32(7.0)
        scale = np.maximum(amax * seventh, np.float32(2.0 ** -20)).astype(np.float16)
        q = x / scale.astype(np.float32)[..., None]
        steps = np.minimum(np.floor(np.abs(q) + np.float32(0.5)), np.float32(7.0))
        return np.where(np.isnan(q), 0, np.copysign(steps, q)).astype(np.int64), scale


def random_pool(gen, pages, heads, device, scale=0.3):
    """A pool of random codes in [-7, 7] and scales in (0, 2 * scale)."""
    low = torch.randint(1, 16, (pages, heads, 2, 1024), generator=gen)
    high = torch.randint(1, 16, (pages, heads, 2, 1024), generator=gen)
    scales = torch.rand(pages, heads, 4, 2, 4, generator=gen) * 2 * scale + 2.0 ** -12
    return (low | high << 4).to(torch.uint8).to(device), scales.half().to(device)


def attention(q, k, v, center, sm_scale):
    """One request in float64: q [Hq, 128], k and v [T, Hkv, 128] -> (out, lse,
    bound): ``bound`` [Hq] is what float32 may be off by before the output's
    rounding, as test_gpu_int4_decode derives it."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    hq, hkv = q.shape[0], k.shape[1]
    group = hq // hkv
    out = np.zeros((hq, 128))
    lse = np.full(hq, -np.inf)
    bound = np.zeros(hq)
    spread = np.zeros(hq)
    for h in range(hq):
        kh, vh = k[:, h // group], v[:, h // group]
        if len(kh):
            s = kh @ q[h] * sm_scale * np.log2(np.e)
            m = s.max()
            p = np.exp2(s - m)
            out[h] = p @ vh / p.sum()
            lse[h] = m + np.log2(p.sum())
            spread[h] = (np.abs(kh) @ np.abs(q[h])).max() * sm_scale * np.log2(np.e)
            weight = np.log(2.0) * 136 * 2.0 ** -24 * spread[h] + 2.0 ** -20
            bound[h] = 2 * weight * np.abs(vh).max()
    if center is not None:
        out += np.repeat(np.asarray(center, np.float64), group, axis=0)
    return out, lse, bound, 136 * 2.0 ** -24 * spread
