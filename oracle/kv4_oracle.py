"""The 4-bit paged cache in numpy, in 64 bits, from the definitions in ``include/mi_kv4.h``.

A group of 32 values of one token and head: m = bf16(min), s = bf16(fp32((max - m) / 15)),
c = clamp(round((x - m) / s), 0, 15), a zero m being +0; it stands for m + s * c.
"""

from __future__ import annotations

import numpy as np

GROUP = 32


def bf16(x: np.ndarray) -> np.ndarray:
    """float32 values rounded to bfloat16 (nearest even), as float32."""
    x = np.ascontiguousarray(x, dtype=np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000
    out = u.astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), out)


def quantise(x: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """x [..., D] -> (codes [..., D/32, 32] uint8, steps, minima [..., D/32] float32)."""
    x = np.asarray(x, dtype=np.float64)
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(all="ignore"):
        m = bf16(g.min(-1).astype(np.float32)) + np.float32(0)  # a zero minimum is +0
        s = bf16(((g.max(-1) - m.astype(np.float64)) / 15).astype(np.float32))
        bad = ~np.isfinite(g).all(-1) | ~np.isfinite(m) | ~np.isfinite(s)
        s = np.where(s > 0, s, np.float32(0))
        wide = s[..., None].astype(np.float64)
        c = np.clip(np.rint((g - m[..., None]) / np.where(wide > 0, wide, np.inf)), 0, 15)
        c = np.where(bad[..., None], 0, c).astype(np.uint8)
    return c, np.where(bad, np.float32(0), s), np.where(bad, np.float32(np.nan), m)


def stored(x: np.ndarray) -> np.ndarray:
    """What the cache stands for after x [..., D] was stored, in 64 bits."""
    c, s, m = quantise(x)
    return (m[..., None].astype(np.float64) + s[..., None].astype(np.float64) * c).reshape(np.shape(x))


def page_bytes(block_size: int, head_dim: int) -> int:
    return block_size * head_dim * 5 // 8


def write(pool: np.ndarray, tokens: np.ndarray, slots, block_size: int) -> None:
    """tokens [T, H, D] into pool uint8 [N, H, page bytes] at their slots."""
    d = tokens.shape[-1]
    c, s, m = quantise(tokens)
    ng = d // GROUP
    codes = pool[..., : ng * block_size * 16].reshape(*pool.shape[:2], ng, block_size, 16).copy()
    pars = pool[..., ng * block_size * 16 :].reshape(*pool.shape[:2], block_size, ng, 4).copy()
    pair = c.reshape(*c.shape[:-1], 16, 2)
    packed = pair[..., 0] | (pair[..., 1] << 4)
    words = np.stack((s, m), -1).view(np.uint32) >> 16
    words = np.where(np.isnan(np.stack((s, m), -1)), 0x7FC0, words).astype("<u2")
    for i, slot in enumerate(slots):
        b, o = int(slot) // block_size, int(slot) % block_size
        codes[b, :, :, o] = packed[i]
        pars[b, :, o] = words[i].view(np.uint8).reshape(words.shape[1], ng, 4)
    pool[..., : ng * block_size * 16] = codes.reshape(*pool.shape[:2], -1)
    pool[..., ng * block_size * 16 :] = pars.reshape(*pool.shape[:2], -1)


def read(pool: np.ndarray, blocks, block_size: int, head_dim: int) -> np.ndarray:
    """Blocks of a pool as values [len(blocks), bs, H, D] in 64 bits."""
    ng = head_dim // GROUP
    p = pool[np.asarray(blocks, dtype=np.int64)]
    codes = p[..., : ng * block_size * 16].reshape(*p.shape[:2], ng, block_size, 16)
    c = np.stack((codes & 15, codes >> 4), -1).reshape(*codes.shape[:-1], GROUP)
    par = np.ascontiguousarray(p[..., ng * block_size * 16 :]).view("<u2").reshape(*p.shape[:2], block_size, ng, 2)
    sm = (par.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    v = sm[..., 1][..., None] + sm[..., 0][..., None] * c.transpose(0, 1, 3, 2, 4)
    return v.reshape(*v.shape[:3], head_dim).transpose(0, 2, 1, 3)


def decode(q: np.ndarray, k_pool, v_pool, tables, ctx, scale: float, block_size: int) -> np.ndarray:
    """q [B, Hq, D] -> [B, Hq * D]: attention over the first ctx[b] positions (zeros where there are none)."""
    q = np.asarray(q, dtype=np.float64)
    b, hq, d = q.shape
    h = k_pool.shape[1]
    out = np.zeros((b, hq, d))
    for i in range(b):
        n = int(ctx[i])
        if n <= 0:
            continue
        ids = tables[i, : -(-n // block_size)]
        k = read(k_pool, ids, block_size, d).reshape(-1, h, d)[:n].repeat(hq // h, axis=1)
        v = read(v_pool, ids, block_size, d).reshape(-1, h, d)[:n].repeat(hq // h, axis=1)
        s = np.einsum("hd,thd->ht", q[i], k) * scale
        p = np.exp(s - s.max(-1, keepdims=True))
        out[i] = np.einsum("ht,thd->hd", p / p.sum(-1, keepdims=True), v)
    return out.reshape(b, hq * d)
