"""Plain 64-bit forms of the 4-bit page format and of what attends and evicts it."""

from __future__ import annotations

import math

import torch

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantise(x):
    """(codes, scale bytes) of rows (..., D): the format's definition in 64 bits."""
    blocks = x.double().reshape(*x.shape[:-1], -1, 32)
    finite = torch.isfinite(blocks).all(-1)
    safe = torch.where(finite[..., None], blocks, 0.0)
    amax = safe.abs().amax(-1)
    byte = torch.ones_like(amax, dtype=torch.int64)
    for e in range(1, 252):  # the smallest scale of which amax is at most 7 times
        byte = torch.where(amax > 7.0 * 2.0 ** (e - 127), torch.full_like(byte, e + 1), byte)
    y = safe.abs() / torch.exp2(byte.double() - 127)[..., None]
    gaps = (y[..., None] - LEVELS.to(x.device)).abs()
    best = gaps.amin(-1, keepdim=True)
    near = gaps == best  # two levels at halfway: the even code
    code = torch.arange(8, device=x.device)
    pick = torch.where(near & (code % 2 == 0), code, torch.where(near, code + 8, 99)).amin(-1)
    pick = torch.where(pick >= 8, pick - 8, pick)
    sign = torch.signbit(safe).long()  # of a zero too
    codes = pick + 8 * sign
    byte = torch.where(finite, byte, 255)
    return codes.reshape(x.shape), byte


def values(codes, byte):
    """fp64 rows of codes (..., D) and scale bytes (..., D / 32)."""
    v = LEVELS.to(codes.device)[codes & 7] * (1 - 2 * (codes >> 3).double())
    s = torch.where(byte == 255, math.nan, torch.exp2(byte.double() - 127))
    return (v.reshape(*v.shape[:-1], -1, 32) * s[..., None]).reshape(v.shape)


def stored(x):
    return values(*quantise(x))


def parts(pool):
    """Views (K codes, V codes, K scales, V scales) of a 4-bit pool."""
    n, H, P, row = pool.shape
    D = row * 16 // 17
    out, at = [], 0
    for width in (D // 2, D // 2, D // 32, D // 32):
        out.append(torch.as_strided(pool, (n, H, P, width), (pool.stride(0), pool.stride(1), width, 1),
                                    pool.storage_offset() + at))
        at += P * width
    return out


def read_pool(pool):
    """(k, v) codes and scale bytes as (codes, byte) of all pages (n, Hkv, P, D)."""
    kc, vc, ks, vs = parts(pool)
    return [(torch.stack([c & 15, c >> 4], -1).flatten(-2).long(), s.long()) for c, s in ((kc, ks), (vc, vs))]


def fill_pool(pool, k, v):
    """Write rows k, v (n, Hkv, P, D) into the pages of a pool."""
    for x, c, s in zip((k, v), parts(pool)[:2], parts(pool)[2:]):
        codes, byte = quantise(x)
        c.copy_((codes[..., 0::2] + 16 * codes[..., 1::2]).to(torch.uint8))
        s.copy_(byte.to(torch.uint8))


def rows_of(pages, table_row, n):
    """Rows [0, n) (Hkv, n, D) of a sequence whose pages are (num_pages, Hkv, P, D)."""
    P = pages.shape[2]
    ids = table_row[:-(-n // P)].long()
    return pages[ids].transpose(0, 1).reshape(pages.shape[1], -1, pages.shape[3])[:, :n]


def attention(q, k, v, scale):
    """q (Hq, D), k, v (Hkv, n, D) in fp64: (o, lse, sum of p |v|, largest sum of |q k|)."""
    Hkv, n, D = k.shape
    qg = q.double().view(Hkv, -1, D)
    s = qg @ k.transpose(1, 2).contiguous() * scale
    p = torch.softmax(s, -1)
    spread = (qg.abs() @ k.abs().transpose(1, 2).contiguous() * scale).amax(-1)
    return ((p @ v).reshape(-1, D), torch.logsumexp(s, -1).reshape(-1), (p @ v.abs()).reshape(-1, D),
            spread.reshape(-1))


def key_weights(q, k, lse, scale, causal=True):
    """q (Hq, S, D), k (Hkv, n, D), lse (Hq, S): (Hkv, n) in fp64."""
    Hkv, n, D = k.shape
    Hq, S, _ = q.shape
    s = (q.double().reshape(Hkv, -1, D) @ k.double().transpose(1, 2).contiguous() * scale).view(Hq, S, n)
    l = lse.double()[..., None]
    p = torch.where(l == -math.inf, 0.0, torch.exp(s - torch.where(l == -math.inf, 0.0, l)))
    if causal and S > 1:
        p = p * torch.ones(S, n, dtype=torch.bool, device=p.device).tril(n - S)
    return p.view(Hkv, Hq // Hkv, S, n).sum((1, 2))


def select(w, n, keep, recent, first):
    """The rows a head keeps, by sorting: w (W,) fp32."""
    if n <= keep:
        return list(range(n)) + [-1] * (keep - n)
    middle = list(range(first, n - recent))
    vals = w.tolist()
    order = sorted(middle, key=lambda i: (0 if vals[i] != vals[i] else 1, -vals[i] if vals[i] == vals[i] else 0.0, i))
    chosen = order[:keep - first - recent]
    return list(range(first)) + sorted(chosen) + list(range(n - recent, n))
