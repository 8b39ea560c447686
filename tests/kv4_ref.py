"""Plain numpy forms of the 4-bit cache's formulas, for its tests: the Q4_0 rule
in fp32, the page layout, and attention in 64 bits."""
import numpy as np


def quantise(x):
    """(codes uint8 [..., D], scales fp16 [..., D/32]) of fp32 rows."""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    m = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)
    d = (m / np.float32(-8)).astype(np.float32)
    with np.errstate(divide="ignore", over="ignore", invalid="ignore"):
        r = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        y = (b * r).astype(np.float32) + np.float32(8.5)
        y = np.where(np.isnan(y), 0, np.clip(y, 0, 15))
        scale = d[..., 0].astype(np.float16)
    return np.trunc(y).astype(np.uint8).reshape(x.shape), scale


def values(codes, scales):
    """What codes stand for, in 64 bits."""
    c = codes.reshape(*codes.shape[:-1], -1, 32).astype(np.float64) - 8
    with np.errstate(invalid="ignore"):
        return (c * scales.astype(np.float64)[..., None]).reshape(codes.shape)


def group_bytes(D):
    return 16 * 2 * (D // 2 + D // 16)


def place(pool, page, head, off, is_v, D, page_len, codes, scales):
    """Writes one row into a pool [n_pages, Hkv, page_len / 16, group_bytes]."""
    g = pool[page, head, off // 16]
    r, base = off % 16, (group_bytes(D) // 2 if is_v else 0)
    nb = D // 32
    row = np.zeros(D // 4, np.uint16)
    for b in range(nb):
        for q in range(8):
            w = 0
            for i in range(4):
                w |= int(codes[32 * b + 4 * q + i]) << (4 * i)
            row[q * nb + b] = w
    g[base + r * D // 2: base + (r + 1) * D // 2] = row.view(np.uint8)
    s = base + 8 * D + r * nb * 2
    g[s:s + 2 * nb] = scales.view(np.uint8)


def attention(q, k, v):
    """q [Hq, D], k and v [n, Hkv, D] -> (out [Hq, D], bound [Hq, D], largest |score|)
    in 64 bits.

    bound: how far an fp32 evaluation by the kernel's steps may be off.  A
    score's inputs carry 22 bits and it takes, per block of 32 dims, two matrix
    instructions started at -8 sum q, so terms up to |q| (15 + 8) |d| in size, each
    instruction rounding or cutting its sum by at most 2^-21 of the terms' sum,
    and four more fp32 steps: 2^-22 + 2 * 2^-21 + 4 * 2^-24 < 2^-19 of A = sum over
    blocks of |d| 23 sum |q| / sqrt(D).  A probability is then off by that and
    the exponential's 2^-21, numerator and denominator both; the sum over the
    keys adds at most one instruction's 2^-21 per 16 keys of the longest chain,
    which the caller states through `steps`."""
    n, hkv, D = k.shape
    hq = q.shape[0]
    out = np.zeros((hq, D))
    bound = np.zeros((hq, D))
    top = 0.0
    if n == 0:
        return out, bound, top
    q = q.astype(np.float64)
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)], v[:, h // (hq // hkv)]
        s = kk @ q[h] / np.sqrt(D)
        top = max(top, np.abs(s).max())
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vv
        # |d| of a block is at least its largest value / 8
        dk = np.abs(kk).reshape(n, -1, 32).max(-1) / 8
        A = (dk * 23 * np.abs(q[h]).reshape(-1, 32).sum(-1)).sum(-1).max() / np.sqrt(D)
        bound[h] = 2 * (2.0 ** -19 * A + 2.0 ** -21) * (p @ np.abs(vv))
    return out, bound, top


def steps_bound(v, n, chain):
    """The accumulation's part: `chain` matrix instructions, 2^-21 each, of the
    terms |p d (n - 8)|, at most the largest |v|."""
    return chain * 2.0 ** -21 * (np.abs(v).max() if n else 0.0)
