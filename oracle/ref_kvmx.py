"""CPU restatement, in 64 bits, of the KV cache in blocks of 32 elements with a shared power-of-two scale, and of
single-token attention over it (numpy). TEST INFRASTRUCTURE ONLY: nothing in the product path may import this file.

The number types are the 4-bit e2m1 and 8-bit e4m3 floats of the public OCP microscaling specification with its e8m0
scale; the rule for the scale (no element further than half a step from its code) is this framework's. The reference has
no quantised cache: the attention is that of transformers models/qwen3/modeling_qwen3.py:259-279 with q_len = 1."""
import numpy as np

GRID = {"mxfp4": np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6]),
        "mxfp8": np.array([m / 512 for m in range(8)] + [(1 + m / 8) * 2.0 ** (x - 7) for x in range(1, 16)
                                                         for m in range(8)][:-1])}
EDGE = {"mxfp4": 7.0, "mxfp8": 464.0}
MOST = {"mxfp4": 252, "mxfp8": 246}


def quantise(x, fmt):
    """x [..., D] fp64 (bf16 numbers) -> (codes uint8 [..., D] one per element, scale bytes uint8 [..., D/32])."""
    blocks = np.asarray(x, np.float64).reshape(*np.shape(x)[:-1], np.shape(x)[-1] // 32, 32)
    grid, bits = GRID[fmt], 3 if fmt == "mxfp4" else 7
    finite = np.isfinite(blocks).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(blocks), blocks, 0)).max(-1), 0)
    e = np.ones(top.shape, np.int64)
    for cand in range(1, MOST[fmt]):                       # the smallest exponent whose range holds the largest element
        e = np.where(top > EDGE[fmt] * 2.0 ** (cand - 127), cand + 1, e)
    y = np.where(finite[..., None], blocks, 0) / 2.0 ** (e[..., None] - 127)
    dist = np.abs(np.abs(y)[..., None] - grid)
    best = dist.argmin(-1)                                 # the lower code of a tie
    up = np.minimum(best + 1, len(grid) - 1)
    tie = (np.take_along_axis(dist, best[..., None], -1)[..., 0] == np.take_along_axis(dist, up[..., None], -1)[..., 0])
    code = np.where(tie & (best % 2 == 1), up, best) | (np.signbit(y).astype(np.int64) << bits)
    code = np.where(finite[..., None], code, 0)
    return (code.reshape(np.shape(x)).astype(np.uint8), np.where(finite, e, 255).astype(np.uint8))


def pack(code, fmt):
    """Codes one per element -> stored bytes (two to a byte in 4 bits, the even element in the low half)."""
    return code if fmt == "mxfp8" else (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def values(stored, scales, fmt):
    """Stored bytes [..., D or D/2] and scale bytes [..., D/32] -> fp64 [..., D]."""
    stored = np.asarray(stored).astype(np.int64)
    code = stored if fmt == "mxfp8" else np.stack([stored & 15, stored >> 4], -1).reshape(*stored.shape[:-1], 2 * stored.shape[-1])
    bits = 3 if fmt == "mxfp4" else 7
    grid = GRID[fmt] if fmt == "mxfp4" else np.append(GRID[fmt], np.nan)
    v = grid[code & ((1 << bits) - 1)] * np.where(code >> bits, -1.0, 1.0)
    s = np.where(np.asarray(scales) == 255, np.nan, 2.0 ** (np.asarray(scales).astype(np.float64) - 127))
    return v * np.repeat(s, 32, -1)


def attend(q, k, v, scale):
    """One stream: q [H, D], k/v [KVH, n, D] fp64 -> (out [H, D], bound [H, D]): bound is what an fp32 evaluation with a
    bf16 result may be off by. n = 0: zeros.

    Half a step of the result is 2^-8 |o| (bf16). A score is a sum of D products held in fp32 and two more roundings: off
    by at most (D + 4) 2^-24 S with S = scale max_j sum_d |q_d k_jd|, so a weight by that relative amount, plus 2^-21 for
    the exponential of a difference whose log2 is off by its own rounding (|s| 2^-24 each way, |s| <= S), plus n 2^-24 for
    each of the two sums over the keys; weights enter numerator and denominator: twice, on sum_j p_j |v_j|. The split of
    the keys adds one rounding a split (at most 64).
    With several query heads a kv head a weight w in [1, 2) enters the numerator as two bf16 numbers: the first is off by at
    most 2^-8, so what it leaves is at most that and the second is off by at most 2^-17 (half a step below 2^-8): that once.
    Weights are taken against a maximum that may lag the true one by 2^8 and are lost below fp32's smallest normal number
    (so are the factors that join waves and splits, each on a sum of at most n weights of at most 2^8), while the
    denominator is at least 1: n 2^8 2^-126 max_j |v_j| twice."""
    H, D = q.shape
    kvh, n = k.shape[:2]
    if n == 0:
        return np.zeros((H, D)), np.zeros((H, D))
    out, bound = np.empty((H, D)), np.empty((H, D))
    for h in range(H):
        kk, vv = k[h // (H // kvh)], v[h // (H // kvh)]
        s = scale * (kk @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ vv
        S = scale * (np.abs(kk) @ np.abs(q[h])).max()
        rel = (D + 4) * 2.0 ** -24 * S + 2 * S * 2.0 ** -24 + 2.0 ** -21 + (n + 64) * 2.0 ** -24
        two = 2.0 ** -17 if H > kvh else 0.0
        bound[h] = (2.0 ** -8 * np.abs(out[h]) + (2 * rel + two) * (p @ np.abs(vv))
                    + n * 2.0 ** -117 * np.abs(vv).max(0))
    return out, bound
