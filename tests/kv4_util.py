"""The 4-bit cache and attention over it in 64 bits (numpy), as the header defines them."""
import numpy as np

GROUP = 32


def groups(size):
    n = -(-size // GROUP)
    return 8 if n > 4 else n


def row_bytes(size):
    return 20 * groups(size)


def pack(x):
    """Rows for values [..., size], given as float64 that hold the inputs' values exactly."""
    size, ng = x.shape[-1], groups(x.shape[-1])
    x = np.clip(np.nan_to_num(x, nan=0.0, posinf=65504.0, neginf=-65504.0), -65504.0, 65504.0)
    codes = np.full(x.shape[:-1] + (ng * GROUP,), 8, dtype=np.int64)
    params = np.zeros(x.shape[:-1] + (ng, 2), dtype=np.float16)
    for g in range(-(-size // GROUP)):
        part = x[..., g * GROUP:min(size, (g + 1) * GROUP)]
        lo, hi = part.min(-1, keepdims=True), part.max(-1, keepdims=True)
        scale = ((hi - lo) / 15).astype(np.float32).astype(np.float16)
        zero = (lo + 8 * scale.astype(np.float64)).astype(np.float32).astype(np.float16)
        s, z = scale.astype(np.float64), zero.astype(np.float64)
        code = np.where(s > 0, np.rint((part - z) / np.where(s > 0, s, 1.0)) + 8, 8)
        codes[..., g * GROUP:g * GROUP + part.shape[-1]] = np.clip(code, 0, 15)
        params[..., g, 0], params[..., g, 1] = scale[..., 0], zero[..., 0]
    both = (codes[..., 0::2] | codes[..., 1::2] << 4).astype(np.uint8)
    return np.concatenate([both, params.reshape(x.shape[:-1] + (-1,)).view(np.uint8)], -1)


def unpack(rows, size):
    """(values, scales, zeros) of rows, each [..., size], in 64 bits."""
    ng = groups(size)
    b = rows[..., :ng * 16].astype(np.int64)
    codes = np.stack([b & 15, b >> 4], -1).reshape(rows.shape[:-1] + (ng * GROUP,))
    params = np.ascontiguousarray(rows[..., ng * 16:]).view(np.float16).astype(np.float64).reshape(rows.shape[:-1] + (ng, 2))
    s, z = np.repeat(params[..., 0], GROUP, -1), np.repeat(params[..., 1], GROUP, -1)
    return (z + s * (codes - 8))[..., :size], s[..., :size], z[..., :size]


def attention(q, k_rows, v_rows, lens, scale, half_probabilities):
    """Results [batch, heads, size], sums [batch, kv heads, capacity] of the softmax, and bounds of the error of either.

    Bounds, u = 2^-24: a score is a sum of `size` products with codes, scales and zeros in FP32, off by at most (size + 16) u of the sum of
    magnitudes; a probability is off by that twice (its own score and the sum's) and by the exponential (4 u), and by half a step of FP16
    (2^-11; hi + lo: 2^-21) where it meets a value's distance from the zero; sums over positions go through the tensor cores' accumulators,
    a tile of 16 positions per step and at most one tile in 128 positions behind another, with 2 u each, and 64 more where warps and
    runs are put together."""
    batch, heads, size = q.shape
    kv, cap = k_rows.shape[1:3]
    gqa, u = heads // kv, 2.0 ** -24
    out, bound = np.zeros((batch, heads, size)), np.zeros((batch, heads, size))
    sums, sums_bound = np.zeros((batch, kv, cap)), np.zeros((batch, kv, cap))
    for b in range(batch):
        n = int(lens[b])
        if n == 0:
            continue
        for h in range(kv):
            k, ks, kz = unpack(k_rows[b, h, :n], size)
            v, vs, vz = unpack(v_rows[b, h, :n], size)
            qh = q[b, h * gqa:(h + 1) * gqa]
            x = qh @ k.T * scale
            dx = (size + 16) * u * (np.abs(qh) @ (16 * ks + np.abs(kz)).T) * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            # of p: own score, exponent's rounding, and the weighted mean of the same for the sum
            dp = dx + (np.abs(x) + np.abs(x).max(-1, keepdims=True) + 8) * 2 * u
            dp = np.expm1(dp + (dp * p).sum(-1, keepdims=True)) + (2 * (n / 128) + 64) * 2 * u
            out[b, h * gqa:(h + 1) * gqa] = p @ v
            bound[b, h * gqa:(h + 1) * gqa] = (p * dp) @ (np.abs(v - vz) + np.abs(vz)) + p @ np.abs(v - vz) * (2.0 ** -11 if half_probabilities else 2.0 ** -21) \
                + n * 2.0 ** -33 * (p @ np.abs(v - vz)).max(-1, keepdims=True)
            sums[b, h, :n] = p.sum(0)
            sums_bound[b, h, :n] = (p * dp).sum(0)
    return out, bound, sums, sums_bound


def keep_rows(sums, n, keep, recent):
    """Positions that stay of the first n of one head."""
    if n <= keep:
        return list(range(n))
    old = max(0, n - recent)
    w = [-np.inf if np.isnan(x) else x for x in sums[:old]]
    some = sorted(range(old), key=lambda i: (-w[i], i))[:keep - (n - old)]
    return sorted(some) + list(range(old, n))
