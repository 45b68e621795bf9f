"""Plain forms of the paged KV cache's operators for the tests: the cache's
layout from its description, its values from the host encoders, and the
attention of token trees in 64 bits."""
import numpy as np

PAGE = 64
Q8_LIMIT = 65024.0


def bf16_bits(x):
    """f32 -> bf16 bits, round to nearest even (finite values)."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    return ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) >> 16).astype(np.uint16)


def q8_blocks(lrs, x):
    """Codes [..., hd] and f16 scales [..., hd / 32] of the host's Q8_0 encoder."""
    x = np.clip(np.nan_to_num(np.asarray(x, np.float32), nan=0.0, posinf=Q8_LIMIT, neginf=-Q8_LIMIT),
                -Q8_LIMIT, Q8_LIMIT)
    hd = x.shape[-1]
    n = x.size // hd
    q = lrs.QuantTensor.quantize(x.ravel(), n, hd, lrs.QuantType.Q8_0)
    assert q.quant_type == lrs.QuantType.Q8_0
    b = q.data.reshape(n, hd // 32, 34)
    d = np.ascontiguousarray(b[:, :, :2]).view(np.float16).reshape(x.shape[:-1] + (hd // 32,))
    c = np.ascontiguousarray(b[:, :, 2:]).view(np.int8).reshape(x.shape)
    return c, d


def held(lrs, dtype, x):
    """The f64 values a cache of the type holds for f32 rows x."""
    x = np.asarray(x, np.float32)
    if dtype == lrs.KvType.F32:
        return x.astype(np.float64)
    if dtype == lrs.KvType.BF16:
        return (bf16_bits(x).astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    c, d = q8_blocks(lrs, x)
    return c.astype(np.float64) * np.repeat(d.astype(np.float64), 32, axis=-1)


def pack(lrs, dtype, x, is_v):
    """Tiles [pages, heads, bytes] of rows x [pages, heads, 64, hd]."""
    p, h, _, hd = x.shape
    if dtype == lrs.KvType.F32:
        return np.ascontiguousarray(x, np.float32).view(np.uint8).reshape(p, h, -1)
    if dtype == lrs.KvType.BF16:
        return bf16_bits(x).view(np.uint8).reshape(p, h, -1)
    c, d = q8_blocks(lrs, x)
    if is_v:
        codes = c.reshape(p, h, PAGE // 4, 4, hd).transpose(0, 1, 2, 4, 3)
        scale = d.transpose(0, 1, 3, 2)
    else:
        codes = c.reshape(p, h, PAGE, hd // 16, 16).transpose(0, 1, 3, 2, 4)
        scale = d
    return np.concatenate([np.ascontiguousarray(codes).view(np.uint8).reshape(p, h, -1),
                           np.ascontiguousarray(scale).view(np.uint8).reshape(p, h, -1)], axis=2)


def random_tree(rng, n):
    """Masks of a random tree of n nodes: node i hangs on one before it."""
    masks = [1]
    for i in range(1, n):
        masks.append(masks[int(rng.integers(0, i))] | 1 << i)
    return masks[:n]


def attention(q, k, v, ctx, masks, scale):
    """One tree in 64 bits: q [nodes, heads, hd], k / v [kv heads, positions, hd]
    -> (out [nodes, heads, hd], err): err bounds what f32 products and sums may
    do to each row (derivation in the caller's tolerance)."""
    n, nh, hd = q.shape
    nkv = k.shape[0]
    out = np.zeros((n, nh, v.shape[2]))
    err = np.zeros((n, nh, 1))
    for i in range(n):
        seen = list(range(ctx)) + [ctx + j for j in range(n) if masks[i] >> j & 1]
        if not seen:
            continue
        for h in range(nh):
            kk, vv = k[h // (nh // nkv)][seen], v[h // (nh // nkv)][seen]
            s = (kk @ q[i, h].astype(np.float64)) * scale
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv
            # a score: hd products summed in f32, in any order, with truncating
            # sums (2^-23 a step), its scaling and exponential (4 more)
            ds = (hd + 4) * 2.0 ** -23 * abs(scale) * (np.abs(kk) @ np.abs(q[i, h].astype(np.float64))).max()
            # the weights move by at most e^(2 ds) - 1; their sums and the
            # products with V add a truncation a step of 32 positions, and 64 more
            err[i, h] = (np.expm1(2 * ds) + (len(seen) / 32 + 64) * 2.0 ** -23) * np.abs(vv).max()
    return out, err
