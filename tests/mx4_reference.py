"""Plain 64-bit forms of the four-bit operators and of the mixture-of-experts layer (numpy)."""
import numpy as np

CODES = np.array([0, .5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantize(x):
    """Rows of float64 values -> (codes, scales), by distance to the eight magnitudes."""
    rows, cols = x.shape
    blocks = -(-cols // 32)
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = x
    v = v.reshape(rows, blocks, 32)
    codes = np.zeros((rows, blocks, 32), np.uint8)
    scales = np.zeros((rows, blocks), np.uint8)
    for r in range(rows):
        for b in range(blocks):
            a = np.abs(v[r, b])
            if not np.isfinite(a).all():
                scales[r, b] = 255
                continue
            top = a.max()
            e = -127 if top == 0 else max(-127, int(np.frexp(top)[1]) - 1 - 2)
            scales[r, b] = e + 127
            d = np.abs(np.ldexp(a, -e)[:, None] - CODES[None])
            low = d.argmin(1)                      # the lower one of two at the same distance
            tie = (low < 7) & (d[np.arange(32), low] == d[np.arange(32), np.minimum(low + 1, 7)])
            c = np.where(tie & (low % 2 == 1), low + 1, low)
            codes[r, b] = c | np.where(np.signbit(v[r, b]), 8, 0)
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(rows, blocks * 16), scales


def values(codes, scales, cols):
    """float64 values of codes [..., blocks * 16] and scales [..., blocks]."""
    c = np.stack((codes & 15, codes >> 4), -1).reshape(*scales.shape, 32)
    v = np.where(c >= 8, -CODES[c & 7], CODES[c & 7])
    s = np.ldexp(1.0, scales.astype(np.int64) - 127)
    s = np.where(scales == 255, np.nan, s)
    return (v * s[..., None]).reshape(*scales.shape[:-1], scales.shape[-1] * 32)[..., :cols]


def select(logits, topk):
    """[tokens, topk] indices: NaN first, then by value, ties to the lowest index."""
    key = np.where(np.isnan(logits), np.inf, logits)
    first = ~np.isnan(logits)
    idx = np.broadcast_to(np.arange(logits.shape[1]), logits.shape)
    order = np.stack([np.lexsort((idx[t], -key[t], first[t])) for t in range(logits.shape[0])])
    return order[:, :topk]


def route(x, router, topk, renormalize):
    """(ids, weights) of each token."""
    logits = x @ router.T
    ids = select(logits, topk)
    z = np.exp(logits - np.take_along_axis(logits, ids[:, :1], 1))
    w = np.take_along_axis(z, ids, 1)
    return ids, w / (w if renormalize else z).sum(1, keepdims=True)


def moe(x, router, gate, up, down, topk, renormalize, half_eps, gamma):
    """(y, bound, ids, weights): the layer, and how far a kernel may be from y that sums in fp32
    (gamma(K): relative to the sum of magnitudes of K products), rounds h once to a type whose
    rounding is half_eps relative, and takes the softmax in fp32 (2^-20 relative)."""
    ids, w = route(x, router, topk, renormalize)
    y, bound = np.zeros_like(x), np.zeros_like(x)
    gk, gi = gamma(x.shape[1]), gamma(down.shape[2])
    for t in range(x.shape[0]):
        for e, share in zip(ids[t], w[t]):
            g, u = gate[e] @ x[t], up[e] @ x[t]
            dg, du = gk * (np.abs(gate[e]) @ np.abs(x[t])), gk * (np.abs(up[e]) @ np.abs(x[t]))
            sig = 1 / (1 + np.exp(-g))
            h = g * sig * u
            # |silu'| <= 1.1, and silu itself to 2^-21 relative in fp32
            dh = 1.1 * dg * np.abs(u) + np.abs(g * sig) * du + 1.1 * dg * du + 2.0 ** -21 * np.abs(h)
            dh = dh * (1 + half_eps) + half_eps * np.abs(h) + 2.0 ** -25  # fp16's subnormal half step
            y[t] += share * (down[e] @ h)
            bound[t] += share * (np.abs(down[e]) @ dh + (gi + 2.0 ** -20) * (np.abs(down[e]) @ (np.abs(h) + dh)))
    return y, bound, ids, w
