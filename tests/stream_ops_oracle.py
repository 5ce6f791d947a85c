"""Plain 64-bit statements of the multi-axis rotary, dropout and group norm ops, in numpy on the CPU
(test infrastructure)."""
import numpy as np


def philox4x32(counter, key, rounds):
    """Philox4x32 (Salmon et al. 2011) of arrays of counter words c0..c3 under a 2-word key, word by word in
    Python-sized integers: uint64 arrays whose values stay below 2^32."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        p0, p1 = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(p1 >> half) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> half) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def dropout_bits(count, seed, offset, first=0):
    """The 16 random bits of elements first .. first+count-1 (first a multiple of 8)."""
    block = np.arange(first // 8, first // 8 + (count + 7) // 8, dtype=np.uint64)
    seed, offset = seed & (2 ** 64 - 1), offset & (2 ** 64 - 1)
    words = philox4x32((block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), np.full_like(block, offset & 0xFFFFFFFF),
                        np.full_like(block, offset >> 32)), (seed & 0xFFFFFFFF, seed >> 32), 7)
    halves = []
    for w in words:
        halves += [w & np.uint64(0xFFFF), w >> np.uint64(16)]
    return np.stack(halves, -1).reshape(-1)[:count].astype(np.int64)


def dropout(x, threshold, seed, offset, residual=None):
    """64 bits; x any shape of float64."""
    keep = dropout_bits(x.size, seed, offset).reshape(x.shape) >= threshold
    scale = 65536.0 / (65536.0 - threshold) if threshold < 65536 else 0.0
    y = np.where(keep, x * scale if threshold < 65536 else 0.0, 0.0)
    return y if residual is None else residual + y


def pair_axes(sections, order):
    if order == "blocks":
        return [a for a in range(len(sections)) for _ in range(sections[a])]
    left, out = list(sections), []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def rope_axes(x, table, positions, sections, half, order, backward):
    """x (tokens, heads, d) float64, table (rows, d) float64, positions (tokens, axes): loops over pairs."""
    tokens, heads, d = x.shape
    y = np.empty_like(x)
    rows = table.shape[0]
    for j, axis in enumerate(pair_axes(sections, order)):
        i1, i2 = (j, j + d // 2) if half else (2 * j, 2 * j + 1)
        pos = positions[:, axis].astype(np.int64)
        ok = (pos >= 0) & (pos < rows)
        at = np.where(ok, pos, 0)
        c, s = np.where(ok, table[at, 2 * j], np.nan)[:, None], np.where(ok, table[at, 2 * j + 1], np.nan)[:, None]
        if backward:
            s = -s
        y[:, :, i1] = x[:, :, i1] * c - x[:, :, i2] * s
        y[:, :, i2] = x[:, :, i2] * c + x[:, :, i1] * s
    return y


def sigmoid(z):
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1.0 / (1.0 + e), e / (1.0 + e))


def group_norm(x, weight, bias, groups, eps, activation):
    """x (N, S, C) float64 -> (y, stats (N, G, 2))."""
    N, S, C = x.shape
    v = x.reshape(N, S, groups, C // groups)
    mean = v.mean((1, 3))
    var = ((v - mean[:, None, :, None]) ** 2).mean((1, 3))
    rstd = 1.0 / np.sqrt(var + eps)
    z = ((v - mean[:, None, :, None]) * rstd[:, None, :, None]).reshape(N, S, C) * weight + bias
    return (z * sigmoid(z) if activation == "silu" else z), np.stack([mean, rstd], -1)


def group_norm_backward(dout, x, weight, bias, stats, groups, activation):
    N, S, C = x.shape
    v = x.reshape(N, S, groups, C // groups)
    mean, rstd = stats[:, None, :, None, 0], stats[:, None, :, None, 1]
    h = ((v - mean) * rstd).reshape(N, S, C)
    dz = dout
    if activation == "silu":
        z = h * weight + bias
        dz = dout * sigmoid(z) * (1.0 + z * sigmoid(-z))
    g = (dz * weight).reshape(N, S, groups, C // groups)
    hg = h.reshape(N, S, groups, C // groups)
    dx = rstd * (g - g.mean((1, 3), keepdims=True) - hg * (g * hg).mean((1, 3), keepdims=True))
    return dx.reshape(N, S, C), (dz * h).sum((0, 1)), dz.sum((0, 1))
