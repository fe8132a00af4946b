"""A cache in 4 bits in plain numpy: rounding, codes, pages, and what a page's bytes stand for."""
import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def scale_byte(block):
    """The scale's byte of 32 (or fewer) numbers."""
    if not np.isfinite(block).all():
        return 255
    top = float(np.abs(block).max())
    if top == 0.0:
        return 8
    frac, expo = np.frexp(top)                      # frac in [0.5, 1)
    e = expo - 1 - 2 + (1 if 2 * frac > 1.75 else 0)
    return int(np.clip(e, -119, 125)) + 127


def codes_of(block, byte):
    if byte == 255:
        return np.zeros(len(block), dtype=np.uint8)
    y = np.asarray(block, dtype=np.float64) / 2.0 ** (byte - 127)
    a = np.minimum(np.abs(y), 6.0)
    d = np.abs(a[:, None] - LEVELS)
    best = d.min(axis=1)
    near = d == best[:, None]
    even = near & (np.arange(8) % 2 == 0)           # a tie goes to the even code
    code = np.where(even.any(axis=1), even.argmax(axis=1), near.argmax(axis=1))
    return (code + 8 * np.signbit(y)).astype(np.uint8)


def rounded(x):
    """(codes [..., D], bytes [..., blocks], the numbers they stand for) of the last axis."""
    x = np.asarray(x)
    D, nb = x.shape[-1], -(-x.shape[-1] // 32)
    flat = x.reshape(-1, D)
    codes, scales = np.zeros(flat.shape, dtype=np.uint8), np.zeros((len(flat), nb), dtype=np.uint8)
    for r in range(len(flat)):
        for b in range(nb):
            part = flat[r, 32 * b:32 * b + 32]
            scales[r, b] = scale_byte(part)
            codes[r, 32 * b:32 * b + 32] = codes_of(part, int(scales[r, b]))
    codes, scales = codes.reshape(x.shape), scales.reshape(x.shape[:-1] + (nb,))
    return codes, scales, numbers(codes, scales)


def numbers(codes, scales):
    x = LEVELS[codes & 7] * np.where(codes & 8, -1.0, 1.0)
    byte = np.repeat(scales, 32, axis=-1)[..., :codes.shape[-1]].astype(np.float64)
    with np.errstate(over="ignore"):
        return np.where(byte == 255, np.nan, x * 2.0 ** (byte - 127))


def random_sequence(rng, n, heads, dim, spread=1.0):
    """Codes and scales as if written: a head's numbers with deviations of their own."""
    x = rng.normal(size=(n, heads, dim)) * np.exp(rng.normal(size=(1, heads, dim)) * 0.5) * spread
    return fast_rounded(x)


def fast_rounded(x):
    """``rounded`` of finite numbers of many rows at once (heads in whole blocks or not)."""
    D, nb = x.shape[-1], -(-x.shape[-1] // 32)
    pad = np.zeros(x.shape[:-1] + (nb * 32,))
    pad[..., :D] = x
    blocks = pad.reshape(x.shape[:-1] + (nb, 32))
    frac, expo = np.frexp(np.abs(blocks).max(-1))
    byte = np.clip(expo - 3 + (2 * frac > 1.75), -119, 125).astype(np.int64) + 127
    byte = np.where(frac == 0, 8, byte)
    y = blocks / 2.0 ** (byte[..., None] - 127.0)
    a = np.abs(y)
    code = ((a > 0.25).astype(np.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).astype(np.uint8)
    code = (code + 8 * np.signbit(y)).astype(np.uint8).reshape(pad.shape)[..., :D]
    scales = byte.astype(np.uint8)
    return code, scales, numbers(code, scales)


def fill_pages(seqs, tables, n_pages, page, values, junk=None):
    """Page bytes ``(codes, scales)`` that hold ``seqs[b] = (codes, scales, _)`` of every request under its table; ``junk``: a generator whose bytes
    stand wherever nothing was written."""
    heads, D = seqs[0][0].shape[1:]
    nb = -(-D // 32)
    cshape = (n_pages, heads, page // 8, D // 2, 8) if values else (n_pages, heads, page, D // 2)
    sshape = (n_pages, heads, page // 8, nb, 8)
    codes, scales = ((junk.integers(0, 256, size=s, dtype=np.uint8) if junk is not None else np.zeros(s, dtype=np.uint8)) for s in (cshape, sshape))
    for (c, s, _), table in zip(seqs, tables):
        for i in range(len(c)):
            p, off = table[i // page], i % page
            if p < 0:
                continue
            both = c[i, :, 0::2] | (c[i, :, 1::2] << 4)
            if values:
                codes[p, :, off // 8, :, off % 8] = both
            else:
                codes[p, :, off] = both
            scales[p, :, off // 8, :, off % 8] = s[i]
    return codes, scales


def pages_rows(codes, scales, table, positions, page, values):
    """Numbers ``[n, heads, D]`` of a request's positions."""
    out = []
    for pos in positions:
        p, off = table[pos // page], pos % page
        both = codes[p, :, off // 8, :, off % 8] if values else codes[p, :, off]
        c = np.stack([both & 15, both >> 4], axis=-1).reshape(both.shape[0], -1)
        out.append(numbers(c, scales[p, :, off // 8, :, off % 8]))
    return np.stack(out)
