"""Plain 64-bit restatement of rotary positions, head norms, the 4-bit cache's rows and a serving step's tables (numpy, on the
host), with the bounds of what an f32 evaluation may be off by."""
import math

import numpy as np

SCALE_MIN = np.float32(2.0 ** -64)


# ------------------------------------------------------------------ rotary positions, norms


def frequencies(n, base, scaling="plain", factor=1.0, original=0.0, low=0.0, high=0.0):
    """Radians a position adds to each of n / 2 pairs, and the amplitude."""
    if scaling == "base" and n > 2:
        base = base * factor ** (n / (n - 2))
    out = []
    for i in range(n // 2):
        w = base ** (-2 * i / n)
        if scaling == "linear":
            w /= factor
        elif scaling == "bands":
            wave = 2 * math.pi / w
            if wave > original / low:
                w /= factor
            elif wave > original / high:
                t = (original / wave - low) / (high - low)
                w = (1 - t) * w / factor + t * w
        elif scaling == "ramp":
            pair = lambda turns: n * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
            a, b = max(math.floor(pair(high)), 0), min(math.ceil(pair(low)), n - 1)
            t = min(max((i - a) / max(b - a, 0.001), 0), 1)
            w = w / factor * t + w * (1 - t)
        out.append(w)
    return np.array(out), 0.1 * math.log(factor) + 1 if scaling == "ramp" else 1.0


def pairs(first, n, layout):
    i = np.arange(n // 2)
    return (first + i, first + n // 2 + i) if layout == "half" else (first + 2 * i, first + 2 * i + 1)


def rotate(x, positions, w, amplitude, left, right, inverse=False):
    """x [rows, heads, dim] f64; the result, and how far the cosines and sines of an f32 evaluation may be off at most.

    The angle in quarter turns, position * (w 2 / pi), is off by two roundings of 2^-53 in 64 bits; its fraction is rounded to
    f32 (below a half: 2^-26); the series of its sine and cosine add a rounding or two of 2^-24 a step, of terms that fall off by a factor
    of 3 and more, and end at 2e-9: 4 * 2^-24 in all.  The amplitude is rounded to f32 and multiplied: 2 * 2^-24 of it."""
    t = positions.astype(np.float64)[:, None] * w
    # the reference's own reduction: in long double where numpy has it
    t = np.asarray(np.fmod(positions.astype(np.longdouble)[:, None] * w.astype(np.longdouble), 2 * np.pi * np.longdouble(1)), np.float64) if \
        np.finfo(np.longdouble).nmant > 60 and np.abs(t).max(initial=0) < 1e5 else t
    c, s = (amplitude * f(t)[:, None] for f in (np.cos, np.sin))
    if inverse:
        s = -s
    y = x.copy()
    y[..., left], y[..., right] = x[..., left] * c - x[..., right] * s, x[..., right] * c + x[..., left] * s
    off = amplitude * (np.pi / 2 * (2.0 ** -26 + np.abs(positions).max(initial=0) * w.max(initial=0) * 2.0 ** -51) + 6 * 2.0 ** -24)
    return y, off


def norm(x, gamma, eps):
    return x if gamma is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * np.asarray(gamma, np.float64)


# An f32 norm: the sum of D squares a lane of 8 at a time and then pairwise is off by 8 + 6 roundings of 2^-24, its mean and eps by 2
# more, the root halves that, the reciprocal root is good to 2^-23, and two products round: (16 / 2 + 2 + 2) 2^-24.
NORM = 12 * 2.0 ** -24


def heads(x, positions, q_heads, q_gamma, k_gamma, eps, w, amplitude, left, right, out_eps, inverse=False):
    """Norm and rotation of rows x [rows, heads, dim], and the bound of what a result of a type may be off by."""
    n = np.concatenate([norm(x[:, :q_heads], q_gamma, eps), norm(x[:, q_heads:], k_gamma, eps)], 1)
    # the angle's own error in this restatement is one rounding of position * w in 64 bits, within what rotate counts
    y, off = rotate(n, positions, w, amplitude, left, right, inverse)
    size = np.abs(n)
    both = np.zeros_like(size)
    both[..., left] = both[..., right] = size[..., left] + size[..., right]
    normed = np.zeros(x.shape[1], bool)
    normed[:q_heads], normed[q_heads:] = q_gamma is not None, k_gamma is not None
    # the products and their sum round twice: 2 * 2^-24 of |l| + |r|
    tol = (off + 2 * 2.0 ** -24 + amplitude * NORM * normed[None, :, None]) * both
    still = both == 0
    tol = np.where(still, NORM * normed[None, :, None] * size, tol)
    return y, tol + out_eps / 2 * np.abs(y) + (2.0 ** -25 if out_eps > 1e-5 else 2.0 ** -149)


# ------------------------------------------------------------------ rows in 4 bits


def quantize4(x, half_even=False):
    """Codes times units (f64, whole numbers) and f32 scales of the last axis; NaN scale and zeros for rows with Inf / NaN."""
    x = np.asarray(x, np.float32)
    finite = np.isfinite(x).all(-1)
    x = np.where(finite[..., None], x, np.float32(0))
    s = np.maximum(np.abs(x).max(-1) * (np.float32(1) / np.float32(1785)), SCALE_MIN).astype(np.float32)
    out = np.zeros(x.shape)
    for g in range(0, x.shape[-1], 32):
        y = x[..., g:g + 32]
        u = np.ceil(np.abs(y).max(-1) * (np.float32(1) / s) * (np.float32(1) / np.float32(7)))
        u = np.clip(u, 1, 255).astype(np.float32)
        y = (y * (np.float32(1) / (u * s))[..., None]).astype(np.float32).astype(np.float64)
        c = np.rint(y) if half_even else np.trunc(y + np.copysign(0.5, y))
        out[..., g:g + 32] = np.clip(c, -7, 7) * u[..., None]
    return out, np.where(finite, s, np.float32(np.nan))


# ------------------------------------------------------------------ a serving step's tables


def step(change, length, table, free, page, pages, rows, max_new, max_len, prefix=0):
    """One step on lists: new lengths, table and free list (its free part), row starts, (slot, position, page slot) of the rows, refused."""
    shared = prefix // page
    length, table, free = list(length), [list(t) for t in table], list(free)
    held = [max(-(-n // page), shared) for n in length]
    for i, c in enumerate(change):
        if c < 0:
            length[i] = max(length[i] + c, 0)
            keep = max(-(-length[i] // page), shared)
            for j in range(keep, held[i]):
                free.append(table[i][j])
                table[i][j] = -1
    starts, maps, refused, asked_rows, asked_pages, stock = [0], [], 0, 0, 0, len(free)
    for i, c in enumerate(change):
        n = max(c, 0)
        if n > max_new or length[i] + n > max_len or n > rows:
            n = 0
        asked_rows += n
        if asked_rows > rows:
            n = 0
        need = max(-(-(length[i] + n) // page), shared) - held[i] if n else 0
        asked_pages += need
        if need and asked_pages > stock:
            n = need = 0
        refused += c > 0 and n == 0
        for j in range(need):
            table[i][held[i] + j] = free.pop()
        for p in range(length[i], length[i] + n):
            maps.append((i, p, table[i][p // page] * page + p % page))
        length[i] += n
        starts.append(starts[-1] + n)
    return length, table, free, starts, maps, refused
