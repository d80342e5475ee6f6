"""Plain 64-bit restatement of the key/value cache and its attention (numpy, on the host), and the bound
of what an f32 / fp16 evaluation of the same formulas may be off by."""
import numpy as np

SCALE_MIN = np.float32(2.0 ** -64)


def quantize(x, half_even=False):
    """Codes (as f64) and f32 scales of the last axis; NaN scale and zero codes for rows with Inf / NaN."""
    x = np.asarray(x, np.float32)
    finite = np.isfinite(x).all(-1)
    x = np.where(finite[..., None], x, np.float32(0))
    s = np.maximum(np.abs(x).max(-1) * (np.float32(1) / np.float32(127)), SCALE_MIN).astype(np.float32)
    y = (x * (np.float32(1) / s)[..., None]).astype(np.float32).astype(np.float64)
    c = np.rint(y) if half_even else np.trunc(y + np.copysign(0.5, y))
    return np.clip(c, -127, 127), np.where(finite, s, np.float32(np.nan))


def attend(q, kc, ks, vc, vs, seen, scale, limbs, out_eps):
    """Rows q [rows, q_heads, D] (f64 values of their type) over codes kc, vc [tokens, kv_heads, D] and scales
    [tokens, kv_heads]; row r sees the first seen[r] tokens.  Returns the result and the error bound.

    The bound counts, for one row and head with p_j the probabilities and A_d = sum_j p_j |v_jd|:
      eta    the error of an exponent, natural units.  Its sum of D f32 products is off by at most (D + 8) steps of
             2^-23 (a truncating adder) of B = max_j scale sum_d |q_d k_jd|, and its logarithms, maxima and
             differences by 4 steps of 2^-23 of the largest exponent in bits, L; it acts on numerator and
             denominator: 2 eta A.  Queries kept to 22 bits add 2^-21 B.
      P      rounded to limbs * 11 bits before it meets V: half a step, 2^-11 (one limb) or 2^-22 relative, A each; and to a
             step of 2^-24 absolute below the fp16 normals, half of it at most, P being scaled by 2^8: 2^-33 of the
             largest p_j s^V_j a token, with codes up to 127.
      sums   of P over n tokens in f32, numerator and denominator: 2 (n / 8 + 64) 2^-23 A (32 tokens a step, a
             quarter of the steps a wave, joined by a few additions).
      result half a step of its type: out_eps / 2 |o|, and for fp16 half the subnormal step 2^-25."""
    rows, hq, D = q.shape
    hk = kc.shape[1]
    out, tol = np.zeros((rows, hq, D)), np.zeros((rows, hq, D))
    k, v = kc * ks[..., None].astype(np.float64), vc * vs[..., None].astype(np.float64)
    for r in range(rows):
        n = int(seen[r])
        if n <= 0:
            continue
        for g in range(hq):
            h = g // (hq // hk)
            kk, vv, s = k[:n, h], v[:n, h], vs[:n, h].astype(np.float64)
            l = kk @ q[r, g] * scale
            if not (np.isfinite(l).all() and np.isfinite(s).all()):
                out[r, g] = np.nan
                continue
            e = np.exp(l - l.max())
            p = e / e.sum()
            out[r, g] = p @ vv
            B = (np.abs(kk) @ np.abs(q[r, g])).max() * abs(scale)
            L = np.abs(l).max() * 1.4427 + np.abs(np.log2(s)).max() + 8
            eta = 2.0 ** -23 * ((D + 8) * B + 4 * L) + 2.0 ** -21 * B
            A = p @ np.abs(vv)
            P = 2.0 ** (-11 * limbs)
            sums = 2 * (n / 8 + 64) * 2.0 ** -23
            tiny = n * 2.0 ** -33 * (p * s).max() * 127 / (1 if limbs == 1 else 2.0 ** 5)
            tol[r, g] = (2 * eta + P + sums) * A + tiny + out_eps / 2 * np.abs(out[r, g]) + (2.0 ** -25 if out_eps > 1e-5 else 0)
    return out, tol
