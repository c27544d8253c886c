"""64-bit restatement (numpy) of the decoding operators of pero_ocr_amd/decode_ops.py, with bounds on what 32-bit sums may be off by.
Test infrastructure only."""
import math

import numpy as np

U32 = 2.0 ** -24            # half a step of float32, relative
HALF_STEP = {"fp32": 2.0 ** -24, "bf16": 2.0 ** -8, "fp16": 2.0 ** -11}      # the same of an output's type


def round_to(x, bits, min_exp):
    """float64 -> nearest value with `bits` significant bits (ties to even), fixed point below 2 ** min_exp"""
    x = np.asarray(x, np.float64)
    m, e = np.frexp(np.where(np.isfinite(x), np.abs(x), 0.0))
    step = np.ldexp(1.0, np.maximum(e - 1, min_exp) - (bits - 1))
    with np.errstate(invalid="ignore"):
        return np.where(np.isfinite(x), np.rint(x / step) * step, x)


def quantise_rows(x):
    """[..., D] -> (e4m3 codes as float64, exponents): the smallest power of two that brings the largest finite |value| within 448"""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x)
    big = np.where(fine, np.abs(x), 0.0).max(-1)
    exp = np.full(big.shape, 27, np.int64)
    for i in np.ndindex(big.shape):
        while big[i] > 448 * 2.0 ** (exp[i] - 127):
            exp[i] += 1
    y = np.where(fine, x, 0.0) / (2.0 ** (exp - 127.0))[..., None]
    return np.where(fine, round_to(y, 4, -6), np.nan), exp


def cache_values(codes, exp):
    """the numbers a cache's rows stand for"""
    codes = np.asarray(codes, np.float64)
    return codes if exp is None else codes * (2.0 ** (np.asarray(exp, np.float64) - 127))[..., None]


def visible(i, n, length, mask_row):
    """which of the `length` positions new token i of n sees (mask_row: list of 64-bit words as Python ints, or None)"""
    out = np.zeros(length, bool)
    for j in range(length):
        d = j - (length - n)
        out[j] = d < 0 or (d <= i if mask_row is None else (d // 64 < len(mask_row) and bool(mask_row[d // 64] >> (d % 64) & 1)))
    return out


def attention(q, k, v, table, lengths, starts, mask=None, scale=None, out_type="fp32", planes=2.0 ** -24):
    """q [T][H][D]; k, v: the cache's values [pages][Hk][P][D] -> out, lse and how far each may be off: tol [T][H][D], lse_tol [T][H].

    With u = 2^-24, D-term dot products in 32 bits are off by at most D u sum|q_d k_d| scale =: ds; the exponent's argument and exp add
    4 u (1 + max|s - m|); the L-term sums add 2 L u; the probabilities enter the second product rounded by `planes`; the result is
    rounded to its type once.  Errors of p count twice in sum p v / sum p."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    T, H, D = q.shape
    pages, hk, P, _ = k.shape
    scale = D ** -0.5 if scale is None else scale
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    lse, lse_tol = np.full((T, H), -math.inf), np.zeros((T, H))
    for s in range(len(lengths)):
        a, b = int(starts[s]), int(starts[s + 1])
        n, length = b - a, int(min(max(lengths[s], 0), len(table[s]) * P))
        ids = [int(table[s][j // P]) for j in range(length)]
        there = np.array([0 <= p < pages for p in ids], bool)
        at = np.array([(p if t else 0) for p, t in zip(ids, there)], int), np.arange(length) % P
        for i in range(n):
            see = visible(i, n, length, None if mask is None else [int(w) & (1 << 64) - 1 for w in mask[a + i]]) & there
            if not see.any():
                continue
            for h in range(H):
                kk, vv = (t[at[0][see], h // (H // hk), at[1][see]] for t in (k, v))
                with np.errstate(all="ignore"):
                    sc = kk @ q[a + i, h] * scale
                    m = sc.max()
                    p = np.exp(sc - m)
                    z = p.sum()
                    out[a + i, h] = (p @ vv) / z
                    lse[a + i, h] = m + math.log(z)
                    ds = D * U32 * (np.abs(kk) @ np.abs(q[a + i, h])).max() * abs(scale)
                    ep = ds + 4 * U32 * (1 + np.abs(sc - m).max())
                    o = (p @ np.abs(vv)) / z
                    tol[a + i, h] = (2 * ep + 2 * len(p) * U32 + planes) * o + HALF_STEP[out_type] * np.abs(out[a + i, h]) + 1e-30
                    lse_tol[a + i, h] = ep + ds + len(p) * U32 + 4 * U32 * (1 + abs(lse[a + i, h]) + abs(m))
    return out, lse, tol, lse_tol


def logprobs(x, tokens, top):
    """[R][C], [R][g] -> logprob, entropy, top_logprob, top_index, and how far logprob and entropy of a row may be off (a logprob by
    another 4 u of itself).

    u = 2^-24: a term exp(d) is off by 2 u (1 + |d|) of itself, so the sums by 2 u (1 + E|d|) of Z plus C / 64 + 16 additions in a row; log Z
    by that and 2 u of itself; the two subtractions by u of their results."""
    x = np.asarray(x, np.float64)
    R, C = x.shape
    lp, ent = np.zeros(tokens.shape), np.zeros(R)
    tlp, tid = np.zeros((R, top)), np.zeros((R, top), np.int64)
    lp_tol, ent_tol = np.zeros(R), np.zeros(R)
    adds = C / 64 + 16
    for r in range(R):
        row = x[r]
        key = np.where(np.isnan(row), np.inf, row)
        order = np.lexsort((np.arange(C), -key, ~np.isnan(row)))[:top]
        tid[r] = order
        with np.errstate(all="ignore"):
            m = np.nan if np.isnan(row).any() else row.max()
            if m == -math.inf:
                logp = np.full(C, -math.inf)
                ent[r] = 0.0
            else:
                d = row - m
                p = np.exp(d)
                z = p.sum()
                logp = d - np.log(z)
                w = np.where(p > 0, p * d, 0.0) / z
                ent[r] = np.log(z) - w.sum()
                spread = np.abs(w).sum()
                if np.isfinite(z):
                    lp_tol[r] = U32 * (adds + 2 * (1 + spread) + 4 * abs(math.log(z)))
                    ent_tol[r] = U32 * ((adds + 2 * (1 + spread)) * (1 + spread) + 2 * np.abs(w * d)[p > 0].sum() + 4 * (math.log(z) + spread) + 2)
        tlp[r] = logp[order]
        for g in range(tokens.shape[1]):
            t = int(tokens[r, g])
            lp[r, g] = 0.0 if t < 0 else (np.nan if t >= C else logp[t])
    beyond = float(np.finfo(np.float32).max)
    lp, tlp = (np.where(t < -beyond, -math.inf, t) for t in (lp, tlp))          # (what float32 holds of them)
    return lp, ent, tlp, tid, lp_tol, ent_tol
