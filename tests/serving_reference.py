"""Plain 64-bit forms of the drafted-decoding operators (numpy), for the tests."""

import numpy as np

PAGE = 64
SCALE_MIN, PEAK_MAX = 2.0**-60, 2.0**40


def quantise(x, kind):
    """(codes as the numbers they are, scales) of rows x [..., dim] (any float array), in float64."""
    x = np.asarray(x, dtype=np.float64)
    peak = np.abs(x).max(-1)
    held = np.isfinite(x).all(-1) & (peak <= PEAK_MAX)
    safe = np.where(held & (peak > 0), peak, 1.0)
    if kind == "int8":
        scale = (safe.astype(np.float32) * (np.float32(1) / np.float32(127))).astype(np.float64)
        scale = np.maximum(scale, SCALE_MIN)
        clean = np.where(held[..., None], x, 0.0)
        codes = np.clip(np.rint(clean / scale[..., None]), -127, 127)
    else:
        part, e = np.frexp(safe)  # 448 = 0.875 * 2^9
        scale = np.exp2(np.maximum(e - 9 + (part > 0.875), -60).astype(np.float64))
        codes = e4m3(np.where(held[..., None], x, 0.0) / scale[..., None])
    scale = np.where(held, np.where(peak > 0, scale, 1.0), np.nan)
    return codes, scale


def e4m3(y):
    """y rounded to the nearest e4m3 number, halves to even, saturating at 448."""
    a = np.abs(y)
    step = np.exp2(np.floor(np.log2(np.maximum(a, 2.0**-6))) - 3)
    return np.copysign(np.minimum(np.rint(a / step) * step, 448.0), y)


def attend(query, keys, codes, scales, rows, lengths, prefix, scale):
    """query [rows][heads][dim]; keys and the values' codes [prefix + sum(lengths)][kv][dim] and scales [..][kv]: the
    prefix's positions, then each sequence's. Returns the result and, for each of its elements, the sum of p |v|, the
    largest sum of |q k| and the largest p vs times the sum of the codes' sizes."""
    heads, dim = query.shape[1:]
    kv = keys.shape[1]
    out = np.zeros(query.shape)
    mass = np.zeros(query.shape)
    size = np.zeros(query.shape[:2] + (1,))
    least = np.zeros(query.shape)
    row, at = 0, prefix
    for r, t in zip(rows, lengths):
        index = np.concatenate([np.arange(prefix), np.arange(at, at + t)]).astype(int)
        for i in range(r):
            seen = index[: prefix + t - r + i + 1]
            for h in range(heads):
                j = h // (heads // kv)
                q = query[row + i, h].astype(np.float64)
                if not seen.size:
                    continue
                k, v = keys[seen, j], codes[seen, j] * scales[seen, j, None]
                with np.errstate(invalid="ignore"):
                    s = k @ q * scale
                    p = np.exp(s - s.max())
                    p /= p.sum()
                    out[row + i, h] = p @ v
                    mass[row + i, h] = p @ np.abs(v)
                    least[row + i, h] = (p * scales[seen, j]).max() * np.abs(codes[seen, j]).sum(0)
                    size[row + i, h] = (np.abs(k) @ np.abs(q)).max() * abs(scale)
        row, at = row + r, at + t
    return out, mass, size, least


def unpack(words, vocab):
    return np.unpackbits(np.ascontiguousarray(words).view(np.uint8), bitorder="little")[:vocab].astype(bool)


def verify(logits, tokens, accept, sample, q=None, counts=None, mask=None, temperature=1.0):
    """tokens [n][drafts + 1] (-1 behind the last), accepted [n]."""
    n, rows, vocab = logits.shape
    out = np.full((n, rows), -1, dtype=np.int64)
    kept = np.zeros(n, dtype=np.int64)
    for b in range(n):
        k = rows - 1 if counts is None else min(max(int(counts[b]), 0), rows - 1)
        for i in range(k + 1):
            x = logits[b, i].astype(np.float64)
            x = np.where(np.isnan(x), -np.inf, np.minimum(x, float(np.finfo(np.float32).max)))
            if mask is not None:
                allowed = unpack(mask[b, i], vocab)
                if allowed.any():
                    x = np.where(allowed, x, -np.inf)
            if x.max() == -np.inf:
                break
            last = i == k
            d = -1 if last else int(tokens[b, i])
            known = 0 <= d < vocab
            if temperature == 0:
                best = int(np.argmax(x))
                out[b, i] = best
                if last or d != best:
                    break
                kept[b] += 1
                continue
            p = np.exp((x - x.max()) / temperature)
            p /= p.sum()
            if not last and known and float(accept[b, i]) * (1.0 if q is None else float(q[b, i, d])) < p[d]:
                out[b, i] = d
                kept[b] += 1
                continue
            share = p
            if not last:
                less = np.zeros(vocab)
                if q is not None:
                    less = q[b, i].astype(np.float64)
                elif known:
                    less[d] = 1.0
                share = np.maximum(p - less, 0.0)
                if not share.sum() > 0:
                    share = p
            upto = np.cumsum(share)
            past = np.nonzero((upto > float(sample[b]) * upto[-1]) & (share > 0))[0]
            out[b, i] = past[0] if past.size else np.nonzero(share > 0)[0][-1]
            break
    return out, kept
