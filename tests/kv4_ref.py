"""The 4-bit KV cache, its attention and beam search's selection from their
definitions (include/g4cuda.h), in 64 bits on the CPU: what the GPU tests
compare with. Plain numpy, no code of the library."""
import numpy as np

REC, GROUP = 16, 64


def bf16(x):
    """Non-negative float64 -> the nearest bf16 value, ties to even."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(m * 256), e - 8)


def bf16_bits(x):
    return (np.asarray(x, np.float64).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16)


def quantise(x):
    """x[..., hd] (float64) -> codes [..., hd] and scales [..., hd / 64]."""
    y = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, GROUP)
    amax = np.max(np.abs(y), -1)
    bad = ~np.isfinite(amax) | (amax >= 2.0 ** 127)
    s = np.where(bad, np.nan, np.where(amax < 2.0 ** -100, 0, bf16(np.where(bad, 1, amax) / 7)))
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s[..., None] > 0, np.clip(np.rint(y / s[..., None]), -7, 7), 0)
    return c.reshape(x.shape).astype(np.int64), s


def stored(x):
    """The values that x's codes stand for, float64."""
    c, s = quantise(x)
    return c * np.repeat(s, GROUP, -1)


class Cache:
    """A pool of pages on the CPU: [pages][kv][page / 16][17 * hd] bytes."""

    def __init__(self, pages, page, kv, hd, fill=0xFF):
        self.page, self.kv, self.hd = page, kv, hd
        self.bytes = np.full((pages, kv, page // REC, 17 * hd), fill, np.uint8)

    def put(self, page, slot, h, k, v):
        """One token's key and value of head h."""
        rec, t, hd = self.bytes[page, h, slot // REC], slot % REC, self.hd
        g = hd // GROUP
        for x, at, unit, place in ((k, 0, 16, lambda u: (t & 7) * 64 + u * 16 + (t >> 3) * 8),
                                   (v, 8 * hd, 8, lambda u: u * 64 + (t >> 1 & 3) * 16 + (t >> 3) * 8 + (t & 1) * 4)):
            c, s = quantise(x)
            n = (c + 8).astype(np.uint8)
            for grp in range(g):
                for u in range(GROUP // unit):
                    d = n[grp * GROUP + u * unit:grp * GROUP + (u + 1) * unit]
                    o = at + grp * 512 + place(u)
                    rec[o:o + unit // 2] = d[0::2] | (d[1::2] << 4)
                bits = 0x7fc0 if np.isnan(s[grp]) else bf16_bits(s[grp])
                o = 16 * hd + 2 * (t * g + grp) if at == 0 else \
                    16 * hd + 32 * g + 2 * (grp * 16 + (t >> 1 & 3) * 4 + (t >> 3) * 2 + (t & 1))
                rec[o:o + 2] = np.array([bits], np.uint16).view(np.uint8)


def attention(q, keys, values, pos, scale, window):
    """One row: q[heads, hd], keys / values [n, kv, hd] (float64) with NaN rows
    for tokens that are not there; returns out[heads, hd] and what the error
    bound of `tolerance` needs."""
    heads, hd = q.shape
    kv = keys.shape[1] if keys.ndim == 3 else 1
    out = np.zeros((heads, hd))
    mag = np.zeros((heads, hd))          # sum of p |v|, and 2^-18 of the sum of |v| (see `tolerance`)
    first = max(0, pos - window + 1) if window else 0
    last = min(pos, keys.shape[0] - 1)
    if last < first:
        return out, mag, np.zeros(heads), 0
    k, v = keys[first:last + 1], values[first:last + 1]
    there = ~np.isnan(k[:, 0, 0])
    k, v = k[there], v[there]
    if not len(k):
        return out, mag, np.zeros(heads), 0
    delta = np.zeros(heads)
    for h in range(heads):
        j = h * kv // heads
        s = scale * (k[:, j] @ q[h])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[h] = p @ v[:, j]
        mag[h] = p @ np.abs(v[:, j]) + 2.0 ** -18 * np.abs(v[:, j]).sum(0)
        # |q| against the largest code and the offset of the unsigned ones: 15 scales
        top = np.abs(k[:, j]).reshape(len(k), -1, GROUP).max(-1) / 7 * 15
        delta[h] = abs(scale) * (np.repeat(top, GROUP, -1) @ np.abs(q[h])).max()
    return out, mag, delta, len(k)


def tolerance(out, mag, delta, n, eps):
    """How far the kernel may be from `out`. Scores: q keeps 22 bits (2^-22), a
    group of 64 dimensions is up to 8 tensor-core steps that may truncate at
    fp32 (8 * 2^-23), 8 groups are added: below 2^-19 of the sum of magnitudes
    `delta`; a probability moves by that much, its sum too (factor 2). Each
    probability keeps 16 bits (high and low parts: 2^-17), exp2 and its
    argument 2^-20: together below 2^-15. In fp16 parts of 2^14 p, taken from a
    reference up to 2^6 above the largest, the step is 2^-24 at least: an error of
    2^-25 2^-14 2^6 = 2^-33 per key however small p is, 2^-15 of the 2^-18 sum |v|
    that `mag` holds. Sums over n keys add 2^-23 each.
    The result is rounded once: eps / 2."""
    return mag * (2 * 2.0 ** -19 * delta[:, None] + 2.0 ** -15 + n * 2.0 ** -23) + np.abs(out) * eps / 2 * 1.01 + 1e-30


def beam(logits, scores, finished, eos):
    """One group: logits[beams, vocab] (float64), -> scores, parents, tokens, finished."""
    w, vocab = logits.shape
    x = np.where(np.isnan(logits), -np.inf, logits)
    cand = np.full((w, vocab), -np.inf)
    for b in range(w):
        if not np.isfinite(scores[b]):
            continue
        if finished is not None and finished[b]:
            cand[b, eos] = scores[b]
            continue
        m = x[b].max()
        if np.isfinite(m):
            cand[b] = scores[b] + (x[b] - (m + np.log(np.exp(x[b] - m).sum())))
    at = np.lexsort((np.arange(w * vocab), -cand.ravel()))[:w]
    parents, tokens = at // vocab, at % vocab
    ended = np.array([(finished is not None and bool(finished[p])) or t == eos for p, t in zip(parents, tokens)])
    return cand.ravel()[at], parents, tokens, ended
