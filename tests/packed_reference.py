"""64-bit definitions of the packed-batch operators, for their tests."""
import numpy as np

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def pack(grids, capacity, lead, normalized):
    offsets, image, pos = [0], [], []
    for i, (t, h, w) in enumerate(grids):
        if min(t, h, w) <= 0:
            offsets.append(offsets[-1])
            continue
        rows = [(0.0, 0.0, 0.0)] * lead
        for c in np.ndindex(t, h, w):
            rows.append(tuple((2 * a + 1 - n) / n for a, n in zip(c, (t, h, w))) if normalized
                        else tuple(float(a) for a in c))
        pos += rows
        image += [i] * len(rows)
        offsets.append(min(offsets[-1] + len(rows), capacity))
    left = capacity - len(pos)
    pos = (pos + [(0.0, 0.0, 0.0)] * max(left, 0))[:capacity]
    image = (image + [-1] * max(left, 0))[:capacity]
    return np.array(offsets), np.array(image), np.array(pos)


def pairs(head_dim, sections, pairing):
    """(axis, place within the axis, low element, high element) of each pair."""
    out, p, total = [], 0, sum(sections)
    for a, n in enumerate(sections):
        first = p
        for k in range(n):
            lo, hi = {"half": (p, p + total), "adjacent": (2 * p, 2 * p + 1),
                      "axis_half": (2 * first + k, 2 * first + k + n)}[pairing]
            out.append((a, k, lo, hi))
            p += 1
    return out


def rope(x, pos, sections, theta, pairing, inverse, shared=False, freqs=None):
    """(result, bound on what 32-bit arithmetic may be off before rounding)."""
    x, pos = np.asarray(x, np.float64), np.asarray(pos, np.float64)
    y, off = x.copy(), np.zeros_like(x)
    for p, (a, k, lo, hi) in enumerate(pairs(x.shape[-1], sections, pairing)):
        f = (freqs[p] if freqs is not None
             else theta ** (-p / sum(sections)) if shared else theta ** (-k / sections[a]))
        ang = pos[:, a] * f
        c, s = np.cos(ang)[:, None], np.sin(ang)[:, None] * (-1.0 if inverse else 1.0)
        u, v = x[..., lo], x[..., hi]
        y[..., lo], y[..., hi] = u * c - v * s, v * c + u * s
        # the reduced angle to 32 bits (2^-25 half turns = 9.4e-8), sincospif within 2 ulp
        # (1.2e-7), a product and a sum (2^-24 each); 64-bit angles add |angle| 2^-51
        b = (np.abs(u) + np.abs(v)) * (4e-7 + np.abs(ang)[:, None] * 2.0 ** -50)
        off[..., lo] = off[..., hi] = b
    return y, off


def spans(batch, tokens, offsets=None, lengths=None):
    if offsets is not None:
        return [(int(b), int(e)) for b, e in zip(offsets[:-1], offsets[1:])]
    return [(s * tokens, s * tokens + (int(lengths[s]) if lengths is not None else tokens))
            for s in range(batch)]


def attention(q, k, v, where, *, scale=0.125, last_rows=0, mask=None, prefix=None, cap=None,
              slopes=None, positions=None, probs_f16=True):
    """``q`` [rows][heads][64], ``k``/``v`` [rows][kv_heads][64] float64, NaN
    where nothing may be read. Returns (result, bound, written): the bound is
    on the error before the last rounding."""
    rows, heads = q.shape[:2]
    group = heads // k.shape[1]
    out = np.zeros((rows, heads, 64))
    off = np.zeros((rows, heads, 64))
    written = np.zeros(rows, bool)
    for s, (b, e) in enumerate(where):
        n = e - b
        first = max(0, n - last_rows) if last_rows else 0
        if n <= first:
            continue
        written[b + first:e] = True
        i, j = np.arange(first, n)[:, None], np.arange(n)[None]
        seen = np.ones((n - first, n), bool)
        if mask is not None:
            p = min(max(int(prefix[s]), 0), n) if mask == "prefix" else 0
            seen = (j <= i) | (j < p)
        for h in range(heads):
            kk, vv = k[b:e, h // group], v[b:e, h // group]
            x = scale * (q[b + first:e, h] @ kk.T)
            big = scale * (np.abs(q[b + first:e, h]) @ np.abs(kk).T)
            if cap:
                x = cap * np.tanh(x / cap)
            # a score: 64 products and sums in 32 bits; a cap: some 2^-23 of it in absolute
            # terms (two approximate functions of 2 ulp each); a distance: its product
            err = 66 * 2.0 ** -24 * big + (16 * 2.0 ** -24 * cap if cap else 0.0)
            if slopes is not None:
                if positions is not None:
                    d = positions[b + first:e, None] - positions[None, b:e]
                    far = np.sqrt((d * d).sum(-1))
                else:
                    far = np.abs(i - j).astype(float)
                x = x - slopes[h] * far
                err = err + 4 * 2.0 ** -23 * abs(slopes[h]) * far
            err = err + 2.0 ** -23 * np.abs(x) * 2 + 2.0 ** -21  # log2 units, the exponential
            x = np.where(seen, x, -np.inf)
            m = x.max(1, keepdims=True)
            # the running maximum's own rounding shifts numerator and sum alike
            p = np.exp(x - m)
            total = p.sum(1, keepdims=True)
            out[b + first:e, h] = (p / total) @ vv
            # each probability is off by its exponent's error (and the sum by as much), by a
            # rounding to f16 where the tensor cores take it (2^-11 of it, or half the least
            # f16 step where it is below the normal range), and the sums by 2^-24 a term
            w = p / total * np.where(seen, err, 0.0)
            rel = 2.0 ** -11 if probs_f16 else 0.0
            tiny = n * 2.0 ** -25 if probs_f16 else 0.0
            # an error that all probabilities share cancels; the weighted mean bounds the rest
            vmax = np.abs(vv).max(0)[None]
            off[b + first:e, h] = ((p / total) @ np.abs(vv)) * rel + vmax * (
                2 * w.sum(1, keepdims=True) + tiny + 2.0 ** -20)
    return out, off, written
