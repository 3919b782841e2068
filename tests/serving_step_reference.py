"""The calls of a serving step over several sequences (packed attention, the int8 block cache, logit rules) in 64 bits, with the
bounds that their results may be off by."""
import numpy as np

HALF_STEP = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}


def attend(q, k, v, limits, scale, dtype, weight_half):
    """Rows q [m, dim] over k [n, dim] and v [n, vdim], row i seeing keys [0, limits[i]). Returns the result and how far a kernel may be from it:

      half a step of the stored type, relative to the value;
      weights: each is off by its rounding to the products' type (weight_half) and by its score's error;
      scores: a dot product of dim terms in f32 is off by (dim + 4) 2^-24 sum |q k| (products, sums, scale, maximum), and twice that
        moves a weight against the sum of weights;
      exponentials and sums in f32: 2^-21 for 2^x and its rescaling, n 2^-24 for the sum over n keys.
    All errors of weights apply to sum w |v|. Weights below the smallest normal f16 (2^-14 of a maximum of at least 2^-8) are off by 2^-25 of the
    largest weight each. A tenth more covers products of errors.
    """
    m, n = q.shape[0], k.shape[0]
    out, off = np.zeros((m, v.shape[1])), np.zeros((m, v.shape[1]))
    for i in range(m):
        e = min(int(limits[i]), n)
        if e <= 0:
            continue
        s = k[:e] @ q[i] * scale
        if np.max(s) == -np.inf:
            continue
        w = np.exp(s - np.max(s))
        total = w.sum()
        out[i] = w @ v[:e] / total
        spread = (q.shape[1] + 4) * 2.0 ** -24 * np.max(np.abs(k[:e]) @ np.abs(q[i])) * scale
        each = weight_half + 2 * spread + 2.0 ** -21 + e * 2.0 ** -24
        tiny = 2.0 ** -16 * np.abs(v[:e]).sum(0) / total * (2.0 ** -9 if dtype != "bf16" else 0.0)
        off[i] = 1.1 * (HALF_STEP[dtype] * np.abs(out[i]) + each * (w @ np.abs(v[:e])) / total + tiny) + 1e-30
    return out, off


def encode(x, scale):
    """Codes of x under the f32 `scale`: the nearest integer, ties to even."""
    if scale == 0:
        return np.zeros(x.shape, dtype=np.int8)
    with np.errstate(invalid="ignore"):
        c = np.clip(np.rint(x.astype(np.float64) / np.float64(scale)), -127, 127)
    return np.where(np.isnan(c), 0, c).astype(np.int8)


def write_plane(x, codes, scales, starts, lengths, table, block):
    """New rows x [rows, kv_heads, dim] into codes [blocks, kv_heads, block, dim] and scales [blocks, kv_heads], in place."""
    for s in range(len(lengths)):
        n = int(lengths[s])
        first = n - int(starts[s + 1] - starts[s])
        if first == n:
            continue
        for j in range(first // block, -(-n // block)):
            b, lo, hi = int(table[s, j]), max(first, j * block) - j * block, min(n, (j + 1) * block) - j * block
            at = int(starts[s]) + j * block + lo - first
            for h in range(x.shape[1]):
                new = x[at:at + hi - lo, h].astype(np.float32)
                size = np.abs(new[np.isfinite(new)])
                now = np.float32(np.float64(size.max() if size.size else 0.0) / 127.0)
                if lo:
                    before = scales[b, h]
                    now = max(now, before)
                    if now > before:
                        codes[b, h, :lo] = encode(codes[b, h, :lo].astype(np.float64) * np.float64(before), now)
                codes[b, h, lo:hi] = encode(new, now)
                scales[b, h] = now


def rules(z, history, spans, params, bias, allowed):
    """One row of logits: history a list, spans (prompt, total), params (repetition, presence, frequency, temperature), bias a list of
    (token, value), allowed a truth value per token or None. Also how far f32 may be off: 2^-24 of every intermediate value, seven roundings."""
    z = z.astype(np.float64).copy()
    size = np.abs(z)
    again, presence, frequency, temperature = (float(p) for p in params)
    prompt, total = spans
    count, seen = np.zeros(z.size), np.zeros(z.size, dtype=bool)
    for i, t in enumerate(history[:total]):
        if 0 <= t < z.size:
            seen[t] = True
            count[t] += i >= prompt
    z = np.where(seen, np.where(z > 0, z / again, z * again), z)
    size = np.maximum(size, np.abs(z))
    z = z - np.where(count > 0, frequency * count + presence, 0.0)
    size = np.maximum(size, np.abs(z)) + np.where(count > 0, np.abs(frequency) * count + np.abs(presence), 0.0)
    values = {}
    for t, b in bias:
        if 0 <= t < z.size:
            values[t] = float(b)
    for t, b in values.items():
        z[t] += b
        size[t] += abs(b)
    if temperature > 0:
        z, size = z / temperature, size / temperature
    if allowed is not None:
        z = np.where(allowed, z, -np.inf)
    return z, 7 * 2.0 ** -24 * size
