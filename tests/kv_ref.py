"""The quantized key/value cache in numpy: ggml's conversions, the cache's
bytes as include/s3e.h documents them, and attention in 64 bits."""
import numpy as np

Q4_0, Q8_0 = 2, 8


def quantize(t, x):
    """Rows [..., D] of f32 → codes (uint8 0..15 or int8) of that shape and the scales [..., D/32] as fp16 bits."""
    x = np.asarray(x, np.float32)
    b = x.reshape(*x.shape[:-1], -1, 32)
    a = np.abs(b)
    bad = ~np.isfinite(b).all(-1)
    with np.errstate(all="ignore"):
        if t == Q4_0:
            lead = np.take_along_axis(b, a.argmax(-1)[..., None], -1)[..., 0]  # argmax: the first of equals
            lead = np.where(lead == 0, np.float32(0), lead)  # of a block of zeros, -0 too, ggml's scale is 0 / -8
            d = (lead / np.float32(-8)).astype(np.float32)
            inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
        else:
            top = a.max(-1)
            d = (top / np.float32(127)).astype(np.float32)
            inv = np.where(top > 0, np.float32(127) / top, np.float32(0)).astype(np.float32)
        inv = np.where(bad | ~np.isfinite(inv), np.float32(0), inv)
        y = np.where(bad[..., None], np.float32(0), b * inv[..., None]).astype(np.float32)
        if t == Q4_0:
            q = np.minimum(15, np.floor((y + np.float32(8.5)).astype(np.float32))).astype(np.uint8)
        else:
            q = np.rint(y).astype(np.int8)
        d16 = np.where(bad, np.float16(np.nan), d.astype(np.float16)).view(np.uint16)
    d16 = np.where(bad, np.uint16(0x7E00), d16).astype(np.uint16)
    return q.reshape(x.shape), d16


def values(t, q, d16):
    """float64 values of codes and scale bits."""
    c = q.astype(np.float64) - (8 if t == Q4_0 else 0)
    with np.errstate(all="ignore"):
        v = c.reshape(*d16.shape, 32) * d16.view(np.float16).astype(np.float64)[..., None]
    return v.reshape(q.shape)


def chunk_bytes(t, D):
    return (36 if t == Q4_0 else 68) * D


def _word_at(t, NB, w, lane):
    B = 4 if t == Q4_0 else 8
    per = 16 // B
    p = w // per
    width = min(per, 2 * NB - p * per)
    return p * per * 64 * B + (lane * width + w % per) * B


def place(t, D, page, heads, slot, head, tensor, ch):
    """(byte offset of the code, nibble shift or None, byte offset of its scale) in the cache's memory."""
    NB, ck = D // 32, chunk_bytes(t, D)
    codes = 64 * 2 * NB * (4 if t == Q4_0 else 8)
    base = (((slot // page) * heads + head) * (page // 32) + slot % page // 32) * ck + tensor * (ck // 2)
    key = slot % 32
    if tensor == 0:
        b, g, j = ch // 32, ch % 32 // 8, ch % 8
        a, tt, i = key // 8, key % 8 // 4, key % 4
        at = base + _word_at(t, NB, tt * NB + b, 16 * g + 4 * a + i)
    else:
        j = key % 8
        at = base + _word_at(t, NB, ch // 16, 16 * (key // 8) + ch % 16)
    scale = base + codes + (ch // 32 * 32 + key) * 2
    if t == Q8_0:
        return at + j, None, scale
    n = (j >> 1) + 4 * (j & 1)
    return at + n // 2, 4 * (n & 1), scale


def write(mem, t, D, page, heads, slots, k, v):
    """Rows k, v [n][heads][D] (f32) into the cache's bytes, row by row; rows whose slot the cache lacks are left out."""
    total = len(mem) * 8 // (heads * D * (9 if t == Q4_0 else 17))
    for tensor, x in enumerate((k, v)):
        q, d = quantize(t, x)
        for r, s in enumerate(slots):
            if not 0 <= s < total:
                continue
            for h in range(heads):
                for ch in range(D):
                    at, shift, scale = place(t, D, page, heads, int(s), h, tensor, ch)
                    c = int(q[r, h, ch])
                    if shift is None:
                        mem[at] = c & 0xFF
                    else:
                        mem[at] = (int(mem[at]) & ~(15 << shift) & 0xFF) | (c << shift)
                    if ch % 32 == 0:
                        mem[scale], mem[scale + 1] = int(d[r, h, ch // 32]) & 0xFF, int(d[r, h, ch // 32]) >> 8


def attention(t, kq, kd, vq, vd, q, scale, see, mask=None):
    """One sequence: codes and scale bits [len][heads][..], q [nq][nh][D], see [nq][len] bool.  → (o, bound) float64,
    where bound is, per output value, Σ p·|v| and A, per row, the largest Σ|q·k|·scale of a seen key."""
    K, V = values(t, kq, kd), values(t, vq, vd)
    nq, nh, D = q.shape
    G = nh // K.shape[1] if K.shape[0] else 1
    o, mag, A = np.zeros((nq, nh, D)), np.zeros((nq, nh, D)), np.zeros((nq, nh))
    for h in range(nh):
        for i in range(nq):
            use = see[i].copy()
            if mask is not None:
                use &= ~np.isneginf(mask[i])
            if not use.any():
                continue
            k, v = K[use, h // G], V[use, h // G]
            qi = q[i, h].astype(np.float64)
            s = k @ qi * scale
            A[i, h] = (np.abs(k) @ np.abs(qi)).max() * abs(scale)
            if mask is not None:
                s = s + mask[i][use].astype(np.float64)
                A[i, h] = max(A[i, h], np.abs(s).max())
            p = np.exp(s - s.max())
            p /= p.sum()
            o[i, h], mag[i, h] = p @ v, p @ np.abs(v)
    return o, mag, A


def largest(t, vq, vd):
    """V's largest finite magnitude."""
    v = np.abs(values(t, vq, vd))
    return v[np.isfinite(v)].max(initial=0)


def attention_bound(f32, o, mag, A, n_keys, D, vmax):
    """How far a result may be off, value by value, from the roundings the operator makes (u = 2^-24):
    F16: the output's rounding to fp16 (2^-11) and each P·d's (2^-11);
    F32: pairs of fp16 carry 22 bits: 2^-22 of q and of P·d, and the output's own u.
    Either way a P·d below fp16's normal numbers is off by up to 2^-25, in units where the largest weight (at most 1)
    times 2^ed, the power of two above V's largest scale, is 2^7: times the code that is at most
    2^-25 · 2^-7 · 2·d_max · |code| a key, and d_max times the largest code is V's largest value: 2^-31 of that a key.
    Both: scores are sums of D products in fp32, scaled (D + 4 roundings of at most A·u each), their exponential's
    argument and result (4u·A + 4u), and sums over the keys in fp32 (one rounding a key and lane, at most n/16 + 64)."""
    u = 2.0 ** -24
    score = (D + 8) * u * A + (A * 2.0 ** -22 if f32 else 0)
    rel = 2 * score + 8 * u + (n_keys / 16 + 64) * u + (2.0 ** -22 if f32 else 2.0 ** -11)
    return mag * rel[..., None] + n_keys * 2.0 ** -31 * vmax + np.abs(o) * (u if f32 else 2.0 ** -11) + (1e-38 if f32 else 2.0 ** -25)
