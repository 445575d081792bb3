"""Plain 64-bit attention sublayer (numpy) for the tests: per-head norms and
rotation, the 16-token-block 8-bit cache, and grouped-query attention over it."""
import numpy as np

BLOCK = 16
TINY = np.float32(1e-20)


def norm_rope(x, w, pos, rope_dim, interleaved, theta=None, eps=0.0, mscale=1.0, inv_freq=None):
    """x [T, heads, D] at positions pos [T] -> float64."""
    y = np.asarray(x, dtype=np.float64)
    if w is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * np.asarray(w, dtype=np.float64)
    y = y.copy()
    if rope_dim:
        i = np.arange(rope_dim // 2)
        f = np.asarray(inv_freq, dtype=np.float64) if inv_freq is not None else float(theta) ** (-2.0 * i / rope_dim)
        angle = np.asarray(pos, dtype=np.float64)[:, None] * f
        c, s = np.cos(angle)[:, None] * mscale, np.sin(angle)[:, None] * mscale
        ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rope_dim // 2)
        a, b = y[..., ia].copy(), y[..., ib].copy()
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def quantise(block):
    """block [16, D] f32 -> (int8 [16, D], f32 scale)."""
    x = np.asarray(block, dtype=np.float32)
    fin = np.isfinite(x)
    amax = np.max(np.abs(x[fin]), initial=np.float32(0))
    if not amax >= TINY:
        return np.zeros(x.shape, np.int8), np.float32(0)
    s = np.float32(np.float64(amax) / 127.0)
    with np.errstate(invalid="ignore", over="ignore"):
        q = np.rint(np.where(fin, x.astype(np.float64) / np.float64(s), 0.0))
    q = np.where(np.isposinf(x), 127, np.where(np.isneginf(x), -127, q))
    return q.astype(np.int8), s


class Cache:
    """Sequences' keys and values in f32, quantised by blocks when read."""

    def __init__(self):
        self.k, self.v = {}, {}     # slot -> [n, heads, D] f32

    def append(self, slot, past, k, v):
        for store, x in ((self.k, k), (self.v, v)):
            x = np.asarray(x, dtype=np.float32)
            old = store.get(slot)
            store[slot] = x if old is None else np.concatenate((old[:past], x))

    def blocks(self, slot, which):
        """(q [heads, blocks, 16, D], s [heads, blocks]) of a slot's tokens."""
        x = (self.k if which == "k" else self.v)[slot]
        n, heads, D = x.shape
        nb = -(-n // BLOCK)
        pad = np.zeros((nb * BLOCK, heads, D), np.float32)
        pad[:n] = x
        q, s = np.zeros((heads, nb, BLOCK, D), np.int8), np.zeros((heads, nb), np.float32)
        for h in range(heads):
            for b in range(nb):
                q[h, b], s[h, b] = quantise(pad[b * BLOCK:(b + 1) * BLOCK, h])
        return q, s


def attend(q, kq, ks, vq, vs, past, scale, window, bad=()):
    """q [n, q_heads, D] over quantised blocks (as Cache.blocks): out [n, q_heads, D] in 64 bits,
    with the largest sum of |q_d k_d| * scale and |v| for the error bounds. Blocks in `bad` count as absent."""
    n, hq, D = q.shape
    hk = kq.shape[0]
    k = (kq.astype(np.float64) * ks.astype(np.float64)[..., None, None]).reshape(hk, -1, D)
    v = (vq.astype(np.float64) * vs.astype(np.float64)[..., None, None]).reshape(hk, -1, D)
    out = np.zeros((n, hq, D))
    big = 0.0
    for i in range(n):
        pos = past + i
        lo = max(0, pos - window + 1) if window else 0
        seen = [j for j in range(lo, pos + 1) if j // BLOCK not in bad]
        if not seen:
            continue
        for h in range(hq):
            kv = h // (hq // hk)
            qq = np.asarray(q[i, h], dtype=np.float64)
            e = k[kv][seen] @ qq * scale
            big = max(big, float(np.max(np.abs(k[kv][seen]) @ np.abs(qq)) * abs(scale)))
            p = np.exp(e - e.max())
            out[i, h] = p @ v[kv][seen] / p.sum()
    return out, big, float(np.max(np.abs(v))) if v.size else 0.0


def attend_bound(q, kq, ks, vq, vs, past, scale, window, part, floor):
    """attend's outputs, with a bound on each of them for a kernel whose weights are off by at most `part`
    relative, and by `floor` of the largest p_j * (scale of v_j) of the row where they are small:
    2 part sum p_j |v_j| + floor max(p_j s_j) sum |byte of v_j|. part(A, S): A the row's largest sum |q_d k_d| * scale,
    S its scales' largest |log2 s_j|. Blocks of zeros have no scale: they count with 2^-80, far below any other, which
    their weights are formed with (a floor of 2^-80 p_j floor, absolute)."""
    n, hq, D = q.shape
    hk = kq.shape[0]
    k = (kq.astype(np.float64) * ks.astype(np.float64)[..., None, None]).reshape(hk, -1, D)
    byte = np.abs(vq.astype(np.float64)).reshape(hk, -1, D)
    sv = np.repeat(vs.astype(np.float64), BLOCK, axis=1)
    v = vq.astype(np.float64).reshape(hk, -1, D) * sv[..., None]
    weight = np.where(sv > 0, sv, 2.0 ** -80)
    size = np.abs(np.log2(weight))
    out, tol = np.zeros((n, hq, D)), np.zeros((n, hq, D))
    for i in range(n):
        pos = past + i
        seen = slice(max(0, pos - window + 1) if window else 0, pos + 1)
        for h in range(hq):
            kv = h // (hq // hk)
            qq = np.asarray(q[i, h], dtype=np.float64)
            e = k[kv, seen] @ qq * scale
            A = float(np.max(np.abs(k[kv, seen]) @ np.abs(qq)) * abs(scale))
            p = np.exp(e - e.max())
            p /= p.sum()
            out[i, h] = p @ v[kv, seen]
            tol[i, h] = 2 * part(A, float(size[kv, seen].max())) * (p @ np.abs(v[kv, seen])) + floor * np.max(p * weight[kv, seen]) * byte[kv, seen].sum(0)
    return out, tol
