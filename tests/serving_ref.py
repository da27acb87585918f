"""Definitions in 64 bits of the operators around prompts, 4-bit caches and token scores
(test infrastructure; numpy only, so that the CPU and the GPU tests share it).

Element types are those of the library (F32, F16, BF16); a bf16 array holds its bits.
"""
import numpy as np

U = 2.0 ** -24
F32, F16, BF16 = 0, 1, 2
NAMES = {F32: "f32", F16: "f16", BF16: "bf16"}
STORED = {F32: np.float32, F16: np.float16, BF16: np.uint16}
HALF_ULP = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -25, BF16: 2.0 ** -134}  # half of the smallest number


def tname(t):
    return NAMES.get(t, str(t))


def stored(v, t):
    """Values as an array of type t's elements, rounded once."""
    v = np.asarray(v)
    if t != BF16:
        with np.errstate(over="ignore"):
            return v.astype(STORED[t])
    w = v.astype(np.float32)
    bits = w.view(np.uint32).astype(np.uint64)
    up = ((bits + 0x7FFF + (bits >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(w), np.uint16(0x7FC0), up)


def values(a, t):
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def close(got, ref, tol, what=""):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what
    with np.errstate(invalid="ignore"):
        bad = np.abs(got - ref) > tol
        ratio = np.abs(got - ref) / np.maximum(tol, 1e-300)
    bad &= ~(np.isinf(ref) & (got == ref)) & ~np.isnan(ref)
    assert not bad.any(), (what, int(bad.sum()), float(ratio[bad].max()), np.argwhere(bad)[:4].tolist())


# ------------------------------------------------------------ rows in 4 bits
def row_bytes(dim):
    return dim // 32 * 20


def pack_rows(x):
    """[.., dim] floats (as fp32) to the key row and the value row that hold them: two uint8 arrays [.., row_bytes]."""
    x = np.asarray(x, np.float32)
    dim, groups = x.shape[-1], x.shape[-1] // 32
    g = x.reshape(x.shape[:-1] + (groups, 32))
    bad = ~np.isfinite(g).all(-1)
    g = np.clip(np.where(bad[..., None], np.float32(0), g), np.float32(-65504), np.float32(65504))
    low, high = g.min(-1), g.max(-1)
    step = ((high - low) / np.float32(15)).astype(np.float16)
    least = low.astype(np.float16)
    s, z = step.astype(np.float32)[..., None], least.astype(np.float32)[..., None]
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(s > 0, np.clip(np.rint((g - z) / np.where(s > 0, s, np.float32(1))), 0, 15), 0)
    n = np.where(bad[..., None], 0, n).reshape(x.shape).astype(np.uint8)
    bits = step.view(np.uint16).astype(np.uint32) | least.view(np.uint16).astype(np.uint32) << 16
    bits = np.where(bad, np.uint32(0x7E000000), bits).astype("<u4")
    meta = np.ascontiguousarray(bits).view(np.uint8).reshape(x.shape[:-1] + (4 * groups,))
    rows = []
    for key in (True, False):
        nib = np.zeros(x.shape, np.uint8)  # by nibble of the row
        for d in range(dim):
            nib[..., spot(d, dim, key)] = n[..., d]
        rows.append(np.concatenate([nib[..., ::2] | nib[..., 1::2] << 4, meta], -1))
    return rows


def spot(d, dim, key):
    """The nibble of a row that holds element d."""
    groups = dim // 32
    return 8 * (d % 32 // 8 * groups + d // 32) + d % 8 if key else 2 * groups * (d % 16) + d // 16


def unpack_rows(rows, dim, key):
    """n * s + z of rows in 4 bits, in 64 bits, and |n s| + |z|."""
    groups = dim // 32
    nib = np.stack([rows[..., :16 * groups] & 15, rows[..., :16 * groups] >> 4], -1).reshape(rows.shape[:-1] + (dim,))
    half = np.ascontiguousarray(rows[..., 16 * groups:]).view("<f2").astype(np.float64)
    out, mag = np.empty(rows.shape[:-1] + (dim,)), np.empty(rows.shape[:-1] + (dim,))
    for d in range(dim):
        s, z = half[..., 2 * (d // 32)], half[..., 2 * (d // 32) + 1]
        out[..., d] = nib[..., spot(d, dim, key)] * s + z
        mag[..., d] = nib[..., spot(d, dim, key)] * s + np.abs(z)
    return out, mag


# ---------------------------------------------------------------- attention
def attention(q, keys, vals, pos, *, scale, cap=0.0, slopes=None, seen=None, positions=None, key_mag=None, val_mag=None, weight=2.0 ** -20):
    """One request and all its heads: q [n, heads, dim] at positions pos, keys and vals [m, kv, dim] at `positions`,
    seen [n, m].  Outputs [n, heads, dim] and how far off they may be, rounding to the output's type aside:
    scores by (2^-21 + 4 sqrt(D) u) sum |q k| scale, 6 u of the cap and of the bias, 2 u of themselves; weights by `weight`,
    sums by 8 sqrt(m) u, both of sum p |v|."""
    n, heads, dim = q.shape
    kv = keys.shape[1]
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    key_mag = np.abs(keys) if key_mag is None else key_mag
    val_mag = np.abs(vals) if val_mag is None else val_mag
    away = np.abs(pos[:, None] - positions[None, :]).astype(np.float64)
    for h in range(heads):
        k, v = keys[:, h // (heads // kv)], vals[:, h // (heads // kv)]
        for i in range(n):
            at = np.flatnonzero(seen[i])
            if not len(at):
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                x = k[at] @ q[i, h] * scale
                err = (2.0 ** -21 + 4 * np.sqrt(dim) * U) * (key_mag[:, h // (heads // kv)][at] @ np.abs(q[i, h])) * abs(scale)
                s = cap * np.tanh(x / cap) if cap else x
                if cap:
                    err = err + 6 * U * cap
                if slopes is not None:
                    s = s - slopes[h] * away[i, at]
                    err = err + 6 * U * np.abs(slopes[h]) * away[i, at]
                err = err + 2 * U * np.abs(s)
                most = s.max()
                if most == -np.inf:
                    continue
                p = np.exp(s - most)
                p /= p.sum()
                out[i, h] = p @ v[at]
                tol[i, h] = (2 * np.max(np.where(np.isfinite(err), err, 0)) + weight + 8 * np.sqrt(len(at)) * U) * (p @ val_mag[:, h // (heads // kv)][at])
    return out, tol


def sees(pos, positions, prefix, window):
    m = (positions[None, :] <= pos[:, None]) | (positions[None, :] < prefix)
    return m & (positions[None, :] > pos[:, None] - window) if window else m


# ----------------------------------------------------------------- logprobs
def logprobs(x, tokens, top):
    """log p of the tokens, entropy, ids and log p of the best, of rows x (64 bits)."""
    rows, cols = x.shape
    lp, ent = np.zeros(rows), np.zeros(rows)
    ids, best = np.full((rows, top), -1, np.int64), np.full((rows, top), -np.inf)
    for r in range(rows):
        v = x[r]
        bad = np.isnan(v).any() or (v == np.inf).any()
        none = not bad and (cols == 0 or (v == -np.inf).all())
        with np.errstate(invalid="ignore"):
            if bad:
                logp, ent[r] = np.full(cols, np.nan), np.nan
            elif none:
                logp = np.full(cols, -np.inf)
            else:
                e = np.exp(v - v.max())
                logp = v - v.max() - np.log(e.sum())
                ent[r] = -(np.where(e > 0, e / e.sum() * np.where(e > 0, logp, 0), 0)).sum()
        lp[r] = logp[tokens[r]] if 0 <= tokens[r] < cols else 0.0
        order = [i for i in np.lexsort((np.arange(cols), -np.where(np.isnan(v), -np.inf, v))) if not np.isnan(v[i])][:top]
        ids[r, :len(order)] = order
        best[r, :len(order)] = logp[order]
    return lp, ent, ids, best
