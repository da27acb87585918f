"""Calls at the edges of the operators around prompts and 4-bit caches, written once for the CPU build
(tests/cpu_emu/lanes.py) and for the GPU (`GpuProgram`): `program` is a class of either.

Tolerances are those of serving_ref.attention, derived there, but for caps: cap * tanh(x / cap) is
off by 6 u of the smaller of the cap and 3 |x| (a series below |x / cap| = 0.35), not of the cap.
Outputs of 16 bits of prompts may use a form that is 12 u of the cap off where that is an eighth of
their weights' own rounding at most.
"""
import numpy as np

import serving_ref as ref
from serving_ref import BF16, F16, F32, HALF_ULP, STORED, TINY, close, stored, values
from test_cpu_serving_more import Cache, rows_back, rows_of

COMBOS = [(F32, F32), (F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)]


class GpuProgram:
    """lanes.Program's interface on the GPU: calls run as they are made."""

    def __init__(self, cus=None, reverse=False):
        self.buffers, self.shapes, self.codes, self.messages = [], [], [], []

    def buf(self, array):
        import torch
        a = np.ascontiguousarray(array)
        self.buffers.append(torch.from_numpy(a.reshape(-1).view(np.uint8).copy()).cuda())
        self.shapes.append((a.dtype, a.shape))
        return len(self.buffers) - 1

    def call(self, name, *args):
        from tomoul_amd import _abi
        given = [self.buffers[a[1]].data_ptr() + (a[2] if len(a) > 2 else 0) if isinstance(a, tuple) else a for a in args]
        self.codes.append(getattr(_abi.lib(), f"tml_hip_{name}_dev")(*given))
        self.messages.append("")

    def run(self):
        import torch
        torch.cuda.synchronize()
        return [b.cpu().numpy().view(t).reshape(shape) for b, (t, shape) in zip(self.buffers, self.shapes)]


def expected(q, keys, vals, pos, cap, weight, **kw):
    """serving_ref.attention with the cap's tolerance as above."""
    if not cap:
        return ref.attention(q, keys, vals, pos, weight=weight, **kw)
    want, wide = ref.attention(q, keys, vals, pos, cap=cap, weight=weight, **kw)
    with np.errstate(invalid="ignore"):  # the largest score without the cap
        x = max([np.abs(keys[:, h // (q.shape[1] // keys.shape[1])] @ q[:, h].T).max(initial=0) for h in range(q.shape[1])]) * abs(kw["scale"])
    if not cap > 3 * x:
        return want, wide
    # (6 u of 3 |x| is 18 u |x|; the tolerance without a cap has 2 u |s| of it)
    _, tol = ref.attention(q, keys, vals, pos, weight=weight + 36 * ref.U * x, **kw)
    return want, tol


def prompt(program, q_t, cache_t, both, heads, kv, dim, block, layout="thd", prefix=None, window=0, cap=0.0, slopes=False, scale=None, pad=2, lost=(), odd=(),
           odd_q=(), seed=0, cus=256, reverse=False, loud=1.5, lens=None):
    """both: (context, new tokens) of each request; odd_q: (row, element, number) of q; lens: of the caches, where not their sums."""
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in both] if lens is None else lens
    cache = Cache(rng, cache_t, lens, kv, dim, block, layout, 0, lost)
    cache.put(odd)
    starts = np.concatenate([[0], np.cumsum([n for _, n in both])]).astype(np.int32)
    tokens = int(starts[-1]) + pad
    q = stored(loud * rng.standard_normal((tokens, heads * dim)), q_t)
    for row, d, x in odd_q:
        q[row, d] = stored(np.array([x]), q_t)[0]
    sl = (2.0 ** -rng.uniform(0, 8, heads)).astype(np.float32) if slopes else None
    qs, os_ = heads * dim + 3, heads * dim + 1
    scale = float(np.float32(1 / np.sqrt(dim) if scale is None else scale))
    p = program(cus, reverse)
    bq, bo = p.buf(rows_of(q, qs, STORED[q_t](1))), p.buf(np.full((tokens - 1) * os_ + heads * dim, 7, STORED[q_t]))
    bk, bv, bt = p.buf(cache.bytes[0]), p.buf(cache.bytes[1]), p.buf(cache.table)
    bl, bs = p.buf(np.array(lens, np.int32)), p.buf(starts)
    bp = p.buf(np.array(prefix, np.int32)) if prefix is not None else None
    bsl = p.buf(sl) if slopes else None
    p.call("prompt_attention", q_t, cache_t, tokens, len(both), heads, kv, dim, ("b", bq), qs, ("b", bk), ("b", bv), cache.n_blocks, block, *cache.strides,
           ("b", bt), cache.width, cache.width, ("b", bs), ("b", bl), None if bp is None else ("b", bp), window, scale, cap, ("b", bsl) if slopes else None,
           ("b", bo), os_, None)
    got = p.run()
    assert p.codes == [0], p.messages
    out = rows_back(got[bo], tokens, heads * dim, os_)
    for r in range(tokens - 1):
        assert (got[bo][r * os_ + heads * dim:(r + 1) * os_] == 7).all()
    assert (out[starts[-1]:] == 7).all()
    weight = 2.0 ** -20 if q_t == F32 else HALF_ULP[q_t] * (1.125 if cap else 1.0)
    for r, (_, n) in enumerate(both):
        if n == 0:
            continue
        pos = np.arange(lens[r] - n, lens[r])
        t, k, v, _, _ = cache.of(r, lens[r])
        want, tol = expected(values(q[starts[r]:starts[r + 1]], q_t).reshape(n, heads, dim), k, v, pos, cap, weight, scale=scale, slopes=sl,
                             seen=ref.sees(pos, t, prefix[r] if prefix else 0, window if window < 1 << 62 else 0), positions=t)
        mine = values(out[starts[r]:starts[r + 1]], q_t).reshape(want.shape)
        # (an infinite value's element is infinite or NaN in those who see it; a weight may underflow here or there)
        infinite = np.repeat(np.isinf(v), heads // kv, 1).astype(float)
        sees_one = np.einsum("nt,thd->nhd", ref.sees(pos, t, prefix[r] if prefix else 0, window if window < 1 << 62 else 0).astype(float), infinite) > 0
        mine = np.where(sees_one & ~np.isfinite(want) & ~np.isfinite(mine), want, mine)
        close(mine, want, tol + HALF_ULP[q_t] * (np.abs(want) + tol) + TINY[q_t], f"request {r}")


def decode(program, q_t, cache_t, lens, heads, kv, dim, block, cap=0.0, slopes=False, scale=None, odd=(), odd_q=(), seed=0, cus=256, loud=1.5, window=0, spoil=()):
    """One new token a request; cache_t None: in 4 bits.  spoil: (request, position, key or value, head, group) whose group is NaN."""
    rng = np.random.default_rng(seed)
    cache = Cache(rng, cache_t, lens, kv, dim, block, "thd", window)
    cache.put(odd)
    for r, pos, w, h, g in spoil:
        page, at = cache.table[r, pos // block], pos % block
        cache.values[w][page, at, h, 32 * g:32 * g + 32] = np.nan
        b, tk, hd = cache.strides
        word = page * b + at * tk + h * hd + dim // 2 + 4 * g
        cache.bytes[w][word:word + 4] = np.frombuffer(np.uint32(0x7E000000).tobytes(), np.uint8)
    batch = len(lens)
    q = stored(loud * rng.standard_normal((batch, heads * dim)), q_t)
    for row, d, x in odd_q:
        q[row, d] = stored(np.array([x]), q_t)[0]
    sl = (2.0 ** -rng.uniform(0, 8, heads)).astype(np.float32) if slopes else None
    scale = float(np.float32(1 / np.sqrt(dim) if scale is None else scale))
    p = program(cus)
    bq, bo = p.buf(q), p.buf(np.full((batch, heads * dim), 7, STORED[q_t]))
    bk, bv, bt, bl = p.buf(cache.bytes[0]), p.buf(cache.bytes[1]), p.buf(cache.table), p.buf(np.array(lens, np.int32))
    bs = p.buf(sl) if slopes else None
    p.call("paged_attention_q4" if cache_t is None else "paged_attention_ex", *((q_t,) if cache_t is None else (q_t, cache_t)), batch, heads, kv, dim, ("b", bq),
           heads * dim, ("b", bk), ("b", bv), cache.n_blocks, block, *cache.strides, ("b", bt), cache.width, cache.width, ("b", bl), window, scale, cap,
           ("b", bs) if slopes else None, ("b", bo), heads * dim, None)
    got = p.run()
    assert p.codes == [0], p.messages
    weight = 2.0 ** -16 if cache_t == BF16 and q_t == BF16 else 2.0 ** -11 if cache_t is None and q_t != F32 else 2.0 ** -20
    for r, length in enumerate(lens):
        pos = np.array([length - 1])
        t, k, v, km, vm = cache.of(r, length)
        its_q = values(q[r], q_t).reshape(1, heads, dim)
        if cache_t is None:
            its_q = np.where(np.isinf(its_q), np.nan, its_q)  # (an infinite element makes its head NaN)
        want, tol = expected(its_q, k, v, pos, cap, weight, scale=scale, slopes=sl, seen=ref.sees(pos, t, 0, window), positions=t, key_mag=km, val_mag=vm)
        close(values(got[bo][r], q_t).reshape(want[0].shape), want[0], tol[0] + HALF_ULP[q_t] * (np.abs(want[0]) + tol[0]) + TINY[q_t], f"request {r}")


# ------------------------------------------------------------------------ caps
CAPS = [2.0 ** -100, 0.5, 60.0, 65.0, 400.0, 600.0, 1e4, 1e6, 1e9, 2.0 ** 100]


def prompt_caps(program, q_t, cache_t, cap):
    prompt(program, q_t, cache_t, [(20, 50), (0, 3)], 4, 2, 64, 16, cap=cap, seed=11)
    # (loud scores: some reach the caps of the middle)
    prompt(program, q_t, cache_t, [(5, 30)], 2, 1, 40, 8, cap=cap, slopes=True, loud=30.0, seed=12)


def prompt_cap_of_large_scale(program, q_t, cache_t):
    """scale / cap is no number here; a product of 0 is a score of 0 all the same."""
    prompt(program, q_t, cache_t, [(5, 30)], 2, 1, 64, 8, cap=2.0 ** -100, scale=2.0 ** 40, odd_q=[(3, d, 0.0) for d in range(64)], seed=13)


def decode_caps(program, q_t, cache_t, cap):
    decode(program, q_t, cache_t, [70, 3, 0], 4, 2, 64, 16, cap=cap, seed=14)


# ------------------------------------------------- more new tokens than the cache has
def prompt_before_the_cache(program, q_t, cache_t, window):
    """Tokens that stand before position 0 see the prefix all the same, as one sequence attends to another's cache."""
    prompt(program, q_t, cache_t, [(0, 30), (0, 12)], 4, 2, 64, 16, lens=[9, 40], prefix=[9, 20], window=window, seed=21)
    prompt(program, q_t, cache_t, [(0, 150)], 2, 1, 40, 8, lens=[70], prefix=[50], window=window, slopes=True, seed=22)


WINDOWS = [0, 5, 60, 70, 1 << 31, 1 << 40, (1 << 63) - 1]


# --------------------------------------------------------- infinities and NaN
def sprinkled(rng, lens, kv, dim, what, share, kinds):
    """Odd numbers at a share of the elements of keys (0) or values (1)."""
    odd = []
    for r, n in enumerate(lens):
        for _ in range(max(1, int(share * n))):
            odd.append((r, int(rng.integers(n)), what, int(rng.integers(kv)), int(rng.integers(dim)), float(rng.choice(kinds))))
    return odd


ODD_MASKS = [dict(), dict(window=30), dict(prefix=[110, 0, 64]), dict(window=45, prefix=[130, 70, 0], cap=20.0), dict(slopes=True, lost=[(0, 2, -1), (0, 6, 1 << 30)])]


def prompt_odd_values(program, q_t, cache_t, dim, mask, cus=256, shares=(0.02, 0.5)):
    """Infinite and NaN values reach those who see them and no one else, few and many of them, at the tiles' ends too."""
    both, inf, nan = [(60, 90), (0, 70), (130, 3)], np.inf, np.nan
    lens = [c + n for c, n in both]
    rng = np.random.default_rng(dim)
    for share in shares:
        odd = sprinkled(rng, lens, 2, dim, 1, share, [inf, -inf, nan])
        odd += [(0, p, 1, 0, dim - 1, inf) for p in (63, 64, 127, 128, 149)] + [(1, 69, 1, 1, 0, nan)]
        # (a page that is no block of the cache holds no values)
        odd = [o for o in odd if (o[0], o[1] // 16) not in [(r, i) for r, i, _ in mask.get("lost", ())]]
        prompt(program, q_t, cache_t, both, 4, 2, dim, 16, odd=odd, seed=31, cus=cus, **mask)
    if len(shares) < 2 and mask:
        return
    # (one head's rows: a workgroup of 128 tokens, whose first and last see tiles far apart)
    prompt(program, q_t, cache_t, [(300, 140)], 1, 1, dim, 32, odd=sprinkled(rng, [440], 1, dim, 1, 0.05, [inf, -inf, nan]), window=mask.get("window", 0), seed=32, cus=cus)


KEY_MASKS = [dict(), dict(cap=20.0), dict(cap=1e4, slopes=True), dict(window=40), dict(prefix=[100, 0, 133], cap=5.0), dict(scale=-0.2), dict(scale=-0.3, cap=3.0)]


def prompt_odd_keys(program, q_t, cache_t, dim, mask, cus=256, which=slice(None)):
    """A score of -inf weighs nothing, one of +inf makes its row NaN, a capped one is the cap: whatever the terms of q are."""
    both, inf, nan = [(60, 90), (0, 70), (130, 3)], np.inf, np.nan
    lens = [c + n for c, n in both]
    # few infinite keys (rows with scores of -inf alone stay numbers), elements of q that are 0, tiny next to the others, or both signs
    rng = np.random.default_rng(dim)
    tiny = 1e-6 if q_t == F16 else 1e-20 if q_t == F32 and cache_t != BF16 else 1e-35
    odd_q = [(int(rng.integers(160)), int(rng.integers(4)) * dim + 3, x) for x in (0.0, -0.0, tiny, -tiny, 1.0, -2.0, 0.3) * 6]
    sets = ([(0, 30, 0, 0, 3, inf)], [(0, 5, 0, 0, 3, -inf), (0, 100, 0, 1, 3, -inf), (1, 3, 0, 1, 3, inf), (2, 131, 0, 0, 3, inf)],
            [(0, 64, 0, 0, 3, inf), (0, 64, 0, 0, 4, inf), (0, 70, 0, 0, 3, -inf)], [(0, 20, 0, 0, 3, inf), (0, 120, 0, 0, 5, nan), (1, 0, 0, 0, 3, inf)],
            [(0, 20, 0, 0, 3, inf), (0, 130, 1, 0, 7, -inf)])
    for odd in sets[which]:
        prompt(program, q_t, cache_t, both, 4, 2, dim, 16, odd=odd, odd_q=odd_q, seed=41, cus=cus, **mask)


def prompt_odd_q(program, q_t, cache_t, dim):
    """Infinite and NaN elements of q give what their scores give: NaN, or under a cap the cap."""
    odd_q = [(3, 5, np.nan), (40, dim + 1, np.nan), (70, 3 * dim, np.nan), (7, 2 * dim + 1, np.inf), (90, 9, -np.inf), (91, 9, np.inf), (91, 10, np.inf), (92, dim, -np.inf)]
    for cap in (0.0, 20.0):
        prompt(program, q_t, cache_t, [(60, 90), (0, 70)], 4, 2, dim, 16, odd_q=odd_q, cap=cap, seed=42)
        prompt(program, q_t, cache_t, [(60, 90), (0, 70)], 4, 2, dim, 16, odd_q=odd_q, odd=[(0, 30, 0, 0, 3, np.inf)], cap=cap, slopes=True, seed=43)


def decode_odd_q_and_keys(program, q_t, cache_t, cap):
    """Infinite and NaN elements of q, infinite keys (float caches), NaN groups (4-bit caches)."""
    inf, nan = np.inf, np.nan
    odd_q = [(0, 5, nan), (0, 64 + 9, inf), (2, 128, -inf), (2, 3 * 64 + 1, nan)]
    if cache_t is None:
        decode(program, q_t, None, [70, 3, 40], 4, 2, 64, 16, cap=cap, odd_q=odd_q, seed=51)
        # a key's group: the heads that look at it; a value's: its 32 elements
        decode(program, q_t, None, [70, 3, 40], 4, 2, 64, 16, cap=cap, spoil=[(0, 33, 0, 0, 1), (1, 2, 1, 1, 0), (2, 39, 1, 0, 1)], seed=52)
    else:
        decode(program, q_t, cache_t, [70, 3, 40], 4, 2, 64, 16, cap=cap, odd_q=odd_q, seed=53)
        odd = [(0, 30, 0, 0, 3, inf), (0, 69, 0, 1, 3, -inf), (1, 1, 0, 0, 7, -inf), (2, 0, 0, 1, 7, inf), (2, 20, 0, 1, 9, inf)]
        decode(program, q_t, cache_t, [70, 3, 40], 4, 2, 64, 16, cap=cap, slopes=cap > 0, odd=odd, seed=54)


# ---------------------------------------------------------------- other scales
SCALES = [-0.3, 0.0, -1e-4, 2.0]


def other_scales(program, q_t, cache_t, scale):
    """Negative scales, one of 0 (every token alike), one that leaves few tokens with a weight."""
    decode(program, q_t, cache_t, [70, 3, 0], 4, 2, 64, 16, scale=scale, seed=61)
    decode(program, q_t, cache_t, [70, 3, 0], 4, 2, 64, 16, scale=scale, cap=4.0, slopes=True, seed=62)
    if cache_t is not None:
        prompt(program, q_t, cache_t, [(60, 90), (0, 20)], 4, 2, 64, 16, scale=scale, seed=63)
        prompt(program, q_t, cache_t, [(60, 90), (0, 20)], 4, 2, 40, 16, scale=scale, cap=4.0, slopes=True, window=50, seed=64)


# ------------------------------------------------------ more workgroups than CUs
MANY_MASKS = [dict(), dict(window=77), dict(some_prefix=True), dict(lost=[(0, 2, -1), (1, 5, 1 << 30), (2, 0, 99999)], layout="htd"), dict(odd=True)]


def prompt_many(program, q_t, cache_t, dim, mask, cus, requests):
    """More workgroups than CUs: prompts in 16 bits then go by one team of waves each."""
    rng = np.random.default_rng(dim)
    both = [(0, 150), (300, 40), (64, 64), (0, 0), (200, 130)] + [(int(rng.integers(40)), int(rng.integers(1, 6))) for _ in range(requests)]
    tokens, kv = sum(n for _, n in both) + 2, 4
    assert (tokens // 128 + len(both)) * kv > cus
    more = {k: v for k, v in mask.items() if k not in ("some_prefix", "odd")}
    if "some_prefix" in mask:
        more["prefix"] = [int(rng.integers(c + n + 1)) for c, n in both]
    if "odd" in mask:
        more["odd"] = sprinkled(rng, [c + n for c, n in both[:3]], kv, dim, 1, 0.05, [np.inf, -np.inf, np.nan])
    prompt(program, q_t, cache_t, both, kv, kv, dim, 16, seed=71, cus=cus, **more)


# ------------------------------------------------------------- nothing weighs
def nothing_weighs(program, q_t, cache_t):
    """Scores of -inf alone: zeros, whatever the values are."""
    inf, nan = np.inf, np.nan
    lens, kv, heads, dim = [1, 2, 70, 33], 2, 4, 64
    odd = [(r, p, 0, h, 3, inf) for r, n in enumerate(lens) for p in range(n) for h in range(kv)]
    odd += [(0, 0, 1, 0, 5, inf), (1, 1, 1, 1, 6, nan), (2, 3, 1, 0, 7, -inf), (2, 69, 1, 1, 8, nan), (3, 20, 1, 0, 9, inf)]
    decode(program, q_t, cache_t, lens, heads, kv, dim, 16, odd=odd, odd_q=[(r, h * dim + 3, -1.0) for r in range(4) for h in range(heads)], seed=91)
    both = [(0, 1), (1, 1), (60, 10), (0, 33)]
    prompt(program, q_t, cache_t, both, heads, kv, dim, 16, odd=odd, odd_q=[(r, h * dim + 3, -1.0) for r in range(45) for h in range(heads)], seed=92)

