"""The operators around prompts, 4-bit caches and token scores on the CPU, lane by lane
(tests/cpu_emu/lanes.py), against definitions in 64 bits (tests/serving_ref.py), every
operand in an allocation of exactly the size that the header gives it.

Tolerances, fixed by derivation before the first run (u = 2^-24; a result of f16 / bf16 is
rounded once more):
  4-bit rows  bit for bit; loaded values are n s + z rounded once
  attention   serving_ref.attention; weights 2^-20, or a 16-bit type's half step (2^-11,
              2^-8) where prompts' weights are rounded to it
  logprobs    a sum's roundings 8 sqrt(cols) u at most, 4 u (1 + |log p|) for the logarithm
              and the differences; 2 u |x - m| of each exponent, at most 2 u of the mean of
              |x - m| e^(x - m), below u
CPU only; needs /opt/rocm/llvm/bin/clang++ and an x86-64 (skipped without them).
"""
import os
import platform
import sys

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import serving_ref as ref  # noqa: E402
from serving_ref import BF16, F16, F32, HALF_ULP, STORED, TINY, U, close, stored, tname, values  # noqa: E402

CLANG = "/opt/rocm/llvm/bin/clang++"
pytestmark = pytest.mark.skipif(not os.path.exists(CLANG) or platform.machine() != "x86_64", reason="no clang++ for the CPU build, or not x86-64")
INVALID_SHAPE, SHAPE_MISMATCH, INVALID_FORMAT, INVALID_ARG = -1, -2, -4, -5


@pytest.fixture(scope="module")
def lanes():
    sys.path.insert(0, os.path.join(HERE, "cpu_emu"))
    import lanes as emu_lanes  # tests/cpu_emu/lanes.py
    emu_lanes.build()
    return emu_lanes


def rows_of(a, stride, fill):
    """A 2-D array's rows `stride` apart, ending with the last row's last element."""
    n, m = a.shape
    flat = np.full((n - 1) * stride + m if n else 0, fill, a.dtype)
    for r in range(n):
        flat[r * stride:r * stride + m] = a[r]
    return flat


def rows_back(flat, n, m, stride):
    return np.stack([flat[r * stride:r * stride + m] for r in range(n)]) if n else np.zeros((0, m), flat.dtype)


def pool_strides(layout, block, heads, row):
    """(block, token, head) strides of a cache of whole rows."""
    return (block * heads * row, heads * row, row) if layout == "thd" else (block * heads * row, row, block * row)


def pool_index(layout, n_blocks, block, heads, row):
    """Where [block, token, head] rows begin."""
    b, t, h = pool_strides(layout, block, heads, row)
    return (np.arange(n_blocks)[:, None, None] * b + np.arange(block)[None, :, None] * t + np.arange(heads)[None, None, :] * h)


# --------------------------------------------------------------- 4-bit rows
def wild(rng, shape):
    """Groups of every kind: ordinary, constant, tiny, huge, with an infinity or a NaN."""
    x = rng.standard_normal(shape)
    g = x.reshape(-1, 32)
    for i in range(len(g)):
        kind = rng.integers(9)
        if kind == 0:
            g[i] = g[i, 0]
        elif kind == 1:
            g[i] *= 2.0 ** -22
        elif kind == 2:
            g[i] *= 2.0 ** 15
        elif kind == 3:
            g[i, rng.integers(32)] = rng.choice([np.inf, -np.inf, np.nan])
        elif kind == 4:
            g[i] += 100.0
        elif kind == 5:
            g[i] = np.round(g[i]) + 0.5  # quotients at the halves
    return x


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("tokens,heads,dim,block,layout", [(1, 1, 32, 1, "thd"), (5, 3, 64, 8, "htd"), (23, 2, 96, 16, "thd"), (9, 5, 128, 4, "htd"),
                                                           (7, 1, 160, 3, "thd"), (3, 2, 192, 8, "htd"), (4, 1, 224, 8, "thd"), (11, 1, 256, 5, "htd")])
def test_store_and_load(lanes, t, tokens, heads, dim, block, layout):
    rng = np.random.default_rng(tokens * dim + t)
    n_blocks, row = -(-tokens // block) + 1, ref.row_bytes(dim)
    ks, vs = heads * dim + 3, 2 * heads * dim + 1
    k, v = (stored(wild(rng, (tokens, heads * dim)), t) for _ in range(2))
    slots = rng.permutation(n_blocks * block)[:tokens].astype(np.int64)
    if tokens > 2:
        slots[1], slots[2] = -1, n_blocks * block
    b, tk, h = pool_strides(layout, block, heads, row)
    p = lanes.Program()
    bk, bv, bs = p.buf(rows_of(k, ks, STORED[t](1))), p.buf(rows_of(v, vs, STORED[t](1))), p.buf(slots)
    ck, cv = p.buf(np.full(n_blocks * b, 0xAB, np.uint8)), p.buf(np.full(n_blocks * b, 0xCD, np.uint8))
    p.call("kv_store_q4", t, tokens, heads, dim, ("b", bk), ("b", bv), ks, vs, ("b", bs), ("b", ck), ("b", cv), n_blocks, block, b, tk, h, None)
    again = np.concatenate([slots, slots[:1], [-5]]).astype(np.int64)  # one of them twice, and one that is none
    n = len(again)
    outs = []
    for out_t in (F32, F16, BF16):
        so = heads * dim + out_t
        ok, ov, ba = p.buf(np.full((n - 1) * so + heads * dim, 9, STORED[out_t])), p.buf(np.full((n - 1) * so + heads * dim, 9, STORED[out_t])), p.buf(again)
        p.call("kv_load_q4", out_t, n, heads, dim, ("b", ck), ("b", cv), n_blocks, block, b, tk, h, ("b", ba), ("b", ok), ("b", ov), so, so, None)
        outs.append((out_t, so, ok, ov))
    got = p.run()
    assert p.codes == [0] * 4, p.messages
    index = pool_index(layout, n_blocks, block, heads, row)
    want = [np.full(n_blocks * b, 0xAB, np.uint8), np.full(n_blocks * b, 0xCD, np.uint8)]
    held = {}
    for i, slot in enumerate(slots):
        if 0 <= slot < n_blocks * block:
            for w, x, key in ((0, k, 0), (1, v, 1)):
                rows = ref.pack_rows(values(x[i], t).astype(np.float32).reshape(heads, dim))[key]
                for hd in range(heads):
                    at = index[slot // block, slot % block, hd]
                    want[w][at:at + row] = rows[hd]
                held[w, slot] = ref.unpack_rows(rows, dim, key == 0)[0].reshape(-1)
    assert np.array_equal(got[ck], want[0]) and np.array_equal(got[cv], want[1])
    for out_t, so, ok, ov in outs:
        for w, o in ((0, ok), (1, ov)):
            back = rows_back(got[o], n, heads * dim, so)
            for i, slot in enumerate(again):
                if (w, slot) in held:
                    with np.errstate(over="ignore"):
                        expect = stored(held[w, slot].astype(np.float32), out_t)
                    assert np.array_equal(values(back[i], out_t), values(expect, out_t), equal_nan=True)
                else:
                    assert (back[i] == 9).all()


def test_rows_are_near_what_they_hold():
    # the header's bound, on the definition that the kernels meet bit for bit
    x = np.random.default_rng(1).standard_normal((500, 64)).astype(np.float32)
    x *= np.float32(10) ** np.random.default_rng(2).uniform(-4, 4, (500, 1)).astype(np.float32)
    x = np.clip(x, -65504, 65504)
    for key, rows in enumerate(ref.pack_rows(x)):
        got = ref.unpack_rows(rows, 64, key == 0)[0].reshape(500, 2, 32)
        step = np.ascontiguousarray(rows[:, 32:]).view("<f2").astype(np.float64).reshape(500, 2, 2)[..., :1]
        g = x.astype(np.float64).reshape(500, 2, 32)
        low, high = g.min(2, keepdims=True), g.max(2, keepdims=True)
        assert (np.abs(got - g) <= step / 2 + 2.0 ** -11 * (np.abs(low) + high - low) + 2.0 ** -21).all()


# ------------------------------------------------------ one token a request
class Cache:
    """A paged cache of random rows, its bytes and what they stand for; what no one may look at is NaN."""

    def __init__(self, rng, t, lens, kv, dim, block, layout, window=0, lost=()):
        self.t, self.kv, self.dim, self.block = t, kv, dim, block
        blocks = [-(-v // block) for v in lens]
        self.n_blocks, self.width = max(1, sum(blocks)), max(1, max(blocks))
        self.row = ref.row_bytes(dim) if t is None else dim
        self.strides = pool_strides(layout, block, kv, self.row)
        if t is not None:  # rows of floats start on 16-byte boundaries
            size = 4 if t == F32 else 2
            assert self.row * size % 16 == 0
        index = pool_index(layout, self.n_blocks, block, kv, self.row)
        order = rng.permutation(self.n_blocks)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        first = 0
        for r, b in enumerate(blocks):
            gone = max(0, lens[r] - window) // block if window else 0
            for i in range(gone, b):
                self.table[r, i] = order[first + i]
            first += b
        for r, i, page in lost:  # pages that are no block of the cache
            if i < self.width:
                self.table[r, i] = page
        live = np.zeros((self.n_blocks, block), bool)
        for r, v in enumerate(lens):
            for pos in range(v):
                page = self.table[r, pos // block]
                if 0 <= page < self.n_blocks:
                    live[page, pos % block] = True
        self.bytes, self.values, self.mags = [], [], []
        for key in (True, False):
            x = rng.standard_normal((self.n_blocks, block, kv, dim))
            if t is None:
                rows = ref.pack_rows(x)[0 if key else 1]
                rows[~live] = 255
                val, mag = ref.unpack_rows(rows, dim, key)
                flat = np.zeros(self.n_blocks * block * kv * self.row, np.uint8)
            else:
                rows = stored(x, t)
                rows[~live] = stored(np.full(1, np.nan), t)[0]
                val, mag = values(rows, t), None
                flat = np.zeros(self.n_blocks * block * kv * self.row, STORED[t])
            for b in range(self.n_blocks):
                for i in range(block):
                    for h in range(kv):
                        flat[index[b, i, h]:index[b, i, h] + self.row] = rows[b, i, h]
            self.bytes.append(flat)
            self.values.append(val)
            self.mags.append(mag)

    def put(self, odd):
        """(request, position, key or value (0, 1), head, d, number) into a cache of floats."""
        for r, pos, w, h, d, x in odd:
            page, at = self.table[r, pos // self.block], pos % self.block
            self.values[w][page, at, h, d] = x
            b, tk, hd = self.strides
            self.bytes[w][page * b + at * tk + h * hd + d] = stored(np.array([x]), self.t)[0]

    def of(self, r, length):
        """Positions of request r that are in the cache, their keys and values, and magnitudes."""
        t = np.arange(length)
        page = self.table[r, t // self.block] if length else t
        t = t[(page >= 0) & (page < self.n_blocks)]
        page, at = self.table[r, t // self.block], t % self.block
        return (t, *(x[page, at] for x in self.values), *(None if m is None else m[page, at] for m in self.mags))


def decode_program(lanes, cache_t, q_t, lens, heads, kv, dim, block, layout="thd", window=0, cap=0.0, slopes=False, lost=(), seed=0, cus=256, reverse=False):
    rng = np.random.default_rng(seed)
    cache = Cache(rng, cache_t, lens, kv, dim, block, layout, window, lost)
    batch = len(lens)
    q = stored(1.5 * rng.standard_normal((batch, heads * dim)), q_t)
    sl = (2.0 ** -rng.uniform(0, 8, heads)).astype(np.float32) if slopes else None
    qs, os_ = heads * dim + 3, heads * dim + 1
    scale = 1 / np.sqrt(dim)
    p = lanes.Program(cus, reverse)
    bq, bo = p.buf(rows_of(q, qs, STORED[q_t](1))), p.buf(np.full((batch - 1) * os_ + heads * dim, 7, STORED[q_t]))
    bk, bv, bt, bl = p.buf(cache.bytes[0]), p.buf(cache.bytes[1]), p.buf(cache.table), p.buf(np.array(lens, np.int32))
    bs = p.buf(sl) if slopes else None
    types = (q_t,) if cache_t is None else (q_t, cache_t)
    name = "paged_attention_q4" if cache_t is None else "paged_attention_ex"
    p.call(name, *types, batch, heads, kv, dim, ("b", bq), qs, ("b", bk), ("b", bv), cache.n_blocks, block, *cache.strides, ("b", bt), cache.width,
           cache.width, ("b", bl), window, float(np.float32(scale)), cap, ("b", bs) if slopes else None, ("b", bo), os_, None)
    got = p.run()
    assert p.codes == [0], p.messages
    out = rows_back(got[bo], batch, heads * dim, os_)
    for r in range(batch - 1):
        assert (got[bo][r * os_ + heads * dim:(r + 1) * os_] == 7).all()
    # (over a 4-bit cache the weights of 16-bit outputs are rounded to f16)
    weight = 2.0 ** -16 if cache_t == BF16 and q_t == BF16 else 2.0 ** -11 if cache_t is None and q_t != F32 else 2.0 ** -20
    for r, length in enumerate(lens):
        pos = np.array([length - 1])
        t, k, v, km, vm = cache.of(r, length)
        want, tol = ref.attention(values(q[r], q_t).reshape(1, heads, dim), k, v, pos, scale=float(np.float32(scale)), cap=cap, slopes=sl,
                                  seen=ref.sees(pos, t, 0, window), positions=t, key_mag=km, val_mag=vm, weight=weight)
        close(values(out[r], q_t).reshape(want[0].shape), want[0], tol[0] + HALF_ULP[q_t] * (np.abs(want[0]) + tol[0]) + TINY[q_t], f"request {r}")


@pytest.mark.parametrize("q_t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_q4(lanes, q_t, dim):
    decode_program(lanes, None, q_t, [0, 1, 33, 70], 4, 2, dim, 16, seed=dim)
    decode_program(lanes, None, q_t, [40, 5], 3, 3, dim, 7, layout="htd", cus=1, reverse=True, seed=dim + 1)


@pytest.mark.parametrize("case", [
    dict(lens=[90, 2, 33], heads=17, kv=1, block=1), dict(lens=[64, 31], heads=40, kv=2, block=32, layout="htd"),
    dict(lens=[100, 20], heads=2, kv=1, block=8, window=19), dict(lens=[70, 3], heads=4, kv=2, block=16, cap=20.0),
    dict(lens=[70, 3], heads=4, kv=4, block=16, slopes=True), dict(lens=[70, 64], heads=4, kv=1, block=50, cap=2.0, slopes=True, window=40),
    dict(lens=[50, 60], heads=2, kv=2, block=8, lost=[(0, 0, -1), (0, 3, 1 << 30), (1, 7, 99)]),
    dict(lens=[16, 8], heads=1, kv=1, block=8, lost=[(0, 0, -1), (0, 1, -7)]),
    dict(lens=[700, 0, 1300], heads=3, kv=1, block=16, cus=2), dict(lens=[900], heads=2, kv=2, block=64, cus=3, reverse=True, slopes=True)],
    ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items() if k != "lost").replace(" ", ""))
def test_attention_q4_shapes(lanes, case):
    decode_program(lanes, None, F32, dim=64, seed=5, **case)
    decode_program(lanes, None, BF16, dim=32, seed=6, **case)


@pytest.mark.parametrize("q_t,cache_t", [(F32, F32), (F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)], ids=tname)
@pytest.mark.parametrize("case", [dict(lens=[70, 3, 0], heads=4, kv=2, cap=20.0), dict(lens=[33, 40], heads=3, kv=3, slopes=True, layout="htd"),
                                  dict(lens=[50, 7], heads=4, kv=1, cap=1.5, slopes=True, window=21), dict(lens=[600, 20], heads=2, kv=1, cap=50.0, cus=2),
                                  dict(lens=[20, 30], heads=2, kv=1)],
                         ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items()).replace(" ", ""))
def test_attention_ex(lanes, q_t, cache_t, case):
    decode_program(lanes, cache_t, q_t, dim=40, block=16, seed=8, **case)


# ------------------------------------------------------------------ prompts
def prompt_program(lanes, q_t, cache_t, both, heads, kv, dim, block, layout="thd", prefix=None, window=0, cap=0.0, slopes=False, pad=2, lost=(), seed=0,
                   reverse=False, odd=()):
    """both: (context, new tokens) of each request."""
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in both]
    cache = Cache(rng, cache_t, lens, kv, dim, block, layout, 0, lost)
    cache.put(odd)
    starts = np.concatenate([[0], np.cumsum([n for _, n in both])]).astype(np.int32)
    tokens = int(starts[-1]) + pad
    q = stored(1.5 * rng.standard_normal((tokens, heads * dim)), q_t)
    sl = (2.0 ** -rng.uniform(0, 8, heads)).astype(np.float32) if slopes else None
    qs, os_ = heads * dim + 3, heads * dim + 1
    scale = float(np.float32(1 / np.sqrt(dim)))
    p = lanes.Program(reverse=reverse)
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
    weight = 2.0 ** -20 if q_t == F32 else HALF_ULP[q_t]
    for r, (ctx, n) in enumerate(both):
        if n == 0:
            continue
        pos = np.arange(ctx, ctx + n)
        t, k, v, _, _ = cache.of(r, lens[r])
        want, tol = ref.attention(values(q[starts[r]:starts[r + 1]], q_t).reshape(n, heads, dim), k, v, pos, scale=scale, cap=cap, slopes=sl,
                                  seen=ref.sees(pos, t, prefix[r] if prefix else 0, window), positions=t, weight=weight)
        mine = values(out[starts[r]:starts[r + 1]], q_t).reshape(want.shape)
        mine = np.where(np.isinf(want) & ~np.isfinite(mine), want, mine)  # (an infinite value's element is infinite or NaN)
        close(mine, want, tol + HALF_ULP[q_t] * (np.abs(want) + tol) + TINY[q_t], f"request {r}")


COMBOS = [(F32, F32), (F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)]


@pytest.mark.parametrize("q_t,cache_t", COMBOS, ids=tname)
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 136, 256])
def test_prompt_attention(lanes, q_t, cache_t, dim):
    prompt_program(lanes, q_t, cache_t, [(0, 5), (3, 0), (70, 9), (0, 1)], 4, 2, dim, 16, seed=dim, layout="htd" if dim % 16 else "thd")


@pytest.mark.parametrize("case", [
    dict(both=[(0, 150)], heads=1, kv=1, block=16), dict(both=[(30, 40), (0, 3), (0, 33)], heads=5, kv=1, block=8, layout="htd"),
    dict(both=[(10, 70)], heads=2, kv=2, block=100, prefix=[80]), dict(both=[(0, 90), (5, 20)], heads=2, kv=1, block=16, prefix=[40, 0]),
    dict(both=[(100, 40), (0, 20)], heads=2, kv=1, block=16, window=33), dict(both=[(0, 100)], heads=1, kv=1, block=1, window=7, prefix=[60]),
    dict(both=[(20, 50)], heads=2, kv=2, block=16, cap=3.0), dict(both=[(20, 50)], heads=2, kv=2, block=16, slopes=True, prefix=[70]),
    dict(both=[(64, 64), (0, 0), (1, 1)], heads=3, kv=3, block=64, cap=30.0, slopes=True, window=50, prefix=[100, 5, 2]),
    dict(both=[(60, 20), (0, 30)], heads=2, kv=2, block=8, lost=[(0, 0, -1), (0, 5, 1 << 30), (1, 2, 99)]),
    dict(both=[(0, 16)], heads=1, kv=1, block=8, lost=[(0, 0, -1), (0, 1, -7)]), dict(both=[(0, 1)] * 70, heads=2, kv=1, block=4)],
    ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items() if k != "lost").replace(" ", "")[:60])
def test_prompt_attention_shapes(lanes, case):
    prompt_program(lanes, F16, F16, dim=64, seed=3, **case)
    prompt_program(lanes, F32, BF16, dim=40, seed=4, reverse=True, **case)
    prompt_program(lanes, F32, F32, dim=64, seed=5, **case)


ODD = [(0, 100, 1, 0, 3, np.inf), (0, 120, 1, 0, 3, -np.inf), (0, 130, 1, 1, 70 % 40, np.nan), (0, 90, 1, 0, 0, -np.inf), (0, 140, 0, 0, 5, np.nan),
       (0, 64, 0, 1, 2, np.inf), (0, 149, 1, 1, 1, np.inf)]


@pytest.mark.parametrize("q_t,cache_t", COMBOS, ids=tname)
def test_prompt_attention_infinities_and_nan_are_for_those_who_see_them(lanes, q_t, cache_t):
    # an infinity or a NaN of a later (or of a left) position reaches no one else
    odd = [o for o in ODD if o[2] == 1 or np.isnan(o[5]) or q_t == cache_t]
    prompt_program(lanes, q_t, cache_t, [(60, 90)], 4, 2, 40, 16, odd=odd, seed=7)
    prompt_program(lanes, q_t, cache_t, [(60, 90)], 2, 2, 40, 16, odd=odd, window=30, prefix=[110], seed=8)


@pytest.mark.parametrize("starts,lens", [([0, 100, 5], [9, 9]), ([-3, 4, 4], [9, 30000]), ([5, 2, 7], [-4, 3]), ([0, 7, 0x7FFFFFFF], [9, 0x7FFFFFFF]),
                                         ([7, -2 ** 31, 7], [1, 9]), ([0, 7, 7], [3, 9])])
def test_prompt_attention_lengths_that_do_not_fit(lanes, starts, lens):
    # whatever the lengths say, nothing outside the operands is touched (exact results only where they make sense)
    tokens, heads, dim, block = 7, 2, 64, 4
    for t in (F16, F32):
        cache = Cache(np.random.default_rng(1), t, [9, 9], 1, dim, block, "thd")
        p = lanes.Program()
        bq, bo = p.buf(np.ones(tokens * heads * dim, STORED[t])), p.buf(np.zeros(tokens * heads * dim, STORED[t]))
        bk, bv, bt = p.buf(cache.bytes[0]), p.buf(cache.bytes[1]), p.buf(cache.table)
        bs, bl, bp = p.buf(np.array(starts, np.int32)), p.buf(np.array(lens, np.int32)), p.buf(np.array([-1, 0x7FFFFFFF], np.int32))
        p.call("prompt_attention", t, t, tokens, 2, heads, 1, dim, ("b", bq), heads * dim, ("b", bk), ("b", bv), cache.n_blocks, block, *cache.strides,
               ("b", bt), cache.width, cache.width, ("b", bs), ("b", bl), ("b", bp), 0, 0.1, 0.0, None, ("b", bo), heads * dim, None)
        p.run()
        assert p.codes == [0], p.messages


# ----------------------------------------------------------------- logprobs
def logprobs_program(lanes, t, x, top, tokens, stride_pad=1, reverse=False):
    x = stored(x, t)
    rows, cols = x.shape
    p = lanes.Program(reverse=reverse)
    bx, bt = p.buf(rows_of(x, cols + stride_pad, STORED[t](1))), p.buf(np.array(tokens, np.int32))
    bl, be = p.buf(np.full(rows, 5, np.float32)), p.buf(np.full(rows, 5, np.float32))
    bi, bp = p.buf(np.full((rows, top), 77, np.int32)), p.buf(np.full((rows, top), 5, np.float32))
    p.call("token_logprobs", t, rows, cols, ("b", bx), cols + stride_pad, ("b", bt), ("b", bl), ("b", be), top, ("b", bi), ("b", bp), None)
    got = p.run()
    assert p.codes == [0], p.messages
    check_logprobs(values(x, t), tokens, top, got[bl], got[be], got[bi], got[bp])


def check_logprobs(x, tokens, top, lp, ent, ids, best):
    rows, cols = x.shape
    want_lp, want_ent, want_ids, want_best = ref.logprobs(x, tokens, top)
    sums = 8 * np.sqrt(max(cols, 1)) * U
    with np.errstate(invalid="ignore"):
        close(lp, want_lp, sums + 4 * U * (1 + np.abs(np.where(np.isfinite(want_lp), want_lp, 0))) + 2 * U, "log p")
        close(ent, want_ent, 2 * sums * (1 + np.log(max(cols, 2))) + 8 * U * (1 + np.abs(want_ent)), "entropy")
        if top:
            assert np.array_equal(ids, want_ids)
            close(best, want_best, sums + 4 * U * (1 + np.abs(np.where(np.isfinite(want_best), want_best, 0))) + 2 * U, "best")


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("cols,top", [(1, 0), (1, 3), (7, 7), (8, 1), (9, 64), (63, 5), (511, 64), (520, 20), (2049, 5), (2500, 64), (8195, 20), (9000, 64)])
def test_logprobs(lanes, t, cols, top):
    rng = np.random.default_rng(cols + top)
    x = 3 * rng.standard_normal((3, cols))
    x[1] = np.round(x[1])  # equal ones
    x[2, rng.integers(cols)] += 30
    logprobs_program(lanes, t, x, top, [cols // 2, -1 if cols > 1 else 0, cols], reverse=cols % 2 == 0)


@pytest.mark.parametrize("cols,top", [(70, 5), (600, 64), (2100, 3), (9000, 8)])
def test_logprobs_odd_rows(lanes, cols, top):
    lowest = -3.38e38
    inf = np.inf
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((10, cols))
    x[0] = 2.5  # all equal
    x[1] = np.arange(cols) / 100  # rising
    x[2] = -np.arange(cols) / 100
    x[3] = -inf
    x[4, rng.permutation(cols)[:cols - 2]] = -inf  # fewer than asked for are left
    x[5] = lowest
    x[6, :-1] = lowest  # one is not masked, and it is the last
    x[7, 3] = np.nan
    x[8, 4] = inf
    x[9] = np.nan
    logprobs_program(lanes, F32, x, top, [0] * 10)
    logprobs_program(lanes, BF16, x, top, [cols - 1] * 10)
    # zeros of both signs are equal
    y = np.zeros((1, cols))
    y[0, ::2] = -0.0
    logprobs_program(lanes, F16, y, top, [1])


def test_logprobs_more_candidates_than_are_held(lanes):
    # 63 lanes of a wave hold nothing but the maximum, the 64th's largest is below it: thousands reach that
    cols = 16 * 64 * 8 * 4
    x = np.full(cols, -1.0).reshape(-1, 1024, 8)
    x[:, :63] = 2.0
    x[:, 63] = 1.5
    logprobs_program(lanes, F16, x.reshape(1, cols), 64, [5])


# ----------------------------------------------------------------- refusals
def refusals(lanes, name, good, bad):
    """Each of `bad`: (index or indices, value or values, code); all other arguments as in `good`."""
    p = lanes.Program()
    b = p.buf(np.zeros(1 << 16, np.uint8))
    args = [("b", b) if a == "buf" else a for a in good]
    p.call(name, *args)
    for where, value, _ in bad:
        a = list(args)
        for i, v in zip(where if isinstance(where, tuple) else (where,), value if isinstance(where, tuple) else (value,)):
            a[i] = ("b", b, v[1]) if isinstance(v, tuple) and v[0] == "buf" else v
        p.call(name, *a)
    p.run()
    assert p.codes == [0] + [c for _, _, c in bad], list(zip(p.codes, p.messages))
    assert all(m for m in p.messages[1:])


def test_refusals_store(lanes):
    good = [F16, 0, 2, 64, "buf", "buf", 128, 128, "buf", "buf", "buf", 2, 4, 320, 80, 40, None]
    bad = [(0, 3, INVALID_FORMAT), (1, -1, INVALID_SHAPE), (2, -1, INVALID_SHAPE), (3, -32, INVALID_SHAPE), (12, 0, INVALID_ARG), (11, -1, INVALID_SHAPE)]
    bad += [((1, *([w] if not isinstance(w, tuple) else w)), (2, *([v] if not isinstance(w, tuple) else v)), c) for w, v, c in
            [(3, 48, INVALID_SHAPE), (3, 288, INVALID_SHAPE), (4, None, INVALID_ARG), (5, None, INVALID_ARG), (8, None, INVALID_ARG), (9, None, INVALID_ARG),
             (10, None, INVALID_ARG), (6, 127, INVALID_SHAPE), (7, 100, INVALID_SHAPE), (13, -4, INVALID_SHAPE), (14, 81, INVALID_ARG), (15, 42, INVALID_ARG),
             (13, 322, INVALID_ARG), (9, ("buf", 2), INVALID_ARG), (10, ("buf", 1), INVALID_ARG), (12, 1 << 31, INVALID_SHAPE), (11, 1 << 31, INVALID_SHAPE)]]
    refusals(lanes, "kv_store_q4", good, bad)
    load = [F16, 0, 2, 64, "buf", "buf", 2, 4, 320, 80, 40, "buf", "buf", "buf", 128, 128, None]
    bad = [(0, 4, INVALID_FORMAT), (1, -1, INVALID_SHAPE), (7, 0, INVALID_ARG), ((1, 14), (2, 127), INVALID_SHAPE), ((1, 13), (2, None), INVALID_ARG),
           ((1, 12), (2, None), INVALID_ARG), ((1, 11), (2, None), INVALID_ARG), ((1, 4), (2, ("buf", 2)), INVALID_ARG), ((1, 10), (2, 41), INVALID_ARG),
           ((1, 3), (2, 40), INVALID_SHAPE)]
    refusals(lanes, "kv_load_q4", load, bad)


def test_refusals_attention(lanes):
    good = [F32, 0, 4, 2, 64, "buf", 256, "buf", "buf", 2, 4, 320, 80, 40, "buf", 3, 3, "buf", 0, 0.1, 0.0, None, "buf", 256, None]
    one = [((1, *([w] if not isinstance(w, tuple) else w)), (2, *([v] if not isinstance(w, tuple) else v)), c) for w, v, c in
           [(0, 3, INVALID_FORMAT), (3, 3, SHAPE_MISMATCH), (4, 40, INVALID_SHAPE), (4, 288, INVALID_SHAPE), (5, None, INVALID_ARG), (7, None, INVALID_ARG),
            (8, None, INVALID_ARG), (14, None, INVALID_ARG), (17, None, INVALID_ARG), (22, None, INVALID_ARG), (6, 255, INVALID_SHAPE), (23, 1, INVALID_SHAPE),
            (16, 2, INVALID_SHAPE), (11, -4, INVALID_SHAPE), (12, 81, INVALID_ARG), (13, 2, INVALID_ARG), (7, ("buf", 2), INVALID_ARG), (18, -1, INVALID_SHAPE),
            (20, -1.0, INVALID_ARG), (20, 1e38, INVALID_ARG), (20, 1e-38, INVALID_ARG), (20, float("nan"), INVALID_ARG), (10, 0, INVALID_ARG),
            (15, 1 << 30, INVALID_SHAPE)]]
    refusals(lanes, "paged_attention_q4", good, one + [(1, -1, INVALID_SHAPE), (1, 1 << 16, INVALID_SHAPE)])
    ex = [F16, F16, 0, 4, 2, 64, "buf", 256, "buf", "buf", 2, 4, 512, 128, 64, "buf", 3, 3, "buf", 0, 0.1, 0.0, None, "buf", 256, None]
    refusals(lanes, "paged_attention_ex", ex, [(21, -1.0, INVALID_ARG), (21, float("inf"), INVALID_ARG), (0, BF16, INVALID_FORMAT), ((2, 13), (2, 4), INVALID_ARG)])
    prompt = [F16, F16, 0, 1, 4, 2, 64, "buf", 256, "buf", "buf", 2, 4, 512, 128, 64, "buf", 3, 3, "buf", "buf", None, 0, 0.1, 0.0, None, "buf", 256, None]
    bad = [((2, *([w] if not isinstance(w, tuple) else w)), (2, *([v] if not isinstance(w, tuple) else v)), c) for w, v, c in
           [(0, BF16, INVALID_FORMAT), (1, 3, INVALID_FORMAT), (4, 3, SHAPE_MISMATCH), (6, 60, INVALID_SHAPE), (6, 264, INVALID_SHAPE), (7, None, INVALID_ARG),
            (9, None, INVALID_ARG), (10, None, INVALID_ARG), (16, None, INVALID_ARG), (19, None, INVALID_ARG), (20, None, INVALID_ARG), (26, None, INVALID_ARG),
            (8, 255, INVALID_SHAPE), (27, 255, INVALID_SHAPE), ((3, 18), (2, 2), INVALID_SHAPE), (13, -8, INVALID_SHAPE), (14, 4, INVALID_ARG),
            (15, 12, INVALID_ARG), (9, ("buf", 8), INVALID_ARG), (22, -1, INVALID_SHAPE), (24, -2.0, INVALID_ARG), (24, 1e35, INVALID_ARG), (12, 0, INVALID_ARG),
            (17, 1 << 30, INVALID_SHAPE), (3, 1 << 16, INVALID_SHAPE), (3, -1, INVALID_SHAPE)]]
    refusals(lanes, "prompt_attention", prompt, bad + [(2, 1 << 24, INVALID_SHAPE), (2, -1, INVALID_SHAPE)])


def test_refusals_logprobs(lanes):
    good = [F16, 2, 8, "buf", 8, "buf", "buf", "buf", 2, "buf", "buf", None]
    refusals(lanes, "token_logprobs", good, [
        (0, 3, INVALID_FORMAT), (1, -1, INVALID_SHAPE), (2, -1, INVALID_SHAPE), (8, -1, INVALID_SHAPE), (8, 65, INVALID_SHAPE), (2, 1 << 31, INVALID_SHAPE),
        (3, None, INVALID_ARG), (4, 7, INVALID_SHAPE), (5, None, INVALID_ARG), (6, None, INVALID_ARG), ((9, 10), (None, None), INVALID_ARG)])


@pytest.mark.parametrize("q_t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("dim,heads,kv", [(32, 5, 1), (64, 12, 2), (96, 17, 1), (128, 6, 1), (128, 16, 2), (160, 7, 1), (256, 9, 1)])
def test_attention_q4_wide_groups(lanes, q_t, dim, heads, kv):
    decode_program(lanes, None, q_t, [70, 0, 600], heads, kv, dim, 16, cus=2, cap=20.0 if dim == 128 else 0.0, slopes=dim == 64, seed=dim + heads)
