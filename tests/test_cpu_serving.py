"""The serving operators on the CPU, lane by lane (tests/cpu_emu/lanes.py), against
definitions in 64 bits, every operand in an allocation of exactly the size that the
header gives it: an access outside one, a matrix instruction with a lane missing or any
undefined behaviour fails the case.

Tolerances (u = 2^-24; a result of f16 / bf16 is rounded once more), fixed by
derivation before the first run:
  rmsnorm    |dy| <= 32 u |y|; 8 bits: half a step and 127 * 80 u of rounding before it
  matvec     (2^-23 + 8 sqrt(K) u) sum |x w|
  attention  scores (2^-21 + 4 sqrt(D) u) sum |q k| * scale, weights 2^-16 (16-bit output
             of a bf16 cache) or 2^-20, sums 8 sqrt(len) u, of sum p |v|

CPU only; needs /opt/rocm/llvm/bin/clang++ and an x86-64 (skipped without them).
"""
import os
import platform
import sys

import numpy as np
import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = "/opt/rocm/llvm/bin/clang++"
pytestmark = pytest.mark.skipif(not os.path.exists(CLANG) or platform.machine() != "x86_64", reason="no clang++ for the CPU build, or not x86-64")

U = 2.0 ** -24
F32, F16, BF16, I8 = 0, 1, 2, 3
NAMES = {F32: "f32", F16: "f16", BF16: "bf16", I8: "i8"}
STORED = {F32: np.float32, F16: np.float16, BF16: np.uint16, I8: np.int8}
SIZE = {F32: 4, F16: 2, BF16: 2, I8: 1}
HALF_ULP = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}


@pytest.fixture(scope="module")
def lanes():
    sys.path.insert(0, os.path.join(HERE, "cpu_emu"))
    import lanes as emu_lanes  # tests/cpu_emu/lanes.py
    emu_lanes.build()
    return emu_lanes


def tname(t):
    return NAMES.get(t, str(t))


def stored(v, t):
    """Values as an array of type t's elements."""
    v = np.asarray(v, np.float64)
    if t != BF16:
        with np.errstate(over="ignore"):
            return v.astype(STORED[t])
    bits = v.astype(np.float32).view(np.uint32).astype(np.uint64)
    nan = np.isnan(v)
    up = ((bits + 0x7FFF + (bits >> 16 & 1)) >> 16).astype(np.uint16)
    return np.where(nan, np.uint16(0x7FC0), up)


def values(a, t):
    if t == BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def rows_of(a, stride, fill):
    """A 2-D array's rows `stride` apart, ending with the last row's last element."""
    n, m = a.shape
    flat = np.full((n - 1) * stride + m if n else 0, fill, a.dtype)
    for r in range(n):
        flat[r * stride:r * stride + m] = a[r]
    return flat


def rows_back(flat, n, m, stride):
    return np.stack([flat[r * stride:r * stride + m] for r in range(n)]) if n else np.zeros((0, m), flat.dtype)


def close(got, ref, tol, what=""):
    got, ref = np.asarray(got, np.float64), np.asarray(ref, np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(ref)), what
    with np.errstate(invalid="ignore"):
        bad = np.abs(got - ref) > tol
    bad &= ~(np.isinf(ref) & (got == ref)) & ~np.isnan(ref)
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist())


# ---------------------------------------------------------------- rmsnorm
def norm_program(lanes, t, rows, cols, out_t, group=0, residual=True, weight=True, alias=None, seed=1, short=None, cus=256, reverse=False):
    rng = np.random.default_rng(seed)
    sx, sr, ss, so = cols + 3, cols + 1, cols + 2, cols + (1 if out_t == I8 else 0)
    x, r = stored(rng.standard_normal((rows, cols)), t), stored(2 * rng.standard_normal((rows, cols)), t)
    w = (1 + 0.2 * rng.standard_normal(cols)).astype(np.float32)
    noise = STORED[t](5)
    p = lanes.Program(cus, reverse)

    def make(name, a):
        return p.buf(a, short=16 if short == name else 0)

    bx = make("x", rows_of(x, sx, noise))
    br = make("residual", rows_of(r, sr, noise)) if residual else None
    bw = make("weight", w) if weight else None
    bs, ss = (bx, sx) if alias == "x" else (br, sr) if alias == "residual" else (make("sum", rows_of(np.zeros_like(x), ss, noise)), ss)
    bo = make("out", rows_of(np.zeros((rows, cols), STORED[out_t]), so, 7))
    groups = (-(-cols // group) if group else 1)
    bg = make("scales", np.full(rows * groups, -1, np.float32)) if out_t == I8 else None

    def at(b):
        return None if b is None else ("b", b)

    p.call("rmsnorm", t, rows, cols, at(bx), sx, at(br), sr, at(bw), 1e-6, at(bs), ss, out_t, at(bo), so, at(bg), group, None)
    got = p.run()
    assert p.codes == [0], p.messages
    h = values(x, t) + (values(r, t) if residual else 0.0)
    y = h / np.sqrt((h * h).mean(1, keepdims=True) + 1e-6) * (w.astype(np.float64) if weight else 1.0)
    sums = values(rows_back(got[bs], rows, cols, ss), t)
    close(sums, h, HALF_ULP[t] * 1.001 * np.abs(h) + 1e-30, "sum")
    out = rows_back(got[bo], rows, cols, so)
    for r0 in range(rows - 1):  # what lies between rows stays
        assert (got[bo][r0 * so + cols:(r0 + 1) * so] == 7).all()
    if out_t != I8:
        close(values(out, out_t), y, (HALF_ULP[out_t] * 1.001 + 32 * U) * np.abs(y) + 2.0 ** -25 * (out_t == F16), "out")
        return
    scales = got[bg].reshape(rows, groups)
    width = group or cols
    for g in range(groups):
        part = y[:, g * width:(g + 1) * width]
        most = np.abs(part).max(1)
        close(scales[:, g], most / 127, 40 * U * most / 127, "scale")
        assert (np.abs(out[:, g * width:(g + 1) * width] - part / (most / 127)[:, None]) <= 0.5 + 127 * 80 * U).all()


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("rows,cols", [(3, 1), (3, 7), (5, 8), (6, 9), (3, 511), (2, 513), (9, 1237), (2, 2049), (1, 8193), (1, 33001)])
def test_rmsnorm(lanes, t, rows, cols):
    norm_program(lanes, t, rows, cols, t)
    norm_program(lanes, t, rows, cols, F32, residual=False, weight=False, reverse=True)
    norm_program(lanes, t, rows, cols, t, alias="x", cus=1)  # (one unit: a wave a row where rows fit one)
    norm_program(lanes, t, rows, cols, t, alias="residual")


@pytest.mark.parametrize("t", [F32, BF16], ids=tname)
@pytest.mark.parametrize("rows,cols,group", [(3, 7, 0), (2, 7, 3), (4, 64, 8), (2, 1280, 128), (3, 1237, 0), (3, 1237, 64), (2, 5120, 512), (2, 5120, 96),
                                             (1, 8200, 1024), (1, 33000, 128), (5, 40, 1), (6, 96, 96), (5, 1000, 64)])
def test_rmsnorm_8_bits(lanes, t, rows, cols, group):
    norm_program(lanes, t, rows, cols, I8, group=group)
    norm_program(lanes, t, rows, cols, I8, group=group, cus=1, reverse=True)


def tie_weights(cols, most, seed):
    """Values at and next to the halves between the steps of a group whose largest is `most`."""
    rng = np.random.default_rng(seed)
    step = np.float32(most) / np.float32(127)
    w = ((rng.integers(-127, 127, cols) + 0.5) * np.float64(step)).astype(np.float32)
    w = (w.view(np.int32) + rng.integers(-2, 3, cols)).astype(np.int32).view(np.float32)
    w[rng.integers(cols)] = most
    return w


@pytest.mark.parametrize("cols,group", [(1280, 0), (1280, 128), (1237, 0), (1237, 96), (7, 0), (33000, 0)])
def test_rmsnorm_8_bits_at_the_halves(lanes, cols, group):
    # x of ones and no epsilon: out is the weight itself, so the quotient is known to its last bit
    rng = np.random.default_rng(17)
    width = group or cols
    w = np.concatenate([tie_weights(min(width, cols - g), np.float32(m), g) for g, m in
                        zip(range(0, cols, width), np.exp(rng.uniform(-8, 8, -(-cols // width))))])
    groups = -(-cols // width)
    p = lanes.Program()
    bx, bw = p.buf(np.ones(cols, np.float32)), p.buf(w)
    bo, bs = p.buf(np.zeros(cols, np.int8)), p.buf(np.zeros(groups, np.float32))
    p.call("rmsnorm", F32, 1, cols, ("b", bx), cols, None, 0, ("b", bw), 0.0, None, 0, I8, ("b", bo), cols, ("b", bs), group, None)
    got = p.run()
    assert p.codes == [0], p.messages
    for g in range(groups):
        part = w[g * width:(g + 1) * width]
        scale = np.abs(part).max() / np.float32(127)
        assert got[bs][g] == scale
        want = np.rint(part / scale)
        wrong = got[bo][g * width:(g + 1) * width] != want
        assert not wrong.any(), (g, int(wrong.sum()), part[wrong][:3] / scale, want[wrong][:3])


@pytest.mark.parametrize("what", ["x", "residual", "weight", "sum", "out", "scales"])
def test_rmsnorm_short_operand_is_reported(lanes, what):
    with pytest.raises(lanes.Fault):
        norm_program(lanes, BF16, 5, 1237, I8, group=64, short=what)


# ---------------------------------------------------------------- kv_plan
def plan_ref(block, ctx, new, free, table, max_tokens):
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    slots, req, pos, seq, start, used, wide = [], [], [], [], [0], 0, 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        need = -(-(c + n) // block)
        wide += need > width
        for col in range(min(-(-c // block), width), min(need, width)):
            table[r][col] = free[used] if used < len(free) else -1
            used += 1
        for j in range(n):
            col = (c + j) // block
            page = table[r][col] if col < width else -1
            slots.append(page * block + (c + j) % block if page >= 0 else -1)
            req.append(r)
            pos.append(c + j)
        seq.append(c + n)
        start.append(start[-1] + n)
    pad = [-1] * max(0, max_tokens - len(slots))
    return table, slots + pad, req + pad, pos + pad, seq, start, [start[-1], used, wide]


PLANS = [(1, 16, 5, 7, 3, 0), (64, 16, 500, 1, 0, 0), (300, 16, 300, 40, 17, 0), (257, 7, 64, 9, 100, 0), (5, 32, 100, 900, 11, 0),
         (33, 16, 200, 60, 9, 40), (12, 4, 40, 30, 2, 1000000), (600, 16, 40, 0, 4, 0)]


def plan_inputs(n, block, ctx_most, new_most, short, narrow=0):
    rng = np.random.default_rng(n * 1000 + block)
    low = -2 if n > 3 else 0
    ctx = [int(v) for v in rng.integers(low, ctx_most + 1, n)]
    new = [int(v) for v in rng.integers(low, new_most + 1, n)] if n > 1 else [new_most]
    width = max(1, -(-(ctx_most + new_most) // block) - narrow)
    need = sum(-(-(max(c, 0) + max(v, 0)) // block) for c, v in zip(ctx, new))
    pool = [int(v) for v in rng.permutation(need + 50)]
    table = [[-1] * width for _ in range(n)]
    for r, c in enumerate(ctx):
        for col in range(min(width, -(-max(c, 0) // block))):
            table[r][col] = pool.pop()
    return ctx, new, pool[:max(0, len(pool) - 40 - short)], table


def plan_program(lanes, block, ctx, new, free, table, max_tokens, gap=2, reverse=False, short=None, in_place=None):
    n, width = len(ctx), len(table[0])
    p = lanes.Program(reverse=reverse)
    i32, i64 = np.int32, np.int64

    def make(name, a):
        return p.buf(a, short=8 if short == name else 0)

    bc, bn, bf = make("ctx", np.array(ctx, i32)), make("new", np.array(new, i32)), make("free", np.array(free, i32))
    bt = make("table", rows_of(np.array(table, i32), width + gap, -77))
    bs = make("slots", np.full(max_tokens, -9, i64))
    outs = [make(name, np.full(k, -9, i32)) for name, k in (("request", max_tokens), ("position", max_tokens), ("seq_len", n), ("query_start", n + 1))]
    bl = make("totals", np.full(3, -9, i64))
    if in_place is not None:
        outs[2] = {"ctx": bc, "new": bn}[in_place]
    p.call("kv_plan", n, block, ("b", bc), ("b", bn), ("b", bf) if free else None, len(free), ("b", bt), width, width + gap, max_tokens, ("b", bs),
           *[("b", o) for o in outs], ("b", bl), None)
    got = p.run()
    assert p.codes == [0], p.messages
    return [rows_back(got[bt], n, width, width + gap).tolist(), got[bs].tolist(), *[got[o].tolist() for o in outs], got[bl].tolist()]


@pytest.mark.parametrize("n,block,ctx_most,new_most,pad,short", PLANS)
def test_kv_plan(lanes, n, block, ctx_most, new_most, pad, short):
    ctx, new, free, table = plan_inputs(n, block, ctx_most, new_most, short, 2 if n == 33 else 0)
    tokens = sum(max(v, 0) for v in new) + pad
    ref = plan_ref(block, ctx, new, free, table, tokens)
    for reverse in (False, True):
        got = plan_program(lanes, block, ctx, new, free, table, tokens, reverse=reverse)
        for what, g, r in zip(("table", "slots", "request", "position", "seq_len", "query_start", "totals"), got, ref):
            assert g == [list(v) for v in r] if what == "table" else g == list(r), what


@pytest.mark.parametrize("n,block,ctx_most,new_most,pad,short", PLANS)
@pytest.mark.parametrize("which", ["ctx", "new"])
def test_kv_plan_lengths_in_place(lanes, which, n, block, ctx_most, new_most, pad, short):
    # seq_len over one of the lengths it is made of: no workgroup may read it after it was written
    ctx, new, free, table = plan_inputs(n, block, ctx_most, new_most, short, 2 if n == 33 else 0)
    tokens = sum(max(v, 0) for v in new) + pad
    ref = plan_ref(block, ctx, new, free, table, tokens)
    for reverse in (False, True):
        got = plan_program(lanes, block, ctx, new, free, table, tokens, reverse=reverse, in_place=which)
        for what, g, r in zip(("table", "slots", "request", "position", "seq_len", "query_start", "totals"), got, ref):
            assert g == [list(v) for v in r] if what == "table" else g == list(r), what


def test_kv_plan_refuses_outputs_over_inputs(lanes):
    # one buffer of ints: ctx at 0, new at 8, free blocks at 16, a table of 2 x 3 with rows 8 apart at 32, the outputs behind
    n, tokens = 2, 4
    good = dict(ctx=0, new=8, free=16, table=32, slots=64, request=80, position=88, seq_len=96, query_start=104, totals=112)

    def code(**over):
        at = {**good, **over}
        p = lanes.Program()
        b = p.buf(np.concatenate([[5, 3], np.zeros(6), [3, 1], np.zeros(6), np.arange(16), np.zeros(128)]).astype(np.int32))
        a = {k: ("b", b, 4 * v) for k, v in at.items()}
        p.call("kv_plan", n, 4, a["ctx"], a["new"], a["free"], 5, a["table"], 3, 8, tokens, a["slots"], a["request"], a["position"], a["seq_len"],
               a["query_start"], a["totals"], None)
        p.run()
        return p.codes[0]

    assert code() == 0 and code(seq_len=0) == 0 and code(seq_len=8) == 0
    assert code(free=35) == 0 and code(ctx=36, new=44) == 0  # (between the table's rows)
    for over in (dict(seq_len=1), dict(seq_len=7), dict(seq_len=17), dict(query_start=0), dict(query_start=6), dict(query_start=20), dict(slots=2),
                 dict(slots=10), dict(request=1), dict(position=9), dict(position=13 + 5), dict(totals=4), dict(totals=6), dict(free=34), dict(free=38),
                 dict(ctx=41), dict(new=31), dict(new=34), dict(table=1), dict(table=18)):
        assert code(**over) == -5, over


def test_kv_plan_more_tokens_than_room(lanes):
    ctx, new, free, table = plan_inputs(300, 16, 300, 40, 0)
    tokens = sum(max(v, 0) for v in new)
    _, slots, req, pos, seq, start, totals = plan_ref(16, ctx, new, free, table, tokens)
    got = plan_program(lanes, 16, ctx, new, free, table, tokens - 1000)
    assert got[1:4] == [slots[:-1000], req[:-1000], pos[:-1000]] and got[4:] == [seq, start, totals]


@pytest.mark.parametrize("what", ["ctx", "new", "free", "table", "slots", "request", "position", "seq_len", "query_start", "totals"])
def test_kv_plan_short_operand_is_reported(lanes, what):
    ctx, new, free, table = plan_inputs(5, 8, 100, 900, 0)
    if what == "table":
        ctx[-1], new[-1] = 0, 8 * len(table[0])  # the last row is used to its end
    need = sum(-(-(c + v) // 8) - -(-c // 8) for c, v in zip(ctx, new))
    free = (free * 3)[:need]
    with pytest.raises(lanes.Fault):
        plan_program(lanes, 8, ctx, new, free, table, sum(new), short=what)


# --------------------------------------------------------------- kv_store
def cache_strides(layout, block, heads, dim):
    """Of a block, a token and a head, in elements."""
    return (block * heads * dim, heads * dim, dim) if layout == "thd" else (heads * block * dim, dim, block * dim)


def store_program(lanes, t, ct, tokens, heads, dim, block, layout, short=None):
    rng = np.random.default_rng(7)
    n_blocks = -(-tokens // block) + 1
    k, v = (stored(300 * rng.standard_normal((tokens, heads * dim)), t) for _ in range(2))
    k[0, 0], v[0, -1] = stored([1e6, 3e-6], t)  # past f16's range, and among its subnormals
    slots = rng.permutation(n_blocks * block)[:tokens].astype(np.int64)
    slots[0] = n_blocks * block - 1
    slots[1:][slots[1:] == slots[0]] = -1
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, n_blocks * block, -(2 ** 40)
    sk, sv = heads * dim + 5, heads * dim
    p = lanes.Program()

    def make(name, a):
        return p.buf(a, short=8 if short == name else 0)

    bk, bv, bs = make("k", rows_of(k, sk, STORED[t](1))), make("v", rows_of(v, sv, STORED[t](1))), make("slots", slots)
    size = n_blocks * block * heads * dim
    bkc, bvc = (make(name, np.full(size, STORED[ct](7))) for name in ("k_cache", "v_cache"))
    sb, st, sh = cache_strides(layout, block, heads, dim)
    p.call("kv_store", t, ct, tokens, heads, dim, ("b", bk), ("b", bv), sk, sv, ("b", bs), ("b", bkc), ("b", bvc), n_blocks, block, sb, st, sh, None)
    got = p.run()
    assert p.codes == [0], p.messages
    for src, b in ((k, bkc), (v, bvc)):
        ref = np.full(size, STORED[ct](7))
        for tok, slot in enumerate(slots.tolist()):
            if 0 <= slot < n_blocks * block:
                for h in range(heads):
                    at = slot // block * sb + slot % block * st + h * sh
                    ref[at:at + dim] = stored(values(src[tok, h * dim:(h + 1) * dim], t), ct)
        assert np.array_equal(got[b], ref)


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("ct", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("tokens,heads,dim,block,layout", [(1, 1, 8, 1, "thd"), (5, 3, 64, 16, "htd"), (70, 2, 20, 7, "thd"), (9, 1, 3, 4, "htd"),
                                                           (33, 5, 80, 24, "thd")])
def test_kv_store(lanes, t, ct, tokens, heads, dim, block, layout):
    store_program(lanes, t, ct, tokens, heads, dim, block, layout)


@pytest.mark.parametrize("dim", [64, 3])
@pytest.mark.parametrize("what", ["k", "v", "slots", "k_cache", "v_cache"])
def test_kv_store_short_operand_is_reported(lanes, dim, what):
    with pytest.raises(lanes.Fault):
        store_program(lanes, F32, BF16, 9, 3, dim, 4, "thd", short=what)


# -------------------------------------------------------- paged attention
def attention_problem(qt, ct, heads, kv, dim, block, lens, layout="thd", window=0, holes=(), widen=0, seed=3):
    rng = np.random.default_rng(seed)
    n = [-(-max(v, 0) // block) for v in lens]
    width, n_blocks, batch = max([1, *n]) + widen, sum(n) + 1, len(lens)
    order = rng.permutation(n_blocks)
    sb, st, sh = cache_strides(layout, block, kv, dim)
    caches = [np.full(n_blocks * block * kv * dim, stored([np.nan], ct)[0]) for _ in range(2)]
    table = np.full((batch, width), -1, np.int32)
    q = stored(rng.standard_normal((batch, heads, dim)), qt)
    scale = float(np.float32(1 / np.sqrt(dim)))
    rows, at = [], 0
    for r, length in enumerate(lens):
        pages = order[at:at + n[r]]
        at += n[r]
        table[r, :n[r]] = pages
        keys = [stored(rng.standard_normal((max(length, 0), kv, dim)), ct) for _ in range(2)]
        for tok in range(max(length, 0)):
            for cache, part in zip(caches, keys):
                for h in range(kv):
                    to = pages[tok // block] * sb + tok % block * st + h * sh
                    cache[to:to + dim] = part[tok, h]
        for col in holes:
            if col < n[r]:
                table[r, col] = -1 if col % 2 else n_blocks + 3
        rows.append(keys)
    return dict(qt=qt, ct=ct, heads=heads, kv=kv, dim=dim, block=block, lens=list(lens), window=window, holes=holes, n_blocks=n_blocks, width=width,
                strides=(sb, st, sh), caches=caches, table=table, q=q, scale=scale, rows=rows, batch=batch)


def attention_ref(a):
    qt, ct, dim, heads = a["qt"], a["ct"], a["dim"], a["heads"]
    ref, tol = np.zeros((a["batch"], heads, dim)), np.zeros((a["batch"], heads, dim))
    term = 2.0 ** -16 if ct == BF16 and qt == BF16 else 2.0 ** -20
    for r, length in enumerate(a["lens"]):
        seen = [t for t in range(max(length, 0)) if t // a["block"] not in a["holes"] and (not a["window"] or t >= length - a["window"])]
        if not seen:
            continue
        key, val = (np.repeat(values(x[seen], ct), heads // a["kv"], 1) for x in a["rows"][r])
        q = values(a["q"][r], qt)
        with np.errstate(invalid="ignore", over="ignore"):
            s = np.einsum("hd,thd->ht", q, key) * a["scale"]
            top = s.max(1, keepdims=True)
            p = np.exp(s - np.where(top == -np.inf, 0.0, top))
            total = p.sum(1, keepdims=True)
            p /= np.where(total == 0, 1.0, total)
            err = ((2.0 ** -21 + 4 * np.sqrt(dim) * U) * np.einsum("hd,thd->ht", np.abs(q), np.where(np.isfinite(key), np.abs(key), 0.0)) * abs(a["scale"])).max(1)
            ref[r] = np.einsum("ht,thd->hd", p, val)
            tol[r] = (2 * err[:, None] + term + 8 * np.sqrt(length) * U) * np.einsum("ht,thd->hd", p, np.abs(val))
    return ref, np.nan_to_num(tol) + HALF_ULP[qt] * 1.001 * np.nan_to_num(np.abs(ref)) + (2.0 ** -25 if qt == F16 else 1e-30)


def attention_run(lanes, a, cus=4, short=None, reverse=False, calls=1):
    heads, dim, batch, width = a["heads"], a["dim"], a["batch"], a["width"]
    sq, so, st = heads * dim + 8, heads * dim, width + 2
    p = lanes.Program(cus, reverse)

    def make(name, arr):
        return p.buf(arr, short=16 if short == name else 0)

    bq = make("q", rows_of(a["q"].reshape(batch, -1), sq, STORED[a["qt"]](1)))
    bk, bv = make("k", a["caches"][0]), make("v", a["caches"][1])
    bt, bl = make("table", rows_of(a["table"], st, 99)), make("lens", np.array(a["lens"], np.int32))
    bo = make("out", np.full(batch * so, STORED[a["qt"]](9)))
    for _ in range(calls):
        p.call("paged_attention", a["qt"], a["ct"], batch, heads, a["kv"], dim, ("b", bq), sq, ("b", bk), ("b", bv), a["n_blocks"], a["block"],
               *a["strides"], ("b", bt), width, st, ("b", bl), a["window"], a["scale"], ("b", bo), so, None)
    got = p.run()
    assert p.codes == [0] * calls, p.messages
    return values(got[bo].reshape(batch, heads, dim), a["qt"])


def attention_check(lanes, a, **kw):
    ref, tol = attention_ref(a)
    got = attention_run(lanes, a, **kw)
    close(got, ref, tol, "attention")
    return got


PAIRS = [(F32, F32), (F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)]


def pair(p):
    return NAMES[p[0]] + "_" + NAMES[p[1]] if isinstance(p, tuple) else None


@pytest.mark.parametrize("types", PAIRS, ids=pair)
@pytest.mark.parametrize("heads,kv,dim,block,lens,layout", [
    (1, 1, 64, 16, [1], "thd"), (4, 4, 8, 1, [0, 3, 33], "htd"), (6, 2, 40, 7, [31, 32, -5, 129], "thd"), (3, 1, 80, 50, [600, 5], "htd"),
    (3, 1, 136, 16, [100, 513], "thd"), (2, 2, 256, 32, [70, 530], "thd"),
    # groups of more heads than a workgroup takes, whole and split; the largest LDS
    (34, 2, 96, 16, [40, 700], "htd"), (16, 1, 256, 16, [20, 540], "thd")])
def test_paged_attention(lanes, types, heads, kv, dim, block, lens, layout):
    attention_check(lanes, attention_problem(*types, heads, kv, dim, block, lens, layout))


@pytest.mark.parametrize("types", [(F32, F16), (BF16, BF16), (F32, F32)], ids=pair)
def test_paged_attention_window_and_missing_blocks(lanes, types):
    attention_check(lanes, attention_problem(*types, 4, 2, 64, 16, [0, 1, 29, 400, 900], window=100))
    attention_check(lanes, attention_problem(*types, 2, 1, 64, 16, [29, 1500], window=700), reverse=True)
    got = attention_check(lanes, attention_problem(*types, 4, 2, 40, 8, [100, 300, 16, 9], holes=(0, 1, 5, 6, 7, 8, 20), widen=3))
    assert (got[2] == 0).all()


@pytest.mark.parametrize("types", PAIRS, ids=pair)
@pytest.mark.parametrize("dim,length", [(64, 50), (80, 50), (40, 33), (128, 600), (136, 40)])
def test_paged_attention_infinite_keys_and_queries(lanes, types, dim, length):
    # a score of -inf weighs nothing, one of +inf or NaN makes the head NaN, whatever
    # the head size and the types; nothing but scores of -inf: zeros
    inf = np.inf
    for scale in (0.125, -0.125):
        a = attention_problem(*types, 6, 2, dim, 16, [length, length, 1, length], seed=21)
        a["scale"], low = scale, -np.sign(scale)
        qt, ct = types
        q = np.abs(values(a["q"], qt)) + 0.1  # all of one sign, in d 0 and the last one of both
        q[:, 1, 0] *= -1
        q[1, 2, dim - 1] *= -1
        q[1, 3, 5] = 0
        q[1, 4, 5] = 1e-30 if qt == F32 else 1e-3  # (little next to the others, but something)
        q[3, 0, 7], q[3, 1, 7], q[3, 4, 7] = inf, -inf, np.nan
        a["q"] = stored(q, qt)
        puts = [(0, 7, 0, 0, low * inf), (0, 20, 1, dim - 1, low * inf), (1, 3, 0, dim - 1, low * inf), (1, 32, 1, 5, low * inf), (1, 4, 1, 0, low * inf),
                (2, 0, 0, 3, low * inf), (2, 0, 1, 3, -low * inf), (3, 9, 1, 8, low * inf)]
        sb, st, sh = a["strides"]
        for r, tok, h, d, v in puts:
            a["rows"][r][0][tok, h, d] = stored([v], ct)[0]
            a["caches"][0][a["table"][r, tok // 16] * sb + tok % 16 * st + h * sh + d] = stored([v], ct)[0]
        ref, tol = attention_ref(a)
        assert np.isnan(ref[0, 1]).all() and np.isfinite(ref[0, 0]).all() and np.isfinite(ref[0, 3:]).all()
        assert np.isnan(ref[1, 2]).all() and np.isnan(ref[1, 3]).all() and np.isfinite(ref[1, [0, 1, 4, 5]]).all()
        assert (ref[2, [0, 2]] == 0).all() and np.isnan(ref[2, 3:]).all()
        close(attention_run(lanes, a), ref, tol, (scale,))


@pytest.mark.parametrize("cus", [1, 4, 16, 256])
def test_paged_attention_splits(lanes, cus):
    # lists shared by one workgroup and by many, whole ones between split ones, empty requests among them
    attention_check(lanes, attention_problem(F16, F16, 2, 1, 64, 16, [700, 0, 33, 1200, 0, 520], widen=1), cus=cus)
    attention_check(lanes, attention_problem(BF16, BF16, 2, 2, 8, 16, [(i * 37) % 60 for i in range(70)]), cus=cus, reverse=True)


def test_paged_attention_has_a_workspace_of_its_own(lanes):
    # an attention on one stream must not write where a split GEMM's sums are on another
    a = attention_problem(F16, F16, 2, 1, 64, 16, [700])
    p = lanes.Program(cus=4)
    p.env["TML_GEMM_SPLIT"] = "4"
    gemm = [p.buf(np.zeros(n, np.float32)) for n in (32 * 2048, 2048 * 64, 32 * 64)]
    b = [p.buf(v) for v in (a["q"], a["caches"][0], a["caches"][1], a["table"], np.array(a["lens"], np.int32), np.zeros_like(a["q"]))]
    for _ in range(2):
        p.call("gemm", 0, 32, 64, 2048, ("b", gemm[0]), ("b", gemm[1]), 1.0, None, 0, None, ("b", gemm[2]), 1.0, 0.0, None)
        p.call("paged_attention", F16, F16, 1, 2, 1, 64, ("b", b[0]), 128, ("b", b[1]), ("b", b[2]), a["n_blocks"], 16, *a["strides"], ("b", b[3]),
               a["width"], a["width"], ("b", b[4]), 0, a["scale"], ("b", b[5]), 128, None)
    p.run()
    assert p.codes == [0] * 4, p.messages
    first, second, third, fourth = p.allocations
    assert second == first + 1 and second == third == fourth, p.allocations


@pytest.mark.parametrize("what", ["q", "k", "v", "table", "lens", "out"])
def test_paged_attention_short_operand_is_reported(lanes, what):
    a = attention_problem(F32, F16, 4, 2, 40, 8, [90, 96])
    # every block is used, the last one to its end
    a.update(n_blocks=24, caches=[c[:24 * 8 * 80] for c in a["caches"]], table=np.arange(24, dtype=np.int32).reshape(2, 12))
    with pytest.raises(lanes.Fault):
        attention_run(lanes, a, short=what)


# ------------------------------------------------------------- matvec_q4g
def matvec_program(lanes, xt, m, n, k, group, x_group=0, width=None, offset=0, yt=F32, bias=True, short=None, cus=256, reverse=False, edit=None):
    rng = np.random.default_rng(11)
    groups, x_groups = -(-k // group), -(-k // x_group) if x_group else 1
    x = rng.integers(-128, 128, (m, k)).astype(np.int8) if xt == I8 else stored(rng.standard_normal((m, k)), xt)
    xs = (0.01 * (0.5 + rng.random((m, x_groups)))).astype(np.float32)
    q, s = rng.integers(-8, 8, (n, k)), (0.01 * (0.5 + rng.random((n, groups)))).astype(np.float32)
    b = rng.standard_normal(n).astype(np.float32)
    if edit is not None:
        edit(q, s)
    width = -(-k // 32) * 16 if width is None else width
    rows = rng.integers(0, 256, (n, width)).astype(np.uint8)  # what follows a row's nibbles is noise
    u = (np.concatenate([q, np.full((n, k % 2), 10)], 1) & 15).astype(np.uint8)
    rows[:, :(k + 1) // 2] = u[:, 0::2] | u[:, 1::2] << 4
    p = lanes.Program(cus, reverse)

    def make(name, a):
        return p.buf(a, short=8 if short == name else 0)

    sx, sy = k + 1, n + 3
    bx = make("x", rows_of(x, sx, STORED[xt](1)))
    bxs = make("x_scales", xs) if xt == I8 else None
    bw = make("w", np.concatenate([np.zeros(offset, np.uint8), rows.reshape(-1)]))
    bs, bb = make("w_scales", s), make("bias", b) if bias else None
    by = make("y", rows_of(np.zeros((m, n), STORED[yt]), sy, STORED[yt](9)))

    def at(buf, off=0):
        return None if buf is None else ("b", buf, off)

    p.call("matvec_q4g", xt, m, n, k, at(bx), sx, at(bxs), x_group, at(bw, offset), width, at(bs), group, at(bb), yt, at(by), sy, None)
    got = p.run()
    assert p.codes == [0], p.messages
    xv = values(x, xt) * (xs.astype(np.float64)[:, np.arange(k) // (x_group or max(k, 1))] if xt == I8 else 1.0)
    w = q * s.astype(np.float64)[:, np.arange(k) // group]
    y, mass = xv @ w.T, np.abs(xv) @ np.abs(w).T
    if bias:
        y, mass = y + b, mass + np.abs(b)
    for r0 in range(m - 1):
        assert (got[by][r0 * sy + n:(r0 + 1) * sy] == STORED[yt](9)).all()
    out = values(rows_back(got[by], m, n, sy), yt)
    if edit is None:
        close(out, y, (2.0 ** -23 + 8 * np.sqrt(k) * U) * mass + HALF_ULP[yt] * 1.001 * np.abs(y) + (2.0 ** -25 if yt == F16 else 1e-30), (m, n, k))
    return out, q, s, xv


@pytest.mark.parametrize("xt", [F32, F16, BF16, I8], ids=tname)
@pytest.mark.parametrize("m,n,k,group,x_group", [
    (1, 1, 1, 32, 0), (1, 16, 32, 32, 32), (2, 17, 33, 32, 32), (3, 15, 127, 64, 0), (4, 33, 129, 32, 64), (5, 50, 1000, 96, 96), (1, 40, 1312, 32, 0),
    (8, 35, 640, 64, 64), (9, 20, 640, 128, 0), (16, 17, 512, 128, 128), (17, 20, 256, 32, 32), (33, 18, 96, 5000, 0), (2, 90, 200, 200, 0)])
def test_matvec_q4g(lanes, xt, m, n, k, group, x_group):
    matvec_program(lanes, xt, m, n, k, group, x_group)
    matvec_program(lanes, xt, m, n, k, group, x_group, cus=1, bias=False, yt=xt if xt != I8 else BF16, reverse=True)


@pytest.mark.parametrize("xt,m,k", [(F32, 1, 40000), (F32, 8, 6000), (BF16, 16, 6000), (I8, 16, 9300)])
def test_matvec_q4g_x_past_one_fill(lanes, xt, m, k):
    matvec_program(lanes, xt, m, 20, k, 64, 64 if xt == I8 else 0)


@pytest.mark.parametrize("xt", [F32, BF16, I8], ids=tname)
@pytest.mark.parametrize("k,width,offset", [(100, 50, 0), (101, 51, 0), (64, 32, 1), (1000, 501, 3), (33, 17, 0), (31, 16, 16), (40, 24, 0)])
def test_matvec_q4g_rows_anywhere(lanes, xt, k, width, offset):
    matvec_program(lanes, xt, 3, 21, k, 32, 32 if xt == I8 else 0, width=width, offset=offset)


@pytest.mark.parametrize("xt", [F32, F16, BF16, I8], ids=tname)
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
def test_matvec_q4g_infinite_scales(lanes, xt, group):
    # a scale multiplies the sum over each 32 of its group's columns (of f32 x, of each of
    # its terms), and these are added then
    k, n = 256, 18

    def edit(q, s):
        s[3, 0], s[7, -1] = np.inf, -np.inf

    y, q, s, x = matvec_program(lanes, xt, 2, n, k, group, bias=False, edit=edit)
    with np.errstate(invalid="ignore"):
        parts = np.einsum("mck,nck->mnc", x.reshape(2, k // 32, 32), q.reshape(n, k // 32, 32).astype(np.float64))
        want = (parts * s.astype(np.float64)[:, np.arange(k // 32) * 32 // group]).sum(2)
    assert not np.isfinite(want[:, [3, 7]]).any() and (group == 256 or np.isinf(want[:, [3, 7]]).any() or np.isnan(want).any())
    ok = np.isfinite(want)
    assert np.array_equal(np.isfinite(y), ok)
    if xt != F32:
        assert np.array_equal(np.isnan(y), np.isnan(want)) and np.array_equal(y[np.isinf(want)], want[np.isinf(want)])
    assert (np.abs(y[ok] - want[ok]) <= 1e-4 * np.abs(want[ok]) + 1e-3).all()


@pytest.mark.parametrize("width", [None, 501])
@pytest.mark.parametrize("what", ["x", "x_scales", "w", "w_scales", "bias", "y"])
def test_matvec_q4g_short_operand_is_reported(lanes, width, what):
    with pytest.raises(lanes.Fault):
        matvec_program(lanes, I8, 3, 21, 992, 32, 32, width=width and 496, offset=0 if width is None else 3, short=what)


# -------------------------------------------------------- quantize_groups
def quantize_program(lanes, n, k, group, short=None):
    rng = np.random.default_rng(13)
    w = rng.standard_normal((n, k)).astype(np.float32)
    w[0, :min(k, group)] = 0
    sw, sq, groups = k + 3, (k + 1) // 2 + 2, -(-k // group)
    p = lanes.Program()

    def make(name, a):
        return p.buf(a, short=4 if short == name else 0)

    bw, bq = make("w", rows_of(w, sw, np.float32(np.nan))), make("q", rows_of(np.zeros((n, (k + 1) // 2), np.uint8), sq, 0xEE))
    bs = make("scales", np.zeros((n, groups), np.float32))
    p.call("quantize_groups", n, k, group, ("b", bw), sw, ("b", bq), sq, ("b", bs), None)
    got = p.run()
    assert p.codes == [0], p.messages
    packed = rows_back(got[bq], n, (k + 1) // 2, sq)
    q = np.stack([packed & 15, packed >> 4], 2).reshape(n, -1)[:, :k].astype(np.int64)
    q = np.where(q > 7, q - 16, q)
    for g in range(groups):
        part = w[:, g * group:(g + 1) * group]
        most = np.abs(part).max(1)
        scale = np.where(most == 0, np.float32(1), most / np.float32(7))
        assert np.array_equal(got[bs][:, g], scale)
        assert (np.abs(q[:, g * group:(g + 1) * group] * scale[:, None].astype(np.float64) - part) <= scale[:, None] * (0.5 + 1e-5)).all()


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 33, 32), (5, 200, 64), (2, 700, 128), (9, 96, 96), (4, 50, 2),
                                       (3, 50, 2 ** 63 - 1), (2, 51, 2 ** 63 - 1)])
def test_quantize_groups(lanes, n, k, group):
    quantize_program(lanes, n, k, group)


@pytest.mark.parametrize("what", ["w", "q", "scales"])
def test_quantize_groups_short_operand_is_reported(lanes, what):
    with pytest.raises(lanes.Fault):
        quantize_program(lanes, 3, 65, 32, short=what)
