"""The operators around prompts, 4-bit caches and token scores on the GPU against
definitions in 64 bits (tests/serving_ref.py, and torch in float64 where sizes are large).

Tolerances, fixed by derivation (u = 2^-24; a result of f16 / bf16 is rounded once more):
  4-bit rows  bit for bit
  attention   serving_ref.attention: scores (2^-21 + 4 sqrt(D) u) sum |q k| scale, weights
              2^-20 (2^-16 for 16-bit outputs of a bf16 cache; a 16-bit type's half step
              where prompts' weights are rounded to it), sums 8 sqrt(len) u
  logprobs    sums 8 sqrt(cols) u, 4 u (1 + |log p|)
"""
import os
import sys

import numpy as np
import pytest

from tomoul_amd import _abi

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import serving_ref as ref  # noqa: E402
from serving_ref import BF16, F16, F32, HALF_ULP, STORED, TINY, close, stored, tname, values  # noqa: E402
from test_cpu_serving_more import COMBOS, ODD, Cache, check_logprobs, pool_index, pool_strides, rows_back, rows_of, wild  # noqa: E402

pytestmark = pytest.mark.gpu


def gpu(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a).view({2: np.int16, 4: np.int32}.get(a.dtype.itemsize, a.dtype) if a.dtype.kind in "fu" else a.dtype)).cuda()


def back(t, dtype):
    return t.cpu().numpy().view(dtype)


def sync():
    import torch
    torch.cuda.synchronize()


# --------------------------------------------------------------- 4-bit rows
@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("tokens,heads,dim,block,layout", [(1, 1, 32, 1, "thd"), (5, 3, 64, 8, "htd"), (333, 2, 96, 16, "thd"), (900, 5, 128, 4, "htd"),
                                                           (70, 1, 160, 3, "thd"), (30, 2, 192, 8, "htd"), (40, 1, 224, 8, "thd"), (111, 3, 256, 5, "htd")])
def test_store_and_load(t, tokens, heads, dim, block, layout):
    rng = np.random.default_rng(tokens * dim + t)
    n_blocks, row = -(-tokens // block) + 1, ref.row_bytes(dim)
    ks, vs = heads * dim + 3, 2 * heads * dim + 1
    k, v = (stored(wild(rng, (tokens, heads * dim)), t) for _ in range(2))
    slots = rng.permutation(n_blocks * block)[:tokens].astype(np.int64)
    if tokens > 2:
        slots[1], slots[2] = -1, n_blocks * block
    b, tk, h = pool_strides(layout, block, heads, row)
    gk, gv, gs = gpu(rows_of(k, ks, STORED[t](1))), gpu(rows_of(v, vs, STORED[t](1))), gpu(slots)
    ck, cv = gpu(np.full(n_blocks * b, 0xAB, np.uint8)), gpu(np.full(n_blocks * b, 0xCD, np.uint8))
    _abi.kv_store_q4_dev(t, tokens, heads, dim, gk.data_ptr(), gv.data_ptr(), ks, vs, gs.data_ptr(), ck.data_ptr(), cv.data_ptr(), n_blocks, block, b, tk, h)
    index = pool_index(layout, n_blocks, block, heads, row)
    want = [np.full(n_blocks * b, 0xAB, np.uint8), np.full(n_blocks * b, 0xCD, np.uint8)]
    live = [i for i, s in enumerate(slots) if 0 <= s < n_blocks * block]
    floats = []
    for w, x in ((0, k), (1, v)):
        rows = ref.pack_rows(values(x, t).astype(np.float32).reshape(tokens, heads, dim))[w]
        for i in live:
            for hd in range(heads):
                at = index[slots[i] // block, slots[i] % block, hd]
                want[w][at:at + row] = rows[i, hd]
        floats.append(ref.unpack_rows(rows, dim, w == 0)[0].reshape(tokens, -1))
    sync()
    assert np.array_equal(back(ck, np.uint8), want[0]) and np.array_equal(back(cv, np.uint8), want[1])
    for out_t in (F32, F16, BF16):
        so = heads * dim + out_t
        ok, ov = (gpu(np.full((tokens - 1) * so + heads * dim, 9, STORED[out_t])) for _ in range(2))
        _abi.kv_load_q4_dev(out_t, tokens, heads, dim, ck.data_ptr(), cv.data_ptr(), n_blocks, block, b, tk, h, gs.data_ptr(), ok.data_ptr(), ov.data_ptr(), so, so)
        sync()
        for w, o in ((0, ok), (1, ov)):
            got = rows_back(back(o, STORED[out_t]), tokens, heads * dim, so)
            with np.errstate(over="ignore"):
                expect = stored(floats[w].astype(np.float32), out_t)
            assert np.array_equal(values(got[live], out_t), values(expect[live], out_t), equal_nan=True)
            assert all((got[i] == 9).all() for i in range(tokens) if i not in set(live))


# ------------------------------------------------------ one token a request
def decode(cache_t, q_t, lens, heads, kv, dim, block, layout="thd", window=0, cap=0.0, slopes=False, lost=(), seed=0):
    rng = np.random.default_rng(seed)
    cache = Cache(rng, cache_t, lens, kv, dim, block, layout, window, lost)
    batch, scale = len(lens), float(np.float32(1 / np.sqrt(dim)))
    q = stored(1.5 * rng.standard_normal((batch, heads * dim)), q_t)
    sl = (2.0 ** -rng.uniform(0, 8, heads)).astype(np.float32) if slopes else None
    qs, os_ = heads * dim + 3, heads * dim + 1
    gq, go = gpu(rows_of(q, qs, STORED[q_t](1))), gpu(np.full((batch - 1) * os_ + heads * dim, 7, STORED[q_t]))
    gk, gv, gt, gl = gpu(cache.bytes[0]), gpu(cache.bytes[1]), gpu(cache.table), gpu(np.array(lens, np.int32))
    gs = gpu(sl) if slopes else None
    f = _abi.paged_attention_q4_dev if cache_t is None else _abi.paged_attention_ex_dev
    f(*((q_t,) if cache_t is None else (q_t, cache_t)), batch, heads, kv, dim, gq.data_ptr(), qs, gk.data_ptr(), gv.data_ptr(), cache.n_blocks, block, *cache.strides,
      gt.data_ptr(), cache.width, cache.width, gl.data_ptr(), scale, go.data_ptr(), os_, window=window, cap=cap, slopes_ptr=gs.data_ptr() if slopes else None)
    sync()
    flat = back(go, STORED[q_t])
    out = rows_back(flat, batch, heads * dim, os_)
    for r in range(batch - 1):
        assert (flat[r * os_ + heads * dim:(r + 1) * os_] == 7).all()
    # (over a 4-bit cache the weights of 16-bit outputs are rounded to f16)
    weight = 2.0 ** -16 if cache_t == BF16 and q_t == BF16 else 2.0 ** -11 if cache_t is None and q_t != F32 else 2.0 ** -20
    for r, length in enumerate(lens):
        pos = np.array([length - 1])
        t, k, v, km, vm = cache.of(r, length)
        want, tol = ref.attention(values(q[r], q_t).reshape(1, heads, dim), k, v, pos, scale=scale, cap=cap, slopes=sl, seen=ref.sees(pos, t, 0, window),
                                  positions=t, key_mag=km, val_mag=vm, weight=weight)
        close(values(out[r], q_t).reshape(want[0].shape), want[0], tol[0] + HALF_ULP[q_t] * (np.abs(want[0]) + tol[0]) + TINY[q_t], f"request {r}")


@pytest.mark.parametrize("q_t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_attention_q4(q_t, dim):
    decode(None, q_t, [0, 1, 33, 700, 2050], 4, 2, dim, 16, seed=dim)
    decode(None, q_t, [400, 5], 5, 5, dim, 7, layout="htd", seed=dim + 1)


SHAPES = [dict(lens=[900, 2, 333], heads=17, kv=1, block=1), dict(lens=[640, 31], heads=40, kv=2, block=32, layout="htd"),
          dict(lens=[1000, 20], heads=2, kv=1, block=8, window=190), dict(lens=[700, 3], heads=4, kv=2, block=16, cap=20.0),
          dict(lens=[700, 3], heads=4, kv=4, block=16, slopes=True), dict(lens=[700, 64], heads=4, kv=1, block=50, cap=2.0, slopes=True, window=400),
          dict(lens=[500, 600], heads=2, kv=2, block=8, lost=[(0, 0, -1), (0, 3, 1 << 30), (1, 7, 99999)]),
          dict(lens=[16, 8], heads=1, kv=1, block=8, lost=[(0, 0, -1), (0, 1, -7)]), dict(lens=[7000, 0, 13000], heads=3, kv=1, block=16),
          dict(lens=[1, 0, 40] * 70, heads=2, kv=2, block=16)]


@pytest.mark.parametrize("case", SHAPES, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items() if k != "lost").replace(" ", "")[:50])
def test_attention_q4_shapes(case):
    decode(None, F32, dim=64, seed=5, **case)
    decode(None, BF16, dim=128, seed=6, **case)


@pytest.mark.parametrize("q_t,cache_t", COMBOS, ids=tname)
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
def test_attention_ex(q_t, cache_t, dim):
    decode(cache_t, q_t, [700, 3, 0, 1300], 4, 2, dim, 16, cap=20.0, seed=dim)
    decode(cache_t, q_t, [333, 40], 3, 3, dim, 8, layout="htd", slopes=True, seed=dim + 1)
    decode(cache_t, q_t, [900, 70], 4, 1, dim, 16, cap=1.5, slopes=True, window=600, seed=dim + 2)


# ------------------------------------------------------------------ prompts
def prompt(q_t, cache_t, both, heads, kv, dim, block, layout="thd", prefix=None, window=0, cap=0.0, slopes=False, pad=2, lost=(), seed=0, odd=()):
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in both]
    cache = Cache(rng, cache_t, lens, kv, dim, block, layout, 0, lost)
    cache.put(odd)
    starts = np.concatenate([[0], np.cumsum([n for _, n in both])]).astype(np.int32)
    tokens, scale = int(starts[-1]) + pad, float(np.float32(1 / np.sqrt(dim)))
    q = stored(1.5 * rng.standard_normal((tokens, heads * dim)), q_t)
    sl = (2.0 ** -rng.uniform(0, 8, heads)).astype(np.float32) if slopes else None
    qs, os_ = heads * dim + 3, heads * dim + 1
    gq, go = gpu(rows_of(q, qs, STORED[q_t](1))), gpu(np.full((tokens - 1) * os_ + heads * dim, 7, STORED[q_t]))
    gk, gv, gt, gl, gst = gpu(cache.bytes[0]), gpu(cache.bytes[1]), gpu(cache.table), gpu(np.array(lens, np.int32)), gpu(starts)
    gs = gpu(sl) if slopes else None
    gp = gpu(np.array(prefix, np.int32)) if prefix is not None else None
    _abi.prompt_attention_dev(q_t, cache_t, tokens, len(both), heads, kv, dim, gq.data_ptr(), qs, gk.data_ptr(), gv.data_ptr(), cache.n_blocks, block, *cache.strides,
                              gt.data_ptr(), cache.width, cache.width, gst.data_ptr(), gl.data_ptr(), scale, go.data_ptr(), os_, window=window, cap=cap,
                              prefix_len_ptr=None if gp is None else gp.data_ptr(), slopes_ptr=gs.data_ptr() if slopes else None)
    sync()
    flat = back(go, STORED[q_t])
    out = rows_back(flat, tokens, heads * dim, os_)
    for r in range(tokens - 1):
        assert (flat[r * os_ + heads * dim:(r + 1) * os_] == 7).all()
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


@pytest.mark.parametrize("q_t,cache_t", COMBOS, ids=tname)
@pytest.mark.parametrize("dim", [8, 64, 80, 128, 136, 256])
def test_prompt_attention(q_t, cache_t, dim):
    prompt(q_t, cache_t, [(0, 5), (3, 0), (70, 9), (0, 1), (500, 130)], 4, 2, dim, 16, seed=dim, layout="htd" if dim % 16 else "thd")


PROMPTS = [dict(both=[(0, 450)], heads=1, kv=1, block=16), dict(both=[(300, 40), (0, 3), (0, 133)], heads=5, kv=1, block=8, layout="htd"),
           dict(both=[(10, 270)], heads=2, kv=2, block=300, prefix=[280]), dict(both=[(0, 190), (5, 20)], heads=2, kv=1, block=16, prefix=[100, 0]),
           dict(both=[(400, 140), (0, 20)], heads=2, kv=1, block=16, window=133), dict(both=[(0, 200)], heads=1, kv=1, block=1, window=7, prefix=[60]),
           dict(both=[(20, 150)], heads=2, kv=2, block=16, cap=3.0), dict(both=[(20, 150)], heads=2, kv=2, block=16, slopes=True, prefix=[70]),
           dict(both=[(64, 164), (0, 0), (1, 1)], heads=3, kv=3, block=64, cap=30.0, slopes=True, window=50, prefix=[100, 5, 2]),
           dict(both=[(160, 120), (0, 130)], heads=2, kv=2, block=8, lost=[(0, 0, -1), (0, 5, 1 << 30), (1, 2, 99999)]),
           dict(both=[(0, 16)], heads=1, kv=1, block=8, lost=[(0, 0, -1), (0, 1, -7)]), dict(both=[(0, 1)] * 170, heads=2, kv=1, block=4),
           dict(both=[(2000, 1), (1500, 1), (0, 1)], heads=16, kv=2, block=16)]


@pytest.mark.parametrize("case", PROMPTS, ids=lambda c: "-".join(f"{k}{v}" for k, v in c.items() if k != "lost").replace(" ", "")[:50])
def test_prompt_attention_shapes(case):
    prompt(F16, F16, dim=64, seed=3, **case)
    prompt(BF16, BF16, dim=128, seed=3, **case)
    prompt(F32, BF16, dim=40, seed=4, **case)
    prompt(F32, F32, dim=64, seed=5, **case)


@pytest.mark.parametrize("q_t,cache_t", COMBOS, ids=tname)
def test_prompt_attention_infinities_and_nan_are_for_those_who_see_them(q_t, cache_t):
    odd = [o for o in ODD if o[2] == 1 or np.isnan(o[5]) or q_t == cache_t]
    for dim in (40, 64, 128, 256):
        prompt(q_t, cache_t, [(60, 90)], 4, 2, dim, 16, odd=odd, seed=7)
        prompt(q_t, cache_t, [(60, 90)], 2, 2, dim, 16, odd=odd, window=30, prefix=[110], seed=8)


# ----------------------------------------------------------------- logprobs
def logprobs(t, x, top, tokens, stride_pad=1):
    import torch
    x = stored(x, t)
    rows, cols = x.shape
    gx, gt = gpu(rows_of(x, cols + stride_pad, STORED[t](1))), gpu(np.array(tokens, np.int32))
    gl, ge = torch.full((rows,), 5.0, device="cuda"), torch.full((rows,), 5.0, device="cuda")
    gi, gp = torch.full((rows, max(top, 1)), 77, dtype=torch.int32, device="cuda"), torch.full((rows, max(top, 1)), 5.0, device="cuda")
    _abi.token_logprobs_dev(t, rows, cols, gx.data_ptr(), cols + stride_pad, tokens_ptr=gt.data_ptr(), logprobs_ptr=gl.data_ptr(), entropy_ptr=ge.data_ptr(),
                            top=top, top_ids_ptr=gi.data_ptr(), top_logprobs_ptr=gp.data_ptr())
    sync()
    check_logprobs(values(x, t), tokens, top, gl.cpu().numpy(), ge.cpu().numpy(), gi.cpu().numpy(), gp.cpu().numpy())


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("cols,top", [(1, 0), (1, 3), (7, 7), (8, 1), (9, 64), (63, 5), (511, 64), (520, 20), (2049, 5), (2500, 64), (8195, 20), (51866, 5),
                                      (51866, 0), (131072, 64)])
def test_logprobs(t, cols, top):
    rng = np.random.default_rng(cols + top)
    x = 3 * rng.standard_normal((3, cols))
    x[1] = np.round(x[1])  # equal ones
    x[2, rng.integers(cols)] += 30
    logprobs(t, x, top, [cols // 2, -1 if cols > 1 else 0, cols])


@pytest.mark.parametrize("cols,top", [(70, 5), (600, 64), (2100, 3), (9000, 8)])
def test_logprobs_odd_rows(cols, top):
    inf = np.inf
    rng = np.random.default_rng(cols)
    x = rng.standard_normal((10, cols))
    x[0] = 2.5
    x[1] = np.arange(cols) / 100
    x[2] = -np.arange(cols) / 100
    x[3] = -inf
    x[4, rng.permutation(cols)[:cols - 2]] = -inf
    x[5] = -3.38e38
    x[6, :-1] = -3.38e38
    x[7, 3] = np.nan
    x[8, 4] = inf
    x[9] = np.nan
    logprobs(F32, x, top, [0] * 10)
    logprobs(BF16, x, top, [cols - 1] * 10)
    y = np.zeros((1, cols))
    y[0, ::2] = -0.0
    logprobs(F16, y, top, [1])


def test_logprobs_more_candidates_than_are_held():
    cols = 16 * 64 * 8 * 4
    x = np.full(cols, -1.0).reshape(-1, 1024, 8)
    x[:, :63] = 2.0
    x[:, 63] = 1.5
    logprobs(F16, x.reshape(1, cols), 64, [5])


def test_logprobs_many_rows():
    x = np.random.default_rng(5).standard_normal((1100, 9001))
    logprobs(BF16, x, 0, list(range(1100)))


@pytest.mark.parametrize("q_t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("dim,heads,kv", [(32, 5, 1), (64, 12, 2), (96, 17, 1), (128, 6, 1), (128, 16, 2), (160, 7, 1), (256, 9, 1)])
def test_attention_q4_wide_groups(q_t, dim, heads, kv):
    decode(None, q_t, [70, 0, 1600, 33], heads, kv, dim, 16, cap=20.0 if dim == 128 else 0.0, slopes=dim == 64, seed=dim + heads)
