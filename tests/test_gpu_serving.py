"""The serving operators (kv_plan, kv_store, paged_attention, rmsnorm,
matvec_q4g, quantize_groups) on the GPU against plain implementations in 64
bits or whole numbers.

Tolerances, fixed by derivation (u = 2^-24, the unit roundoff of fp32; a result
of f16 / bf16 is rounded once more, by 2^-11 / 2^-8 of itself):
  rmsnorm    h one rounding; the sum of squares of n columns in a tree of runs
             of at most 32, relative error <= (32 + 16) u, halved by the root;
             four more roundings: |dy| <= 32 u |y|
  matvec     2^-23 of each |x w| for the split (f16, bf16, 8 bits: none), and the
             sum's roundings: at most K / 8 additions into one fp32 of a lane,
             random in sign, 8 sqrt(K) u of sum |x w| bounds them with room
  attention  scores: (2^-21 + 4 sqrt(D) u) sum |q k| * scale absolute, that is
             relative to the weights; values: the weights' terms (2^-16 for
             16-bit outputs of a bf16 cache, 2^-20 else) and the sum's roundings
             8 sqrt(len) u, of sum p |v|
"""
import math

import numpy as np
import pytest

from tomoul_amd import _abi

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, F16, BF16, I8 = _abi.TYPE_F32, _abi.TYPE_F16, _abi.TYPE_BF16, _abi.TYPE_I8
NAMES = {F32: "f32", F16: "f16", BF16: "bf16", I8: "i8"}
HALF_ULP = {F32: U, F16: 2.0 ** -11, BF16: 2.0 ** -8}


def tname(t):
    return NAMES[t]


def dt(t):
    import torch
    return {F32: torch.float32, F16: torch.float16, BF16: torch.bfloat16, I8: torch.int8}[t]


def gen(seed):
    import torch
    g = torch.Generator()
    g.manual_seed(seed)
    return g


def randn(seed, *shape):
    import torch
    return torch.randn(*shape, generator=gen(seed), dtype=torch.float64)


def padded(x, pad, fill):
    """x (2-D, CPU) on the GPU with rows `pad` elements further apart, and its row stride."""
    import torch
    big = torch.full((x.shape[0], x.shape[1] + pad), fill, dtype=x.dtype, device="cuda")
    big[:, :x.shape[1]] = x.cuda()
    return big, big.stride(0)


def ptr(t):
    return None if t is None else t.data_ptr()


def close(got, ref, tol, what=""):
    import torch
    got, ref = got.double().cpu(), ref.double().cpu()
    assert torch.equal(torch.isnan(got), torch.isnan(ref)), what
    bad = (got - ref).abs() > tol
    bad &= ~(torch.isinf(ref) & (got == ref)) & ~torch.isnan(ref)
    assert not bad.any(), (what, int(bad.sum()), float(((got - ref).abs() / tol.clamp(min=1e-300))[bad].max()))


# ---------------------------------------------------------------- rmsnorm
def norm_ref(x, r, w, eps):
    h = x.double() + (r.double() if r is not None else 0.0)
    y = h / torch_sqrt(h.square().mean(1, keepdim=True) + eps)
    return h, y * w.double() if w is not None else y


def torch_sqrt(v):
    import torch
    return torch.sqrt(v)


def run_norm(t, x, r, w, eps, out_t, group=0, pad=0, alias=None):
    import torch
    rows, cols = x.shape
    gx, sx = padded(x, pad, float("nan"))
    gr, sr = padded(r, pad + 1, float("nan")) if r is not None else (None, 0)
    gw = w.float().cuda() if w is not None else None
    if alias == "x":
        gs, ss = gx, sx
    elif alias == "r":
        gs, ss = gr, sr
    elif alias == "none":
        gs, ss = None, 0
    else:
        gs, ss = padded(torch.zeros(rows, cols, dtype=dt(t)), 3, 7.0)
    go, so = padded(torch.zeros(rows, cols, dtype=dt(out_t)), pad, 5)
    width = group if group else max(cols, 1)
    scales = torch.full((rows, -(-cols // width)), -1.0, device="cuda") if out_t == I8 else None
    _abi.rmsnorm_dev(t, rows, cols, gx.data_ptr(), sx, ptr(gw), eps, out_t, go.data_ptr(), so, residual_ptr=ptr(gr),
                     residual_stride=sr, sum_ptr=ptr(gs), sum_stride=ss, scales_ptr=ptr(scales), group=group)
    torch.cuda.synchronize()
    if alias is None:
        assert (gs[:, cols:] == 7).all()
    assert (go[:, cols:] == 5).all()
    return (None if gs is None else gs[:, :cols].cpu()), go[:, :cols].cpu(), None if scales is None else scales.cpu()


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 8), (5, 9), (1, 100), (3, 511), (2, 513), (1, 1280), (1030, 1237), (3, 2049), (2, 5120),
                                       (1, 8192), (2, 8193), (1, 20011), (1, 32768), (1, 33001), (2050, 1032)])
def test_rmsnorm(t, rows, cols):
    x, r, w = randn(1, rows, cols).to(dt(t)), (3 * randn(2, rows, cols)).to(dt(t)), 1 + 0.2 * randn(3, cols)
    for res, wt, alias in ((r, w, None), (None, None, "none"), (r, w, "x"), (r, None, "r")):
        s, y, _ = run_norm(t, x, res, wt, 1e-6, t, pad=cols % 3, alias=alias)
        h, ref = norm_ref(x, res, wt.float() if wt is not None else None, 1e-6)
        if s is not None:
            close(s, h, HALF_ULP[t] * 1.001 * h.abs() + 1e-30, "sum")
        close(y, ref, (HALF_ULP[t] * 1.001 + 32 * U) * ref.abs() + 2.0 ** -25 * (t == F16), "out")


@pytest.mark.parametrize("t,out_t", [(BF16, F32), (F16, BF16), (F32, F16)], ids=tname)
def test_rmsnorm_other_output_type(t, out_t):
    x = randn(4, 4, 300).to(dt(t))
    _, y, _ = run_norm(t, x, None, None, 1e-5, out_t, alias="none")
    _, ref = norm_ref(x, None, None, 1e-5)
    close(y, ref, (HALF_ULP[out_t] * 1.001 + 32 * U) * ref.abs() + 2.0 ** -25)


@pytest.mark.parametrize("t", [F32, BF16], ids=tname)
@pytest.mark.parametrize("rows,cols,group", [(1, 1, 0), (3, 7, 0), (2, 7, 3), (4, 64, 8), (2, 1280, 128), (1100, 1280, 32), (3, 1237, 0), (3, 1237, 64),
                                             (2, 4096, 4096), (2, 5120, 0), (2, 5120, 512), (3, 5120, 96), (1, 8200, 1024), (1, 33000, 128), (1, 40, 1),
                                             (1, 96, 100), (1100, 1000, 64)])
def test_rmsnorm_8_bits(t, rows, cols, group):
    import torch
    x, r, w = randn(5, rows, cols).to(dt(t)), (2 * randn(6, rows, cols)).to(dt(t)), 1 + 0.2 * randn(7, cols)
    _, q, scales = run_norm(t, x, r, w, 1e-6, I8, group=group)
    _, ref = norm_ref(x, r, w.float(), 1e-6)
    width = min(group, cols) if group else cols
    for g in range(scales.shape[1]):
        part = ref[:, g * width:(g + 1) * width]
        most = part.abs().amax(1)
        close(scales[:, g], most / 127, 40 * U * most / 127, "scale")
        exact = part / (most / 127)[:, None]
        # off by at most the half that rounding takes, and the error of y and the scale
        assert ((q[:, g * width:(g + 1) * width].double() - exact).abs() <= 0.5 + 127 * 80 * U).all()
        assert (q[:, g * width:(g + 1) * width].abs().amax(1) == 127).all()
    assert torch.equal(q, q.clamp(-127, 127))


def test_rmsnorm_zeros_infinities_nan():
    import torch
    nan, inf = float("nan"), float("inf")
    x = torch.ones(6, 256, dtype=torch.float32)
    x[0] = 0
    x[1, 5] = nan
    x[2, 9] = inf
    x[3] = 1e-30
    x[4, 128:] = 0
    _, y, _ = run_norm(F32, x, None, None, 0.0, F32, alias="none")
    assert torch.isnan(y[0]).all() and torch.isnan(y[1]).all() and torch.isnan(y[2, 9]) and (y[2, :9] == 0).all()
    for eps, group in ((1e-6, 0), (1e-6, 64), (1e-6, 96)):
        _, q, s = run_norm(F32, x, None, None, eps, I8, group=group)
        assert (q[0] == 0).all() and (s[0] == 1).all()
        assert (q[1] == 0).all() and torch.isnan(s[1]).all()
        assert torch.isnan(s[2, 0]) and (q[2] == 0).all()
        assert (q[5] == 127).all()
        if group == 64:
            assert (s[4, 2:] == 1).all() and (q[4, 128:] == 0).all() and (q[4, :128] == 127).all()


def test_rmsnorm_refusals():
    import torch
    x = torch.ones(4, 64, device="cuda")
    p = x.data_ptr()

    def call(code, *a, **kw):
        with pytest.raises(_abi.TmlError) as e:
            _abi.rmsnorm_dev(*a, **kw)
        assert e.value.code == code, str(e.value)

    call(_abi.TML_ERR_INVALID_FORMAT, I8, 4, 64, p, 64, None, 1e-6, F32, p, 64)
    call(_abi.TML_ERR_INVALID_FORMAT, F32, 4, 64, p, 64, None, 1e-6, 9, p, 64)
    call(_abi.TML_ERR_INVALID_SHAPE, F32, -1, 64, p, 64, None, 1e-6, F32, p, 64)
    call(_abi.TML_ERR_INVALID_SHAPE, F32, 4, 64, p, 63, None, 1e-6, F32, p, 64)
    call(_abi.TML_ERR_INVALID_SHAPE, F32, 4, 64, p, 64, None, 1e-6, F32, p, 64, residual_ptr=p, residual_stride=9)
    call(_abi.TML_ERR_INVALID_ARG, F32, 4, 64, None, 64, None, 1e-6, F32, p, 64)
    call(_abi.TML_ERR_INVALID_ARG, F32, 4, 64, p, 64, None, 1e-6, I8, p, 64)
    call(_abi.TML_ERR_INVALID_SHAPE, F32, 4, 64, p, 64, None, 1e-6, I8, p, 64, scales_ptr=p, group=-1)
    call(_abi.TML_ERR_INVALID_SHAPE, F32, 1, 40000, p, 40000, None, 1e-6, I8, p, 40000, scales_ptr=p, group=2)
    _abi.rmsnorm_dev(F32, 0, 64, None, 64, None, 1e-6, F32, None, 64)
    _abi.rmsnorm_dev(F32, 4, 0, None, 64, None, 1e-6, F32, None, 64)


# ---------------------------------------------------------------- kv_plan
def plan_ref(block, ctx, new, free, table, max_tokens):
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    slots, req, pos, seq, start = [], [], [], [], [0]
    used = wide = 0
    for r, (c, n) in enumerate(zip(ctx, new)):
        c, n = max(c, 0), max(n, 0)
        need = -(-(c + n) // block)
        wide += need > width
        for col in range(min(-(-c // block), width), min(need, width)):
            table[r][col] = free[used] if used < len(free) else -1
            used += 1
        for j in range(n):
            p = c + j
            col = p // block
            page = table[r][col] if col < width else -1
            slots.append(page * block + p % block if page >= 0 else -1)
            req.append(r)
            pos.append(p)
        seq.append(c + n)
        start.append(start[-1] + n)
    pad = [-1] * (max_tokens - len(slots))
    return table, slots + pad, req + pad, pos + pad, seq, start, [start[-1], used, wide]


def run_plan(block, ctx, new, free, table, max_tokens, stride_pad=0, optional=True):
    import torch
    n, width = len(ctx), len(table[0]) if table else 0
    i32 = dict(dtype=torch.int32, device="cuda")
    big = torch.full((n, width + stride_pad), -77, **i32)
    if n and width:
        big[:, :width] = torch.tensor(table, dtype=torch.int32)
    c, f, fr = torch.tensor(ctx, **i32), torch.tensor(new, **i32), torch.tensor(free, **i32)
    slots = torch.full((max_tokens + 1,), -9, dtype=torch.int64, device="cuda")
    outs = [torch.full((k + 1,), -9, **i32) for k in (max_tokens, max_tokens, n, n + 1)]
    totals = torch.full((4,), -9, dtype=torch.int64, device="cuda")
    _abi.kv_plan_dev(n, block, ptr(c), ptr(f), ptr(fr), len(free), big.data_ptr(), width, width + stride_pad, max_tokens, slots.data_ptr(),
                     **(dict(token_request_ptr=ptr(outs[0]), positions_ptr=ptr(outs[1]), seq_len_ptr=ptr(outs[2]), query_start_ptr=ptr(outs[3]),
                             totals_ptr=ptr(totals)) if optional else {}))
    torch.cuda.synchronize()
    for o in [slots, *outs, totals]:
        assert int(o[-1]) == -9  # nothing past the end
    assert (big[:, width:] == -77).all()
    return [big[:, :width].tolist(), slots[:-1].tolist(), *[o[:-1].tolist() for o in outs], totals[:-1].tolist()]


@pytest.mark.parametrize("n,block,ctx_most,new_most,pad,short", [
    (1, 16, 0, 1, 0, 0), (1, 1, 5, 7, 3, 0), (64, 16, 500, 1, 0, 0), (300, 16, 300, 40, 17, 0), (257, 7, 64, 9, 1000, 0), (700, 100, 900, 3, 5, 0),
    (5, 32, 100, 3000, 11, 0), (33, 16, 200, 60, 9, 40), (12, 4, 40, 30, 2, 1000000), (1000, 16, 40, 0, 4, 0)])
def test_kv_plan(n, block, ctx_most, new_most, pad, short):
    rng = np.random.default_rng(n * 1000 + block)
    ctx = [int(v) for v in rng.integers(-2 if n > 3 else 0, ctx_most + 1, n)]
    new = [int(v) for v in rng.integers(-1 if n > 3 else 0, new_most + 1, n)]
    if n == 1:
        new = [new_most]
    width = max(1, -(-(ctx_most + new_most) // block) - (2 if n == 33 else 0))
    need = sum(-(-(max(c, 0) + max(v, 0)) // block) for c, v in zip(ctx, new))
    pool = [int(v) for v in rng.permutation(need + 50)]
    table = [[-1] * width for _ in range(n)]
    for r, c in enumerate(ctx):
        for col in range(min(width, -(-max(c, 0) // block))):
            table[r][col] = pool.pop()
    if n > 20:
        table[7][0] = -5  # an evicted block
    free = pool[:max(0, len(pool) - 40 - short)]
    tokens = sum(max(v, 0) for v in new)
    ref = plan_ref(block, ctx, new, free, table, tokens + pad)
    got = run_plan(block, ctx, new, free, table, tokens + pad, stride_pad=n % 3)
    for what, g, r in zip(("table", "slots", "request", "position", "seq_len", "query_start", "totals"), got, ref):
        assert g == [list(v) for v in r] if what == "table" else g == list(r), what
    # a second call on its own result finds the same blocks and hands out the same slots
    again = run_plan(block, ctx, new, free, got[0], tokens + pad, optional=False)
    assert again[:2] == got[:2]


def test_kv_plan_edges():
    import torch
    got = run_plan(16, [], [], [], [], 5)
    assert got[1] == [-1] * 5 and got[5] == [0] and got[6] == [0, 0, 0]
    got = run_plan(16, [3, 4], [2, 1], [9], [[1], [2]], 0)  # no room for tokens: the totals still say so
    assert got[6] == [3, 0, 0] and got[0] == [[1], [2]]
    big = 2 ** 31 - 1
    got = run_plan(16, [big, 0], [big, 2], [4, 5], [[3], [6]], 1)
    assert got[6] == [big + 2, 1, 1] and got[4] == [big, 2] and got[1] == [-1] and got[3] == [big] and got[0] == [[3], [6]]
    p = torch.zeros(8, dtype=torch.int64, device="cuda").data_ptr()
    for code, a in ((_abi.TML_ERR_INVALID_SHAPE, (-1, 16, p, p, p, 1, p, 1, 1, 1, p)), (_abi.TML_ERR_INVALID_ARG, (1, 0, p, p, p, 1, p, 1, 1, 1, p)),
                    (_abi.TML_ERR_INVALID_ARG, (1, 16, None, p, p, 1, p, 1, 1, 1, p)), (_abi.TML_ERR_INVALID_ARG, (1, 16, p, p, None, 1, p, 1, 1, 1, p)),
                    (_abi.TML_ERR_INVALID_ARG, (1, 16, p, p, p, 1, p, 1, 1, 1, None)), (_abi.TML_ERR_INVALID_SHAPE, (2, 16, p, p, p, 1, p, 4, 3, 1, p))):
        with pytest.raises(_abi.TmlError) as e:
            _abi.kv_plan_dev(*a)
        assert e.value.code == code


# --------------------------------------------------------------- kv_store
def cache_like(t, n_blocks, block, heads, dim, layout, fill):
    """[block, token, head, dim] on the GPU in either order."""
    import torch
    if layout == "thd":
        return torch.full((n_blocks, block, heads, dim), fill, dtype=dt(t), device="cuda")
    return torch.full((n_blocks, heads, block, dim), fill, dtype=dt(t), device="cuda").permute(0, 2, 1, 3)


@pytest.mark.parametrize("t", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("ct", [F32, F16, BF16], ids=tname)
@pytest.mark.parametrize("tokens,heads,dim,block,layout", [(1, 1, 8, 1, "thd"), (5, 3, 64, 16, "htd"), (70, 2, 20, 7, "thd"), (33, 5, 80, 24, "htd"),
                                                           (9, 1, 3, 4, "htd"), (300, 8, 128, 16, "thd")])
def test_kv_store(t, ct, tokens, heads, dim, block, layout):
    import torch
    n_blocks = -(-tokens // block) + 2
    k, v = (randn(s, tokens, heads * dim) * 300 for s in (8, 9))
    k[0, 0], v[0, -1] = 1e6, 3e-6  # past f16's range, and among its subnormals
    k, v = k.to(dt(t)), v.to(dt(t))
    gk, sk = padded(k, 5, 1.0)
    gv, sv = padded(v, 0, 1.0)
    slots = torch.randperm(n_blocks * block, generator=gen(10))[:tokens]
    if tokens > 3:
        slots[1], slots[2], slots[3] = -1, n_blocks * block, -(2 ** 40)
    kc, vc = (cache_like(ct, n_blocks, block, heads, dim, layout, 7.0) for _ in range(2))
    _abi.kv_store_dev(t, ct, tokens, heads, dim, gk.data_ptr(), gv.data_ptr(), sk, sv, slots.cuda().data_ptr(), kc.data_ptr(), vc.data_ptr(), n_blocks,
                      block, kc.stride(0), kc.stride(1), kc.stride(2))
    torch.cuda.synchronize()
    for src, got in ((k, kc), (v, vc)):
        ref = torch.full((n_blocks * block, heads, dim), 7.0, dtype=dt(ct))
        ok = (slots >= 0) & (slots < n_blocks * block)
        ref[slots[ok]] = src[ok].view(-1, heads, dim).to(dt(ct))
        assert torch.equal(got.cpu().reshape(-1, heads, dim), ref)


def test_kv_store_refusals():
    import torch
    x = torch.zeros(64, device="cuda")
    p = x.data_ptr()
    ok = [F32, F32, 2, 1, 8, p, p, 8, 8, p, p, p, 2, 2, 16, 8, 8]
    for at, value, code in ((0, I8, _abi.TML_ERR_INVALID_FORMAT), (1, 7, _abi.TML_ERR_INVALID_FORMAT), (2, -1, _abi.TML_ERR_INVALID_SHAPE),
                            (5, None, _abi.TML_ERR_INVALID_ARG), (9, None, _abi.TML_ERR_INVALID_ARG), (13, 0, _abi.TML_ERR_INVALID_ARG),
                            (7, 7, _abi.TML_ERR_INVALID_SHAPE), (14, -16, _abi.TML_ERR_INVALID_SHAPE), (12, 2 ** 31, _abi.TML_ERR_INVALID_SHAPE)):
        a = list(ok)
        a[at] = value
        with pytest.raises(_abi.TmlError) as e:
            _abi.kv_store_dev(*a)
        assert e.value.code == code, at
    a = list(ok)
    a[2], a[5] = 0, None
    _abi.kv_store_dev(*a)


# -------------------------------------------------------- paged attention
class Attn:
    """One attention problem: the cache, its tables, and the result in 64 bits."""

    def __init__(self, qt, ct, heads, kv, dim, block, lens, layout="thd", window=0, seed=1, holes=(), widen=0, loud=1.0):
        import torch
        self.qt, self.ct, self.heads, self.kv, self.dim, self.block, self.window = qt, ct, heads, kv, dim, block, window
        self.batch = len(lens)
        self.lens = lens
        n = [-(-max(v, 0) // block) for v in lens]
        width = max([1, *n]) + widen
        self.n_blocks = sum(n) + 2
        order = torch.randperm(self.n_blocks, generator=gen(seed)).to(torch.int32)
        self.k, self.v = (cache_like(ct, self.n_blocks, block, kv, dim, layout, float("nan")) for _ in range(2))
        self.table = torch.full((self.batch, width), -1, dtype=torch.int32)
        self.q = (loud * randn(seed + 1, self.batch, heads, dim)).to(dt(qt))
        self.scale = 1 / math.sqrt(dim)
        self.out = torch.full((self.batch, heads * dim + 8), 9.0, dtype=dt(qt), device="cuda")
        ref, tol = torch.zeros(self.batch, heads, dim, dtype=torch.float64), torch.zeros(self.batch, heads, dim, dtype=torch.float64)
        at = 0
        for r, length in enumerate(lens):
            self.table[r, :n[r]] = order[at:at + n[r]]
            at += n[r]
            if length <= 0:
                continue
            pages = self.table[r, :n[r]].long()
            key, val = (randn(seed * 100 + r + s, length, kv, dim).to(dt(ct)) for s in (10, 50))
            for cache, rows in ((self.k, key), (self.v, val)):
                full = torch.full((n[r] * block, kv, dim), float("nan"), dtype=dt(ct))
                full[:length] = rows
                cache[pages.cuda()] = full.view(n[r], block, kv, dim).cuda()
            for col in holes:
                if col < n[r]:
                    self.table[r, col] = -1 if col % 2 else self.n_blocks + 3
            t = torch.arange(length)
            hole = torch.tensor([c in holes for c in range(n[r])])[t // block]
            seen = ~hole & (t >= length - window if window else True)
            t = t[seen]
            if not len(t):
                continue
            q = self.q[r].double()
            kk = key[t].double().repeat_interleave(heads // kv, 1)
            vv = val[t].double().repeat_interleave(heads // kv, 1)
            s = torch.einsum("hd,thd->ht", q, kk) * self.scale
            p = torch.softmax(s, 1)
            ref[r] = torch.einsum("ht,thd->hd", p, vv)
            mass = torch.einsum("ht,thd->hd", p, vv.abs())
            score_err = ((2.0 ** -21 + 4 * math.sqrt(dim) * U) * torch.einsum("hd,thd->ht", q.abs(), kk.abs()) * self.scale).amax(1)
            term = 2.0 ** -16 if ct == BF16 and qt == BF16 else 2.0 ** -20
            tol[r] = (2 * score_err[:, None] + term + 8 * math.sqrt(length) * U) * mass
        self.ref, self.tol = ref, tol + HALF_ULP[qt] * 1.001 * ref.abs() + (2.0 ** -25 if qt == F16 else 1e-30)
        self.gq, self.gt = self.q.reshape(self.batch, -1).cuda(), self.table.cuda()
        self.gl = torch.tensor(lens, dtype=torch.int32, device="cuda")

    def args(self):
        return (self.qt, self.ct, self.batch, self.heads, self.kv, self.dim, self.gq.data_ptr(), self.gq.stride(0), self.k.data_ptr(), self.v.data_ptr(),
                self.n_blocks, self.block, self.k.stride(0), self.k.stride(1), self.k.stride(2), self.gt.data_ptr(), self.gt.shape[1],
                self.gt.stride(0), self.gl.data_ptr(), self.scale, self.out.data_ptr(), self.out.stride(0))

    def run(self, stream=None):
        import torch
        _abi.paged_attention_dev(*self.args(), window=self.window, stream=stream)
        torch.cuda.synchronize()
        assert (self.out[:, self.heads * self.dim:] == 9).all()
        return self.out[:, :self.heads * self.dim].reshape(self.batch, self.heads, self.dim).cpu()

    def check(self):
        got = self.run()
        close(got, self.ref, self.tol, "attention")
        return got


TYPES = [(F32, F32), (F32, F16), (F16, F16), (F32, BF16), (BF16, BF16)]


def pair(p):
    return NAMES[p[0]] + "_" + NAMES[p[1]] if isinstance(p, tuple) else None


@pytest.mark.parametrize("types", TYPES, ids=pair)
@pytest.mark.parametrize("heads,kv,dim,block,lens,layout", [
    (1, 1, 64, 16, [1], "thd"), (4, 4, 8, 1, [0, 3, 33], "htd"), (6, 2, 40, 7, [31, 32, 0, 129], "thd"), (20, 20, 64, 16, [448], "thd"),
    (8, 1, 80, 50, [1000, 5], "htd"), (16, 1, 128, 16, [2000, 64], "thd"), (34, 2, 96, 16, [260, 300, 1], "htd"), (3, 1, 136, 16, [100, 513], "thd"),
    (2, 2, 256, 32, [70, 1030], "thd"), (32, 8, 128, 16, [0, 17, 900, 256, 1], "thd")])
def test_paged_attention(types, heads, kv, dim, block, lens, layout):
    Attn(*types, heads, kv, dim, block, lens, layout).check()


@pytest.mark.parametrize("types", TYPES, ids=pair)
@pytest.mark.parametrize("window", [1, 30, 100, 5000])
def test_paged_attention_window(types, window):
    Attn(*types, 8, 2, 64, 16, [0, 1, 29, 31, 400, 1500], window=window, seed=3).check()


@pytest.mark.parametrize("types", TYPES, ids=pair)
def test_paged_attention_missing_blocks(types):
    # negative and out-of-range entries; request 2 has nothing else
    p = Attn(*types, 4, 2, 64, 8, [100, 300, 16, 9], holes=(0, 1, 5, 6, 7, 8, 20), seed=5, widen=3)
    got = p.check()
    assert (got[2] == 0).all()


def test_paged_attention_long_and_many():
    Attn(F32, F16, 8, 1, 128, 64, [40000, 3, 0, 7000], seed=7).check()
    Attn(BF16, BF16, 2, 1, 64, 16, [(i * 37) % 130 for i in range(700)], seed=8).check()  # over 64 requests a strip, many empty
    Attn(F32, F32, 5, 5, 64, 16, [1] * 70 + [0] * 80 + [600], seed=9).check()


def test_paged_attention_bits_do_not_vary():
    import torch
    p = Attn(F32, BF16, 16, 2, 128, 16, [9000, 100, 4097], seed=11)
    first = p.run()
    for _ in range(4):
        assert torch.equal(p.run(), first)


def test_paged_attention_loud_queries():
    # scores of hundreds: the running maximum moves, weights under- and overflow without it
    for types in TYPES:
        Attn(*types, 4, 2, 64, 16, [700, 40], seed=13, loud=60.0).check()
        p = Attn(*types, 4, 2, 64, 16, [700, 40], seed=14, loud=1e-6 if types[0] != F16 else 1e-3)
        p.check()


def test_paged_attention_offsets_past_32_bits():
    import torch
    heads, kv, dim, block = 4, 2, 64, 16
    stride = 1 << 30  # elements between blocks: the third starts past 2^32 bytes
    k, v = (torch.empty(4 * stride, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    small = Attn(BF16, BF16, heads, kv, dim, block, [40], seed=15)
    table = torch.tensor([[3, 0, 2]], dtype=torch.int32)
    for big, src in ((k, small.k), (v, small.v)):
        for i, blk in enumerate(table[0].tolist()):
            big[blk * stride:blk * stride + block * kv * dim] = src[int(small.table[0, i])].reshape(-1)
    small.gt = table.cuda()
    a = list(small.args())
    a[8], a[9], a[10], a[12] = k.data_ptr(), v.data_ptr(), 4, stride
    _abi.paged_attention_dev(*a)
    torch.cuda.synchronize()
    close(small.out[:, :heads * dim].reshape(1, heads, dim), small.ref, small.tol)
    # and the store, to the last block
    rows = torch.arange(2 * kv * dim, dtype=torch.float32, device="cuda").view(2, -1) % 64
    slots = torch.tensor([3 * block + 15, 2 * block], device="cuda")
    _abi.kv_store_dev(F32, BF16, 2, kv, dim, rows.data_ptr(), rows.data_ptr(), kv * dim, kv * dim, slots.data_ptr(), k.data_ptr(), v.data_ptr(), 4,
                      block, stride, kv * dim, dim)
    torch.cuda.synchronize()
    for big in (k, v):
        assert torch.equal(big[3 * stride + 15 * kv * dim:3 * stride + 16 * kv * dim].float(), rows[0])
        assert torch.equal(big[2 * stride:2 * stride + kv * dim].float(), rows[1])


def test_paged_attention_nan_scores_and_values():
    import torch
    for types in TYPES:
        p = Attn(*types, 2, 1, 64, 16, [50, 60], seed=17)
        p.gq[0, 3] = float("nan")  # head 0 of request 0
        got = p.run()
        assert torch.isnan(got[0, 0]).all()
        close(got[0, 1], p.ref[0, 1], p.tol[0, 1])
        close(got[1], p.ref[1], p.tol[1])
        p = Attn(*types, 2, 1, 64, 16, [50], seed=17)
        p.v[int(p.table[0, 1]), 4, 0, 7] = float("nan")
        got = p.run()
        assert torch.isnan(got[0, :, 7]).all()
        ok = torch.arange(64) != 7
        close(got[:, :, ok], p.ref[:, :, ok], p.tol[:, :, ok])


def test_paged_attention_streams_and_graph():
    import torch
    p = Attn(F32, F16, 8, 2, 64, 16, [900, 33], seed=19)
    first = p.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    assert torch.equal(p.run(stream=side.cuda_stream), first)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        _abi.paged_attention_dev(*p.args(), stream=side.cuda_stream)
    long = p.gl.clone()
    for lens in ([900, 33], [500, 33], [0, 7], [900, 33]):
        p.gl.copy_(torch.tensor(lens, dtype=torch.int32))
        eager = p.run()
        p.out.fill_(9.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(p.out[:, :512].reshape(2, 8, 64).cpu(), eager)
    assert torch.equal(long, p.gl) and torch.equal(eager, first)


def test_paged_attention_growth_refused_during_capture():
    # a fresh library context has no workspace: a call that may split must not allocate inside a capture
    import torch
    p = Attn(F32, F16, 8, 2, 64, 16, [900, 33], seed=19)
    short = Attn(F32, F16, 8, 2, 64, 16, [300, 33], seed=20)
    torch.cuda.synchronize()
    _abi.shutdown()
    _abi.init()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError) as e:
        with torch.cuda.graph(g, stream=side):
            _abi.paged_attention_dev(*p.args(), stream=side.cuda_stream)
    assert "eagerly" in str(e.value)
    del g
    torch.cuda.synchronize()
    # rows of at most 512 positions need none
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        _abi.paged_attention_dev(*short.args(), stream=side.cuda_stream)
    for _ in range(3):
        short.out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        close(short.out[:, :512].reshape(2, 8, 64), short.ref, short.tol)
    p.check()


def test_paged_attention_refusals():
    p = Attn(F32, F16, 4, 2, 64, 16, [40])
    ok = list(p.args())
    E = _abi
    for at, value, code in ((0, BF16, E.TML_ERR_INVALID_FORMAT), (1, I8, E.TML_ERR_INVALID_FORMAT), (2, -1, E.TML_ERR_INVALID_SHAPE),
                            (3, 5, E.TML_ERR_SHAPE_MISMATCH), (5, 60, E.TML_ERR_INVALID_SHAPE), (5, 264, E.TML_ERR_INVALID_SHAPE),
                            (6, None, E.TML_ERR_INVALID_ARG), (8, None, E.TML_ERR_INVALID_ARG), (8, ok[8] + 2, E.TML_ERR_INVALID_ARG),
                            (11, 0, E.TML_ERR_INVALID_ARG), (13, ok[13] + 1, E.TML_ERR_INVALID_ARG), (12, -16, E.TML_ERR_INVALID_SHAPE),
                            (15, None, E.TML_ERR_INVALID_ARG), (18, None, E.TML_ERR_INVALID_ARG), (20, None, E.TML_ERR_INVALID_ARG)):
        a = list(ok)
        a[at] = value
        with pytest.raises(_abi.TmlError) as e:
            _abi.paged_attention_dev(*a)
        assert e.value.code == code, (at, str(e.value))
    a = list(ok)
    a[2] = 0
    _abi.paged_attention_dev(*a)
    a = list(ok)
    a[10] = 0  # a cache of no blocks: nothing to look at
    _abi.paged_attention_dev(*a)
    import torch
    torch.cuda.synchronize()
    assert (p.out[:, :256] == 0).all()


# ------------------------------------------------------------- matvec_q4g
def weights(seed, n, k, group):
    """Nibbles as integers [n, k] and scales [n, groups]."""
    import torch
    q = torch.randint(-8, 8, (n, k), generator=gen(seed))
    s = 0.01 * (0.5 + torch.rand(n, -(-k // group) if k else 0, generator=gen(seed + 1)))
    return q, s


def pack(q, width, offset):
    """Rows of nibbles, `width` bytes apart, `offset` bytes into an allocation; what follows a row is noise."""
    import torch
    n, k = q.shape
    u = torch.cat([q & 15, torch.zeros(n, k % 2, dtype=q.dtype)], 1).to(torch.uint8)
    rows = torch.randint(0, 256, (n, width), dtype=torch.uint8, generator=gen(3))
    rows[:, :(k + 1) // 2] = u[:, 0::2] | (u[:, 1::2] << 4)
    if k % 2 and k:
        rows[:, k // 2] |= 0xA0  # the odd nibble's other half may be anything
    whole = torch.empty(n * width + offset, dtype=torch.uint8, device="cuda")
    whole[offset:] = rows.reshape(-1).cuda()
    return whole


def run_matvec(xt, x, xs, q, s, group, x_group=0, bias=None, yt=F32, width=None, offset=0, pad=0):
    import torch
    m, k = x.shape
    n = q.shape[0]
    width = -(-k // 32) * 16 if width is None else width
    w = pack(q, max(width, 1), offset)
    gx, sx = padded(x, pad, 1 if xt == I8 else float("nan"))
    y = torch.full((m, n + pad), 9.0, dtype=dt(yt), device="cuda")
    gs, gxs, gb = s.float().cuda(), None if xs is None else xs.float().cuda(), None if bias is None else bias.float().cuda()
    _abi.matvec_q4g_dev(xt, m, n, k, gx.data_ptr(), sx, w.data_ptr() + offset, width, gs.data_ptr(), group, yt, y.data_ptr(), y.stride(0),
                        x_scales_ptr=ptr(gxs), x_group=x_group, bias_ptr=ptr(gb))
    torch.cuda.synchronize()
    assert (y[:, n:] == 9).all()
    return y[:, :n].cpu()


def matvec_ref(xt, x, xs, q, s, group, x_group=0, bias=None, yt=F32):
    import torch
    k = x.shape[1]
    x = x.double()
    if xs is not None:
        x = x * xs.float().double()[:, torch.arange(k) // (x_group or max(k, 1))]
    w = q.double() * s.float().double()[:, torch.arange(k) // group]
    y, mass = x @ w.T, x.abs() @ w.abs().T
    if bias is not None:
        y = y + bias.float().double()
        mass = mass + bias.abs()
    tol = (2.0 ** -23 + 8 * math.sqrt(k) * U) * mass + HALF_ULP[yt] * 1.001 * y.abs() + (2.0 ** -25 if yt == F16 else 1e-30)
    return y, tol


def make_x(xt, seed, m, k, x_group=0):
    import torch
    if xt != I8:
        return randn(seed, m, k).to(dt(xt)), None
    x = torch.randint(-128, 128, (m, k), generator=gen(seed), dtype=torch.int8)
    return x, 0.01 * (0.5 + torch.rand(m, -(-k // x_group) if x_group else 1, generator=gen(seed + 1)))


@pytest.mark.parametrize("xt", [F32, F16, BF16, I8], ids=tname)
@pytest.mark.parametrize("m,n,k,group,x_group", [
    (1, 1, 1, 32, 0), (1, 16, 32, 32, 32), (2, 17, 33, 32, 32), (3, 15, 127, 64, 0), (1, 300, 128, 128, 128), (4, 33, 129, 32, 64), (5, 100, 1000, 96, 96),
    (1, 1280, 5120, 32, 0), (8, 700, 1280, 64, 64), (9, 64, 640, 128, 0), (16, 50, 4096, 128, 128), (17, 40, 256, 32, 32), (33, 20, 96, 5000, 0),
    (1, 4099, 200, 200, 0), (2, 5000, 384, 32, 0), (8, 9000, 100, 128, 0)])
def test_matvec_q4g(xt, m, n, k, group, x_group):
    x, xs = make_x(xt, 21, m, k, x_group)
    q, s = weights(22, n, k, group)
    bias = randn(23, n)
    for b, yt, pad in ((None, F32, 0), (bias, xt if xt != I8 else BF16, 3)):
        got = run_matvec(xt, x, xs, q, s, group, x_group, b, yt, pad=pad)
        ref, tol = matvec_ref(xt, x, xs, q, s, group, x_group, b, yt)
        close(got, ref, tol, (m, n, k))


@pytest.mark.parametrize("xt", [F32, I8], ids=tname)
@pytest.mark.parametrize("m,n,k", [(1, 70, 40000), (8, 300, 6000), (16, 5000, 14336), (3, 20, 131072), (16, 17, 12500)])
def test_matvec_q4g_long_k(xt, m, n, k):
    # x past one fill of LDS: more phases than one, with fewer runs than waves in the last
    x, xs = make_x(xt, 24, m, k, 64)
    q, s = weights(25, n, k, 64)
    got = run_matvec(xt, x, xs, q, s, 64, 64 if xt == I8 else 0)
    close(got, *matvec_ref(xt, x, xs, q, s, 64, 64))


@pytest.mark.parametrize("xt", [F32, BF16, I8], ids=tname)
@pytest.mark.parametrize("k,width,offset", [(100, 50, 0), (101, 51, 0), (64, 32, 1), (1000, 501, 3), (4096, 2048, 8), (33, 17, 0), (31, 16, 16), (40, 24, 0)])
def test_matvec_q4g_rows_anywhere(xt, k, width, offset):
    x, xs = make_x(xt, 26, 3, k, 32)
    q, s = weights(27, 45, k, 32)
    got = run_matvec(xt, x, xs, q, s, 32, 32 if xt == I8 else 0, width=width, offset=offset, pad=1)
    close(got, *matvec_ref(xt, x, xs, q, s, 32, 32))


def test_matvec_q4g_ranges():
    # loud, faint and mixed activations; no chunk may lose its precision to another
    import torch
    q, s = weights(28, 60, 512, 32)
    base = randn(29, 5, 512)
    mult = torch.ones(5, 512, dtype=torch.float64)
    mult[0], mult[1], mult[2, 64:96], mult[3, ::7], mult[4] = 1e30, 1e-30, 1e20, 1e-3, torch.logspace(-12, 12, 512, dtype=torch.float64)
    for xt in (F32, BF16):
        x = (base * mult).to(dt(xt))
        got = run_matvec(xt, x, None, q, s, 32)
        y, _ = matvec_ref(xt, x, None, q, s, 32)
        # (2^-39 of the largest element of each 32, beyond what follows the elements themselves)
        w = (q.double() * s.double().repeat_interleave(32, 1)).abs()
        most = x.double().abs().view(5, 16, 32).amax(2).repeat_interleave(32, 1)
        tol = ((2.0 ** -23 + 8 * math.sqrt(512) * U) * x.double().abs() + 2.0 ** -38 * most) @ w.T
        close(got, y, tol)


def test_matvec_q4g_infinities_nan():
    import torch
    q, s = weights(30, 40, 256, 64)
    q[3, 10] = 0
    for xt in (F32, F16, BF16):
        x = randn(31, 4, 256).to(dt(xt))
        x[1, 10], x[2, 100], x[3, 7] = float("inf"), float("nan"), -float("inf")
        x[3, 9] = 60000.0 if xt == F16 else 3e38
        got = run_matvec(xt, x, None, q, s, 64)
        w = (q.double() * s.double().repeat_interleave(64, 1))
        ref = (x.double()[:, None, :] * w[None]).sum(2)  # inf * 0 is a NaN here too
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(got[1][torch.isinf(ref[1])].double(), ref[1][torch.isinf(ref[1])])
        y, tol = matvec_ref(xt, x[:1], None, q, s, 64)
        close(got[:1], y, tol)


@pytest.mark.parametrize("k,group", [(200, 32), (130, 64), (129, 128), (640, 96)])
def test_matvec_q4g_scales_that_are_no_numbers(k, group):
    # an infinite or NaN scale touches its own column and group alone, chunks past K not at all
    import torch
    q, s = weights(36, 40, k, group)
    q[q == 0] = 3  # (an infinite scale times nothing is a NaN of its own)
    s[2, -1], s[5, 0], s[9, -1] = float("inf"), float("nan"), -float("inf")
    for xt in (F32, F16, I8):
        x, xs = make_x(xt, 37, 2, k, 32 if xt == I8 else 0)
        x = x.abs() + 1 if xt != I8 else x.clamp(min=1)  # one sign: sums of infinities stay infinite or are NaN by q alone
        got = run_matvec(xt, x, xs, q, s, group, 32 if xt == I8 else 0)
        for n in (2, 5, 9):
            lo = 0 if n == 5 else (s.shape[1] - 1) * group
            part = q[n, lo:lo + group]
            if n == 5 or bool((part > 0).any() and (part < 0).any()):
                # (of both signs: the group's sum comes first, and its sign decides)
                assert torch.isnan(got[:, n]).all() if n == 5 else not torch.isfinite(got[:, n]).any()
            else:
                assert torch.isinf(got[:, n]).all()
        rest = [n for n in range(40) if n not in (2, 5, 9)]
        y, tol = matvec_ref(xt, x, xs, q, torch.where(torch.isfinite(s), s, 1.0), group, 32)
        close(got[:, rest], y[:, rest], tol[:, rest])


def test_matvec_q4g_bits_do_not_vary():
    import torch
    x, _ = make_x(F32, 32, 3, 4096)
    q, s = weights(33, 500, 4096, 128)
    first = run_matvec(F32, x, None, q, s, 128)
    for _ in range(3):
        assert torch.equal(run_matvec(F32, x, None, q, s, 128), first)


def test_matvec_q4g_empty_and_refusals():
    import torch
    bias = torch.arange(5, dtype=torch.float32, device="cuda")
    y = torch.full((2, 5), 9.0, device="cuda")
    for xt in (F32, I8):
        ones = torch.ones(2, device="cuda")
        y.fill_(9.0)
        _abi.matvec_q4g_dev(xt, 2, 5, 0, None, 0, None, 0, None, 32, F32, y.data_ptr(), 5, bias_ptr=bias.data_ptr(), x_scales_ptr=ones.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(y, bias.expand(2, 5))
    p = y.data_ptr()
    ok = [F32, 2, 5, 64, p, 64, p, 32, p, 32, F32, p, 5]
    E = _abi
    for at, value, code in ((0, 9, E.TML_ERR_INVALID_FORMAT), (10, I8, E.TML_ERR_INVALID_FORMAT), (1, -1, E.TML_ERR_INVALID_SHAPE),
                            (9, 0, E.TML_ERR_INVALID_ARG), (9, 40, E.TML_ERR_INVALID_SHAPE), (3, 2 ** 21, E.TML_ERR_INVALID_SHAPE),
                            (4, None, E.TML_ERR_INVALID_ARG), (6, None, E.TML_ERR_INVALID_ARG), (8, None, E.TML_ERR_INVALID_ARG),
                            (11, None, E.TML_ERR_INVALID_ARG), (5, 63, E.TML_ERR_INVALID_SHAPE), (7, 31, E.TML_ERR_INVALID_SHAPE),
                            (12, 4, E.TML_ERR_INVALID_SHAPE), (0, I8, E.TML_ERR_INVALID_ARG)):
        a = list(ok)
        a[at] = value
        with pytest.raises(_abi.TmlError) as e:
            _abi.matvec_q4g_dev(*a)
        assert e.value.code == code, (at, str(e.value))
    with pytest.raises(_abi.TmlError):
        _abi.matvec_q4g_dev(I8, *ok[1:], x_scales_ptr=p, x_group=48)
    _abi.matvec_q4g_dev(F32, 0, 5, 64, None, 64, None, 32, None, 32, F32, None, 5)


@pytest.mark.parametrize("n,k,group", [(1, 1, 32), (3, 33, 32), (5, 200, 64), (2, 4096, 128), (70, 96, 96), (4, 50, 2)])
def test_quantize_groups(orc, n, k, group):
    import torch
    w = randn(34, n, k).float()
    w[0, :min(k, group)] = 0
    stride, width = k + 3, (k + 1) // 2 + 2
    gw, _ = padded(w, 3, float("nan"))
    groups = -(-k // group)
    q = torch.full((n, width), 0xEE, dtype=torch.uint8, device="cuda")
    s = torch.empty(n, groups, device="cuda")
    _abi.quantize_groups_dev(n, k, group, gw.data_ptr(), stride, q.data_ptr(), width, s.data_ptr())
    torch.cuda.synchronize()
    q, s = q.cpu().numpy(), s.cpu().numpy()
    assert (q[:, (k + 1) // 2:] == 0xEE).all()
    for r in range(n):
        for g in range(groups):
            part = w[r, g * group:(g + 1) * group].numpy()
            packed, scale = orc.quantize_q4(part)
            assert np.array_equal(q[r, g * group // 2:g * group // 2 + len(packed)], packed) and np.float32(scale) == s[r, g]
    for a in ((-1, k, group), (n, k, 0)):
        with pytest.raises(_abi.TmlError):
            _abi.quantize_groups_dev(*a, gw.data_ptr(), stride, 1, width, 1)
