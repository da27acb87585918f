"""Corners of the serving operators on the GPU: infinite keys and queries, groups of
more heads than a workgroup of the attention takes, the sizes that need the most LDS,
lengths that advance in place, more rows than one launch has room for.

Tolerances are those of test_gpu_serving.py, whose problems these build on.
"""
import math

import numpy as np
import pytest

from test_gpu_serving import BF16, F16, F32, HALF_ULP, I8, TYPES, U, Attn, close, dt, gen, pair
from tomoul_amd import _abi

pytestmark = pytest.mark.gpu


# -------------------------------------------------------- paged attention
def attention_ref(p):
    """The result and its tolerance for the cache, q and scale as they are on the GPU now."""
    import torch
    inf = math.inf
    ref, tol = (torch.zeros(p.batch, p.heads, p.dim, dtype=torch.float64) for _ in range(2))
    term = 2.0 ** -16 if p.ct == BF16 and p.qt == BF16 else 2.0 ** -20
    for r, length in enumerate(p.lens):
        pages = p.table[r, :-(-length // p.block)].long().cuda()
        key, val = (c[pages].reshape(-1, p.kv, p.dim)[:length].double().cpu().repeat_interleave(p.heads // p.kv, 1) for c in (p.k, p.v))
        q = p.gq[r].view(p.heads, p.dim).double().cpu()
        s = (q * key).sum(2).T * p.scale
        top = s.amax(1, keepdim=True)
        e = torch.exp(s - torch.where(top == -inf, 0.0, top))
        total = e.sum(1, keepdim=True)
        w = e / torch.where(total == 0, 1.0, total)
        ref[r] = (w.T[:, :, None] * val).sum(0)
        finite = torch.nan_to_num(q, 0.0, 0.0, 0.0).abs() * torch.nan_to_num(key, 0.0, 0.0, 0.0).abs()
        err = ((2.0 ** -21 + 4 * math.sqrt(p.dim) * U) * finite.sum(2).T * abs(p.scale)).amax(1)
        tol[r] = (2 * err[:, None] + term + 8 * math.sqrt(max(length, 1)) * U) * (w.T[:, :, None] * val.abs()).sum(0)
    tol = torch.nan_to_num(tol) + HALF_ULP[p.qt] * 1.001 * torch.nan_to_num(ref).abs() + (2.0 ** -25 if p.qt == F16 else 1e-30)
    return ref, tol


@pytest.mark.parametrize("types", TYPES, ids=pair)
@pytest.mark.parametrize("dim,length", [(64, 50), (80, 50), (40, 33), (128, 900), (136, 40), (256, 30)])
def test_paged_attention_infinite_keys_and_queries(types, dim, length):
    # a score of -inf weighs nothing, one of +inf or NaN makes the head NaN, whatever
    # the head size and the types; nothing but scores of -inf: zeros
    import torch
    inf = math.inf
    for scale in (0.125, -0.125):
        p = Attn(*types, 6, 2, dim, 16, [length, length, 1, length], seed=21)
        p.scale, low = scale, -math.copysign(1.0, scale)
        q = p.q.double().abs() + 0.1  # all of one sign, in d 0 and the last one of both
        q[:, 1, 0] *= -1
        q[1, 2, dim - 1] *= -1
        q[1, 3, 5] = 0
        q[1, 4, 5] = 1e-30 if types[0] == F32 else 1e-3  # (little next to the others, but something)
        q[3, 0, 7], q[3, 1, 7], q[3, 4, 7] = inf, -inf, math.nan
        p.gq = q.to(dt(types[0])).reshape(p.batch, -1).cuda()
        for r, tok, h, d, v in ((0, 7, 0, 0, low * inf), (0, 20, 1, dim - 1, low * inf), (1, 3, 0, dim - 1, low * inf), (1, 25, 1, 5, low * inf),
                                (1, 4, 1, 0, low * inf), (2, 0, 0, 3, low * inf), (2, 0, 1, 3, -low * inf), (3, 9, 1, 8, low * inf)):
            p.k[int(p.table[r, tok // 16]), tok % 16, h, d] = v
        ref, tol = attention_ref(p)
        assert torch.isnan(ref[0, 1]).all() and torch.isfinite(ref[0, 0]).all() and torch.isfinite(ref[0, 3:]).all()
        assert torch.isnan(ref[1, 2]).all() and torch.isnan(ref[1, 3]).all() and torch.isfinite(ref[1, [0, 1, 4, 5]]).all()
        assert (ref[2, [0, 2]] == 0).all() and torch.isnan(ref[2, 3:]).all()
        close(p.run(), ref, tol, (dim, scale))


def test_paged_attention_infinite_key_against_the_least_query():
    # q's elements that f16 and bf16 cannot hold next to the others still give an infinite key its sign
    import torch
    for ct in (F16, BF16):
        for least in (1e-12, 1e-30, 1e-39, -1e-39):
            p = Attn(F32, ct, 2, 1, 64, 16, [40], seed=23)
            p.gq = p.gq.abs() + 0.5
            p.gq[:, 3] = p.gq[:, 64 + 3] = least
            p.k[int(p.table[0, 1]), 2, 0, 3] = -math.copysign(math.inf, least)
            ref, tol = attention_ref(p)
            assert torch.isfinite(ref).all()
            close(p.run(), ref, tol, (ct, least))


# ---------------------------------------------------------------- rmsnorm
@pytest.mark.parametrize("rows,cols,group", [(1, 1280, 0), (1100, 1280, 128), (1, 1280, 128), (1100, 1237, 0), (3, 1237, 96), (2, 7, 0), (2, 33000, 0), (2, 9000, 64)])
def test_rmsnorm_8_bits_at_the_halves(rows, cols, group):
    # x of ones and no epsilon: out is the weight itself, so the quotient is known to its last bit
    rng = np.random.default_rng(17)
    width = group or cols
    w = np.empty(cols, np.float32)
    for g in range(0, cols, width):
        most = np.float32(np.exp(rng.uniform(-8, 8)))
        part = ((rng.integers(-127, 127, min(width, cols - g)) + 0.5) * np.float64(most / np.float32(127))).astype(np.float32)
        part = (part.view(np.int32) + rng.integers(-2, 3, len(part))).astype(np.int32).view(np.float32)
        part[rng.integers(len(part))] = most
        w[g:g + width] = part
    import torch
    x, gw = torch.ones(rows, cols, device="cuda"), torch.from_numpy(w).cuda()
    q, scales = torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, -(-cols // width), device="cuda")
    _abi.rmsnorm_dev(F32, rows, cols, x.data_ptr(), cols, gw.data_ptr(), 0.0, I8, q.data_ptr(), cols, scales_ptr=scales.data_ptr(), group=group)
    torch.cuda.synchronize()
    scale = np.array([np.abs(w[g:g + width]).max() / np.float32(127) for g in range(0, cols, width)], np.float32)
    want = np.rint(w / np.repeat(scale, width)[:cols])
    assert (scales.cpu().numpy() == scale).all()
    assert (q.cpu().numpy() == want).all()


@pytest.mark.parametrize("t,rows,cols", [(F32, (1 << 22) + 3, 3), (F16, (1 << 26) + 5, 8)], ids=str)
def test_rmsnorm_more_rows_than_a_launch_has_room_for(t, rows, cols):
    import torch
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("needs 12 GiB")
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.empty(rows, cols, dtype=dt(t), device="cuda").normal_(generator=g)
    q, s = torch.zeros(rows, cols, dtype=torch.int8, device="cuda"), torch.zeros(rows, device="cuda")
    total, out = torch.zeros_like(x), torch.zeros_like(x)
    _abi.rmsnorm_dev(t, rows, cols, x.data_ptr(), cols, None, 1e-6, t, out.data_ptr(), cols, residual_ptr=x.data_ptr(), residual_stride=cols,
                     sum_ptr=total.data_ptr(), sum_stride=cols)
    _abi.rmsnorm_dev(t, rows, cols, x.data_ptr(), cols, None, 1e-6, I8, q.data_ptr(), cols, scales_ptr=s.data_ptr())
    torch.cuda.synchronize()
    step = 1 << 22
    for r in range(0, rows, step):
        part = x[r:r + step].float()
        assert torch.equal(total[r:r + step], (2 * part).to(dt(t)))  # (exact: twice a number)
        y = part * torch.rsqrt((part * part).mean(1, keepdim=True) + 1e-6)
        most = y.abs().amax(1)
        assert ((s[r:r + step] - most / 127).abs() <= 60 * U * most / 127).all()
        assert ((q[r:r + step] * s[r:r + step, None] - y).abs() <= (0.5 + 127 * 140 * U) * most[:, None] / 127).all()
        y2 = 2 * part * torch.rsqrt((4 * part * part).mean(1, keepdim=True) + 1e-6)
        assert ((out[r:r + step].float() - y2).abs() <= (HALF_ULP[t] * 1.001 + 60 * U) * y2.abs() + 2.0 ** -25 * (t == F16)).all()


# ------------------------------------------------------------- matvec_q4g
def test_matvec_q4g_more_columns_than_a_launch_has_room_for():
    # two k a column, so that 2^30 columns stay small: rows of a byte
    import torch
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GiB")
    n = (1 << 30) + 7
    g = torch.Generator(device="cuda")
    g.manual_seed(2)
    w = torch.randint(0, 256, (n,), generator=g, device="cuda", dtype=torch.uint8)
    scales, y = torch.ones(n, device="cuda"), torch.full((n,), 99.0, dtype=torch.float16, device="cuda")
    scales[-9:] = 2.0
    x = torch.tensor([[3.0, 0.5]], dtype=torch.float16, device="cuda")
    _abi.matvec_q4g_dev(F16, 1, n, 2, x.data_ptr(), 2, w.data_ptr(), 1, scales.data_ptr(), 32, F16, y.data_ptr(), n)
    torch.cuda.synchronize()
    step = 1 << 27
    for at in range(0, n, step):
        u = w[at:at + step].to(torch.int16)
        want = ((u & 15 ^ 8) - 8).half() * 3 + ((u >> 4 ^ 8) - 8).half() * 0.5  # (exact)
        assert torch.equal(y[at:at + step], want * scales[at:at + step].half())


# ---------------------------------------------------------------- kv_plan
@pytest.mark.parametrize("n,new_most", [(64, 1), (500, 40), (3, 3000), (2000, 3)])
def test_kv_plan_lengths_in_place(n, new_most):
    # the lengths advance over themselves, step after step, eagerly and as a graph
    import torch
    block, steps = 16, 3
    width = -(-steps * max(new_most, 1) // block) + 1
    i32 = dict(dtype=torch.int32, device="cuda")
    new = torch.randint(0, new_most + 1, (n,), generator=gen(5)).to(torch.int32)
    tokens = int(new.sum()) + 7
    free = torch.randperm(n * width, generator=gen(6)).to(torch.int32).cuda()
    ctx, gnew = torch.zeros(n, **i32), new.cuda()
    table = torch.full((n, width), -1, **i32)
    slots, pos = torch.zeros(tokens, dtype=torch.int64, device="cuda"), torch.zeros(tokens, **i32)
    req, totals = torch.zeros(tokens, **i32), torch.zeros(3, dtype=torch.int64, device="cuda")

    def plan(stream):
        _abi.kv_plan_dev(n, block, ctx.data_ptr(), gnew.data_ptr(), free.data_ptr(), free.numel(), table.data_ptr(), width, width, tokens,
                         slots.data_ptr(), token_request_ptr=req.data_ptr(), positions_ptr=pos.data_ptr(), seq_len_ptr=ctx.data_ptr(),
                         totals_ptr=totals.data_ptr(), stream=stream)

    owner = torch.repeat_interleave(torch.arange(n), new.long())
    first = torch.cat([torch.arange(int(v)) for v in new]) if tokens > 7 else torch.zeros(0, dtype=torch.long)
    side = torch.cuda.Stream()
    graph = None
    handed = 0
    for step in range(2 * steps):
        if step == steps:  # the same again from the start, replayed
            ctx.zero_()
            table.fill_(-1)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                plan(side.cuda_stream)
            handed = 0
        pool = torch.roll(torch.arange(n * width, dtype=torch.int32), -handed).cuda()
        free.copy_(pool)
        torch.cuda.synchronize()
        if graph is None:
            plan(None)
        else:
            graph.replay()
        torch.cuda.synchronize()
        done = (step % steps) * new.long()
        assert torch.equal(ctx.cpu().long(), done + new.long())
        assert torch.equal(req[:-7].cpu().long(), owner) and (req[-7:] == -1).all()
        where = done[owner] + first
        assert torch.equal(pos[:-7].cpu().long(), where)
        page = table.cpu().long()[owner, where // block]
        assert (page >= 0).all() and torch.equal(slots[:-7].cpu(), page * block + where % block)
        need = int((-(-(done + new.long()) // block) - -(-done // block)).sum())
        assert totals.tolist() == [tokens - 7, need, 0]
        handed += need
        used = table[table >= 0]
        assert used.unique().numel() == used.numel() == handed


# -------------------------------------------------------- quantize_groups
@pytest.mark.parametrize("k", [50, 51, 4096])
def test_quantize_groups_any_group_past_k(k):
    import torch
    w = torch.randn(3, k, generator=gen(9)).cuda()
    outs = []
    for group in (k, 2 ** 63 - 1):
        q, s = torch.zeros(3, (k + 1) // 2, dtype=torch.uint8, device="cuda"), torch.zeros(3, device="cuda")
        _abi.quantize_groups_dev(3, k, group, w.data_ptr(), k, q.data_ptr(), (k + 1) // 2, s.data_ptr())
        torch.cuda.synchronize()
        outs.append((q.cpu(), s.cpu()))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.equal(outs[0][1], w.abs().amax(1).cpu() / 7)


# ----------------------------------------- paged attention, sizes past the usual
@pytest.mark.parametrize("types", TYPES, ids=pair)
@pytest.mark.parametrize("heads,kv,dim,block,lens,layout,widen", [
    (34, 2, 96, 16, [260, 900, 1], "htd", 0), (48, 1, 64, 16, [1300, 0, 600], "thd", 3),  # groups of more than 16 heads, split
    (16, 1, 256, 16, [70, 1030], "thd", 0), (40, 1, 256, 32, [5, 700], "htd", 0),  # the most LDS a workgroup takes
    (8, 8, 64, 16, [40, 3, 448], "thd", 300), (8, 2, 128, 16, [0, 513, 17], "htd", 1000)])  # a table far wider than its requests
def test_paged_attention_large_groups_and_wide_tables(types, heads, kv, dim, block, lens, layout, widen):
    Attn(*types, heads, kv, dim, block, lens, layout, widen=widen, seed=31).check()


@pytest.mark.parametrize("cols,group", [(49152, 3), (32768, 2), (131072, 8)])
def test_rmsnorm_8_bits_the_most_groups(cols, group):
    # 16384 group maxima in LDS, 64 KiB of them
    import torch
    x = torch.randn(2, cols, generator=gen(41)).cuda()
    q, scales = torch.zeros(2, cols, dtype=torch.int8, device="cuda"), torch.zeros(2, 16384, device="cuda")
    _abi.rmsnorm_dev(F32, 2, cols, x.data_ptr(), cols, None, 1e-6, I8, q.data_ptr(), cols, scales_ptr=scales.data_ptr(), group=group)
    torch.cuda.synchronize()
    y = x.double() / torch.sqrt(x.double().square().mean(1, keepdim=True) + 1e-6)
    most = y.view(2, 16384, group).abs().amax(2)
    assert ((scales - most / 127).abs() <= 40 * U * most / 127).all()
    # (the scale's own error, and half a step)
    assert ((q.view(2, 16384, group) * scales[:, :, None].double() - y.view(2, 16384, group)).abs() <= (0.5 + 127 * 80 * U) * most[:, :, None] / 127).all()
