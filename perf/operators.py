"""Performance cases of the serving operators around a decoder's products.

A case is a dict of plain values; `op` says which operator it goes through:

  plan       _abi.kv_plan_dev          block tables and slot maps from request lengths
  store      _abi.kv_store_dev         new keys and values to their slots in the paged cache
  norm       _abi.rmsnorm_dev          root-mean-square norm with the residual's addition,
                                       its output as floats or in 8 bits with scales
  matvec     _abi.matvec_q4g_dev       products with 4-bit weights and group scales
  attention  _abi.paged_attention_dev  one new token a request over the paged cache

`run` computes an operator in its plain form, elementary torch operations in 32 bits
rounded once at the end, or, where `own` is true, with the framework's kernels on the
same state.  `exact` is the definition in 64 bits, written apart from both.

Sizes are those of the repository's models and benchmark (Whisper large-v3-turbo:
20 heads of 64, 1280 wide, 448 tokens, 51866 words; 1024- and 4096-wide layers)
and generic ones for larger decoders.
"""
import math
import random

import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16), "i8": (3, torch.int8)}


def listed():
    return [
        # One decode step of a full server: 64 requests, a token each, the padded size of a captured graph.
        dict(name="plan_decode_64", op="plan", requests=64, ctx_most=4096, new_most=1, block=16, width=260, pad=0, lengths=11),
        # A mixed batch of prompts and decodes: about 65k new tokens over 512 requests.
        dict(name="plan_mixed_512", op="plan", requests=512, ctx_most=2048, new_most=256, block=16, width=160, pad=301, lengths=12),
        # The same decode step's new keys and values, cut out of one fused projection's f32 output.
        dict(name="store_decode_64", op="store", tokens=64, heads=8, dim=128, block=16, src="f32", cache="f16", layout="thd", pad=3),
        # A prompt batch of 16k tokens into a bf16 cache whose heads come before its tokens.
        dict(name="store_prompt_16k", op="store", tokens=16384, heads=8, dim=128, block=32, src="bf16", cache="bf16", layout="htd", pad=0),
        # The norm before one token's projection, f32, no 8 bits: the smallest call.
        dict(name="norm_one_f32", op="norm", rows=1, cols=1280, type="f32", out="f32", residual=True, group=0),
        # A prompt's 8192 tokens, bf16 stream, in 8 bits with one scale a token for the int8 product.
        dict(name="norm_prompt_i8", op="norm", rows=8192, cols=5120, type="bf16", out="i8", residual=True, group=0),
        # One token's feed-forward down-projection at the turbo decoder's size, f32 activations, groups of 32.
        dict(name="matvec_f32_m1", op="matvec", m=1, n=1280, k=5120, x="f32", y="f32", group=32, xgroup=0, bias=True),
        # Eight sequences through a wide up-projection, activations in 8 bits as the norm leaves them.
        dict(name="matvec_i8_m8", op="matvec", m=8, n=14336, k=4096, x="i8", y="bf16", group=128, xgroup=128, bias=False),
        # The vocabulary projection for four sequences, bf16 activations, f32 logits.
        dict(name="matvec_vocab_m4", op="matvec", m=4, n=51866, k=1280, x="bf16", y="f32", group=64, xgroup=0, bias=False),
        # One speech decoder step over its self-attention cache: 20 heads of 64, f16 cache.
        dict(name="attn_one_448", op="attention", batch=1, heads=20, kv=20, dim=64, least=448, most=448, block=16,
             q="f32", cache="f16", layout="thd", window=0, lengths=21),
        # A full server: 64 requests of ragged length, some of them empty, grouped heads, bf16.
        dict(name="attn_server_64", op="attention", batch=64, heads=32, kv=8, dim=128, least=0, most=4096, block=16,
             q="bf16", cache="bf16", layout="thd", window=0, lengths=22),
        # Two long documents, 40k to 65k tokens, heads before tokens: few rows, so the length is what there is to share out.
        dict(name="attn_long_2", op="attention", batch=2, heads=32, kv=8, dim=128, least=40000, most=65536, block=32,
             q="f16", cache="f16", layout="htd", window=0, lengths=23),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("plan", "store", "norm", "norm", "matvec", "matvec", "attention", "attention"))
    if op == "plan":
        block = rng.choice((1, 8, 16, 32, 64, 100))
        new = rng.choice((1, 3, log(2, 256)))
        ctx = log(8, 4096)
        return dict(op=op, requests=log(1, 512), ctx_most=ctx, new_most=new, block=block, width=max(1, -(-(ctx + new) // block) + rng.randrange(5) - 1),
                    pad=rng.randrange(100), lengths=rng.randrange(1 << 30))
    if op == "store":
        return dict(op=op, tokens=log(1, 16384), heads=rng.choice((1, 2, 5, 8)), dim=rng.choice((64, 80, 96, 128)), block=rng.choice((8, 16, 24, 32)),
                    src=rng.choice(("f32", "f16", "bf16")), cache=rng.choice(("f32", "f16", "bf16")), layout=rng.choice(("thd", "htd")), pad=rng.randrange(8))
    if op == "norm":
        cols = rng.choice((64 * rng.randrange(4, 81), log(100, 5120)))
        out = rng.choice(("f32", "f16", "bf16", "i8"))
        group = rng.choice((0, 32, 64)) if out == "i8" and cols % 64 == 0 else 0
        return dict(op=op, rows=log(1, 8192), cols=cols, type=rng.choice(("f32", "f16", "bf16")) if out == "i8" else out, out=out,
                    residual=rng.random() < 0.7, group=group)
    if op == "matvec":
        m, group = rng.choice((1, 1, 2, 3, 4, 5, 8)), rng.choice((32, 64, 128))
        k = rng.choice((64 * rng.randrange(6, 81), group * rng.randrange(4, 41), log(400, 5120)))
        x = rng.choice(("f32", "f16", "bf16", "i8"))
        return dict(op=op, m=m, n=log(300, 12000), k=k, x=x, y=rng.choice(("f32", "bf16")) if x in ("f32", "i8") else rng.choice(("f32", x)), group=group,
                    xgroup=group if x == "i8" and rng.random() < 0.5 else 0, bias=rng.random() < 0.5)
    kv = rng.choice((1, 2, 8, 12))
    cache = rng.choice(("f16", "bf16", "f32"))
    most = log(16, 16384)
    dim = rng.choice((64, 64, 80, 96, 128, 128))
    batch = max(1, min(64, log(1, 64), 250_000_000 // (most * kv * dim * (4 if cache == "f32" else 2))))
    return dict(op=op, batch=batch, heads=kv * rng.choice((1, 1, 3, 4, 8, 16)), kv=kv, dim=dim,
                least=rng.choice((0, 1, most // 2, most)), most=most, block=rng.choice((1, 8, 16, 16, 32, 50)), q=rng.choice(("f32", cache)),
                cache=cache, layout=rng.choice(("thd", "htd")), window=rng.choice((0, 0, 0, log(1, 4096))), lengths=rng.randrange(1 << 30))


# ------------------------------------------------------------------ inputs
def lengths(case):
    """The ragged lengths of a case: part of the case, alike for every seed."""
    r = random.Random(case["lengths"])
    if case["op"] == "plan":
        return [(r.randrange(case["ctx_most"] + 1), r.randrange(case["new_most"] + 1) if case["new_most"] > 1 else 1) for _ in range(case["requests"])]
    return [r.randint(case["least"], case["most"]) for _ in range(case["batch"])]


def paged(case, n_blocks, heads, gen, fill):
    """A cache [block, token, head, dim], stored in the case's order, with one block after its end that is no part of it."""
    dtype, (b, h, d) = TYPES[case["cache"]][1], (case["block"], heads, case["dim"])
    if case["layout"] == "thd":
        whole = torch.empty(n_blocks + 1, b, h, d, dtype=dtype, device="cuda")
    else:
        whole = torch.empty(n_blocks + 1, h, b, d, dtype=dtype, device="cuda").permute(0, 2, 1, 3)
    if fill is None:
        whole.normal_(generator=gen)
    else:
        whole.fill_(fill)
    return whole


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    s = {"case": case}
    if case["op"] == "plan":
        return prepare_plan(case, gen, s)
    if case["op"] == "store":
        tokens, heads, dim, block = case["tokens"], case["heads"], case["dim"], case["block"]
        n_blocks = -(-tokens // block) + 3
        # keys and values are the middle and the last part of a fused projection's rows
        fused = normal(tokens, 3 * heads * dim, dtype=TYPES[case["src"]][1])
        s["k"], s["v"] = fused[:, heads * dim:2 * heads * dim], fused[:, 2 * heads * dim:]
        slots = torch.randperm(n_blocks * block, generator=gen, device="cuda")[:tokens]
        slots[tokens - min(case["pad"], tokens - 1):] = -1
        s["slots"] = slots.contiguous()
        s["k_all"], s["v_all"] = paged(case, n_blocks, heads, gen, 0.0), paged(case, n_blocks, heads, gen, 0.0)
        s["n_blocks"] = n_blocks
    elif case["op"] == "norm":
        rows, cols, dtype = case["rows"], case["cols"], TYPES[case["type"]][1]
        # a residual stream: most channels near one, a few far out
        loud = torch.where(torch.rand(cols, generator=gen, device="cuda") < 0.01, 12.0, 1.0)
        s["x"] = normal(rows, cols, dtype=dtype)
        s["residual"] = (normal(rows, cols) * loud).to(dtype) if case["residual"] else None
        s["weight"] = 1.0 + 0.1 * normal(cols)
        s["eps"] = 1e-6
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
        s["out"] = torch.empty(rows, cols, dtype=TYPES[case["out"]][1], device="cuda")
        groups = cols // case["group"] if case["group"] else 1
        s["scales"] = torch.empty(rows, groups, device="cuda") if case["out"] == "i8" else None
        s["values"] = torch.empty(rows, groups, cols // groups, dtype=torch.bfloat16, device="cuda") if case["out"] == "i8" else None
    elif case["op"] == "matvec":
        m, n, k, g = case["m"], case["n"], case["k"], case["group"]
        width = -(-k // 32) * 16  # a row's bytes, whole 16-byte chunks
        s["w"] = torch.randint(0, 256, (n, width), generator=gen, device="cuda", dtype=torch.uint8)
        s["w_scales"] = 0.02 / 4.6 * (0.5 + torch.rand(n, -(-k // g), generator=gen, device="cuda"))
        s["bias"] = normal(n) if case["bias"] else None
        if case["x"] == "i8":
            s["x"] = torch.randint(-127, 128, (m, k), generator=gen, device="cuda", dtype=torch.int8)
            s["x_scales"] = 0.01 * (0.5 + torch.rand(m, -(-k // case["xgroup"]) if case["xgroup"] else 1, generator=gen, device="cuda"))
        else:
            s["x"], s["x_scales"] = normal(m, k, dtype=TYPES[case["x"]][1]), None
        s["y"] = torch.empty(m, n, dtype=TYPES[case["y"]][1], device="cuda")
    else:
        lens, block = lengths(case), case["block"]
        blocks = [-(-v // block) for v in lens]
        width = max(1, max(blocks))
        n_blocks = max(1, sum(blocks)) + 2
        s["q"] = normal(case["batch"], case["heads"], case["dim"], dtype=TYPES[case["q"]][1]) * 1.5
        s["k_all"], s["v_all"] = paged(case, n_blocks, case["kv"], gen, None), paged(case, n_blocks, case["kv"], gen, None)
        s["n_blocks"] = n_blocks
        order = torch.randperm(n_blocks, generator=gen, device="cuda").to(torch.int32)
        # a row holds its blocks in the pool's order, whatever the pool last held past its end
        at, live = [], []
        first = 0
        for r, (v, b) in enumerate(zip(lens, blocks)):
            gone = max(0, v - case["window"]) // block if case["window"] else 0  # blocks that the window has left are given back
            at += [(first + i, r, i) for i in range(gone, b)]
            live.append(v % block)
            first += b
        s["table"] = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
        if at:
            pick = torch.tensor(at, device="cuda")
            s["table"][pick[:, 1], pick[:, 2]] = order[pick[:, 0]]
            # memory that no token was written to yet holds anything, NaN among it
            for r, v in enumerate(lens):
                if live[r]:
                    last = s["table"][r, blocks[r] - 1].long()
                    s["k_all"][last, live[r]:] = float("nan")
                    s["v_all"][last, live[r]:] = float("nan")
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["scale"] = 1.0 / math.sqrt(case["dim"])
        s["out"] = torch.empty_like(s["q"])
    return s


def prepare_plan(case, gen, s):
    both, block, width = lengths(case), case["block"], case["width"]
    ctx = torch.tensor([c for c, _ in both], dtype=torch.int32, device="cuda")
    new = torch.tensor([v for _, v in both], dtype=torch.int32, device="cuda")
    have = ((ctx.long() + block - 1) // block).clamp(max=width)
    want = ((ctx.long() + new + block - 1) // block).clamp(max=width)
    pool = torch.randperm(int(want.sum()) + 9, generator=gen, device="cuda").to(torch.int32)
    cols = torch.arange(width, device="cuda")
    old = (have.cumsum(0) - have)[:, None] + cols
    s["table"] = torch.where(cols < have[:, None], pool[old.clamp(max=pool.numel() - 1)], -1).to(torch.int32)
    s["ctx"], s["new"], s["free"] = ctx, new, pool[int(have.sum()):].contiguous()
    t = s["tokens"] = sum(v for _, v in both) + case["pad"]
    n = case["requests"]
    for name, size, dtype in (("slots", t, torch.int64), ("token_request", t, torch.int32), ("positions", t, torch.int32), ("seq_len", n, torch.int32),
                              ("query_start", n + 1, torch.int32), ("totals", 3, torch.int64)):
        s[name] = torch.empty(size, dtype=dtype, device="cuda")
    return s


# -------------------------------------------------------------- plain forms
def plain_plan(s):
    block, (n, width) = s["case"]["block"], s["table"].shape
    ctx, new = s["ctx"].long().clamp(min=0), s["new"].long().clamp(min=0)
    need_ctx, need_all = (ctx + block - 1) // block, (ctx + new + block - 1) // block
    have, want = need_ctx.clamp(max=width), need_all.clamp(max=width)
    need = want - have
    first = need.cumsum(0) - need
    end = new.cumsum(0)
    cols = torch.arange(width, device="cuda")
    at = first[:, None] + cols - have[:, None]
    page = torch.where(at < s["free"].numel(), s["free"][at.clamp(0, s["free"].numel() - 1)], -1)
    table = torch.where((cols >= have[:, None]) & (cols < want[:, None]), page, s["table"])
    t = torch.arange(s["tokens"], device="cuda")
    request = torch.searchsorted(end, t, right=True)
    real = request < n
    r = request.clamp(max=n - 1)
    pos = ctx[r] + t - (end - new)[r]
    col = pos // block
    page = table[r, col.clamp(max=width - 1)]
    slot = torch.where(real & (col < width) & (page >= 0), page * block + pos % block, -1)
    start = torch.cat([torch.zeros_like(end[:1]), end])
    return [table, slot, torch.where(real, r, -1).int(), torch.where(real, pos, -1).int(), (ctx + new).int(), start.int(),
            torch.stack([end[-1], need.sum(), (need_all > width).sum()])]


def plain_store(s):
    block, heads, dim = s["case"]["block"], s["case"]["heads"], s["case"]["dim"]
    # a token without a slot goes to the block after the cache's end
    slot = torch.where(s["slots"] >= 0, s["slots"], s["n_blocks"] * block)
    for src, whole in (("k", "k_all"), ("v", "v_all")):
        s[whole][slot // block, slot % block] = s[src].reshape(-1, heads, dim).to(s[whole].dtype)
    return [s["k_all"][:-1], s["v_all"][:-1]]


def plain_norm(s):
    case = s["case"]
    h = s["x"].float()
    if s["residual"] is not None:
        h = h + s["residual"].float()
    y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + s["eps"]) * s["weight"]
    outs = [h.to(s["x"].dtype)] if s["residual"] is not None else []
    if case["out"] != "i8":
        return outs + [y.to(TYPES[case["out"]][1])]
    y = y.view(s["values"].shape)
    most = y.abs().amax(2, keepdim=True)
    scale = torch.where(most > 0, most / 127.0, 1.0)
    return outs + [(torch.round(y / scale) * scale).to(torch.bfloat16), scale[:, :, 0]]


def plain_matvec(s):
    case = s["case"]
    n, k, g = case["n"], case["k"], case["group"]
    w = s["w"].to(torch.int32)
    q = torch.stack(((w & 15 ^ 8) - 8, (w >> 4 ^ 8) - 8), 2).view(n, -1)[:, :k]
    deq = q.float() * s["w_scales"].repeat_interleave(g, 1)[:, :k]
    x = s["x"].float()
    if s["x_scales"] is not None:
        x = x * (s["x_scales"].repeat_interleave(case["xgroup"], 1)[:, :k] if case["xgroup"] else s["x_scales"])
    y = x @ deq.t()
    return [(y + s["bias"] if s["bias"] is not None else y).to(s["y"].dtype)]


def plain_attention(s):
    case = s["case"]
    batch, kv, dim, block = case["batch"], case["kv"], case["dim"], case["block"]
    table = s["table"]
    t = torch.arange(table.shape[1] * block, device="cuda")
    lens = s["lens"].long()[:, None]
    seen = (t < lens) & (table >= 0).repeat_interleave(block, 1)
    if case["window"]:
        seen = seen & (t >= lens - case["window"])
    page = table.long().clamp(min=0)

    def gathered(whole):  # [batch, kv, tokens, dim], what no one may look at as zeros
        x = whole[page].reshape(batch, -1, kv, dim).permute(0, 2, 1, 3).float()
        return torch.where(seen[:, None, :, None], x, 0.0)

    q = s["q"].float().view(batch, kv, -1, dim)
    score = (q @ gathered(s["k_all"]).transpose(2, 3)) * s["scale"]
    score = torch.where(seen[:, None, None, :], score, -math.inf)
    most = score.amax(3, keepdim=True)
    p = torch.exp(score - torch.where(most > -math.inf, most, 0.0))
    total = p.sum(3, keepdim=True)
    out = (p @ gathered(s["v_all"])) / torch.where(total > 0, total, 1.0)
    return [out.view(batch, case["heads"], dim).to(s["out"].dtype)]


# -------------------------------------------------------- the framework's own
def own_plan(abi, s, stream):
    n, width = s["table"].shape
    abi.kv_plan_dev(n, s["case"]["block"], s["ctx"].data_ptr(), s["new"].data_ptr(), s["free"].data_ptr(), s["free"].numel(), s["table"].data_ptr(), width,
                    width, s["tokens"], s["slots"].data_ptr(), token_request_ptr=s["token_request"].data_ptr(), positions_ptr=s["positions"].data_ptr(),
                    seq_len_ptr=s["seq_len"].data_ptr(), query_start_ptr=s["query_start"].data_ptr(), totals_ptr=s["totals"].data_ptr(), stream=stream)
    return [s["table"], s["slots"], s["token_request"], s["positions"], s["seq_len"], s["query_start"], s["totals"]]


def own_store(abi, s, stream):
    case, k, v, cache = s["case"], s["k"], s["v"], s["k_all"]
    abi.kv_store_dev(TYPES[case["src"]][0], TYPES[case["cache"]][0], case["tokens"], case["heads"], case["dim"], k.data_ptr(), v.data_ptr(), k.stride(0),
                     v.stride(0), s["slots"].data_ptr(), cache.data_ptr(), s["v_all"].data_ptr(), s["n_blocks"], case["block"], cache.stride(0),
                     cache.stride(1), cache.stride(2), stream=stream)
    return [s["k_all"][:-1], s["v_all"][:-1]]


def own_norm(abi, s, stream):
    case, cols = s["case"], s["case"]["cols"]
    residual = s["residual"]
    abi.rmsnorm_dev(TYPES[case["type"]][0], case["rows"], cols, s["x"].data_ptr(), cols, s["weight"].data_ptr(), s["eps"], TYPES[case["out"]][0],
                    s["out"].data_ptr(), cols, residual_ptr=None if residual is None else residual.data_ptr(), residual_stride=cols,
                    sum_ptr=None if residual is None else s["sum"].data_ptr(), sum_stride=cols,
                    scales_ptr=None if s["scales"] is None else s["scales"].data_ptr(), group=case["group"], stream=stream)
    outs = [s["sum"]] if residual is not None else []
    if case["out"] != "i8":
        return outs + [s["out"]]
    torch.mul(s["out"].view(s["values"].shape), s["scales"][:, :, None], out=s["values"])
    return outs + [s["values"], s["scales"]]


def own_matvec(abi, s, stream):
    case, w, bias, xs = s["case"], s["w"], s["bias"], s["x_scales"]
    abi.matvec_q4g_dev(TYPES[case["x"]][0], case["m"], case["n"], case["k"], s["x"].data_ptr(), case["k"], w.data_ptr(), w.stride(0),
                       s["w_scales"].data_ptr(), case["group"], TYPES[case["y"]][0], s["y"].data_ptr(), case["n"],
                       x_scales_ptr=None if xs is None else xs.data_ptr(), x_group=case["xgroup"], bias_ptr=None if bias is None else bias.data_ptr(),
                       stream=stream)
    return [s["y"]]


def own_attention(abi, s, stream):
    case, q, cache, table = s["case"], s["q"], s["k_all"], s["table"]
    abi.paged_attention_dev(TYPES[case["q"]][0], TYPES[case["cache"]][0], case["batch"], case["heads"], case["kv"], case["dim"], q.data_ptr(), q.stride(0),
                            cache.data_ptr(), s["v_all"].data_ptr(), s["n_blocks"], case["block"], cache.stride(0), cache.stride(1), cache.stride(2),
                            table.data_ptr(), table.shape[1], table.stride(0), s["lens"].data_ptr(), s["scale"], s["out"].data_ptr(), s["out"].stride(0),
                            window=case["window"], stream=stream)
    return [s["out"]]


PLAIN = {"plan": plain_plan, "store": plain_store, "norm": plain_norm, "matvec": plain_matvec, "attention": plain_attention}
OWN = {"plan": own_plan, "store": own_store, "norm": own_norm, "matvec": own_matvec, "attention": own_attention}


def run(state):
    op = state["case"]["op"]
    if not own:
        return PLAIN[op](state)
    from tomoul_amd import _abi

    return OWN[op](_abi, state, torch.cuda.current_stream().cuda_stream)


# ------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}
    op = case["op"]
    if op == "plan":
        both, block, width = lengths(case), case["block"], case["width"]
        tokens = sum(v for _, v in both) + case["pad"]
        fresh = sum(min(-(-(c + v) // block), width) - min(-(-c // block), width) for c, v in both)
        return {"bytes": 16 * case["requests"] + 16 * tokens + 8 * fresh + 24, "flops": 0}
    if op == "store":
        row, tokens = case["heads"] * case["dim"], case["tokens"]
        kept = tokens - min(case["pad"], tokens - 1)
        return {"bytes": 2 * kept * row * (size[case["src"]] + size[case["cache"]]) + 8 * tokens, "flops": 0}
    if op == "norm":
        n = case["rows"] * case["cols"]
        streams = (3 if case["residual"] else 1) * size[case["type"]] + size[case["out"]]
        scales = case["rows"] * (case["cols"] // case["group"] if case["group"] else 1) if case["out"] == "i8" else 0
        return {"bytes": n * streams + 4 * scales + 4 * case["cols"], "flops": 6 * n}
    if op == "matvec":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": n * (-(-k // 2)) + 4 * n * -(-k // case["group"]) + m * k * size[case["x"]] + m * n * size[case["y"]], "flops": 2 * m * n * k}
    total = sum(min(v, case["window"]) if case["window"] else v for v in lengths(case))
    return {"bytes": 2 * total * case["kv"] * case["dim"] * size[case["cache"]] + 2 * case["batch"] * case["heads"] * case["dim"] * size[case["q"]],
            "flops": 4 * total * case["heads"] * case["dim"]}


# ------------------------------------------------------- definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers
    if case["op"] == "store":
        outs = []
        for src, whole in ((s["k"], s["k_all"]), (s["v"], s["v_all"])):
            flat = whole[:-1].double().flatten(0, 1)
            live = (s["slots"] >= 0).nonzero()[:, 0]
            flat[s["slots"][live]] = src[live].double().unflatten(1, (case["heads"], case["dim"]))
            outs.append(flat.unflatten(0, (s["n_blocks"], case["block"])))
        return outs
    if case["op"] == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h += s["residual"].double()
        root = torch.sqrt(h.square().sum(1) / case["cols"] + s["eps"])
        y = h / root[:, None] * s["weight"].double()
        outs = [h] if s["residual"] is not None else []
        if case["out"] != "i8":
            return outs + [y]
        y = y.unflatten(1, (s["scales"].shape[1], -1))
        scale = y.abs().max(2).values / 127
        scale[scale == 0] = 1
        return outs + [torch.round(y / scale[:, :, None]) * scale[:, :, None], scale]
    if case["op"] == "matvec":
        k, x = case["k"], s["x"].double()
        if case["x"] == "i8":
            which = torch.arange(k, device="cuda") // (case["xgroup"] or k)
            x = x * s["x_scales"].double()[:, which]
        table = torch.tensor([v if v < 8 else v - 16 for v in range(16)], dtype=torch.float64, device="cuda")
        y = torch.zeros(case["m"], case["n"], dtype=torch.float64, device="cuda")
        for g in range(s["w_scales"].shape[1]):
            for c in range(g * case["group"], min(k, (g + 1) * case["group"]), 32):
                piece = s["w"][:, c // 2:(min(k, c + 32, (g + 1) * case["group"]) + 1) // 2]
                low, high = table[(piece % 16).long()], table[(piece // 16).long()]
                for part, at in ((low, c), (high, c + 1)):
                    cols = x[:, at:min(k, c + 32):2]
                    y += (cols @ part[:, :cols.shape[1]].t().contiguous()) * s["w_scales"][:, g].double()
        return [y if s["bias"] is None else y + s["bias"].double()]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    many = case["heads"] // case["kv"]
    for r, v in enumerate(lengths(case)):
        t = torch.arange(max(0, v - case["window"]) if case["window"] else 0, v, device="cuda")
        if not len(t):
            continue
        page, at = s["table"][r].long()[t // case["block"]], t % case["block"]
        key = s["k_all"][page, at].double().repeat_interleave(many, 1)
        value = s["v_all"][page, at].double().repeat_interleave(many, 1)
        p = torch.softmax((key * s["q"][r].double()).sum(2) * s["scale"], 0)
        out[r] = (p[:, :, None] * value).sum(0)
    return [out]
