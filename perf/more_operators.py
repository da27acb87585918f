"""Performance cases of the operators around prompts, 4-bit caches and token scores.

A case is a dict of plain values; `op` says which operator it goes through:

  store4    _abi.kv_store_q4_dev, _abi.kv_load_q4_dev  new keys and values to their slots of a paged
                                                       cache held in 4 bits, and slots' rows back
  attn4     _abi.paged_attention_q4_dev                one new token a request over that cache
  attn_ex   _abi.paged_attention_ex_dev                one new token a request over a float cache, scores
                                                       capped by a tanh or biased by distance
  prompt    _abi.prompt_attention_dev                  prompts of any length over a float cache: causal,
                                                       windowed or prefix masks, caps, biases
  logprobs  _abi.token_logprobs_dev                    log probabilities of given tokens, entropy, the
                                                       most likely tokens

`run` computes an operator in its plain form, elementary torch operations in 32 bits
rounded once at the end, or, where `own` is true, with the framework's kernels on the
same state.  `exact` is the definition in 64 bits, written apart from both.

A 4-bit row of a head of 32 G elements is 16 G bytes of nibbles, then G words, the f16
step (low half) and the f16 minimum of each 32 elements: x = nibble * step + minimum.
Element d of a key is nibble d % 8 of the little-endian 32-bit word (d % 32 / 8) * G + d / 32,
element d of a value nibble d / 16 of the G bytes from byte (d % 16) * G.

Sizes are those of the repository's models and benchmark (Whisper large-v3-turbo:
20 heads of 64, 1500 frames, 448 tokens, 51866 words) and generic ones for larger decoders.
"""
import math
import random

import torch

own = False

TYPES = {"f32": (0, torch.float32), "f16": (1, torch.float16), "bf16": (2, torch.bfloat16)}


def listed():
    return [
        # One decode step of a full server: 64 requests, a token each, into a 4-bit cache.
        dict(name="store4_decode_64", op="store4", tokens=64, heads=8, dim=128, block=16, src="bf16", layout="htd", pad=3),
        # A prompt batch of 16k tokens, tokens before heads in a block.
        dict(name="store4_prompt_16k", op="store4", tokens=16384, heads=8, dim=128, block=32, src="bf16", layout="thd", pad=0),
        # One speech decoder step over its self-attention cache in 4 bits: 20 heads of 64, f32 activations.
        dict(name="attn4_one_448", op="attn4", batch=1, heads=20, kv=20, dim=64, least=448, most=448, block=16, q="f32", layout="htd", window=0,
             cap=0.0, slopes=False, lengths=31),
        # A full server: 64 requests of ragged length, some of them empty, grouped heads.
        dict(name="attn4_server_64", op="attn4", batch=64, heads=32, kv=8, dim=128, least=0, most=4096, block=16, q="bf16", layout="htd", window=0,
             cap=0.0, slopes=False, lengths=32),
        # Two long documents, the lengths that a cache in 4 bits is for.
        dict(name="attn4_long_2", op="attn4", batch=2, heads=32, kv=8, dim=128, least=40000, most=65536, block=32, q="f16", layout="htd", window=0,
             cap=0.0, slopes=False, lengths=33),
        # Decode of a model that caps its scores: 32 requests, ragged.
        dict(name="attn_cap_32", op="attn_ex", batch=32, heads=16, kv=8, dim=256, least=0, most=4096, block=16, q="bf16", cache="bf16", layout="htd",
             window=0, cap=50.0, slopes=False, lengths=34),
        # Decode of a model without position embeddings: a bias by distance, every head its own keys.
        dict(name="attn_slopes_4", op="attn_ex", batch=4, heads=20, kv=20, dim=64, least=300, most=2000, block=16, q="f32", cache="f16", layout="thd",
             window=0, cap=0.0, slopes=True, lengths=35),
        # The speech encoder's attention: every frame sees every frame.
        dict(name="prompt_encoder_1500", op="prompt", requests=1, heads=20, kv=20, dim=64, new_least=1500, new_most=1500, ctx_most=0, block=1500,
             q="f16", cache="f16", layout="thd", prefix="all", window=0, cap=0.0, slopes=False, pad=0, lengths=36),
        # A mixed batch: decodes and chunks of prompts over contexts to 4096, scores capped.
        dict(name="prompt_mixed_16", op="prompt", requests=16, heads=32, kv=8, dim=128, new_least=1, new_most=256, ctx_most=4096, block=16, q="bf16",
             cache="bf16", layout="htd", prefix="none", window=0, cap=30.0, slopes=False, pad=37, lengths=37),
        # Two long prompts, causal: the matrix cores' case.
        dict(name="prompt_long_2", op="prompt", requests=2, heads=32, kv=8, dim=128, new_least=6000, new_most=8192, ctx_most=0, block=32, q="bf16",
             cache="bf16", layout="htd", prefix="none", window=0, cap=0.0, slopes=False, pad=0, lengths=38),
        # A decode step's scores: four sequences, f32 logits over the speech vocabulary, the five best.
        dict(name="logprobs_step_4", op="logprobs", rows=4, cols=51866, type="f32", top=5),
        # The scores of a prompt's 2048 tokens, bf16 logits.
        dict(name="logprobs_prompt_2k", op="logprobs", rows=2048, cols=51866, type="bf16", top=0),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(("store4", "attn4", "attn4", "attn_ex", "prompt", "prompt", "logprobs"))
    layout = rng.choice(("thd", "htd"))
    if op == "store4":
        return dict(op=op, tokens=log(1, 16384), heads=rng.choice((1, 2, 5, 8)), dim=rng.choice((32, 64, 96, 128, 128)), block=rng.choice((8, 16, 24, 32)),
                    src=rng.choice(("f32", "f16", "bf16")), layout=layout, pad=rng.randrange(8))
    if op == "logprobs":
        cols = log(100, 131072)
        return dict(op=op, rows=max(1, min(log(1, 2048), 100_000_000 // cols)), cols=cols, type=rng.choice(("f32", "f16", "bf16")), top=rng.choice((0, 1, 5, 20, 64)))
    cap, slopes = rng.choice((0.0, 0.0, 20.0, 50.0)), rng.random() < 0.3
    if op == "prompt":
        cache = rng.choice(("f16", "bf16", "f16", "bf16", "f32"))
        kv = rng.choice((1, 2, 8))
        heads = kv * rng.choice((1, 1, 2, 4, 5))
        new, ctx = log(1, 4096), rng.choice((0, log(1, 4096)))
        requests = max(1, min(log(1, 16), 600_000_000 // (heads * new * (new + ctx))))
        return dict(op=op, requests=requests, heads=heads, kv=kv, dim=rng.choice((64, 64, 80, 128, 128, 256)), new_least=rng.choice((0, 1, new // 2, new)), new_most=new,
                    ctx_most=ctx, block=rng.choice((1, 8, 16, 16, 32, 50)), q=rng.choice(("f32", cache, cache)), cache=cache, layout=layout,
                    prefix=rng.choice(("none", "none", "some", "all")), window=rng.choice((0, 0, 0, log(1, 4096))), cap=cap, slopes=slopes,
                    pad=rng.randrange(50), lengths=rng.randrange(1 << 30))
    kv, most = rng.choice((1, 2, 8, 10)), log(16, 16384)
    case = dict(op=op, kv=kv, heads=kv * rng.choice((1, 1, 5, 4, 8, 16)), least=rng.choice((0, 1, most // 2, most)), most=most, block=rng.choice((1, 8, 16, 16, 32, 50)),
                layout=layout, window=rng.choice((0, 0, 0, log(1, 4096))), cap=cap, slopes=slopes, lengths=rng.randrange(1 << 30))
    if op == "attn4":
        case["dim"] = rng.choice((32, 64, 64, 96, 128, 128, 160, 256))
        case["q"] = rng.choice(("f32", "f16", "bf16"))
        wide = 1
    else:
        case["cache"] = rng.choice(("f16", "bf16", "f32"))
        case["dim"] = rng.choice((64, 64, 80, 128, 128, 256))
        case["q"] = rng.choice(("f32", case["cache"]))
        if not case["cap"] and not case["slopes"]:
            case["cap"] = 30.0
        wide = 2 if case["cache"] == "f32" else 1
    case["batch"] = max(1, min(log(1, 64), 200_000_000 // (most * kv * case["dim"] * wide)))
    return case


# ------------------------------------------------------------------ inputs
def lengths(case):
    """The ragged lengths of a case, part of the case and alike for every seed: of a request, or its context, new tokens and prefix."""
    r = random.Random(case["lengths"])
    if case["op"] != "prompt":
        return [r.randint(case["least"], case["most"]) for _ in range(case["batch"])]
    both = []
    for _ in range(case["requests"]):
        ctx, new, part = r.randint(0, case["ctx_most"]), r.randint(case["new_least"], case["new_most"]), r.random()
        both.append((ctx, new, {"none": 0, "all": ctx + new, "some": int(part * (ctx + new))}[case["prefix"]]))
    return both


def pool(case, n_blocks, heads, row, dtype):
    """An empty cache [block, token, head, row], stored in the case's order, with one block after its end that is no part of it."""
    if case["layout"] == "thd":
        return torch.empty(n_blocks + 1, case["block"], heads, row, dtype=dtype, device="cuda")
    return torch.empty(n_blocks + 1, heads, case["block"], row, dtype=dtype, device="cuda").permute(0, 2, 1, 3)


def tables(case, s, lens, gone):
    """Block tables over a shuffled pool, the first gone[r] blocks of a row given back; what lies past a request's end is left."""
    block = case["block"]
    blocks = [-(-v // block) for v in lens]
    n_blocks, width = s["n_blocks"], max(1, max(blocks))
    order = torch.randperm(n_blocks, generator=s["gen"], device="cuda").to(torch.int32)
    s["table"] = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    at, first = [], 0
    for r, b in enumerate(blocks):
        at += [(first + i, r, i) for i in range(min(gone[r], b), b)]
        first += b
    if at:
        pick = torch.tensor(at, device="cuda")
        s["table"][pick[:, 1], pick[:, 2]] = order[pick[:, 0]]
    # memory that no token was written to yet holds anything: NaN here, of bytes with all bits set
    ends = [(r, blocks[r] - 1, v % block) for r, v in enumerate(lens) if v % block]
    if ends:
        e = torch.tensor(ends, device="cuda")
        last = s["table"][e[:, 0], e[:, 1]].long()
        free = torch.arange(block, device="cuda") >= e[:, 2:]
        for whole in ("k_all", "v_all"):
            page = s[whole][last]
            page[free] = 255 if page.dtype == torch.uint8 else float("nan")
            s[whole][last] = page


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    s, op = {"case": case, "gen": gen}, case["op"]
    if op == "store4":
        tokens, heads, dim, block = case["tokens"], case["heads"], case["dim"], case["block"]
        s["n_blocks"] = -(-tokens // block) + 3
        # keys and values are the middle and the last part of a fused projection's rows; some channels of keys are loud
        loud = torch.where(torch.rand(3 * heads * dim, generator=gen, device="cuda") < 0.03, 8.0, 1.0)
        fused = (normal(tokens, 3 * heads * dim) * loud).to(TYPES[case["src"]][1])
        s["k"], s["v"] = fused[:, heads * dim:2 * heads * dim], fused[:, 2 * heads * dim:]
        slots = torch.randperm(s["n_blocks"] * block, generator=gen, device="cuda")[:tokens]
        slots[tokens - min(case["pad"], tokens - 1):] = -1
        s["slots"] = slots.contiguous()
        for name in ("k", "v"):
            s[name + "_all"] = pool(case, s["n_blocks"], heads, 20 * dim // 32, torch.uint8).zero_()
            s[name + "_back"] = torch.zeros(tokens, heads, dim, dtype=torch.bfloat16, device="cuda")
        return s
    if op == "logprobs":
        rows, cols, dtype = case["rows"], case["cols"], TYPES[case["type"]][1]
        # a few words stand out, by more in some rows than in others
        s["logits"] = (normal(rows, cols) * 2.0 + 12.0 * (torch.rand(rows, cols, generator=gen, device="cuda") < 5.0 / cols) * torch.rand(rows, 1, generator=gen, device="cuda")).to(dtype)
        s["tokens"] = torch.where(torch.rand(rows, generator=gen, device="cuda") < 0.5, s["logits"].argmax(1), torch.randint(0, cols, (rows,), generator=gen, device="cuda")).to(torch.int32)
        s["logprobs"], s["entropy"] = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
        if case["top"]:
            s["top_ids"], s["top_logprobs"] = torch.empty(rows, case["top"], dtype=torch.int32, device="cuda"), torch.empty(rows, case["top"], device="cuda")
        return s
    kv, dim, block = case["kv"], case["dim"], case["block"]
    if op == "prompt":
        both = lengths(case)
        lens, gone = [c + n for c, n, _ in both], [0] * len(both)
        s["starts"] = [0]
        for _, n, _ in both:
            s["starts"].append(s["starts"][-1] + n)
        rows = s["starts"][-1] + case["pad"]
        s["query_start"] = torch.tensor(s["starts"], dtype=torch.int32, device="cuda")
        s["prefix"] = torch.tensor([p for _, _, p in both], dtype=torch.int32, device="cuda") if case["prefix"] != "none" else None
        s["most_new"] = max(1, max(n for _, n, _ in both))
    else:
        lens, rows = lengths(case), case["batch"]
        gone = [max(0, v - case["window"]) // block if case["window"] else 0 for v in lens]  # blocks that the window has left are given back
    s["n_blocks"] = max(1, sum(-(-v // block) for v in lens)) + 2
    s["q"] = normal(rows, case["heads"], dim, dtype=TYPES[case["q"]][1]) * 1.5
    for name in ("k_all", "v_all"):
        if op == "attn4":
            s[name] = pool(case, s["n_blocks"], kv, 20 * dim // 32, torch.uint8)
            step = max(1, 50_000_000 // (block * kv * dim))
            for b in range(0, s["n_blocks"] + 1, step):
                part = s[name][b:b + step]
                part.copy_(packed(torch.randn(part.shape[:3] + (dim,), generator=gen, device="cuda"), name == "k_all"))
        else:
            s[name] = pool(case, s["n_blocks"], kv, dim, TYPES[case["cache"]][1]).normal_(generator=gen)
    tables(case, s, lens, gone)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    s["scale"] = 1.0 / math.sqrt(dim)
    s["slopes"] = torch.exp2(-8.0 * torch.arange(1, case["heads"] + 1, device="cuda") / case["heads"]) if case["slopes"] else None
    s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------ rows held in 4 bits
def order(dim, key):
    """Where element d of a row is: its byte, and whether it is the high nibble."""
    d, g = torch.arange(dim, device="cuda"), dim // 32
    if key:
        return 4 * (d % 32 // 8 * g + d // 32) + d % 8 // 2, d % 2
    return d % 16 * g + d // 32, d // 16 % 2


def quantized(x):
    """Nibbles, steps and minima of [.., dim] floats in groups of 32."""
    x = x.clamp(-65504.0, 65504.0).unflatten(-1, (-1, 32))
    low, high = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    step, least = ((high - low) / 15.0).half(), low.half()
    n = torch.where(step > 0, torch.round((x - least.float()) / torch.where(step > 0, step, 1.0).float()), 0.0).clamp(0.0, 15.0)
    return n, step, least


def packed(x, key):
    """The rows that hold the floats x [.., dim] in 4 bits."""
    n, step, least = quantized(x)
    at, high = order(x.shape[-1], key)
    n = n.flatten(-2).to(torch.uint8)
    rows = torch.empty(x.shape[:-1] + (x.shape[-1] // 2,), dtype=torch.uint8, device="cuda")
    rows[..., at[high == 0]] = n[..., high == 0]
    rows[..., at[high == 1]] |= n[..., high == 1] << 4
    return torch.cat([rows, torch.cat([step, least], -1).view(torch.uint8).flatten(-2)], -1)


def unpacked(rows, dim, key):
    """The floats that rows in 4 bits stand for."""
    at, high = order(dim, key)
    n = rows[..., at] >> (4 * high).to(torch.uint8) & 15
    both = rows[..., dim // 2:].contiguous().view(torch.float16).float().unflatten(-1, (-1, 2))
    return (n.float().unflatten(-1, (-1, 32)) * both[..., :1] + both[..., 1:]).flatten(-2)


# -------------------------------------------------------------- plain forms
def plain_store4(s):
    case, block = s["case"], s["case"]["block"]
    # a token without a slot goes to the block after the cache's end
    live = s["slots"] >= 0
    slot = torch.where(live, s["slots"], s["n_blocks"] * block)
    outs = []
    for name in ("k", "v"):
        x = s[name].float().unflatten(1, (case["heads"], case["dim"]))
        s[name + "_all"][slot // block, slot % block] = packed(x, name == "k")
        back = unpacked(s[name + "_all"][slot // block, slot % block], case["dim"], name == "k").to(torch.bfloat16)
        outs.append(torch.where(live[:, None, None], back, s[name + "_back"]))
    return outs


def gathered(s, name, seen):
    """[batch, kv, tokens, dim] of the cache, what no one may look at as zeros."""
    case = s["case"]
    x = s[name][s["table"].long().clamp(min=0)].flatten(1, 2)
    x = unpacked(x, case["dim"], name == "k_all") if case["op"] == "attn4" else x.float()
    return torch.where(seen[:, None, :, None], x.permute(0, 2, 1, 3), 0.0)


def weighted(s, score, away, seen, values):
    """Softmax of the capped and biased scores [batch, kv, group, .., tokens] over the tokens that are seen, times the values."""
    case = s["case"]
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    if s["slopes"] is not None:
        score = score - s["slopes"].view((1, case["kv"], -1) + (1,) * (score.dim() - 3)) * away
    score = torch.where(seen, score, -math.inf)
    most = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(most > -math.inf, most, 0.0))
    total = p.sum(-1, keepdim=True)
    out = (p.flatten(2, -2) @ values).view(p.shape[:-1] + values.shape[-1:])
    return out / torch.where(total > 0, total, 1.0)


def plain_decode(s):
    case, table = s["case"], s["table"]
    t = torch.arange(table.shape[1] * case["block"], device="cuda")
    lens = s["lens"].long()[:, None]
    seen = (t < lens) & (table >= 0).repeat_interleave(case["block"], 1)
    if case["window"]:
        seen = seen & (t >= lens - case["window"])
    q = s["q"].float().view(case["batch"], case["kv"], -1, case["dim"])
    score = (q @ gathered(s, "k_all", seen).transpose(2, 3)) * s["scale"]
    away = (lens - 1 - t).abs()[:, None, None]
    out = weighted(s, score, away, seen[:, None, None], gathered(s, "v_all", seen))
    return [out.view(s["out"].shape).to(s["out"].dtype)]


def plain_prompt(s):
    case, table = s["case"], s["table"]
    kv, dim, n = case["kv"], case["dim"], s["most_new"]
    t = torch.arange(table.shape[1] * case["block"], device="cuda")
    lens, start = s["lens"].long()[:, None], s["query_start"].long()
    there = (t < lens) & (table >= 0).repeat_interleave(case["block"], 1)
    i = torch.arange(n, device="cuda")
    new = (start[1:] - start[:-1])[:, None]
    pos = (lens - new + i)[:, :, None]  # of each new token
    seen = t <= pos
    if s["prefix"] is not None:
        seen = seen | (t < s["prefix"][:, None, None])
    if case["window"]:
        seen = seen & (t > pos - case["window"])
    seen = (seen & there[:, None])[:, None, None]
    row = (start[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][row].float().permute(0, 2, 1, 3).reshape(-1, kv, case["heads"] // kv * n, dim)
    score = (q @ gathered(s, "k_all", there).transpose(2, 3)).view(-1, kv, case["heads"] // kv, n, t.shape[0]) * s["scale"]
    out = weighted(s, score, (pos - t).abs()[:, None, None], seen, gathered(s, "v_all", there))
    out = out.flatten(1, 2).transpose(1, 2).to(s["out"].dtype)
    whole = torch.zeros_like(s["out"])
    live = i < new
    whole[row[live]] = out[live]
    return [whole]


def plain_logprobs(s):
    case = s["case"]
    x = s["logits"].float()
    x = x - x.amax(1, keepdim=True)
    e = torch.exp(x)
    total = e.sum(1, keepdim=True)
    lse = torch.log(total)
    outs = [(x.gather(1, s["tokens"].long()[:, None]) - lse)[:, 0], (lse - (e * x).sum(1, keepdim=True) / total)[:, 0]]
    if case["top"]:
        value, index = torch.sort(x, dim=1, descending=True, stable=True)
        outs += [index[:, :case["top"]].int().contiguous(), value[:, :case["top"]] - lse]
    return outs


# -------------------------------------------------------- the framework's own
def own_store4(abi, s, stream):
    case, k, v, cache, back = s["case"], s["k"], s["v"], s["k_all"], s["k_back"]
    type_, heads, dim, row = TYPES[case["src"]][0], case["heads"], case["dim"], back.stride(0)
    where = (s["n_blocks"], case["block"], cache.stride(0), cache.stride(1), cache.stride(2))
    abi.kv_store_q4_dev(type_, case["tokens"], heads, dim, k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), s["slots"].data_ptr(), cache.data_ptr(),
                        s["v_all"].data_ptr(), *where, stream=stream)
    abi.kv_load_q4_dev(TYPES["bf16"][0], case["tokens"], heads, dim, cache.data_ptr(), s["v_all"].data_ptr(), *where, s["slots"].data_ptr(), back.data_ptr(),
                       s["v_back"].data_ptr(), row, row, stream=stream)
    return [s["k_back"], s["v_back"]]


def cache_of(s):
    case, cache, table = s["case"], s["k_all"], s["table"]
    return (cache.data_ptr(), s["v_all"].data_ptr(), s["n_blocks"], case["block"], cache.stride(0), cache.stride(1), cache.stride(2), table.data_ptr(),
            table.shape[1], table.stride(0))


def more_of(s):
    return dict(window=s["case"]["window"], cap=s["case"]["cap"], slopes_ptr=None if s["slopes"] is None else s["slopes"].data_ptr())


def own_attn4(abi, s, stream):
    case, q, out = s["case"], s["q"], s["out"]
    abi.paged_attention_q4_dev(TYPES[case["q"]][0], case["batch"], case["heads"], case["kv"], case["dim"], q.data_ptr(), q.stride(0), *cache_of(s),
                               s["lens"].data_ptr(), s["scale"], out.data_ptr(), out.stride(0), stream=stream, **more_of(s))
    return [out]


def own_attn_ex(abi, s, stream):
    case, q, out = s["case"], s["q"], s["out"]
    abi.paged_attention_ex_dev(TYPES[case["q"]][0], TYPES[case["cache"]][0], case["batch"], case["heads"], case["kv"], case["dim"], q.data_ptr(), q.stride(0),
                               *cache_of(s), s["lens"].data_ptr(), s["scale"], out.data_ptr(), out.stride(0), stream=stream, **more_of(s))
    return [out]


def own_prompt(abi, s, stream):
    case, q, out, prefix = s["case"], s["q"], s["out"], s["prefix"]
    abi.prompt_attention_dev(TYPES[case["q"]][0], TYPES[case["cache"]][0], q.shape[0], case["requests"], case["heads"], case["kv"], case["dim"], q.data_ptr(),
                             q.stride(0), *cache_of(s), s["query_start"].data_ptr(), s["lens"].data_ptr(), s["scale"], out.data_ptr(), out.stride(0),
                             prefix_len_ptr=None if prefix is None else prefix.data_ptr(), stream=stream, **more_of(s))
    return [out]


def own_logprobs(abi, s, stream):
    case, x, top = s["case"], s["logits"], s["case"]["top"]
    abi.token_logprobs_dev(TYPES[case["type"]][0], case["rows"], case["cols"], x.data_ptr(), x.stride(0), tokens_ptr=s["tokens"].data_ptr(),
                           logprobs_ptr=s["logprobs"].data_ptr(), entropy_ptr=s["entropy"].data_ptr(), top=top,
                           top_ids_ptr=s["top_ids"].data_ptr() if top else None, top_logprobs_ptr=s["top_logprobs"].data_ptr() if top else None, stream=stream)
    return [s["logprobs"], s["entropy"]] + ([s["top_ids"], s["top_logprobs"]] if top else [])


PLAIN = {"store4": plain_store4, "attn4": plain_decode, "attn_ex": plain_decode, "prompt": plain_prompt, "logprobs": plain_logprobs}
OWN = {"store4": own_store4, "attn4": own_attn4, "attn_ex": own_attn_ex, "prompt": own_prompt, "logprobs": own_logprobs}


def run(state):
    op = state["case"]["op"]
    if not own:
        return PLAIN[op](state)
    from tomoul_amd import _abi

    return OWN[op](_abi, state, torch.cuda.current_stream().cuda_stream)


# ------------------------------------------------------------------- work
def pairs(case):
    """Query-key pairs that a prompt case's mask leaves."""
    n = 0
    for ctx, new, prefix in lengths(case):
        for pos in range(ctx, ctx + new):
            n += max(pos + 1, min(prefix, ctx + new)) - (max(0, pos + 1 - case["window"]) if case["window"] else 0)
    return n


def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    op = case["op"]
    if op == "store4":
        elements = case["heads"] * case["dim"]
        kept = case["tokens"] - min(case["pad"], case["tokens"] - 1)
        # stored (source, 5 bits), loaded (5 bits, bf16)
        return {"bytes": 2 * kept * elements * (size[case["src"]] + 2 * 0.625 + 2) + 16 * case["tokens"], "flops": 0}
    if op == "logprobs":
        n = case["rows"] * case["cols"]
        return {"bytes": n * size[case["type"]] + case["rows"] * (12 + 8 * case["top"]), "flops": 4 * n}
    if op == "prompt":
        both = lengths(case)
        tokens, total = sum(n for _, n, _ in both), sum(c + n for c, n, _ in both)
        return {"bytes": 2 * total * case["kv"] * case["dim"] * size[case["cache"]] + 2 * tokens * case["heads"] * case["dim"] * size[case["q"]],
                "flops": 4 * pairs(case) * case["heads"] * case["dim"]}
    total = sum(min(v, case["window"]) if case["window"] else v for v in lengths(case))
    element = 0.625 if op == "attn4" else size[case["cache"]]
    return {"bytes": 2 * total * case["kv"] * case["dim"] * element + 2 * case["batch"] * case["heads"] * case["dim"] * size[case["q"]],
            "flops": 4 * total * case["heads"] * case["dim"]}


# ------------------------------------------------------- definitions in 64 bits
def decoded(rows, dim, key):
    """What [tokens, kv, bytes] rows in 4 bits say, element by element, in 64 bits."""
    g = dim // 32
    halves = rows[..., 16 * g:].contiguous().view(torch.float16).double()
    nibbles = torch.stack([rows[..., :16 * g] % 16, rows[..., :16 * g] // 16], -1).flatten(-2).double()
    out = torch.empty(rows.shape[:-1] + (dim,), dtype=torch.float64, device="cuda")
    for d in range(dim):
        nibble = 8 * ((d % 32) // 8 * g + d // 32) + d % 8 if key else 2 * g * (d % 16) + d // 16
        out[..., d] = nibbles[..., nibble] * halves[..., d // 32 * 2] + halves[..., d // 32 * 2 + 1]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "store4":
        outs = []
        for name in ("k", "v"):
            x = s[name].double().view(case["tokens"], case["heads"], -1, 32)
            low = x.min(3).values
            step, low = ((x.max(3).values - low) / 15).half().double()[..., None], low.half().double()[..., None]
            back = (torch.round((x - low) / step).clamp(0, 15) * step + low).flatten(2)
            back[s["slots"] < 0] = 0
            outs.append(back)
        return outs
    if case["op"] == "logprobs":
        best, x = [], s["logits"].double()
        logp = x - torch.logsumexp(x, 1, keepdim=True)
        if case["top"]:
            best = [None, torch.topk(logp, case["top"], 1).values]
        return [logp[torch.arange(case["rows"], device="cuda"), s["tokens"].long()], -(logp.exp() * logp).sum(1)] + best
    if case["op"] == "prompt" and 4 * pairs(case) * case["heads"] * case["dim"] > 3e12:
        return None
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    many = case["heads"] // case["kv"]
    for r, v in enumerate(lengths(case)):
        ctx, new, prefix = v if case["op"] == "prompt" else (v - 1, 1, 0)
        first = s["starts"][r] if case["op"] == "prompt" else r
        total = ctx + new
        if new == 0 or total <= 0:
            continue
        t = torch.arange(total, device="cuda")
        t = t[s["table"][r].long()[t // case["block"]] >= 0]
        page, at = s["table"][r].long()[t // case["block"]], t % case["block"]
        key, value = s["k_all"][page, at], s["v_all"][page, at]
        if case["op"] == "attn4":
            key, value = decoded(key, case["dim"], True), decoded(value, case["dim"], False)
        for i0 in range(0, new, 1024):
            i1 = min(new, i0 + 1024)
            pos = torch.arange(ctx + i0, ctx + i1, device="cuda")[:, None]
            hidden = (t > pos) & (t >= prefix)
            if case["window"]:
                hidden |= t <= pos - case["window"]
            for h in range(case["heads"]):
                score = s["q"][first + i0:first + i1, h].double() @ key[:, h // many].double().t().contiguous() * s["scale"]
                if case["cap"]:
                    score = torch.tanh(score / case["cap"]) * case["cap"]
                if s["slopes"] is not None:
                    score -= s["slopes"][h].double() * (pos - t).abs()
                score[hidden] = -math.inf
                p = torch.softmax(score, 1).nan_to_num(0.0)
                out[first + i0:first + i1, h] = p @ value[:, h // many].double()
    return [out]
