"""The serving operators one after the other, as a server uses them: a plan of the cache,
new keys and values to a bf16 and a 4-bit cache, attention of the prompts, attention of
the next tokens over both caches, scores of the tokens; eager, captured and replayed,
on two streams.

Tolerances are those of tests/test_gpu_serving_more.py: each operator against its definition in 64 bits
on the inputs that it got, so no error is carried from one to the next."""
import os
import sys

import numpy as np
import pytest

from tomoul_amd import _abi

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, HERE)
import serving_ref as ref  # noqa: E402
from serving_ref import BF16, F32, HALF_ULP, TINY, close, values  # noqa: E402

pytestmark = pytest.mark.gpu

HEADS, KV, DIM, BLOCK, COLS, TOP = 8, 2, 64, 16, 1000, 5
ROW, BYTES = KV * DIM, ref.row_bytes(DIM)
SCALE, CAP = 0.125, 20.0


class Server:
    """Three requests, a bf16 cache [block][token][head][dim] and the same in 4 bits."""

    def __init__(self, new, room=800):
        import torch
        self.requests, self.width = len(new), -(-room // BLOCK)
        self.most, self.n_blocks = sum(new) + 3, self.width * len(new)  # (three tokens of padding)
        rng = np.random.default_rng(5)

        def ints(n, v=0, t=torch.int32):
            return torch.full((n,), v, dtype=t, device="cuda")
        self.ctx, self.new, self.table = ints(self.requests), torch.tensor(new, dtype=torch.int32, device="cuda"), ints(self.requests * self.width, -1)
        self.free = torch.tensor(rng.permutation(self.n_blocks), dtype=torch.int32, device="cuda")
        self.n_free = self.n_blocks
        self.slots, self.totals = ints(self.most, -5, torch.int64), ints(3, 0, torch.int64)
        self.token_request, self.positions, self.seq, self.start = ints(self.most), ints(self.most), ints(self.requests), ints(self.requests + 1)
        self.cache = [torch.zeros(self.n_blocks * BLOCK * ROW, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        self.cache4 = [torch.zeros(self.n_blocks * BLOCK * KV * BYTES, dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.slopes = torch.tensor(2.0 ** -rng.uniform(2, 8, HEADS), dtype=torch.float32, device="cuda")
        self.head = torch.tensor(rng.standard_normal((COLS, HEADS * DIM)) / 8, dtype=torch.bfloat16, device="cuda")
        self.rng = rng
        self.buffers(self.most)

    def buffers(self, tokens):
        import torch

        def floats(cols, t=torch.bfloat16):
            return torch.zeros(tokens, cols, dtype=t, device="cuda")
        self.tokens = tokens
        self.q, self.k, self.v, self.out, self.out4, self.logits = floats(HEADS * DIM), floats(ROW), floats(ROW), floats(HEADS * DIM), floats(HEADS * DIM), floats(COLS)
        self.targets = torch.zeros(tokens, dtype=torch.int32, device="cuda")
        self.lp, self.entropy, self.best = floats(1, torch.float32), floats(1, torch.float32), floats(TOP, torch.float32)
        self.ids = torch.zeros(tokens, TOP, dtype=torch.int32, device="cuda")

    def fill(self, seed):
        import torch
        rng = np.random.default_rng(seed)
        for x in (self.q, self.k, self.v):
            x.copy_(torch.tensor(rng.standard_normal(x.shape), dtype=torch.bfloat16))
        self.targets.copy_(torch.tensor(rng.integers(-1, COLS, self.tokens), dtype=torch.int32))

    def strides(self, row):
        return BLOCK * KV * row, KV * row, row

    def plan(self, s=None):
        _abi.kv_plan_dev(self.requests, BLOCK, self.ctx.data_ptr(), self.new.data_ptr(), self.free.data_ptr(), self.n_free, self.table.data_ptr(), self.width,
                         self.width, self.tokens, self.slots.data_ptr(), token_request_ptr=self.token_request.data_ptr(), positions_ptr=self.positions.data_ptr(),
                         seq_len_ptr=self.seq.data_ptr(), query_start_ptr=self.start.data_ptr(), totals_ptr=self.totals.data_ptr(), stream=s)

    def store(self, s=None):
        at = (self.k.data_ptr(), self.v.data_ptr(), ROW, ROW, self.slots.data_ptr())
        _abi.kv_store_dev(BF16, BF16, self.tokens, KV, DIM, *at, *(c.data_ptr() for c in self.cache), self.n_blocks, BLOCK, *self.strides(DIM), stream=s)
        _abi.kv_store_q4_dev(BF16, self.tokens, KV, DIM, *at, *(c.data_ptr() for c in self.cache4), self.n_blocks, BLOCK, *self.strides(BYTES), stream=s)

    def prompts(self, s=None, out=None, cache=None):
        _abi.prompt_attention_dev(BF16, BF16, self.tokens, self.requests, HEADS, KV, DIM, self.q.data_ptr(), HEADS * DIM, *(c.data_ptr() for c in cache or self.cache),
                                  self.n_blocks, BLOCK, *self.strides(DIM), self.table.data_ptr(), self.width, self.width, self.start.data_ptr(), self.seq.data_ptr(),
                                  SCALE, (self.out if out is None else out).data_ptr(), HEADS * DIM, cap=CAP, slopes_ptr=self.slopes.data_ptr(), stream=s)

    def next_tokens(self, s=None):
        rest = (self.table.data_ptr(), self.width, self.width, self.seq.data_ptr(), SCALE)
        more = dict(cap=CAP, slopes_ptr=self.slopes.data_ptr(), stream=s)
        _abi.paged_attention_ex_dev(BF16, BF16, self.requests, HEADS, KV, DIM, self.q.data_ptr(), HEADS * DIM, *(c.data_ptr() for c in self.cache), self.n_blocks, BLOCK,
                                    *self.strides(DIM), *rest, self.out.data_ptr(), HEADS * DIM, **more)
        _abi.paged_attention_q4_dev(BF16, self.requests, HEADS, KV, DIM, self.q.data_ptr(), HEADS * DIM, *(c.data_ptr() for c in self.cache4), self.n_blocks, BLOCK,
                                    *self.strides(BYTES), *rest, self.out4.data_ptr(), HEADS * DIM, **more)

    def score(self, s=None):
        _abi.token_logprobs_dev(BF16, self.tokens, COLS, self.logits.data_ptr(), COLS, tokens_ptr=self.targets.data_ptr(), logprobs_ptr=self.lp.data_ptr(),
                                entropy_ptr=self.entropy.data_ptr(), top=TOP, top_ids_ptr=self.ids.data_ptr(), top_logprobs_ptr=self.best.data_ptr(), stream=s)

    def after_plan(self):
        """The blocks that the plan took are no longer free."""
        taken = int(self.totals[1])
        self.free = self.free[taken:].contiguous()
        self.n_free -= taken

    def rows_of(self, r, four):
        """Keys and values that request r's table leads to, and their magnitudes, in 64 bits."""
        n = int(self.seq[r])
        blocks = self.table.cpu().numpy().reshape(self.requests, -1)[r]
        at = np.array([blocks[t // BLOCK] * BLOCK + t % BLOCK for t in range(n)], np.int64)
        found = []
        for w in range(2):
            if four:
                rows = self.cache4[w].cpu().numpy().reshape(-1, KV, BYTES)[at]
                found.append(ref.unpack_rows(rows, DIM, w == 0))
            else:
                x = self.cache[w].float().cpu().numpy().astype(np.float64).reshape(-1, KV, DIM)[at]
                found.append((x, np.abs(x)))
        return found

    def check_attention(self, out, four, weight):
        start = self.start.cpu().numpy()
        got, q = out.float().cpu().numpy().astype(np.float64), self.q.float().cpu().numpy().astype(np.float64)
        for r in range(self.requests):
            n = int(self.seq[r])
            (k, km), (v, vm) = self.rows_of(r, four)
            rows = slice(start[r], start[r + 1])
            pos = np.arange(n - (start[r + 1] - start[r]), n)
            t = np.arange(n)
            want, tol = ref.attention(q[rows].reshape(-1, HEADS, DIM), k, v, pos, scale=SCALE, cap=CAP, slopes=self.slopes.cpu().numpy().astype(np.float64),
                                      seen=ref.sees(pos, t, 0, 0), positions=t, key_mag=km, val_mag=vm, weight=weight)
            close(got[rows].reshape(want.shape), want, tol + HALF_ULP[BF16] * (np.abs(want) + tol) + TINY[BF16], f"request {r}")

    def check_scores(self):
        x = self.logits.float().cpu().numpy().astype(np.float64)
        lp, ent, ids, best = ref.logprobs(x, self.targets.cpu().numpy(), TOP)
        sums = 8 * np.sqrt(COLS) * ref.U
        close(self.lp.cpu().numpy()[:, 0], lp, sums + 4 * ref.U * (1 + np.abs(lp)))
        close(self.entropy.cpu().numpy()[:, 0], ent, 4 * sums * (1 + np.abs(ent)))
        close(self.best.cpu().numpy(), best, sums + 4 * ref.U * (1 + np.abs(best)))
        assert np.array_equal(self.ids.cpu().numpy(), ids)

    def project(self):
        import torch
        torch.mm(self.out, self.head.t(), out=self.logits)


def test_prompts_then_tokens():
    import torch
    s = Server([70, 1, 600])
    s.fill(1)
    s.out.fill_(3.0)
    s.plan()
    s.store()
    s.prompts()
    s.after_plan()
    assert s.seq.tolist() == [70, 1, 600] and s.start.tolist() == [0, 70, 71, 671]
    s.check_attention(s.out, False, 2.0 ** -8)
    assert (s.out[671:] == 3.0).all()  # padding: left as it was
    s.project()
    s.score()
    s.check_scores()
    # the 4-bit cache's rows as floats, and the prompts over those
    live = s.slots[:671].contiguous()
    rows = [torch.zeros(671, ROW, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    _abi.kv_load_q4_dev(BF16, 671, KV, DIM, *(c.data_ptr() for c in s.cache4), s.n_blocks, BLOCK, *s.strides(BYTES), live.data_ptr(), *(x.data_ptr() for x in rows), ROW, ROW)
    loaded = [torch.zeros_like(c) for c in s.cache]
    _abi.kv_store_dev(BF16, BF16, 671, KV, DIM, *(x.data_ptr() for x in rows), ROW, ROW, live.data_ptr(), *(c.data_ptr() for c in loaded), s.n_blocks, BLOCK, *s.strides(DIM))
    other = torch.zeros_like(s.out)
    s.prompts(out=other, cache=loaded)
    kept, s.cache = s.cache, loaded
    s.check_attention(other, False, 2.0 ** -8)
    s.cache = kept
    # a second chunk of prompt, of other lengths, then single tokens
    for new in ([1, 40, 100], [1, 1, 1], [1, 1, 1]):
        s.ctx.copy_(s.seq)
        s.new.copy_(torch.tensor(new, dtype=torch.int32))
        s.buffers(sum(new))
        s.fill(sum(new) + int(s.seq.sum()))
        s.plan()
        s.store()
        s.prompts()
        s.check_attention(s.out, False, 2.0 ** -8)
        if new == [1, 1, 1]:
            s.next_tokens()
            s.check_attention(s.out, False, 2.0 ** -16)
            s.check_attention(s.out4, True, 2.0 ** -11)
        s.project()
        s.score()
        s.check_scores()
        s.after_plan()


def test_steps_captured_and_replayed():
    """A graph of a step (plan, stores, both attentions, scores) and one of the attentions alone, which share the
    workspace, replayed in turn with eager steps between: bit for bit what the eager step gives."""
    import torch
    s = Server([70, 1, 600])
    s.fill(1)
    s.plan()
    s.store()
    s.after_plan()
    s.ctx.copy_(s.seq)
    s.new.fill_(1)
    s.buffers(3)
    s.fill(2)
    s.logits.copy_(torch.randn(3, COLS, generator=torch.Generator().manual_seed(1)))
    state = [s.table, s.slots, *s.cache, *s.cache4]
    before = [x.clone() for x in state]
    results = lambda: [x.clone() for x in (s.out, s.out4, s.lp, s.entropy, s.ids, s.best, s.seq, *state)]  # noqa: E731

    def step(stream=None):
        s.plan(stream)
        s.store(stream)
        s.next_tokens(stream)
        s.score(stream)
    step()  # (the workspace grows here)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    with torch.cuda.graph(graphs[0], stream=side):
        step(side.cuda_stream)
    with torch.cuda.graph(graphs[1], stream=side):
        s.next_tokens(side.cuda_stream)
        s.prompts(side.cuda_stream)
    for turn in range(4):
        s.fill(10 + turn)
        s.targets[turn % 3] = COLS + 5  # (no column)
        for x, y in zip(state, before):
            x.copy_(y)
        step()
        torch.cuda.synchronize()
        want = results()
        s.prompts()
        torch.cuda.synchronize()
        want_prompts = s.out.clone()
        for x, y in zip(state, before):
            x.copy_(y)
        for x in (s.out, s.out4, s.lp, s.entropy, s.best):
            x.fill_(9.0)
        torch.cuda.synchronize()
        graphs[0].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(results(), want)), turn
        graphs[1].replay()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(s.out4, want[1]) and torch.equal(s.out, want_prompts), turn
        assert torch.equal(s.lp, want[2]) and torch.equal(s.ids, want[4])


def test_two_streams():
    """The prompts' attention and the scores beside the next tokens' attention on another stream."""
    import torch
    s = Server([70, 1, 600])
    s.fill(1)
    s.plan()
    s.store()
    s.ctx.copy_(s.seq)
    s.logits.copy_(torch.randn(s.tokens, COLS, generator=torch.Generator().manual_seed(1)))
    s.prompts()
    torch.cuda.synchronize()
    want = s.out.clone()
    s.score()
    s.next_tokens()
    torch.cuda.synchronize()
    want_rows, want4, lp = s.out[:3].clone(), s.out4[:3].clone(), s.lp.clone()
    prompts, s.lp = torch.zeros_like(s.out), torch.zeros_like(lp)
    s.out.zero_(), s.out4.zero_()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        s.prompts(one.cuda_stream, out=prompts)
        s.next_tokens(two.cuda_stream)
        s.score(one.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(prompts, want) and torch.equal(s.out[:3], want_rows) and torch.equal(s.out4[:3], want4) and torch.equal(s.lp, lp)


@pytest.mark.parametrize("four", [False, True])
def test_growth_refused_during_capture(four):
    import torch
    s = Server([70, 1, 600])
    s.fill(1)
    s.plan()
    s.store()
    torch.cuda.synchronize()
    _abi.shutdown()
    _abi.init()
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    rest = (s.table.data_ptr(), s.width, s.width, s.seq.data_ptr(), SCALE)
    with pytest.raises(RuntimeError) as e:
        with torch.cuda.graph(g, stream=side):
            if four:
                _abi.paged_attention_q4_dev(BF16, 3, HEADS, KV, DIM, s.q.data_ptr(), HEADS * DIM, *(c.data_ptr() for c in s.cache4), s.n_blocks, BLOCK, *s.strides(BYTES),
                                            *rest, s.out4.data_ptr(), HEADS * DIM, stream=side.cuda_stream)
            else:
                _abi.paged_attention_ex_dev(BF16, BF16, 3, HEADS, KV, DIM, s.q.data_ptr(), HEADS * DIM, *(c.data_ptr() for c in s.cache), s.n_blocks, BLOCK, *s.strides(DIM),
                                            *rest, s.out.data_ptr(), HEADS * DIM, cap=CAP, stream=side.cuda_stream)
    assert "eagerly" in str(e.value)
    del g
    torch.cuda.synchronize()
    # prompts and scores need no workspace
    s.logits.zero_()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        s.prompts(side.cuda_stream)
        s.score(side.cuda_stream)
    g.replay()
    torch.cuda.synchronize()
    s.check_attention(s.out, False, 2.0 ** -8)
    s.check_scores()
    # nor does a window of 512
    _abi.paged_attention_q4_dev(BF16, 3, HEADS, KV, DIM, s.q.data_ptr(), HEADS * DIM, *(c.data_ptr() for c in s.cache4), s.n_blocks, BLOCK, *s.strides(BYTES), *rest,
                                s.out4.data_ptr(), HEADS * DIM, window=512)
    torch.cuda.synchronize()


def test_store_of_many_rows():
    """4-bit rows of many heads, the last workgroup ragged; the same call again gives the same bytes."""
    import torch
    tokens, kv, dim, block = 4099, 13, 96, 7
    row = ref.row_bytes(dim)
    n_blocks = -(-tokens // block)
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(tokens, kv * dim, generator=g).cuda() for _ in range(2))
    slots = torch.randperm(tokens, generator=g).cuda()
    caches = []
    for _ in range(2):
        c = [torch.full((n_blocks * block * kv * row,), 0xEE, dtype=torch.uint8, device="cuda") for _ in range(2)]
        _abi.kv_store_q4_dev(F32, tokens, kv, dim, k.data_ptr(), v.data_ptr(), kv * dim, kv * dim, slots.data_ptr(), c[0].data_ptr(), c[1].data_ptr(), n_blocks, block,
                             block * kv * row, kv * row, row)
        caches.append(c)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(*caches))
    for w, x in ((0, k), (1, v)):
        want = np.full((n_blocks * block, kv, row), 0xEE, np.uint8)
        want[slots.cpu().numpy()] = ref.pack_rows(values(x.cpu().numpy().reshape(tokens, kv, dim), F32))[w]
        assert np.array_equal(caches[0][w].cpu().numpy().reshape(want.shape), want)


def test_offsets_past_32_bits():
    """Caches of over 4 GiB, the requests' blocks at both ends: bit for bit what small caches with the same rows give."""
    import torch
    kv, dim, heads, block, lens = 2, 128, 8, 16, [700, 33, 64]
    row = ref.row_bytes(dim)
    tokens, need = sum(lens), sum(-(-n // block) for n in lens)
    width = 64
    g = torch.Generator().manual_seed(9)
    k, v = (torch.randn(tokens, kv * dim, generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn(tokens, heads * dim, generator=g).bfloat16().cuda()
    start = torch.tensor([0, 700, 733, 797], dtype=torch.int32, device="cuda")
    seq = torch.tensor(lens, dtype=torch.int32, device="cuda")
    results = []
    for large in (False, True):
        out = []
        for four in (False, True):
            size = block * kv * (row if four else 2 * dim)
            n_blocks = (5 << 30) // size if large else need
            caches = [torch.empty(n_blocks * size, dtype=torch.uint8, device="cuda") for _ in range(2)]
            blocks = [i if i % 3 == 0 else n_blocks - need + i for i in range(need)] if large else list(range(need))
            table = torch.full((3, width), -1, dtype=torch.int32)
            slots, at = [], 0
            for r, n in enumerate(lens):
                for i in range(-(-n // block)):
                    table[r, i] = blocks[at]
                    slots += [blocks[at] * block + t for t in range(min(block, n - i * block))]
                    at += 1
            table, slots = table.cuda(), torch.tensor(slots, dtype=torch.int64).cuda()
            strides = (size, kv * row, row) if four else (block * kv * dim, kv * dim, dim)
            pointers = [c.data_ptr() for c in caches]
            rest = (table.data_ptr(), width, width, seq.data_ptr(), SCALE)
            o = torch.zeros(3, heads * dim, dtype=torch.bfloat16, device="cuda")
            if four:
                _abi.kv_store_q4_dev(BF16, tokens, kv, dim, k.data_ptr(), v.data_ptr(), kv * dim, kv * dim, slots.data_ptr(), *pointers, n_blocks, block, *strides)
                _abi.paged_attention_q4_dev(BF16, 3, heads, kv, dim, q.data_ptr(), heads * dim, *pointers, n_blocks, block, *strides, *rest, o.data_ptr(), heads * dim)
                back = [torch.zeros_like(k) for _ in range(2)]
                _abi.kv_load_q4_dev(BF16, tokens, kv, dim, *pointers, n_blocks, block, *strides, slots.data_ptr(), *(x.data_ptr() for x in back), kv * dim, kv * dim)
                out += [o, *back]
            else:
                _abi.kv_store_dev(BF16, BF16, tokens, kv, dim, k.data_ptr(), v.data_ptr(), kv * dim, kv * dim, slots.data_ptr(), *pointers, n_blocks, block, *strides)
                _abi.paged_attention_ex_dev(BF16, BF16, 3, heads, kv, dim, q.data_ptr(), heads * dim, *pointers, n_blocks, block, *strides, *rest, o.data_ptr(), heads * dim, cap=CAP)
                p = torch.zeros_like(q)
                _abi.prompt_attention_dev(BF16, BF16, tokens, 3, heads, kv, dim, q.data_ptr(), heads * dim, *pointers, n_blocks, block, *strides, table.data_ptr(), width, width,
                                          start.data_ptr(), seq.data_ptr(), SCALE, p.data_ptr(), heads * dim)
                out += [o, p]
            torch.cuda.synchronize()
            del caches
        results.append(out)
    for a, b in zip(*results):
        assert torch.isfinite(a.float()).all() and torch.equal(a, b)
