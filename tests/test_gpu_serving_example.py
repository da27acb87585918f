"""examples/decode_step.py: the serving operators together, step after step,
against the same block in 64 bits, and as one captured graph."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decode_step
    finally:
        sys.path.pop(0)
    return decode_step


def reference(block, x, past):
    """One step in 64 bits on the block's own (dequantized) weights; past: each request's keys and values."""
    import torch

    def norm(v, w):
        return v / torch.sqrt(v.square().mean(1, keepdim=True) + 1e-6) * w.double()

    n, hd = block.requests, block.head_dim
    qkv = norm(x, block.norm1) @ block.qkv_w.dequantized().T
    q, k, v = qkv.split([block.heads * hd, block.kv, block.kv], 1)
    past.append((k.view(n, block.kv_heads, hd), v.view(n, block.kv_heads, hd)))
    keys, values = (torch.stack([p[i] for p in past], 2).repeat_interleave(block.heads // block.kv_heads, 1) for i in (0, 1))
    score = (keys * q.view(n, block.heads, 1, hd)).sum(3) * hd ** -0.5
    out = (torch.softmax(score, 2)[..., None] * values).sum(2).reshape(n, -1)
    x = x + out @ block.out_w.dequantized().T
    return x, norm(x, block.norm2)


@pytest.mark.parametrize("requests,heads,kv_heads,head_dim,block", [(3, 8, 2, 64, 4), (1, 4, 4, 80, 16)])
def test_steps_against_64_bits(requests, heads, kv_heads, head_dim, block):
    # 8-bit activations: a value is off by at most 1 / 254 of its group's largest, some
    # 3 times the root mean square of 128 normal ones, uniformly: 0.7 % of it, and the
    # products of it alike; the residual stream adds two such steps: 3 % bounds both outputs
    import torch
    ds = example()
    b = ds.DecoderBlock(requests, 40, width=512, heads=heads, kv_heads=kv_heads, head_dim=head_dim, block=block, seed=3)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    past, used = [], 0
    for step in range(37):
        x = torch.randn(requests, 512, generator=gen, device="cuda")
        ref_x, ref = reference(b, x.double(), past)
        got = b.step(x, b.free[used:])
        used += requests if step % block == 0 else 0
        assert b.totals.tolist() == [requests, requests if step % block == 0 else 0, 0]
        for g, r in ((x, ref_x), (got, ref)):
            assert float((g.double() - r).norm() / r.norm()) < 0.03, step
        b.ctx += 1


def test_step_as_a_graph():
    import torch
    ds = example()
    b = ds.DecoderBlock(5, 64, width=512, heads=8, kv_heads=4, head_dim=64, block=16, seed=5)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    xs = [torch.randn(5, 512, generator=gen, device="cuda") for _ in range(20)]
    x = xs[0].clone()
    b.step(x, b.free)  # the workspace grows outside of the capture
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.step(x, b.free)
    for i, start in enumerate(xs):
        # the same blocks in both runs: lengths inside the first block of each request
        b.ctx.fill_(i % 16)
        x.copy_(start)
        b.table.fill_(-1) if i % 16 == 0 else None
        b.step(x, b.free)
        torch.cuda.synchronize()
        eager = [t.clone() for t in (x, b.normed, b.slots, b.table, b.k_cache, b.v_cache)]
        x.copy_(start)
        b.normed.zero_()
        b.slots.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for e, t in zip(eager, (x, b.normed, b.slots, b.table, b.k_cache, b.v_cache)):
            assert torch.equal(e, t), i


def test_main_runs(capsys, monkeypatch):
    ds = example()
    monkeypatch.setattr(sys, "argv", ["decode_step.py", "4", "20"])
    ds.main()
    assert "tokens/s" in capsys.readouterr().out
