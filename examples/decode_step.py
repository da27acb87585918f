"""One decoder attention block, a token a request, on the serving operators.

    python examples/decode_step.py [requests] [steps]

Each step runs, on the GPU and without the host in between,

  kv_plan          blocks and slots for the new tokens, from the requests' lengths
  rmsnorm          the hidden state to 8 bits with a scale for each 128 columns
  matvec_q4g       queries, keys and values: one product with 4-bit weights
  kv_store         the new keys and values to their slots of the paged cache
  paged_attention  every request's token over its own blocks
  matvec_q4g       the output projection
  rmsnorm          its result added to the residual stream, and normed

with torch holding the buffers.  The sizes are the Whisper large-v3-turbo decoder's
(1280 wide, 20 heads of 64); the weights are random.  Run from the repository's root
on a machine with an MI355X and the built library.
"""
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tomoul_amd import _abi  # noqa: E402

GROUP = 128  # columns of a scale, of the weights and of the 8-bit activations
EPS = 1e-6


class Weight4:
    """4-bit weights with group scales of fp32 rows [n, k], rows padded to 16 bytes."""

    def __init__(self, w):
        self.n, self.k = w.shape
        self.stride = -(-self.k // 32) * 16
        self.q = torch.zeros(self.n, self.stride, dtype=torch.uint8, device="cuda")
        self.scales = torch.empty(self.n, -(-self.k // GROUP), device="cuda")
        _abi.quantize_groups_dev(self.n, self.k, GROUP, w.data_ptr(), self.k, self.q.data_ptr(), self.stride, self.scales.data_ptr(),
                                 stream=torch.cuda.current_stream().cuda_stream)

    def dequantized(self):
        low, high = (self.q.int() & 15 ^ 8) - 8, (self.q.int() >> 4 ^ 8) - 8
        q = torch.stack((low, high), 2).view(self.n, -1)[:, :self.k]
        return q.double() * self.scales.double().repeat_interleave(GROUP, 1)[:, :self.k]

    def product(self, x_type, x, rows, y, stream, x_scales=None):
        _abi.matvec_q4g_dev(x_type, rows, self.n, self.k, x.data_ptr(), self.k, self.q.data_ptr(), self.stride, self.scales.data_ptr(), GROUP,
                            _abi.TYPE_F32, y.data_ptr(), self.n, x_scales_ptr=None if x_scales is None else x_scales.data_ptr(),
                            x_group=0 if x_scales is None else GROUP, stream=stream)


class DecoderBlock:
    def __init__(self, requests, max_len, width=1280, heads=20, kv_heads=20, head_dim=64, block=16, seed=0):
        gen = torch.Generator(device="cuda")
        gen.manual_seed(seed)

        def normal(*shape, std=1.0):
            return torch.randn(*shape, generator=gen, device="cuda") * std

        self.requests, self.width, self.heads, self.kv_heads, self.head_dim, self.block = requests, width, heads, kv_heads, head_dim, block
        self.kv = kv_heads * head_dim
        self.qkv_w = Weight4(normal(heads * head_dim + 2 * self.kv, width, std=width ** -0.5))
        self.out_w = Weight4(normal(width, heads * head_dim, std=(heads * head_dim) ** -0.5))
        self.norm1, self.norm2 = 1 + normal(width, std=0.1), 1 + normal(width, std=0.1)
        self.cols = -(-max_len // block)
        self.n_blocks = requests * self.cols
        # the pool: a block is [heads, tokens, head size], so that a head's tokens are one run
        self.k_cache, self.v_cache = (torch.zeros(self.n_blocks, kv_heads, block, head_dim, dtype=torch.float16, device="cuda") for _ in range(2))
        self.free = torch.randperm(self.n_blocks, generator=gen, device="cuda").to(torch.int32)
        self.table = torch.full((requests, self.cols), -1, dtype=torch.int32, device="cuda")
        self.ctx = torch.zeros(requests, dtype=torch.int32, device="cuda")
        self.one = torch.ones_like(self.ctx)
        self.seq_len = torch.empty_like(self.ctx)
        self.slots = torch.empty(requests, dtype=torch.int64, device="cuda")
        self.totals = torch.zeros(3, dtype=torch.int64, device="cuda")
        self.h8 = torch.empty(requests, width, dtype=torch.int8, device="cuda")
        self.h8_scales = torch.empty(requests, -(-width // GROUP), device="cuda")
        self.qkv = torch.empty(requests, self.qkv_w.n, device="cuda")
        self.attended = torch.empty(requests, heads * head_dim, device="cuda")
        self.projected = torch.empty(requests, width, device="cuda")
        self.normed = torch.empty(requests, width, device="cuda")

    def step(self, x, free):
        """The block on hidden states x [requests, width], which become the residual stream
        after it; `free`: the blocks still to be handed out.  Returns the normed result."""
        s = torch.cuda.current_stream().cuda_stream
        n, w, hd = self.requests, self.width, self.head_dim
        _abi.kv_plan_dev(n, self.block, self.ctx.data_ptr(), self.one.data_ptr(), free.data_ptr(), free.numel(), self.table.data_ptr(), self.cols,
                         self.cols, n, self.slots.data_ptr(), seq_len_ptr=self.seq_len.data_ptr(), totals_ptr=self.totals.data_ptr(), stream=s)
        _abi.rmsnorm_dev(_abi.TYPE_F32, n, w, x.data_ptr(), w, self.norm1.data_ptr(), EPS, _abi.TYPE_I8, self.h8.data_ptr(), w,
                         scales_ptr=self.h8_scales.data_ptr(), group=GROUP, stream=s)
        self.qkv_w.product(_abi.TYPE_I8, self.h8, n, self.qkv, s, self.h8_scales)
        k = self.qkv.data_ptr() + 4 * self.heads * hd
        cache = (self.k_cache.data_ptr(), self.v_cache.data_ptr(), self.n_blocks, self.block, self.kv * self.block, hd, self.block * hd)
        _abi.kv_store_dev(_abi.TYPE_F32, _abi.TYPE_F16, n, self.kv_heads, hd, k, k + 4 * self.kv, self.qkv_w.n, self.qkv_w.n, self.slots.data_ptr(),
                          *cache, stream=s)
        _abi.paged_attention_dev(_abi.TYPE_F32, _abi.TYPE_F16, n, self.heads, self.kv_heads, hd, self.qkv.data_ptr(), self.qkv_w.n, *cache,
                                 self.table.data_ptr(), self.cols, self.cols, self.seq_len.data_ptr(), hd ** -0.5, self.attended.data_ptr(),
                                 self.heads * hd, stream=s)
        self.out_w.product(_abi.TYPE_F32, self.attended, n, self.projected, s)
        _abi.rmsnorm_dev(_abi.TYPE_F32, n, w, self.projected.data_ptr(), w, self.norm2.data_ptr(), EPS, _abi.TYPE_F32, self.normed.data_ptr(), w,
                         residual_ptr=x.data_ptr(), residual_stride=w, sum_ptr=x.data_ptr(), sum_stride=w, stream=s)
        return self.normed


def main():
    requests = int(sys.argv[1]) if len(sys.argv) > 1 else 8
    steps = int(sys.argv[2]) if len(sys.argv) > 2 else 100
    _abi.init()
    block = DecoderBlock(requests, max_len=steps)
    x = torch.randn(requests, block.width, device="cuda")
    used = 0
    block.step(x.clone(), block.free)  # (the workspace, before it is timed)
    torch.cuda.synchronize()
    began = time.perf_counter()
    for step in range(steps):
        block.step(x, block.free[used:])
        # every request is as long as the others here, so the host knows what was handed out;
        # otherwise totals[1] says it
        used += requests if step % block.block == 0 else 0
        block.ctx += 1
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    assert torch.isfinite(block.normed).all()
    print(f"{requests} requests, {steps} steps: {took / steps * 1e6:.1f} us a step, {requests * steps / took:.0f} tokens/s")


if __name__ == "__main__":
    main()
