// kv.hip -- the paged key-value cache's bookkeeping and its filling: block
// tables and slot maps from request lengths, and new keys and values to
// their slots.  Both are a single launch without the host in between.
#include "serving.hpp"

#include <algorithm>

namespace tml {
namespace {

// --------------------------------------------------------------- kv_plan
// Requests r with ctx cached and `fresh` new tokens take
//   have = min(ceil(ctx / B), W) .. want = min(ceil((ctx + fresh) / B), W)
// from the free list in request order, and token t of the batch is position
// ctx + t - start[r] of the request whose range of the exclusive sum `start`
// holds it.
//
// A workgroup owns kSlice tokens.  Each one sums over all requests itself (8
// bytes a request out of L2, 256 requests a step) instead of waiting for a
// launch that does it once: at 64 requests and a token each the whole plan is
// one workgroup, and the launch is what it costs.  Requests whose tokens fall
// into the slice go to a list in LDS, in order, at most one for each token of
// the slice since empty ones are left out; a token finds its request there by
// bisection.  A block is written into the table by the token that is first in
// it, so every entry has one writer, and entries that a token reads (of blocks
// it found) nobody writes.  The lengths are read by all workgroups and seq_len is
// written by the first, so lengths that advance in place take a launch after the
// plan's where that has several workgroups.  Launches in a graph: 64 requests of a token 3.9 us, 512 of
// up to 256 tokens 5.7 us (slices of 512 and 1024 tokens: 6.2, 7.8; workgroups of 1024
// threads, one step of sums for two: 19.3), one of 200000 tokens 3.6.
constexpr int kPlanThreads = 256;
constexpr int kSlice = 256;

struct PlanRequest {
    int64_t first;  // of its new blocks in the free list
    int64_t start;  // first token, less the slice's
    int64_t ctx;
    int64_t have, want;
    int64_t request;
};

// Sums of two lengths stay below 2^32, and 32-bit divisions are a quarter of 64-bit ones.
__device__ __forceinline__ int64_t blocks_of(int64_t tokens, int64_t block) {
    return tokens == 0 ? 0 : (int64_t)((uint32_t)(tokens - 1) / (uint32_t)block) + 1;
}

__device__ __forceinline__ int64_t wave_up(int64_t v, int o) {
    const int lo = __shfl_up((int)(uint32_t)v, o), hi = __shfl_up((int)(v >> 32), o);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}
// Inclusive sum over the workgroup; *total gets the whole.  slots: LDS, a value a wave.
__device__ __forceinline__ int64_t group_scan(int64_t v, int64_t *slots, int64_t *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = wave_up(v, o);
        if (lane >= o) v += u;
    }
    if (lane == 63) slots[wave] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        if (w < wave) before += slots[w];
        all += slots[w];
    }
    *total = all;
    return v + before;
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(KvPlanArgs a) {
    __shared__ PlanRequest list[kSlice];
    __shared__ int64_t scan[3][kPlanThreads / 64];
    const int64_t t0 = (int64_t)blockIdx.x * kSlice, t1 = t0 + kSlice;
    const int64_t B = a.block_size, W = a.table_width;
    int64_t tokens = 0, blocks = 0, wide = 0;  // sums over the requests before this step's
    int listed = 0;
    // the first workgroup writes what there is one of for each request, and the totals
    for (int64_t r0 = 0; r0 < a.requests && (blockIdx.x == 0 || tokens < t1); r0 += kPlanThreads) {
        const int64_t r = r0 + threadIdx.x;
        int64_t ctx = 0, fresh = 0;
        if (r < a.requests) {
            ctx = max(a.ctx_len[r], 0);
            fresh = max(a.new_len[r], 0);
        }
        const int64_t want_all = blocks_of(ctx + fresh, B);
        const int64_t have = min(blocks_of(ctx, B), W), want = min(want_all, W);
        int64_t step_tokens, step_blocks, step_listed, step_wide = 0;
        const int64_t end = tokens + group_scan(fresh, scan[0], &step_tokens);
        const int64_t first = blocks + group_scan(want - have, scan[1], &step_blocks) - (want - have);
        const int64_t start = end - fresh;
        const bool mine = fresh > 0 && start < t1 && end > t0;
        // (both counts in one sum: those of the list below, those too wide above)
        const int64_t both = group_scan((mine ? 1 : 0) + (want_all > W ? (int64_t)1 << 32 : 0), scan[2], &step_listed);
        step_wide = step_listed >> 32;
        step_listed &= 0xFFFFFFFF;
        if (mine) {
            PlanRequest &p = list[listed + (int)(both & 0xFFFFFFFF) - 1];
            p = {first, start - t0, ctx, have, want, r};
        }
        if (blockIdx.x == 0 && r < a.requests) {
            if (a.seq_len != nullptr) a.seq_len[r] = (int)min(ctx + fresh, (int64_t)0x7FFFFFFF);
            if (a.query_start != nullptr) a.query_start[r] = (int)min(start, (int64_t)0x7FFFFFFF);
        }
        tokens += step_tokens;
        blocks += step_blocks;
        wide += step_wide;
        listed += (int)step_listed;
        __syncthreads();  // the sums' slots are written again
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (a.query_start != nullptr) a.query_start[a.requests] = (int)min(tokens, (int64_t)0x7FFFFFFF);
        if (a.totals != nullptr) {
            a.totals[0] = tokens;
            a.totals[1] = blocks;
            a.totals[2] = wide;
        }
    }
    for (int i = threadIdx.x; i < kSlice && t0 + i < a.max_tokens; i += kPlanThreads) {
        int lo = 0, hi = listed;  // the last listed request that starts at or before token i
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (list[mid].start <= i) lo = mid;
            else hi = mid;
        }
        int64_t slot = -1, request = -1, pos = -1;
        if (t0 + i < tokens) {
            const PlanRequest p = list[lo];
            request = p.request;
            pos = p.ctx + i - p.start;
            const int64_t col = (uint32_t)pos / (uint32_t)B, in_block = pos - col * B;
            int64_t block = -1;
            if (col < p.have) {
                block = a.block_table[request * a.table_stride + col];
            } else if (col < p.want) {
                const int64_t at = p.first + col - p.have;
                if (at < a.n_free) block = a.free_blocks[at];
                if (in_block == 0) a.block_table[request * a.table_stride + col] = (int)block;
            }
            if (block >= 0) slot = block * B + in_block;
        }
        const int64_t t = t0 + i;
        a.slots[t] = slot;
        if (a.token_request != nullptr) a.token_request[t] = (int)request;
        if (a.positions != nullptr) a.positions[t] = (int)pos;
    }
}

// Lengths that advance in place while the plan runs in several workgroups: after it.
__global__ __launch_bounds__(256) void kv_lengths_kernel(int64_t requests, const int *ctx_len, const int *new_len, int *seq_len) {
    const int64_t r = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (r < requests) seq_len[r] = (int)min((int64_t)max(ctx_len[r], 0) + max(new_len[r], 0), (int64_t)0x7FFFFFFF);
}

// -------------------------------------------------------------- kv_store
// A thread moves eight elements of one token's keys and the same eight of its
// values, `runs` threads a token.  Bound by memory: each row is read and
// written once, 16 bytes an access of 16-bit types.  16384 tokens of 8 heads of 128
// in bf16 27.5 us (134 MB, 4.9 TB/s), 64 tokens 2.9 us.
struct StoreShape {
    int64_t total;       // tokens * runs
    unsigned runs, per_head;  // runs of eight a token, a head
    bool small;          // the runs and the cache's slots are below 2^32
};
__device__ __forceinline__ int64_t div_any(int64_t a, int64_t b, bool small) {
    return small ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

template <int TS, int TC>
__global__ __launch_bounds__(256) void kv_store_kernel(KvStoreArgs a, StoreShape sh) {
    const int64_t n_slots = a.n_blocks * a.block_size;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < sh.total; i += (int64_t)gridDim.x * 256) {
        const int64_t token = div_any(i, sh.runs, sh.small);
        const unsigned run = (unsigned)(i - token * sh.runs);
        const unsigned head = run / sh.per_head, d = (run - head * sh.per_head) * 8;
        const int64_t slot = a.slots[token];
        const int64_t from = (int64_t)head * a.head_dim + d;
        const SrvRaw<TS> k = srv_load8<TS>(a.k, token * a.k_stride + from);
        const SrvRaw<TS> v = srv_load8<TS>(a.v, token * a.v_stride + from);
        if (slot < 0 || slot >= n_slots) continue;
        const int64_t block = div_any(slot, a.block_size, sh.small), in_block = slot - block * a.block_size;
        const int64_t to = block * a.block_stride + in_block * a.token_stride + head * a.head_stride + d;
        float f[8];
        srv_floats<TS>(k, f);
        srv_store8<TC>(a.k_cache, to, f);
        srv_floats<TS>(v, f);
        srv_store8<TC>(a.v_cache, to, f);
    }
}

// Head sizes that are no multiple of eight: an element a thread.
__global__ __launch_bounds__(256) void kv_store_any_kernel(KvStoreArgs a) {
    const int64_t n_slots = a.n_blocks * a.block_size, row = a.kv_heads * a.head_dim, total = a.tokens * row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t token = i / row, from = i - token * row, head = from / a.head_dim, d = from - head * a.head_dim;
        const int64_t slot = a.slots[token];
        if (slot < 0 || slot >= n_slots) continue;
        const int64_t block = slot / a.block_size, in_block = slot - block * a.block_size;
        const int64_t to = block * a.block_stride + in_block * a.token_stride + head * a.head_stride + d;
        srv_store1(a.cache_type, a.k_cache, to, srv_load1(a.type, a.k, token * a.k_stride + from));
        srv_store1(a.cache_type, a.v_cache, to, srv_load1(a.type, a.v, token * a.v_stride + from));
    }
}

template <int TS>
void launch_store(const KvStoreArgs &a, const StoreShape &sh, dim3 grid, hipStream_t s) {
    if (a.cache_type == TML_TYPE_F32) kv_store_kernel<TS, TML_TYPE_F32><<<grid, dim3(256), 0, s>>>(a, sh);
    else if (a.cache_type == TML_TYPE_F16) kv_store_kernel<TS, TML_TYPE_F16><<<grid, dim3(256), 0, s>>>(a, sh);
    else kv_store_kernel<TS, TML_TYPE_BF16><<<grid, dim3(256), 0, s>>>(a, sh);
}

// Bytes [p, p + bytes); rows > 1: the same every `stride` bytes.
struct Bytes {
    const void *p;
    int64_t bytes;
    int64_t rows = 1, stride = 0;
};
bool meet(const Bytes &a, const Bytes &b) {  // b: one row
    if (a.p == nullptr || b.p == nullptr || a.bytes <= 0 || b.bytes <= 0 || a.rows <= 0) return false;
    const intptr_t off = (intptr_t)b.p - (intptr_t)a.p;  // b's start in a
    if (off + b.bytes <= 0 || off >= (a.rows - 1) * a.stride + a.bytes) return false;
    if (off < 0 || a.rows == 1) return true;
    const intptr_t in_row = off % a.stride;
    return in_row < a.bytes || in_row + b.bytes > a.stride;
}

}  // namespace

Status launch_kv_plan(const KvPlanArgs &a, hipStream_t s) {
    if (a.requests < 0 || a.max_tokens < 0 || a.n_free < 0 || a.table_width < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv plan: negative size");
    if (a.block_size < 1) return Status::Err(TML_ERR_INVALID_ARG, "kv plan: the block size must be positive");
    if (a.requests > 0x7FFFFFFF || a.max_tokens > 0x7FFFFFFF || a.block_size > 0x7FFFFFFF)
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv plan: requests, tokens and block size must be below 2^31");
    if (a.requests > 1 && a.table_stride < a.table_width)
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv plan: the table's row stride is shorter than its width");
    if ((a.requests > 0 && (a.ctx_len == nullptr || a.new_len == nullptr)) || (a.n_free > 0 && a.free_blocks == nullptr) ||
        (a.requests > 0 && a.table_width > 0 && a.block_table == nullptr) || (a.max_tokens > 0 && a.slots == nullptr))
        return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    // Workgroups read all lengths while the first one writes: only seq_len may lie over
    // what it is made of, element on element.
    const int64_t width = std::min(a.table_width, (int64_t)1 << 32);  // (no length reaches further)
    const int64_t free_read = std::min(a.n_free, a.requests * width);
    const Bytes ins[3] = {{a.ctx_len, a.requests * 4}, {a.new_len, a.requests * 4}, {a.free_blocks, free_read * 4}};
    const Bytes outs[6] = {{a.block_table, width * 4, a.requests, a.requests > 1 ? a.table_stride * 4 : 0}, {a.slots, a.max_tokens * 8}, {a.token_request, a.max_tokens * 4},
                           {a.positions, a.max_tokens * 4}, {a.query_start, (a.requests + 1) * 4}, {a.totals, 24}};
    const Bytes lengths{a.seq_len, a.requests * 4};
    bool bad = false;
    for (const Bytes &in : ins) {
        for (const Bytes &out : outs) bad |= meet(out, in);
        bad |= (in.p != a.seq_len || in.p == a.free_blocks) && meet(lengths, in);
    }
    if (bad)
        return Status::Err(TML_ERR_INVALID_ARG, "kv plan: an output overlaps an input (seq_len alone may be ctx_len or new_len itself)");
    const int64_t slices = std::max<int64_t>(1, (a.max_tokens + kSlice - 1) / kSlice);
    const bool after = slices > 1 && a.requests > 0 && a.seq_len != nullptr && (a.seq_len == a.ctx_len || a.seq_len == a.new_len);
    KvPlanArgs plan = a;
    if (after) plan.seq_len = nullptr;
    kv_plan_kernel<<<dim3((unsigned)slices), dim3(kPlanThreads), 0, s>>>(plan);
    TML_HIP_TRY(hipGetLastError());
    if (after) {
        kv_lengths_kernel<<<dim3((unsigned)((a.requests + 255) / 256)), dim3(256), 0, s>>>(a.requests, a.ctx_len, a.new_len, a.seq_len);
        TML_HIP_TRY(hipGetLastError());
    }
    return Status::Ok();
}

Status launch_kv_store(const KvStoreArgs &a, hipStream_t s) {
    if (!float_type(a.type) || !float_type(a.cache_type))
        return Status::Err(TML_ERR_INVALID_FORMAT, "kv store: keys, values and cache must be f32, f16 or bf16");
    if (a.tokens < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.n_blocks < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv store: negative size");
    if (a.block_size < 1) return Status::Err(TML_ERR_INVALID_ARG, "kv store: the block size must be positive");
    if (a.tokens == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.n_blocks == 0) return Status::Ok();
    const int64_t most = (int64_t)1 << 31;
    if (a.kv_heads >= most / a.head_dim || a.tokens >= most || a.n_blocks >= most || a.block_size >= most)
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv store: tokens, heads * size, blocks and block size must be below 2^31");
    if (a.k == nullptr || a.v == nullptr || a.slots == nullptr || a.k_cache == nullptr || a.v_cache == nullptr)
        return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    const int64_t row = a.kv_heads * a.head_dim;
    if (a.tokens > 1 && (a.k_stride < row || a.v_stride < row))
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv store: a token stride is shorter than its heads");
    if (a.block_stride < 0 || a.token_stride < 0 || a.head_stride < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "kv store: negative cache stride");
    if (a.head_dim % 8 != 0) {
        const int64_t groups = std::min<int64_t>((a.tokens * row + 255) / 256, 1 << 20);
        kv_store_any_kernel<<<dim3((unsigned)groups), dim3(256), 0, s>>>(a);
    } else {
        StoreShape sh;
        sh.runs = (unsigned)(row / 8);
        sh.per_head = (unsigned)(a.head_dim / 8);
        sh.total = a.tokens * sh.runs;
        sh.small = sh.total < (int64_t)1 << 32 && a.n_blocks * a.block_size < (int64_t)1 << 32;
        const dim3 grid((unsigned)std::min<int64_t>((sh.total + 255) / 256, 1 << 20));
        if (a.type == TML_TYPE_F32) launch_store<TML_TYPE_F32>(a, sh, grid, s);
        else if (a.type == TML_TYPE_F16) launch_store<TML_TYPE_F16>(a, sh, grid, s);
        else launch_store<TML_TYPE_BF16>(a, sh, grid, s);
    }
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

}  // namespace tml
