// What the attentions of one new token a request over a paged cache share
// (paged_attention.hip, paged_attention_q4.hip): the split of the batch's tiles over
// the workgroups, the waves' and the parts' joining, the scores' caps and biases.
//
// Split.  A request's tiles of 32 tokens, for each key-value head (and the query heads
// of its group that a workgroup takes at once), follow each other in one long list over the batch, which the
// workgroups share evenly: each sums the requests' lengths itself, so the split goes
// by the lengths as they are on the GPU, ragged or not, without the host.  A
// workgroup's share is some whole heads and at most two parts of one; its waves take
// the tiles in turn and join in LDS.  Parts go to the workspace, and a second, small
// kernel adds them up in their order.
#pragma once

#include "serving.hpp"

#include <algorithm>

namespace tml {
namespace {

constexpr int kWaves = 4, kThreads = kWaves * 64;
constexpr int kTile = 32;  // tokens a wave takes at a time
constexpr int kWhole = 16;  // tiles of a list that is not split: four a wave

// A list's parts: the workgroup of the first, how many; none where the list is whole.
struct ListParts {
    int first, count;
};

struct AttnShape {
    int group;      // query heads of a key-value head
    int at_once;    // query heads that a workgroup takes at a time
    int parts;      // of a group
    int heads;      // query heads of a part
    int64_t units;  // key-value heads * parts: a request's lists of tiles
    int64_t positions;  // of a table row
    int grid;  // workgroups
    int part_floats;  // of a part: 16-head part's values, maxima and sums
    float *partials;  // two parts a workgroup
    ListParts *lists;  // [batch][units], or nullptr: no list can be long enough to be split
};

// Values alike in every lane, for the compiler to keep in scalar registers.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)(((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32) | (uint32_t)uniform((int)(uint32_t)v));
}
// a / b of non-negative values that are nearly always below 2^32: a 64-bit
// division is some hundred instructions.
__device__ __forceinline__ int64_t div_short(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}

__device__ __forceinline__ int64_t wave_up64(int64_t v, int o) {
    const int lo = __shfl_up((int)(uint32_t)v, o), hi = __shfl_up((int)(v >> 32), o);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}
__device__ __forceinline__ int64_t wave_at64(int64_t v, int lane) {
    const int lo = __shfl((int)(uint32_t)v, lane), hi = __shfl((int)(v >> 32), lane);
    return (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
}

struct Span {
    int64_t first, len;  // attended positions [first, len), at most 2^31
    int tiles;
};
__device__ __forceinline__ Span span_of(const PagedAttentionArgs &a, const AttnShape &sh, int seq_len) {
    Span s;
    s.len = min((int64_t)max(seq_len, 0), sh.positions);
    s.first = a.window > 0 ? max(s.len - a.window, (int64_t)0) : 0;
    s.tiles = (int)((s.len - s.first + kTile - 1) / kTile);
    return s;
}

// What a part whose maximum is m is multiplied with where the whole's is top.  A
// part without a maximum holds zeros, or the NaN of scores that are none.
__device__ __forceinline__ float rescale(float m, float top) { return m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top); }

// Elements d and d + 1 of a head's output.
__device__ __forceinline__ void store_result(int qt, const PagedAttentionArgs &a, int64_t b, int64_t head, int d, srv_f32x2 sum, float sum_l) {
    // (nothing weighs: zeros, also where a value is infinite or NaN and so its sum is a NaN)
    const bool none = sum_l == 0.0f;
    const float r = 1.0f / sum_l;
    const int64_t to = b * a.out_stride + head * a.head_dim + d;
    srv_store1(qt, a.out, to, none ? 0.0f : sum[0] * r);
    srv_store1(qt, a.out, to + 1, none ? 0.0f : sum[1] * r);
}

// A workgroup's way through its share.
struct ListWalk {
    int64_t u, u_end, share;  // in tiles, or in lists
    bool lists;
    int64_t b, unit;  // the list at hand, from tile t0 on
    int t0;
    Span sp;
};
__device__ __forceinline__ Span span_at(const PagedAttentionArgs &a, const AttnShape &sh, int64_t r) { return span_of(a, sh, uniform(a.seq_len[r])); }

// The first list of this workgroup's share; false where there is none.  Outputs of
// requests with nothing to look at are written on the way.
__device__ __forceinline__ bool first_list(int qt, const PagedAttentionArgs &a, const AttnShape &sh, ListWalk &w) {
    const int lane = threadIdx.x & 63;
    const int64_t D = a.head_dim;
    const int64_t strip = (a.batch + 63) / 64;
    int64_t upto = 0;
    int longest = 0;
    bool none = false;
    for (int64_t i = lane * strip; i < min((lane + 1) * strip, a.batch); ++i) {
        const int tiles = span_of(a, sh, a.seq_len[i]).tiles;
        none |= tiles == 0;
        longest = max(longest, tiles);
        upto += tiles;
    }
    const int64_t own = upto;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t v = wave_up64(upto, o);
        if (lane >= o) upto += v;
    }
    if (__builtin_amdgcn_ballot_w64(none) != 0)  // requests with nothing to look at
        for (int64_t r = blockIdx.x; r < a.batch; r += gridDim.x)
            if (span_at(a, sh, r).tiles == 0) {
                if (sh.lists != nullptr)
                    for (int64_t i = threadIdx.x; i < sh.units; i += kThreads) sh.lists[r * sh.units + i] = ListParts{0, 0};
                for (int i = threadIdx.x; i < (int)(a.q_heads * D); i += kThreads) srv_store1(qt, a.out, r * a.out_stride + i, 0.0f);
            }
    const int64_t total = uniform(wave_at64(upto, 63)) * sh.units;
    if (total == 0) return false;
    // Lists of so few tiles that a part costs more to join than to read stay whole:
    // the workgroups share the lists then, not their tiles.
    w.lists = __builtin_amdgcn_ballot_w64(longest > kWhole) == 0;
    w.share = max(div_short((w.lists ? a.batch * sh.units : total) + gridDim.x - 1, gridDim.x), (int64_t)(w.lists ? 1 : kWhole / 2));
    w.u = (int64_t)blockIdx.x * w.share;
    w.u_end = min(w.u + w.share, w.lists ? a.batch * sh.units : total);
    if (w.u >= w.u_end) return false;
    w.t0 = 0;
    if (w.lists) {
        w.b = div_short(w.u, sh.units);
        w.unit = w.u - w.b * sh.units;
        for (w.sp = span_at(a, sh, w.b); w.sp.tiles == 0; w.sp = span_at(a, sh, ++w.b)) {
            w.u += sh.units - w.unit;
            w.unit = 0;
            if (w.u >= w.u_end) return false;
        }
    } else {
        const int at_lane = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto * sh.units > w.u));
        int64_t rem = w.u - uniform(wave_at64(upto - own, at_lane)) * sh.units;
        w.b = at_lane * strip;
        w.sp = span_at(a, sh, w.b);
        while (rem >= w.sp.tiles * sh.units) {
            rem -= w.sp.tiles * sh.units;
            w.sp = span_at(a, sh, ++w.b);
        }
        w.unit = div_short(rem, w.sp.tiles);
        w.t0 = (int)(rem - w.unit * w.sp.tiles);
    }
    return true;
}
// One past its last tile in the share.
__device__ __forceinline__ int list_end(const ListWalk &w) { return w.lists ? w.sp.tiles : (int)min((int64_t)w.sp.tiles, w.t0 + (w.u_end - w.u)); }
// The next list; false past the last.  (LDS is written again after it.)
__device__ __forceinline__ bool next_list(const PagedAttentionArgs &a, const AttnShape &sh, ListWalk &w, int t1) {
    w.u += w.lists ? 1 : t1 - w.t0;
    if (w.u >= w.u_end) return false;
    __syncthreads();
    w.t0 = 0;
    if (++w.unit == sh.units) {
        w.unit = 0;
        for (w.sp = span_at(a, sh, ++w.b); w.sp.tiles == 0; w.sp = span_at(a, sh, ++w.b))
            if (w.lists && (w.u += sh.units) >= w.u_end) return false;
    }
    return true;
}

// The waves' parts of a list, maxima and sums first: what this wave's values of head
// lane % 16 are multiplied with on their way to LDS.
__device__ __forceinline__ float join_scale(float (&wave_m)[kWaves][16], float (&wave_l)[kWaves][16], int wave, float m, float l) {
    const int l16 = threadIdx.x & 15, c4 = (threadIdx.x & 63) >> 4;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (c4 == 0) {
        wave_m[wave][l16] = m;
        wave_l[wave][l16] = l;
    }
    __syncthreads();
    float top = wave_m[0][l16];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wave_m[w][l16]);
    return rescale(m, top);
}
// Then the values wave_o[wave][head][dp].  The whole list's result goes to the output, a
// part's to the workspace: [heads][D] values, then each head's maximum and sum.  The
// workgroup that a list begins in has it in its second slot, those it goes on in in
// their first.
__device__ __forceinline__ void store_list(int qt, const PagedAttentionArgs &a, const AttnShape &sh, const ListWalk &w, int t1, int64_t head0, int gn, int dp,
                                           float (&wave_m)[kWaves][16], float (&wave_l)[kWaves][16], const float *wave_o) {
    __syncthreads();
    const bool whole = t1 - w.t0 == w.sp.tiles;
    const int row2 = (int)a.head_dim / 2;
    const int64_t part_at = (2 * (int64_t)blockIdx.x + (w.t0 == 0 ? 1 : 0)) * sh.part_floats;
    for (int i = threadIdx.x; i < gn * row2; i += kThreads) {
        const int g = (int)((uint32_t)i / (uint32_t)row2), d = 2 * (i - g * row2);
        float sum_m = wave_m[0][g], sum_l = 0.0f;
        srv_f32x2 sum = {0.0f, 0.0f};
#pragma unroll
        for (int v = 1; v < kWaves; ++v) sum_m = fmaxf(sum_m, wave_m[v][g]);
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            sum += *(const srv_f32x2 *)(wave_o + (v * sh.heads + g) * dp + d);
            sum_l += wave_l[v][g] * rescale(wave_m[v][g], sum_m);
        }
        if (whole) {
            store_result(qt, a, w.b, head0 + g, d, sum, sum_l);
        } else {
            float *const part = sh.partials + part_at;
            *(srv_f32x2 *)(part + g * (int)a.head_dim + d) = sum;
            if (d == 0) *(srv_f32x2 *)(part + sh.heads * (int)a.head_dim + 2 * g) = srv_f32x2{sum_m, sum_l};
        }
    }
    // where the list's parts are, for the kernel that joins them
    if (sh.lists != nullptr && w.t0 == 0 && threadIdx.x == 0)
        sh.lists[w.b * sh.units + w.unit] = whole ? ListParts{0, 0} : ListParts{(int)blockIdx.x, (int)(div_short(w.u + w.sp.tiles - 1, w.share) - blockIdx.x) + 1};
}

// Adds a list's parts up, in their order; a wave a query head, its lanes first the
// parts' maxima and sums, 64 at a time, then pairs of d.
constexpr int kJoinWaves = 4, kJoinBatch = 16;
template <int QT>
__global__ __launch_bounds__(64 * kJoinWaves) void paged_attention_join_kernel(PagedAttentionArgs a, AttnShape sh) {
    const int lane = threadIdx.x & 63;
    const int head = (int)blockIdx.x * kJoinWaves + uniform((int)(threadIdx.x >> 6));
    const int64_t b = blockIdx.y;
    if (head >= (int)a.q_heads) return;
    const int kv = (int)((uint32_t)head / (uint32_t)sh.group), in_group = head - kv * sh.group, part = in_group / sh.at_once, g = in_group - part * sh.at_once;
    const ListParts list = sh.lists[b * sh.units + kv * sh.parts + part];
    const int count = uniform(list.count), D = (int)a.head_dim;
    if (count == 0) return;
    const float *const first = sh.partials + (2 * (int64_t)uniform(list.first) + 1) * sh.part_floats;
    // (later parts are in their workgroups' first slots)
    auto part_of = [&](int i) { return i == 0 ? first : first + (2 * (int64_t)i - 1) * sh.part_floats; };
    float sum_m = -INFINITY, sum_l = 0.0f;
    srv_f32x2 sum[2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};  // pairs lane and lane + 64
    for (int i0 = 0; i0 < count; i0 += 64) {
        const int n = min(64, count - i0);
        const srv_f32x2 ml = *(const srv_f32x2 *)(part_of(i0 + min(lane, n - 1)) + sh.heads * D + 2 * g);
        float peak = fmaxf(ml[0], sum_m);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) peak = fmaxf(peak, __shfl_xor(peak, o));
        const float before = rescale(sum_m, peak), r = lane < n ? rescale(ml[0], peak) : 0.0f;
        sum_m = peak;
        sum_l = sum_l * before + (lane < n ? r * ml[1] : 0.0f);  // (a lane's own parts)
        sum[0] *= before;
        sum[1] *= before;
        for (int i = 0; i < n; i += kJoinBatch) {  // (past the last part: its values again, times zero)
            srv_f32x2 v[kJoinBatch];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (128 * half >= D) break;
                const int d = 2 * lane + 128 * half;
#pragma unroll
                for (int j = 0; j < kJoinBatch; ++j)
                    v[j] = *(const srv_f32x2 *)(part_of(i0 + min(i + j, n - 1)) + g * D + (d < D ? d : 0));
#pragma unroll
                for (int j = 0; j < kJoinBatch; ++j)
                    sum[half] += __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(r), i + j)) * v[j];
            }
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) sum_l += __shfl_xor(sum_l, o);
    if (2 * lane < D) store_result(QT, a, b, head, 2 * lane, sum[0], sum_l);
    if (2 * lane + 128 < D) store_result(QT, a, b, head, 2 * lane + 128, sum[1], sum_l);
}

inline AttnShape shape_of(const PagedAttentionArgs &a, int per_cu, int at_once) {
    AttnShape sh{};
    sh.group = (int)(a.q_heads / a.kv_heads);
    sh.at_once = at_once;
    sh.parts = (sh.group + at_once - 1) / at_once;
    sh.heads = std::min(sh.group, at_once);
    sh.units = a.kv_heads * sh.parts;
    sh.positions = a.table_width * a.block_size;
    sh.grid = per_cu * std::max(1, device_cus());
    sh.part_floats = sh.heads * (int)(a.head_dim + 2);
    return sh;
}

inline bool attn_empty(const PagedAttentionArgs &a) {
    return a.batch <= 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.head_dim <= 0;
}

// Whether a list may be long enough to be split.
inline bool may_split(const PagedAttentionArgs &a) {
    const int64_t positions = a.table_width * a.block_size;
    return (a.window > 0 ? std::min(positions, a.window) : positions) > kWhole * kTile;
}

// Floats of the workspace: the parts, then where each list's parts are.
inline size_t split_floats(const PagedAttentionArgs &a, const AttnShape &sh) {
    return may_split(a) ? (size_t)((int64_t)2 * sh.grid * sh.part_floats + 2 * a.batch * sh.units) : 0;
}
inline Status split_in(const PagedAttentionArgs &a, const Workspace &ws, AttnShape *sh) {
    if (!may_split(a)) return Status::Ok();
    if (ws.partial_floats < split_floats(a, *sh)) return Status::Err(TML_ERR_INVALID_ARG, "paged attention: workspace too small");
    sh->partials = ws.partials;
    sh->lists = (ListParts *)(ws.partials + (int64_t)2 * sh->grid * sh->part_floats);
    return Status::Ok();
}

}  // namespace
}  // namespace tml
