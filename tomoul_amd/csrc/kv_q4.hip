// kv_q4.hip -- a paged key-value cache in 4 bits: new keys and values to their
// slots, and slots' rows back as floats.
//
//   z = f16(min x),  s = f16((max x - min x) / 15),  n = round((x - z) / s) in 0 .. 15,  x ~ n s + z
//
// for each 32 consecutive elements of a head: 16 bytes of nibbles and a word of s and
// z, 5 bits an element.  A row of G groups is 16 G bytes of nibbles, in the order in
// which the attention's lanes take them to the matrix cores without an exchange:
//   keys    lane group c of a token's row multiplies d = 32 w + 8 c + j, all w: its words
//           c G + w follow each other
//   values  lane r of 16 multiplies d = 16 j + r of a token, all j, so that a matrix
//           instruction's 16 rows are of one group: its G bytes follow each other
// then G words of s (low half) and z.
//
// A thread takes eight elements of a key and the same eight of its value, four threads
// a group; rows pass through LDS so that memory is read and written in whole words
// whatever the order in a row.  16384 tokens, 8 heads of 128, bf16, 88 MB: the store takes 29 us
// (3.0 TB/s, bound by its vector instructions, 16100 a SIMD by the counters and 27 us of issue:
// some thirty an element, the group's extremes and the rounding), the load 19 us (4.6 TB/s, memory).
#include "serving.hpp"

#include <algorithm>

namespace tml {
namespace {

constexpr int kThreads = 256;
constexpr int kRowWords = kThreads / 4 * 5;  // of a workgroup's rows: 20 bytes for each four threads

struct Q4Shape {
    unsigned rows;       // tokens * heads of the launch
    unsigned heads;
    bool small;          // the cache's slots are below 2^32
};

// The slot of a row's token: the byte offset of the row in the cache, or -1.
__device__ __forceinline__ int64_t row_offset(const KvStore4Args &a, const Q4Shape &sh, unsigned token, unsigned head) {
    const int64_t slot = a.slots[token];
    if (slot < 0 || slot >= a.n_blocks * a.block_size) return -1;
    const int64_t block = sh.small ? (int64_t)((uint32_t)slot / (uint32_t)a.block_size) : slot / a.block_size;
    return block * a.block_stride + (slot - block * a.block_size) * a.token_stride + head * a.head_stride;
}

// Eight elements of a group (the other 24 in the lanes next to this one): their nibbles,
// element e in bits 4 e, and the group's s and z.
__device__ __forceinline__ uint32_t quantize8(const float (&v)[8], uint32_t *meta) {
    float low = INFINITY, high = -INFINITY;
    bool fine = true;
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        fine &= fabsf(v[e]) < INFINITY;  // (no NaN either)
        x[e] = __builtin_amdgcn_fmed3f(v[e], -65504.0f, 65504.0f);
        low = fminf(low, x[e]);
        high = fmaxf(high, x[e]);
    }
    int bad = !fine;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        low = fminf(low, __shfl_xor(low, o));
        high = fmaxf(high, __shfl_xor(high, o));
        bad |= __shfl_xor(bad, o);
    }
    const uint32_t d = srv_pack_f16((high - low) / 15.0f, low);
    const float s = tml_half_bits(d & 0xFFFFu), z = tml_half_bits(d >> 16);
    *meta = bad ? 0x7E000000u : d;  // (a NaN and no steps)
    uint32_t n = 0;
    if (s > 0.0f && !bad) {
        // (x - z) / s as a division rounds it, from the group's one: the product with 1 / s and its
        // remainder's (Markstein).  With eight divisions store and load of 16384 tokens took 55 us,
        // with these 49.
        const float r = 1.0f / s;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float t = x[e] - z, q = t * r;
            n |= (uint32_t)fminf(fmaxf(rintf(fmaf(fmaf(-q, s, t), r, q)), 0.0f), 15.0f) << (4 * e);
        }
    }
    return n;
}

// A workgroup's rows of G groups, their first and how many.
__host__ __device__ constexpr int rows_here(int groups) { return kThreads / (4 * groups); }
template <int G>
__device__ __forceinline__ int rows_at(const Q4Shape &sh, unsigned *first) {
    *first = blockIdx.x * (unsigned)rows_here(G);
    return (int)min((unsigned)rows_here(G), sh.rows - *first);
}

template <int T, int G>
__global__ __launch_bounds__(kThreads) void kv_store_q4_kernel(KvStore4Args a, Q4Shape sh) {
    __shared__ uint32_t words[2][kRowWords];
    __shared__ int64_t offsets[kThreads / 4];
    constexpr int D = 32 * G;
    unsigned first;
    const int rows = rows_at<G>(sh, &first);
    {
        // (threads past the last row quantize it again: all lanes take part in the exchange)
        const int row = min((int)threadIdx.x / (4 * G), rows - 1), at = (int)threadIdx.x % (4 * G);
        const unsigned token = (first + row) / sh.heads, head = first + row - token * sh.heads;
        const int64_t from = (int64_t)head * D + 8 * at;
        const SrvRaw<T> k = srv_load8<T>(a.k, (int64_t)token * a.k_stride + from);
        const SrvRaw<T> v = srv_load8<T>(a.v, (int64_t)token * a.v_stride + from);
        const int w = at >> 2, c = at & 3;  // d = 32 w + 8 c + e
        if (at == 0) offsets[row] = row_offset(a, sh, token, head);
        float f[8];
        uint32_t meta;
        uint32_t *const to = words[0] + row * 5 * G;
        srv_floats<T>(k, f);
        const uint32_t kn = quantize8(f, &meta);
        to[c * G + w] = kn;
        if (c == 0) to[4 * G + w] = meta;
        srv_floats<T>(v, f);
        const uint32_t vn = quantize8(f, &meta);
        // byte (8 c + e) G + w, c < 2: element 8 c + e low, 16 + 8 c + e high; each lane writes four
        const uint32_t other = (uint32_t)__shfl_xor((int)vn, 2);
        const uint32_t low = c < 2 ? vn : other, high = c < 2 ? other : vn;
        uint8_t *const bytes = (uint8_t *)(words[1] + row * 5 * G);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = (c < 2 ? 0 : 4) + i;
            bytes[(8 * (c & 1) + e) * G + w] = (uint8_t)((low >> (4 * e) & 15) | (high >> (4 * e) & 15) << 4);
        }
        if (c == 0) words[1][row * 5 * G + 4 * G + w] = meta;
    }
    __syncthreads();
    const int n = rows * 5 * G;
    for (int i = threadIdx.x; i < 2 * n; i += kThreads) {
        const int which = i >= n, j = i - which * n, row = j / (5 * G), word = j - row * 5 * G;
        const int64_t off = offsets[row];
        if (off >= 0) *(uint32_t *)((char *)(which ? a.v_cache : a.k_cache) + off + 4 * word) = words[which][j];
    }
}

template <int T, int G>
__global__ __launch_bounds__(kThreads) void kv_load_q4_kernel(KvStore4Args a, Q4Shape sh) {
    __shared__ uint32_t words[2][kRowWords];
    __shared__ int64_t offsets[kThreads / 4];
    constexpr int D = 32 * G;
    unsigned first;
    const int rows = rows_at<G>(sh, &first);
    for (int row = threadIdx.x; row < rows; row += kThreads) {
        const unsigned token = (first + row) / sh.heads;
        offsets[row] = row_offset(a, sh, token, first + row - token * sh.heads);
    }
    __syncthreads();
    const int n = rows * 5 * G;
    for (int i = threadIdx.x; i < 2 * n; i += kThreads) {
        const int which = i >= n, j = i - which * n, row = j / (5 * G), word = j - row * 5 * G;
        const int64_t off = offsets[row];
        if (off >= 0) words[which][j] = *(const uint32_t *)((const char *)(which ? a.v_cache : a.k_cache) + off + 4 * word);
    }
    __syncthreads();
    const int row = (int)threadIdx.x / (4 * G), at = (int)threadIdx.x % (4 * G);
    if (row >= rows || offsets[row] < 0) return;
    const unsigned token = (first + row) / sh.heads, head = first + row - token * sh.heads;
    const int64_t to = (int64_t)head * D + 8 * at;
    const int w = at >> 2, c = at & 3;
    float f[8];
    const uint32_t kn = words[0][row * 5 * G + c * G + w], km = words[0][row * 5 * G + 4 * G + w];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = fmaf((float)(kn >> (4 * e) & 15), tml_half_bits(km & 0xFFFFu), tml_half_bits(km >> 16));
    srv_store8<T>(a.k_out, (int64_t)token * a.k_stride + to, f);
    const uint8_t *const bytes = (const uint8_t *)(words[1] + row * 5 * G);
    const uint32_t vm = words[1][row * 5 * G + 4 * G + w];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = bytes[(8 * (c & 1) + e) * G + w];
        f[e] = fmaf((float)(c < 2 ? b & 15 : b >> 4), tml_half_bits(vm & 0xFFFFu), tml_half_bits(vm >> 16));
    }
    srv_store8<T>(a.v_out, (int64_t)token * a.v_stride + to, f);
}

Status check(const KvStore4Args &a, const void *k, const void *v, bool *empty) {
    if (!float_type(a.type)) return Status::Err(TML_ERR_INVALID_FORMAT, "4-bit cache: keys and values must be f32, f16 or bf16");
    if (a.tokens < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.n_blocks < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "4-bit cache: negative size");
    if (a.block_size < 1) return Status::Err(TML_ERR_INVALID_ARG, "4-bit cache: the block size must be positive");
    *empty = a.tokens == 0 || a.kv_heads == 0 || a.head_dim == 0 || a.n_blocks == 0;
    if (*empty) return Status::Ok();
    if (a.head_dim % 32 != 0 || a.head_dim > 256)
        return Status::Err(TML_ERR_INVALID_SHAPE, "4-bit cache: the head size must be a multiple of 32, at most 256");
    const int64_t most = (int64_t)1 << 31;
    if (a.kv_heads >= most / a.head_dim || a.tokens >= most || a.n_blocks >= most || a.block_size >= most)
        return Status::Err(TML_ERR_INVALID_SHAPE, "4-bit cache: tokens, heads * size, blocks and block size must be below 2^31");
    if (k == nullptr || v == nullptr || a.slots == nullptr || a.k_cache == nullptr || a.v_cache == nullptr)
        return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    const int64_t row = a.kv_heads * a.head_dim;
    if (a.tokens > 1 && (a.k_stride < row || a.v_stride < row))
        return Status::Err(TML_ERR_INVALID_SHAPE, "4-bit cache: a token stride is shorter than its heads");
    if (a.block_stride < 0 || a.token_stride < 0 || a.head_stride < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "4-bit cache: negative cache stride");
    if (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)a.block_stride | (uintptr_t)a.token_stride | (uintptr_t)a.head_stride) % 4 != 0)
        return Status::Err(TML_ERR_INVALID_ARG, "4-bit cache: rows must start on 4-byte boundaries");
    return Status::Ok();
}

Q4Shape shape_of(const KvStore4Args &a) {
    return {(unsigned)(a.tokens * a.kv_heads), (unsigned)a.kv_heads, a.n_blocks * a.block_size < (int64_t)1 << 32};
}
constexpr int64_t kMostRows = (int64_t)1 << 26;  // of a launch: at most 2^23 workgroups of eight and more rows

template <bool LOAD, int T, int G>
void launch_groups(const KvStore4Args &a, const Q4Shape &sh, hipStream_t s) {
    const dim3 grid((unsigned)((sh.rows + rows_here(G) - 1) / rows_here(G))), block(kThreads);
    if (LOAD) kv_load_q4_kernel<T, G><<<grid, block, 0, s>>>(a, sh);
    else kv_store_q4_kernel<T, G><<<grid, block, 0, s>>>(a, sh);
}
template <bool LOAD, int T>
void launch_type(const KvStore4Args &a, const Q4Shape &sh, hipStream_t s) {
    switch (a.head_dim / 32) {
        case 1: launch_groups<LOAD, T, 1>(a, sh, s); break;
        case 2: launch_groups<LOAD, T, 2>(a, sh, s); break;
        case 3: launch_groups<LOAD, T, 3>(a, sh, s); break;
        case 4: launch_groups<LOAD, T, 4>(a, sh, s); break;
        case 5: launch_groups<LOAD, T, 5>(a, sh, s); break;
        case 6: launch_groups<LOAD, T, 6>(a, sh, s); break;
        case 7: launch_groups<LOAD, T, 7>(a, sh, s); break;
        default: launch_groups<LOAD, T, 8>(a, sh, s); break;
    }
}

template <bool LOAD>
Status launch(const KvStore4Args &in, hipStream_t s) {
    bool empty = false;
    TML_TRY(check(in, LOAD ? in.k_out : in.k, LOAD ? in.v_out : in.v, &empty));
    if (empty) return Status::Ok();
    const int64_t tokens_a_launch = std::max<int64_t>(1, kMostRows / in.kv_heads);
    const int64_t size = type_bytes(in.type);
    for (int64_t t = 0; t < in.tokens; t += tokens_a_launch) {
        KvStore4Args a = in;
        a.tokens = std::min(tokens_a_launch, in.tokens - t);
        a.slots += t;
        if (LOAD) {
            a.k_out = (char *)in.k_out + t * in.k_stride * size;
            a.v_out = (char *)in.v_out + t * in.v_stride * size;
        } else {
            a.k = (const char *)in.k + t * in.k_stride * size;
            a.v = (const char *)in.v + t * in.v_stride * size;
        }
        const Q4Shape sh = shape_of(a);
        if (a.type == TML_TYPE_F32) launch_type<LOAD, TML_TYPE_F32>(a, sh, s);
        else if (a.type == TML_TYPE_F16) launch_type<LOAD, TML_TYPE_F16>(a, sh, s);
        else launch_type<LOAD, TML_TYPE_BF16>(a, sh, s);
        TML_HIP_TRY(hipGetLastError());
    }
    return Status::Ok();
}

}  // namespace

Status launch_kv_store_q4(const KvStore4Args &a, hipStream_t s) { return launch<false>(a, s); }
Status launch_kv_load_q4(const KvStore4Args &a, hipStream_t s) { return launch<true>(a, s); }

}  // namespace tml
