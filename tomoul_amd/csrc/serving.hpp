// What the serving operators (rmsnorm.hip, kv.hip, kv_q4.hip, matvec_q4g.hip,
// paged_attention.hip, paged_attention_q4.hip, prompt_attention.hip, logprobs.hip) share: element types, eight elements at a time as
// floats, and the launchers' arguments.
#pragma once

#include "tml_internal.hpp"

namespace tml {

inline bool float_type(int t) { return t == TML_TYPE_F32 || t == TML_TYPE_F16 || t == TML_TYPE_BF16; }
inline int64_t type_bytes(int t) { return t == TML_TYPE_F32 ? 4 : t == TML_TYPE_I8 ? 1 : 2; }

typedef uint32_t srv_u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t srv_u32x2 __attribute__((ext_vector_type(2)));
// The same 16 / 8 bytes on any address: rows of odd length start anywhere.
// The hardware loads and stores them in one instruction all the same.
typedef srv_u32x4 srv_u32x4_any __attribute__((aligned(1)));
typedef srv_u32x2 srv_u32x2_any __attribute__((aligned(1)));
typedef float srv_f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 srv_bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 srv_f16x2 __attribute__((ext_vector_type(2)));

// Two floats to two bf16 / f16, round to nearest even, the first in the low half.
__device__ __forceinline__ uint32_t srv_pack_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((srv_f32x2){a, b}, srv_bf16x2));
}
__device__ __forceinline__ uint32_t srv_pack_f16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((srv_f32x2){a, b}, srv_f16x2));
}

// Eight consecutive elements from element i of p (type T), as loaded.
template <int T>
struct SrvRaw {
    srv_u32x4 d[T == TML_TYPE_F32 ? 2 : 1];
};
template <int T>
__device__ __forceinline__ SrvRaw<T> srv_load8(const void *p, int64_t i) {
    SrvRaw<T> r;
    if constexpr (T == TML_TYPE_F32) {
        const srv_u32x4_any *q = (const srv_u32x4_any *)((const float *)p + i);
        r.d[0] = q[0];
        r.d[1] = q[1];
    } else {
        r.d[0] = *(const srv_u32x4_any *)((const uint16_t *)p + i);
    }
    return r;
}
template <int T>
__device__ __forceinline__ void srv_floats(const SrvRaw<T> &r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (T == TML_TYPE_F32) {
            v[e] = __uint_as_float(r.d[e / 4][e % 4]);
        } else {
            const uint32_t d = r.d[0][e / 2];
            if constexpr (T == TML_TYPE_F16)
                v[e] = tml_half_bits(e % 2 ? d >> 16 : d & 0xFFFFu);
            else
                v[e] = __uint_as_float(e % 2 ? d & 0xFFFF0000u : d << 16);
        }
    }
}
template <int T>
__device__ __forceinline__ void srv_store8(void *p, int64_t i, const float (&v)[8]) {
    if constexpr (T == TML_TYPE_F32) {
        srv_u32x4_any *q = (srv_u32x4_any *)((float *)p + i);
        q[0] = srv_u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])};
        q[1] = srv_u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])};
    } else {
        srv_u32x4 d;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            d[e] = T == TML_TYPE_F16 ? srv_pack_f16(v[2 * e], v[2 * e + 1]) : srv_pack_bf16(v[2 * e], v[2 * e + 1]);
        *(srv_u32x4_any *)((uint16_t *)p + i) = d;
    }
}
// One element.
__device__ __forceinline__ float srv_load1(int type, const void *p, int64_t i) {
    if (type == TML_TYPE_F32) return ((const float *)p)[i];
    const uint32_t d = ((const uint16_t *)p)[i];
    return type == TML_TYPE_F16 ? tml_half_bits(d) : __uint_as_float(d << 16);
}
__device__ __forceinline__ void srv_store1(int type, void *p, int64_t i, float v) {
    if (type == TML_TYPE_F32) ((float *)p)[i] = v;
    else ((uint16_t *)p)[i] = (uint16_t)(type == TML_TYPE_F16 ? srv_pack_f16(v, v) : srv_pack_bf16(v, v));
}

struct RmsNormArgs {
    int type, out_type;
    int64_t rows, cols;
    const void *x, *residual;
    int64_t x_stride, residual_stride;
    const float *weight;
    float eps;
    void *sum, *out;
    int64_t sum_stride, out_stride;
    float *scales;
    int64_t group;  // columns of a scale; cols for one scale a row
};
Status launch_rmsnorm(const RmsNormArgs &a, hipStream_t s);

struct KvPlanArgs {
    int64_t requests, block_size;
    const int *ctx_len, *new_len, *free_blocks;
    int64_t n_free;
    int *block_table;
    int64_t table_width, table_stride, max_tokens;
    int64_t *slots;
    int *token_request, *positions, *seq_len, *query_start;
    int64_t *totals;
};
Status launch_kv_plan(const KvPlanArgs &a, hipStream_t s);

struct KvStoreArgs {
    int type, cache_type;
    int64_t tokens, kv_heads, head_dim;
    const void *k, *v;
    int64_t k_stride, v_stride;
    const int64_t *slots;
    void *k_cache, *v_cache;
    int64_t n_blocks, block_size, block_stride, token_stride, head_stride;
};
Status launch_kv_store(const KvStoreArgs &a, hipStream_t s);

struct Matvec4Args {
    int x_type, y_type;
    int64_t M, N, K;
    const void *x;
    int64_t x_stride;
    const float *x_scales;
    int64_t x_group;  // columns of an x scale (8-bit x), K for one a row
    const uint8_t *w;
    int64_t w_stride;
    const float *w_scales;
    int64_t group;
    const float *bias;
    void *y;
    int64_t y_stride;
};
Status launch_matvec_q4g(const Matvec4Args &a, hipStream_t s);
Status launch_quantize_groups(int64_t N, int64_t K, int64_t group, const float *w, int64_t w_stride, uint8_t *q,
                              int64_t q_stride, float *scales, hipStream_t s);

struct PagedAttentionArgs {
    int q_type, cache_type;
    int64_t batch, q_heads, kv_heads, head_dim;
    const void *q;
    int64_t q_stride;
    const void *k_cache, *v_cache;
    int64_t n_blocks, block_size, block_stride, token_stride, head_stride;
    const int *block_table;
    int64_t table_width, table_stride;
    const int *seq_len;
    int64_t window;
    float scale;
    void *out;
    int64_t out_stride;
    float cap = 0.0f;               // of the scores: 0 for none
    const float *slopes = nullptr;  // [q_heads] of the bias by distance, or nullptr
};
Status check_paged_attention(const PagedAttentionArgs &a);
size_t paged_attention_workspace_floats(const PagedAttentionArgs &a);
Status launch_paged_attention(const PagedAttentionArgs &a, const Workspace &ws, hipStream_t s);

// The same over a cache in 4 bits: cache strides in bytes, cache_type unused.
Status check_paged_attention_q4(const PagedAttentionArgs &a);
size_t paged_attention_q4_workspace_floats(const PagedAttentionArgs &a);
Status launch_paged_attention_q4(const PagedAttentionArgs &a, const Workspace &ws, hipStream_t s);

constexpr float kLog2E = 1.44269504088896341f;

// A cap of the scores: none, or one whose reciprocal is an ordinary number too.
inline bool valid_cap(float cap) { return cap == 0.0f || (cap >= 0x1p-100f && cap <= 0x1p100f); }

// cap * tanh(x / cap): past |z| = 0.35 (1 - t) / (1 + t) of t = e^(-2 |z|), below it the
// series z - z^3 / 3 + 2 z^5 / 15 - .. to z^11 (the next term is below 2^-25 of z there),
// since the first loses the bits that 1 - t does.
__device__ __forceinline__ float cap_score(float x, float cap, float inv_cap) {
    const float z = x * inv_cap, y = z * z;
    const float t = __builtin_amdgcn_exp2f(fabsf(z) * -2.88539008177792681f);
    const float far = __builtin_copysignf(cap * (1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x);
    const float series = -1.0f / 3 + y * (2.0f / 15 + y * (-17.0f / 315 + y * (62.0f / 2835 + y * (-1382.0f / 155925))));
    return fabsf(z) < 0.35f ? x + x * (y * series) : far;
}

struct KvStore4Args {
    int type;
    int64_t tokens, kv_heads, head_dim;
    const void *k, *v;  // (store)
    void *k_out, *v_out;  // (load)
    int64_t k_stride, v_stride;
    const int64_t *slots;
    void *k_cache, *v_cache;
    int64_t n_blocks, block_size, block_stride, token_stride, head_stride;  // bytes
};
Status launch_kv_store_q4(const KvStore4Args &a, hipStream_t s);
Status launch_kv_load_q4(const KvStore4Args &a, hipStream_t s);

struct PromptAttentionArgs {
    int q_type, cache_type;
    int64_t tokens, requests, q_heads, kv_heads, head_dim;
    const void *q;
    int64_t q_stride;
    const void *k_cache, *v_cache;
    int64_t n_blocks, block_size, block_stride, token_stride, head_stride;
    const int *block_table;
    int64_t table_width, table_stride;
    const int *query_start, *seq_len, *prefix_len;
    int64_t window;
    float scale, cap;
    const float *slopes;
    void *out;
    int64_t out_stride;
};
Status launch_prompt_attention(const PromptAttentionArgs &a, hipStream_t s);

struct LogprobsArgs {
    int type;
    int64_t rows, cols;
    const void *logits;
    int64_t stride;
    const int *tokens;
    float *logprobs, *entropy;
    int64_t top;
    int *top_ids;
    float *top_logprobs;
};
Status launch_token_logprobs(const LogprobsArgs &a, hipStream_t s);

}  // namespace tml
