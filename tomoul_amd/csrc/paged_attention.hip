// paged_attention.hip -- attention of one new token a request over a paged
// key-value cache, split over the cache's length and joined.
//
//   s_t = scale * q_h . k_t,   out_h = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),   m = max_t s_t
//
// over the positions t of [max(0, len - window), len) whose block is in the
// cache; none of them: zeros.  Query heads h of a group share a key-value head.
// Keys and values are read once for each 16 query heads of a group, 2 * len * dim
// elements a key-value head, for 4 * group operations an element, so memory bounds it
// from some 100 KB up; the kernel is laid out to have loads in flight, and the matrix
// cores do the arithmetic because they cost nothing next to that, at a group of one too.
//
// One pass with a running maximum and sum.  A wave takes 32 tokens at a time:
//   scores   S = K q^T: 16 tokens are the MFMA's rows, up to 16 query heads its
//            columns; the K operand's lane layout is 16 bytes of a token's row, so
//            it comes straight from memory to registers
//   weights  lane (head, c) then holds the scores of tokens 4 c + i of both 16s,
//            which is the B operand of the next product if its k slots are numbered
//            that way: no exchange between lanes but the maximum's
//   values   O^T += V^T p: a lane loads 16 bytes of eight tokens' rows and turns
//            the 8 x 8 block in registers (one byte permute a pair), its d the
//            product's rows
// Precision: scores and sums are fp32.  q goes in as terms of the cache's type
// (itself where it has that type; two f16 terms scaled by a power of two, or three
// bf16 terms, where it is f32; an infinite key meets the first of them alone), and so
// do the weights: two terms (2^-22 of f16,
// 2^-16 of bf16), three bf16 terms where the output is f32.  An f32 cache runs on
// the fp32 matrix cores.
//
// The batch's tiles are shared by the workgroups as paged_split.hpp says.  FORM: scores capped
// by a tanh or biased by distance, some 20 instructions a score more, which hide behind the loads: bf16,
// 32 requests of up to 4096 tokens, 16 heads on 8 of 256, capped, 126 us (3.9 TB/s); f32 q, f16 cache,
// four of 300 to 2000 tokens, 20 heads of 64, biased, 21 us, of which the second kernel is 4.
//
// Measured on MI355X (launches in a graph): bf16, 64 requests of up to 4096 tokens, 32
// heads on 8 of 128 112 us (4.8 TB/s); f16, two of 40k to 65k tokens 68 us (5.5 TB/s); f32 q,
// f16 cache, one of 448 tokens, 20 heads of 64 8.4 us (10.0 with a table for 4096: the
// second kernel is launched by the table's width and finds nothing to do), of 1500
// 14.2 us; one of 20 tokens 5.6 us; eight of 2k, 32 heads on 8 of 256, bf16 46 us (3.1
// TB/s), f32 112 us (2.6 TB/s).  Long ones are bound by memory, short ones by the chain
// of dependent loads: lengths, table, rows.  The f32 kernel for heads past 128 keeps 36
// vector registers of a lane in scratch, the one for 128 two, the others none.
#include "paged_split.hpp"
#include "terms.hpp"

namespace tml {
namespace {

// q's terms.  The sum over first terms has to be infinite or NaN where the score is,
// so the first is infinite or NaN where the element is, and of its sign otherwise:
//   f16   (|v| < 2^15) the element moved away from zero by f16's smallest number,
//         rounded; a v of 2^-136 still has a sign then
//   bf16  the element cut off, which cannot overflow
template <int CT, int N>
__device__ __forceinline__ void to_query_terms(float (&v)[8], srv_u32x4 (&t)[N]) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        if constexpr (CT == TML_TYPE_F16) {
            const float x = v[e] + __builtin_amdgcn_fmed3f(v[e] * 0x1p112f, -0x1p-24f, 0x1p-24f);
            const float y = v[e + 1] + __builtin_amdgcn_fmed3f(v[e + 1] * 0x1p112f, -0x1p-24f, 0x1p-24f);
            const uint32_t d = srv_pack_f16(x, y);
            t[0][e / 2] = d;
            v[e] -= tml_half_bits(d & 0xFFFFu);
            v[e + 1] -= tml_half_bits(d >> 16);
        } else {
            // (canonical: any NaN has the bit that the cut leaves)
            const uint32_t x = __float_as_uint(__builtin_canonicalizef(v[e])), y = __float_as_uint(__builtin_canonicalizef(v[e + 1]));
            t[0][e / 2] = __builtin_amdgcn_perm(y, x, 0x07060302u);
            v[e] -= __uint_as_float(x & 0xFFFF0000u);
            v[e + 1] -= __uint_as_float(y & 0xFFFF0000u);
        }
    }
    srv_u32x4 rest[N - 1];
    to_terms<CT, N - 1>(v, rest);
#pragma unroll
    for (int n = 1; n < N; ++n) t[n] = rest[n - 1];
}

// 16 bytes of the cache.  ONCE: with the streaming policy, which leaves the
// caches to others.
template <bool ONCE>
__device__ __forceinline__ srv_u32x4 load_cache(const char *p) {
    if constexpr (ONCE) return __builtin_nontemporal_load((const srv_u32x4 *)p);
    else return *(const srv_u32x4 *)p;
}

// CT: the cache's type.  QT: q's and the output's (CT or f32).  DP: the head size
// rounded up to 64, 128 or 256.  FORM: the scores are capped or biased.
template <int CT, int QT, int DP, bool ONCE, bool FORM>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void paged_attention_kernel(PagedAttentionArgs a, AttnShape sh) {
    constexpr bool kF32 = CT == TML_TYPE_F32;
    constexpr int kBytes = kF32 ? 4 : 2;
    constexpr int NQ = QT == CT ? 1 : CT == TML_TYPE_F16 ? 2 : 3;
    constexpr int NP = CT == TML_TYPE_BF16 && QT == TML_TYPE_F32 ? 3 : 2;
    constexpr int kChunk = kF32 ? 16 : 32;           // d of a K load: 16 bytes of each of four lane groups
    constexpr int kChunks = DP / kChunk;
    constexpr int E = kF32 || DP == 64 ? 4 : 8;      // d of a V load
    constexpr int kHalves = DP / (16 * E);           // V loads a token
    constexpr int kOut = DP / 16;                    // accumulators
    // base of the weights' exponent: f16 terms of e^(s - m) reach down to 2^-39 of the largest
    constexpr float kUp = CT == TML_TYPE_F16 ? 14.0f : 0.0f;

    __shared__ __align__(16) int64_t row_off[kWaves][kTile];
    __shared__ float wave_m[kWaves][16], wave_l[kWaves][16];
    TML_DYNAMIC_LDS(floatx4, dyn);
    float *const wave_o = (float *)dyn;  // [wave][head][DP]
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int l16 = lane & 15, c4 = lane >> 4;
    const int64_t D = a.head_dim, P = a.block_size;

    ListWalk walk;
    if (!first_list(QT, a, sh, walk)) return;
    for (;;) {
        const int t1 = list_end(walk);
        const int64_t b = walk.b, unit = walk.unit;
        const Span sp = walk.sp;
        const int64_t kv = sh.parts == 1 ? unit : div_short(unit, sh.parts);
        const int g0 = (int)(unit - kv * sh.parts) * 16, gn = min(16, sh.group - g0);
        const int64_t head0 = kv * sh.group + g0;

        // ---- q as the scores' B operand: lane (head, c) has d = kChunk * chunk + (8 or 4) * c + e
        const int64_t q_at = b * a.q_stride + (head0 + min(l16, gn - 1)) * D;
        float to_score = a.scale;
        srv_u32x4 q[NQ][kChunks];
        if constexpr (kF32) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = c * kChunk + 4 * c4;
                q[0][c] = srv_u32x4{0, 0, 0, 0};
                if (d < D) q[0][c] = *(const srv_u32x4_any *)((const float *)a.q + q_at + d);
            }
        } else if constexpr (QT == CT) {
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = c * kChunk + 8 * c4;
                q[0][c] = srv_u32x4{0, 0, 0, 0};
                if (d < D) q[0][c] = srv_load8<CT>(a.q, q_at + d).d[0];
            }
        } else {
            float v[kChunks][8];
            uint32_t most = 0;
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                const int d = c * kChunk + 8 * c4;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[c][e] = 0.0f;
                if (d < D) srv_floats<QT>(srv_load8<QT>(a.q, q_at + d), v[c]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t g = __float_as_uint(v[c][e]) & 0x7F800000u;
                    most = max(most, g < 0x7F800000u ? g : 0u);
                }
            }
            if constexpr (CT == TML_TYPE_F16) {  // f16's range is short: the largest goes to [2^14, 2^15)
                most = max(most, (uint32_t)__shfl_xor((int)most, 16));
                most = max(most, (uint32_t)__shfl_xor((int)most, 32));
                most = max(most, 27u << 23);
                to_score *= __uint_as_float(most - (14u << 23));
#pragma unroll
                for (int c = 0; c < kChunks; ++c)
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[c][e] *= __uint_as_float((268u << 23) - most);
            }
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
                srv_u32x4 t[NQ];
                to_query_terms<CT, NQ>(v[c], t);
#pragma unroll
                for (int n = 0; n < NQ; ++n) q[n][c] = t[n];
            }
        }

        const float to_log2 = to_score * kLog2E;
        float slope = 0.0f, inv_cap = 0.0f;
        if constexpr (FORM) {
            if (a.slopes != nullptr) slope = a.slopes[head0 + min(l16, gn - 1)] * kLog2E;
            if (a.cap != 0.0f) inv_cap = 1.0f / a.cap;
        }

        float m = -INFINITY, l = 0.0f;  // of this lane's head; l over this lane's tokens alone
        floatx4 o[kOut];
#pragma unroll
        for (int j = 0; j < kOut; ++j) o[j] = floatx4{0, 0, 0, 0};

        // ---- the tiles: lane % 32 looks up a token's row
        auto block_of = [&](int tile) {
            const int64_t tok = sp.first + (int64_t)tile * kTile + (lane & 31);
            return a.block_table[b * a.table_stride + (uint32_t)min(tok, sp.len - 1) / (uint32_t)P];
        };
        // the byte offset of each token's row to LDS; which of the 32 may be looked at
        auto rows_of = [&](int tile, int in_block) {
            const int64_t tok = sp.first + (int64_t)tile * kTile + (lane & 31);
            const bool live = tile < t1 && tok < sp.len && in_block >= 0 && in_block < a.n_blocks;
            // (a token no one may look at reads the cache's first row)
            const int64_t off = live ? (in_block * a.block_stride + (int64_t)((uint32_t)tok % (uint32_t)P) * a.token_stride + kv * a.head_stride) * kBytes : 0;
            row_off[wave][lane & 31] = off;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            return (uint32_t)__builtin_amdgcn_ballot_w64(live);
        };
        srv_u32x4 kr[2][kChunks], vr[8][kHalves];
        auto load_k = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char *row = (const char *)a.k_cache + row_off[wave][16 * h + l16];
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    const int d = c * kChunk + (kChunk / 4) * c4;
                    kr[h][c] = load_cache<ONCE>(row + (d < D ? d : 0) * kBytes);
                }
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const char *row = (const char *)a.v_cache + row_off[wave][16 * (e / 4) + 4 * c4 + e % 4];
#pragma unroll
                for (int f = 0; f < kHalves; ++f) {
                    const int d = f * 16 * E + E * l16;
                    const char *at = row + (d < D ? d : 0) * kBytes;
                    if constexpr (E * kBytes == 16) {
                        vr[e][f] = load_cache<ONCE>(at);
                    } else {
                        const srv_u32x2 half = *(const srv_u32x2 *)at;
                        vr[e][f] = srv_u32x4{half[0], half[1], 0, 0};
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };

        // Keys of the next tile are under way from this tile's scores on, values from
        // its sums on, each into the registers just read.  (No branch around these
        // loads, or the wait for one would be a wait for all: past the last tile they
        // read the cache's first row.)
        int t = walk.t0 + wave;
        uint32_t seen = rows_of(t, block_of(t));
        load_k();
        int block = block_of(t + kWaves);  // (in the loop's order)
        __builtin_amdgcn_sched_barrier(0);
        load_v();
        while (t < t1) {
            // (past the head size there are keys again, and they may be infinite: q's zeros must not meet them)
            if (D < DP) {
#pragma unroll
                for (int c = DP == 64 ? 0 : kChunks / 2; c < kChunks; ++c)
                    if (c * kChunk + (kChunk / 4) * c4 >= D) kr[0][c] = kr[1][c] = srv_u32x4{0, 0, 0, 0};
            }
            // scores: sums over q's first terms, and over the others
            floatx4 lead[2], rest[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                lead[h] = rest[h] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < kChunks; ++c) {
                    if constexpr (kF32) {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            lead[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[h][c][e]), __uint_as_float(q[0][c][e]), lead[h], 0, 0, 0);
                    } else {
                        lead[h] = mma16<CT>(kr[h][c], q[0][c], lead[h]);
#pragma unroll
                        for (int n = 1; n < NQ; ++n) rest[h] = mma16<CT>(kr[h][c], q[n][c], rest[h]);
                    }
                }
            }
            if constexpr (NQ > 1) {
                // an infinite first sum is the score: the others only add infinities of any sign to it
                float peak = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) peak = fmaxf(peak, fabsf(lead[i / 4][i % 4]));
                if (__builtin_amdgcn_ballot_w64(peak == INFINITY) != 0) {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (fabsf(lead[i / 4][i % 4]) == INFINITY) rest[i / 4][i % 4] = 0.0f;
                }
            }
            float s[8];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float score = NQ > 1 ? lead[h][i] + rest[h][i] : lead[h][i];
                    float weight;
                    if constexpr (FORM) {
                        const float x = score * to_score;
                        const int64_t away = sp.len - 1 - sp.first - ((int64_t)t * kTile + 16 * h + 4 * c4 + i);
                        weight = (inv_cap != 0.0f ? cap_score(x, a.cap, inv_cap) : x) * kLog2E - slope * (float)away;
                    } else {
                        weight = score * to_log2;
                    }
                    s[4 * h + i] = (seen >> (16 * h + 4 * c4 + i) & 1) ? weight : -INFINITY;
                }
            t += kWaves;
            const uint32_t seen_now = seen;
            seen = rows_of(t, block);
            load_k();
            block = block_of(t + kWaves);
            float most = s[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) most = fmaxf(most, s[e]);
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            if (__builtin_amdgcn_ballot_w64(most > m) != 0) {
                const float m_new = fmaxf(m, most);
                const float f = rescale(m, m_new);
                m = m_new;
                l *= f;
#pragma unroll
                for (int j = 0; j < kOut; ++j) o[j] *= f;
            }
            const float base = (m == -INFINITY ? 0.0f : m) - kUp;
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(s[e] - base);
                l += p[e];
            }
            // what no one may look at can be anything, and zero times NaN is NaN
            if (seen_now != 0xFFFFFFFFu) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if ((seen_now >> (16 * (e / 4) + 4 * c4 + e % 4) & 1) == 0)
#pragma unroll
                        for (int f = 0; f < kHalves; ++f) vr[e][f] = srv_u32x4{0, 0, 0, 0};
            }
            if constexpr (kF32) {
#pragma unroll
                for (int f = 0; f < kHalves; ++f)
#pragma unroll
                    for (int j = 0; j < E; ++j)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            o[f * E + j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[e][f][j]), p[e], o[f * E + j], 0, 0, 0);
            } else {
                srv_u32x4 w[NP];
                to_terms<CT, NP>(p, w);
#pragma unroll
                for (int f = 0; f < kHalves; ++f)
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        srv_u32x4 vt;  // d = .. + j of the eight tokens
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            vt[e] = __builtin_amdgcn_perm(vr[2 * e + 1][f][j / 2], vr[2 * e][f][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
                        for (int n = 0; n < NP; ++n) o[f * E + j] = mma16<CT>(vt, w[n], o[f * E + j]);
                    }
            }
            load_v();
        }

        // ---- the waves' parts
        const float f = join_scale(wave_m, wave_l, wave, m, l);
        if (l16 < gn) {
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float *to = wave_o + (wave * sh.heads + l16) * DP + h * 16 * E + E * (4 * c4 + i);
#pragma unroll
                    for (int j = 0; j < E; j += 4)
                        *(floatx4 *)(to + j) = floatx4{o[h * E + j][i] * f, o[h * E + j + 1][i] * f, o[h * E + j + 2][i] * f, o[h * E + j + 3][i] * f};
                }
        }
        store_list(QT, a, sh, walk, t1, head0, gn, DP, wave_m, wave_l, wave_o);
        if (!next_list(a, sh, walk, t1)) return;
    }
}

constexpr int kPerCu = 2;  // workgroups
constexpr int kAtOnce = 16;  // query heads: a matrix instruction's columns

// A cache past the GPU's last-level cache is read with the streaming policy, a
// smaller one so that the next step may find it there.  Measured, plain / streaming:
// 64 requests of up to 4096 tokens (533 MB) 118 / 112 us, two of 40k to 65k (377 MB) 76 /
// 68; eight of 2k (72 MB) 25.2 / 27.1, one of 1500 with 20 heads of 64 (8 MB) 14.3 / 14.6.
// The rule goes by the whole pool, the lengths being on the GPU: few short requests in
// a large pool are read with the streaming policy too, at the last two's loss.
constexpr int64_t kLastLevel = (int64_t)256 << 20;

template <int CT, int QT, int DP, bool FORM>
void launch_kernel(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    const size_t lds = (size_t)kWaves * sh.heads * DP * 4;
    const dim3 grid(sh.grid), block(kThreads);
    const double bytes = 2.0 * type_bytes(CT) * a.n_blocks * a.block_size * a.kv_heads * a.head_dim;
    if (bytes > kLastLevel) paged_attention_kernel<CT, QT, DP, true, FORM><<<grid, block, lds, s>>>(a, sh);
    else paged_attention_kernel<CT, QT, DP, false, FORM><<<grid, block, lds, s>>>(a, sh);
}

template <int QT>
Status launch_join(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    if (sh.lists == nullptr) return Status::Ok();
    paged_attention_join_kernel<QT><<<dim3((unsigned)((a.q_heads + kJoinWaves - 1) / kJoinWaves), (unsigned)a.batch), dim3(64 * kJoinWaves), 0, s>>>(a, sh);
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

template <int CT, int QT, bool FORM>
Status launch_dim(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    if (a.head_dim <= 64) launch_kernel<CT, QT, 64, FORM>(a, sh, s);
    else if (a.head_dim <= 128) launch_kernel<CT, QT, 128, FORM>(a, sh, s);
    else launch_kernel<CT, QT, 256, FORM>(a, sh, s);
    TML_HIP_TRY(hipGetLastError());
    return launch_join<QT>(a, sh, s);
}
template <int CT, int QT>
Status launch_form(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    return a.cap != 0.0f || a.slopes != nullptr ? launch_dim<CT, QT, true>(a, sh, s) : launch_dim<CT, QT, false>(a, sh, s);
}

}  // namespace

Status check_paged_attention(const PagedAttentionArgs &a) {
    if (!float_type(a.cache_type) || (a.q_type != a.cache_type && a.q_type != TML_TYPE_F32))
        return Status::Err(TML_ERR_INVALID_FORMAT, "paged attention: the cache is f32, f16 or bf16, q the same or f32");
    if (a.batch < 0 || a.q_heads < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.n_blocks < 0 || a.table_width < 0 || a.window < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "paged attention: negative size");
    if (a.block_size < 1) return Status::Err(TML_ERR_INVALID_ARG, "paged attention: the block size must be positive");
    if (!valid_cap(a.cap)) return Status::Err(TML_ERR_INVALID_ARG, "paged attention: the cap must be 0 or from 2^-100 to 2^100");
    if (attn_empty(a)) return Status::Ok();
    if (a.q_heads % a.kv_heads != 0)
        return Status::Err(TML_ERR_SHAPE_MISMATCH, "paged attention: query heads are no multiple of key-value heads");
    if (a.head_dim % 8 != 0 || a.head_dim > 256)
        return Status::Err(TML_ERR_INVALID_SHAPE, "paged attention: the head size must be a multiple of 8, at most 256");
    const int64_t most = (int64_t)1 << 31;
    if (a.n_blocks >= most || a.block_size >= most || a.batch >= (1 << 16) || a.q_heads >= (1 << 16) ||
        a.table_width >= most || a.table_width * a.block_size > most)
        return Status::Err(TML_ERR_INVALID_SHAPE, "paged attention: requests and heads must be below 2^16, a table's positions at most 2^31");
    if (a.q == nullptr || a.out == nullptr || a.seq_len == nullptr || (a.n_blocks > 0 && (a.k_cache == nullptr || a.v_cache == nullptr)) ||
        (a.table_width > 0 && a.block_table == nullptr))
        return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    if (a.batch > 1 && (a.q_stride < a.q_heads * a.head_dim || a.out_stride < a.q_heads * a.head_dim || a.table_stride < a.table_width))
        return Status::Err(TML_ERR_INVALID_SHAPE, "paged attention: a row stride is shorter than the row");
    if (a.block_stride < 0 || a.token_stride < 0 || a.head_stride < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "paged attention: negative cache stride");
    const int64_t bytes = type_bytes(a.cache_type);
    if (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)(a.block_stride * bytes) | (uintptr_t)(a.token_stride * bytes) |
         (uintptr_t)(a.head_stride * bytes)) % 16 != 0)
        return Status::Err(TML_ERR_INVALID_ARG, "paged attention: the cache's rows must start on 16-byte boundaries");
    return Status::Ok();
}

size_t paged_attention_workspace_floats(const PagedAttentionArgs &a) {
    return attn_empty(a) ? 0 : split_floats(a, shape_of(a, kPerCu, kAtOnce));
}

Status launch_paged_attention(const PagedAttentionArgs &in, const Workspace &ws, hipStream_t s) {
    PagedAttentionArgs a = in;
    if (attn_empty(a)) return Status::Ok();
    if (a.n_blocks == 0) a.table_width = 0;  // no cache: nothing to look at
    AttnShape sh = shape_of(a, kPerCu, kAtOnce);
    TML_TRY(split_in(a, ws, &sh));
    if (a.cache_type == TML_TYPE_F32) return launch_form<TML_TYPE_F32, TML_TYPE_F32>(a, sh, s);
    if (a.cache_type == TML_TYPE_F16)
        return a.q_type == TML_TYPE_F32 ? launch_form<TML_TYPE_F16, TML_TYPE_F32>(a, sh, s) : launch_form<TML_TYPE_F16, TML_TYPE_F16>(a, sh, s);
    return a.q_type == TML_TYPE_F32 ? launch_form<TML_TYPE_BF16, TML_TYPE_F32>(a, sh, s) : launch_form<TML_TYPE_BF16, TML_TYPE_BF16>(a, sh, s);
}

}  // namespace tml
