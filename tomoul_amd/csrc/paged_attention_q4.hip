// paged_attention_q4.hip -- attention of one new token a request over a paged cache in
// 4 bits (kv_q4.hip), split over the cache's length and joined (paged_split.hpp).
//
// With rows x = n s_g + z_g of nibbles n, step s and minimum z for each group g of 32, and
// c_g = z_g + 8 s_g,
//   q . k_t  = sum_g s_tg (q_g . n_tg) + z_tg sum(q_g)
//   out_d    = sum_t (p_t s_tg) (n_td - 8) + sum_t p_t c_tg,   g = d / 32
// so the matrix cores multiply nibbles as f16 numbers, without a conversion.  Keys: a nibble
// alone is a number with no bits but the lowest, n 2^-24 in bits 0 .. 3, n 2^-20 in bits
// 4 .. 7: a shift and four masks for the eight of a word.  Values: or-ed into the lowest bits
// of 1024 it is 1024 + n, four bits higher 1024 + 16 n, and a packed addition takes 1032 or
// 1152 away.  The steps multiply the sums of a group (keys) or the weights (values), minima
// and middles go beside in fp32.  (Values less 8 and the middles, not nibbles and minima: the
// two sums would cancel each other, and the matrix cores round their sums towards zero.  f32
// outputs were 5e-5 off that way at 448 tokens, f16 ones 5e-4 at 65536; a key's sum is of
// one group and loses nothing to speak of.)
//
// Lane layout, a tile of 32 tokens, two halves h of 16 (as paged_attention.hip):
//   scores   MFMA h, w: rows tokens 16 h + lane % 16, k the 32 d of group w, columns heads;
//            the lane's words w of a row follow each other
//   weights  lane (head, c) holds those of tokens 16 h + 4 c + i, the k of the next product
//   values   MFMA j: rows d = 16 j + lane % 16, all of group j / 2; the B operand is p_t s_tg
// Steps and minima or middles of the tile's tokens pass through LDS, where every lane finds
// those of its eight tokens.  f32 q and weights for f32 outputs are two f16 terms each, q of 16
// bits is exact in one, and so are the weights rounded once where the output is of 16 bits:
// that adds to an f16 output about what its own rounding does, to a bf16 one an eighth.
#include "paged_split.hpp"
#include "terms.hpp"

namespace tml {
namespace {

// The eight nibbles of a word: register r holds those r and r + 4, times 2^-24 (r even) or 2^-20.
__device__ __forceinline__ srv_u32x4 nibbles(uint32_t w) {
    const uint32_t up = w >> 8;
    return srv_u32x4{w & 0x000F000Fu, w & 0x00F000F0u, up & 0x000F000Fu, up & 0x00F000F0u};
}
// Nibbles at bits 0 (SHIFT 0) or 4 of both halves of a word, less 8, as two f16; SHIFT 4: times 16.
template <int SHIFT>
__device__ __forceinline__ uint32_t two_nibbles(uint32_t w, uint32_t thousands) {
    const _Float16 less = SHIFT == 0 ? (_Float16)-1032.0f : (_Float16)-1152.0f;
    const uint32_t up = (w & (0x000F000Fu << SHIFT)) | thousands;
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(srv_f16x2, up) + (srv_f16x2){less, less});
}
// 1024 in both halves, in a vector register: one instruction masks and ors then.
__device__ __forceinline__ uint32_t two_thousands() {
    uint32_t v = 0x64006400u;
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("" : "+v"(v));
#endif
    return v;
}

// Two floats in two f16 terms each.
__device__ __forceinline__ void two_terms(float x, float y, uint32_t *first, uint32_t *second) {
    *first = srv_pack_f16(x, y);
    *second = srv_pack_f16(x - tml_half_bits(*first & 0xFFFFu), y - tml_half_bits(*first >> 16));
}

// N consecutive words at p, which may lie on any 4-byte boundary.
template <int N>
struct Words {
    uint32_t w[N];
};
template <int N, bool ONCE>
__device__ __forceinline__ Words<N> load_words(const char *p) {
    Words<N> r;
    typedef srv_u32x4 x4 __attribute__((aligned(4)));
    typedef srv_u32x2 x2 __attribute__((aligned(4)));
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
        const x4 v = ONCE ? __builtin_nontemporal_load((const x4 *)(p + 4 * i)) : *(const x4 *)(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[i + j] = v[j];
    }
    if (N % 4 >= 2) {
        const x2 v = ONCE ? __builtin_nontemporal_load((const x2 *)(p + 4 * (N / 4 * 4))) : *(const x2 *)(p + 4 * (N / 4 * 4));
        r.w[N / 4 * 4] = v[0];
        r.w[N / 4 * 4 + 1] = v[1];
    }
    if (N % 2 == 1) r.w[N - 1] = ONCE ? __builtin_nontemporal_load((const uint32_t *)(p + 4 * (N - 1))) : *(const uint32_t *)(p + 4 * (N - 1));
    return r;
}
// N consecutive bytes at p in (N + 3) / 4 words.  Past the last of a row's 16 lanes lie its
// steps and minima, 4 N bytes, so 3 bytes may be taken as 4 and 5 to 7 as 8.
template <int N, bool ONCE>
__device__ __forceinline__ Words<(N + 3) / 4> load_bytes(const char *p) {
    Words<(N + 3) / 4> r;
    if constexpr (N == 1) {
        r.w[0] = ONCE ? __builtin_nontemporal_load((const uint8_t *)p) : *(const uint8_t *)p;
    } else if constexpr (N == 2) {
        r.w[0] = ONCE ? __builtin_nontemporal_load((const uint16_t *)p) : *(const uint16_t *)p;
    } else if constexpr (N <= 4) {
        typedef uint32_t any __attribute__((aligned(1)));
        r.w[0] = ONCE ? __builtin_nontemporal_load((const any *)p) : *(const any *)p;
    } else {
        const srv_u32x2_any v = ONCE ? __builtin_nontemporal_load((const srv_u32x2_any *)p) : *(const srv_u32x2_any *)p;
        r.w[0] = v[0];
        r.w[1] = v[1];
    }
    return r;
}

// G: groups of a head.  WIDE: q and the output are f32.  FORM: the scores are capped or
// biased.  ONCE: the cache is read with the streaming policy.
template <int G, bool WIDE, bool FORM, bool ONCE>
__global__ __launch_bounds__(kThreads, G > 4 ? 1 : 2) void paged_attention_q4_kernel(PagedAttentionArgs a, AttnShape sh) {
    constexpr int D = 32 * G;
    constexpr int VW = (G + 3) / 4;  // words of a lane's values
    constexpr int NT = WIDE ? 2 : 1;  // terms of q and of the weights
    // The maximum that weights are relative to may fall behind by kBehind (in powers of two)
    // before sums are scaled.  kUp: base of the weights' exponent, their terms reach down to
    // 2^-38 of the largest (f32 outputs) or 2^-23 (and the maximum behind).
    constexpr float kBehind = WIDE ? 0.0f : 8.0f, kUp = WIDE ? 14.0f : 6.0f;

    __shared__ __align__(16) int64_t row_off[kWaves][kTile];
    __shared__ __align__(16) srv_f32x2 meta[kWaves][2][kTile][G];  // steps and minima of keys, steps and middles of values
    __shared__ float wave_m[kWaves][16], wave_l[kWaves][16];
    TML_DYNAMIC_LDS(floatx4, dyn);
    float *const wave_o = (float *)dyn;  // [wave][head][D]
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int l16 = lane & 15, c4 = lane >> 4;
    const int64_t P = a.block_size;
    const uint32_t thousands = two_thousands();

    ListWalk walk;
    if (!first_list(a.q_type, a, sh, walk)) return;
    for (;;) {
        const int t1 = list_end(walk);
        const int64_t b = walk.b, unit = walk.unit;
        const Span sp = walk.sp;
        const int64_t kv = sh.parts == 1 ? unit : div_short(unit, sh.parts);
        const int g0 = (int)(unit - kv * sh.parts) * 16, gn = min(16, sh.group - g0);
        const int64_t head0 = kv * sh.group + g0;

        // ---- q as the scores' B operand: lane (head, c) has d = 32 w + 8 c + e, in the nibbles' order.
        // Scaled by a power of two to [2^14, 2^15) at most, and the odd registers by 2^-4.
        const int64_t q_at = b * a.q_stride + (head0 + min(l16, gn - 1)) * D;
        srv_u32x4 q[NT][G];
        float q_sum[G], to_score = a.scale;
        {
            float v[G][8];
            uint32_t most = 27u << 23;
#pragma unroll
            for (int w = 0; w < G; ++w) {
                const int64_t at = q_at + 32 * w + 8 * c4;
                if (WIDE) srv_floats<TML_TYPE_F32>(srv_load8<TML_TYPE_F32>(a.q, at), v[w]);
                else if (a.q_type == TML_TYPE_F16) srv_floats<TML_TYPE_F16>(srv_load8<TML_TYPE_F16>(a.q, at), v[w]);
                else srv_floats<TML_TYPE_BF16>(srv_load8<TML_TYPE_BF16>(a.q, at), v[w]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t x = __float_as_uint(v[w][e]) & 0x7F800000u;
                    most = max(most, x < 0x7F800000u ? x : 0u);
                }
            }
            most = max(most, (uint32_t)__shfl_xor((int)most, 16));
            most = max(most, (uint32_t)__shfl_xor((int)most, 32));
            to_score *= __uint_as_float(most - (14u << 23)) * 0x1p24f;
            const float up = __uint_as_float((268u << 23) - most);
#pragma unroll
            for (int w = 0; w < G; ++w) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[w][e] *= up;
                    sum += v[w][e];
                }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
                q_sum[w] = sum * 0x1p-24f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = r % 2 ? 0x1p-4f : 1.0f;
                    if constexpr (WIDE) {
                        uint32_t first, second;
                        two_terms(v[w][r] * f, v[w][r + 4] * f, &first, &second);
                        q[0][w][r] = first;
                        q[1][w][r] = second;
                    } else {
                        q[0][w][r] = srv_pack_f16(v[w][r] * f, v[w][r + 4] * f);
                    }
                }
            }
        }
        const float to_log2 = to_score * kLog2E;
        float slope = 0.0f, inv_cap = 0.0f;
        if constexpr (FORM) {
            if (a.slopes != nullptr) slope = a.slopes[head0 + min(l16, gn - 1)] * kLog2E;
            if (a.cap != 0.0f) inv_cap = 1.0f / a.cap;
        }

        float m = -INFINITY, l = 0.0f;  // of this lane's head; l over this lane's tokens alone
        uint32_t peak = 0;              // exponent of the largest step so far, of f32 bits; the weights are in units of it
        floatx4 o[2 * G];
        float middle[G];                // sums of p c over this lane's tokens
#pragma unroll
        for (int j = 0; j < 2 * G; ++j) o[j] = floatx4{0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < G; ++g) middle[g] = 0.0f;

        // ---- the tiles: lane % 32 looks up a token's row
        auto block_of = [&](int tile) {
            const int64_t tok = sp.first + (int64_t)tile * kTile + (lane & 31);
            return a.block_table[b * a.table_stride + (uint32_t)min(tok, sp.len - 1) / (uint32_t)P];
        };
        Words<G> marks;  // steps and minima of the token of lane % 32, of its key or its value
        auto rows_of = [&](int tile, int in_block) {
            const int64_t tok = sp.first + (int64_t)tile * kTile + (lane & 31);
            const bool live = tile < t1 && tok < sp.len && in_block >= 0 && in_block < a.n_blocks;
            // (a token no one may look at reads the cache's first row, its steps and middles are zero)
            const int64_t off = live ? in_block * a.block_stride + (int64_t)((uint32_t)tok % (uint32_t)P) * a.token_stride + kv * a.head_stride : 0;
            row_off[wave][lane & 31] = off;
            marks = load_words<G, ONCE>((const char *)(lane < 32 ? a.k_cache : a.v_cache) + off + 16 * G);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            return (uint32_t)__builtin_amdgcn_ballot_w64(live);
        };
        Words<G> kr[2];
        Words<VW> vr[8];
        auto load_k = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) kr[h] = load_words<G, ONCE>((const char *)a.k_cache + row_off[wave][16 * h + l16] + 4 * G * c4);
        };
        auto load_v = [&]() {
#pragma unroll
            for (int e = 0; e < 8; ++e) vr[e] = load_bytes<G, ONCE>((const char *)a.v_cache + row_off[wave][16 * (e / 4) + 4 * c4 + e % 4] + G * l16);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        };

        int t = walk.t0 + wave;
        uint32_t seen = rows_of(t, block_of(t));
        load_k();
        int block = block_of(t + kWaves);
        __builtin_amdgcn_sched_barrier(0);
        load_v();
        while (t < t1) {
            const bool mine = seen >> (lane & 31) & 1;
            float step_most = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) {
                const uint32_t d = mine ? marks.w[g] : 0u;
                const float step = tml_half_bits(d & 0xFFFFu);
                meta[wave][lane >> 5][lane & 31][g] = srv_f32x2{step, fmaf(step, lane < 32 ? 0.0f : 8.0f, tml_half_bits(d >> 16))};
                step_most = fmaxf(step_most, step);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();

            // ---- scores
            float s[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = 0.0f;
#pragma unroll
            for (int w = 0; w < G; ++w) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const srv_u32x4 n = nibbles(kr[h].w[w]);
                    floatx4 sum = mma16<TML_TYPE_F16>(n, q[0][w], floatx4{0, 0, 0, 0});
                    if constexpr (WIDE) sum = mma16<TML_TYPE_F16>(n, q[1][w], sum);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const srv_f32x2 d = meta[wave][0][16 * h + 4 * c4 + i][w];
                        s[4 * h + i] = fmaf(sum[i], d[0], fmaf(q_sum[w], d[1], s[4 * h + i]));
                    }
                }
                if (G > 4 && w % 2 == 1) __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (FORM) {
                const float from = (float)(sp.len - 1 - sp.first - ((int64_t)t * kTile + 4 * c4));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = s[e] * to_score;
                    s[e] = fmaf(-slope, from - (float)(16 * (e / 4) + e % 4), (inv_cap != 0.0f ? cap_score(x, a.cap, inv_cap) : x) * kLog2E);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) s[e] *= to_log2;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) s[e] = (seen >> (16 * (e / 4) + 4 * c4 + e % 4) & 1) ? s[e] : -INFINITY;
            t += kWaves;
            seen = rows_of(t, block);
            load_k();
            block = block_of(t + kWaves);

            // ---- weights
            float most = s[0];
#pragma unroll
            for (int e = 1; e < 8; ++e) most = fmaxf(most, s[e]);
            most = fmaxf(most, __shfl_xor(most, 16));
            most = fmaxf(most, __shfl_xor(most, 32));
            if (__builtin_amdgcn_ballot_w64(most > m + kBehind) != 0) {
                const float m_new = fmaxf(m, most);
                const float f = rescale(m, m_new);
                m = m_new;
                l *= f;
#pragma unroll
                for (int j = 0; j < 2 * G; ++j) o[j] *= f;
#pragma unroll
                for (int g = 0; g < G; ++g) middle[g] *= f;
            }
            // (a step that is no number, or infinite, counts as none: its weights are what they are)
            uint32_t step_bits = lane < 32 ? 0u : __float_as_uint(step_most) & 0x7F800000u;
            if (step_bits == 0x7F800000u) step_bits = 0u;
            if (__builtin_amdgcn_ballot_w64(step_bits > peak) != 0) {
#pragma unroll
                for (int x = 1; x < 64; x <<= 1) step_bits = max(step_bits, (uint32_t)__shfl_xor((int)step_bits, x));
                const float f = peak == 0u ? 1.0f : __uint_as_float(peak) / __uint_as_float(step_bits);
                peak = step_bits;
#pragma unroll
                for (int j = 0; j < 2 * G; ++j) o[j] *= f;
            }
            // (no step yet: all of them are zero)
            const float unit_step = peak == 0u ? 1.0f : __uint_as_float((253u << 23) - peak);  // 2^-1 / the largest's power of two
            const float base = (m == -INFINITY ? 0.0f : m) - kUp;
            float p[8], in_units[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(s[e] - base);
                l += p[e];
                in_units[e] = p[e] * unit_step;
            }
            // ---- values
            srv_u32x4 pair[2 * VW];  // 16 bits of tokens 2 i and 2 i + 1
#pragma unroll
            for (int x = 0; x < (G + 1) / 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    pair[x][i] = __builtin_amdgcn_perm(vr[2 * i + 1].w[x / 2], vr[2 * i].w[x / 2], x % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                float step[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const srv_f32x2 d = meta[wave][1][16 * (e / 4) + 4 * c4 + e % 4][g];
                    step[e] = d[0];
                    middle[g] = fmaf(p[e], d[1], middle[g]);
                }
                srv_u32x4 weight[NT];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = in_units[2 * i] * step[2 * i], y = in_units[2 * i + 1] * step[2 * i + 1];
                    if constexpr (WIDE) {
                        uint32_t first, second;
                        two_terms(x, y, &first, &second);
                        weight[0][i] = first;
                        weight[1][i] = second;
                    } else {
                        weight[0][i] = srv_pack_f16(x, y);
                    }
                }
#pragma unroll
                for (int j = 2 * g; j < 2 * g + 2; ++j) {
                    srv_u32x4 n;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t two = j % 4 >= 2 ? pair[j / 4][i] >> 8 : pair[j / 4][i];
                        n[i] = j % 2 ? two_nibbles<4>(two, thousands) : two_nibbles<0>(two, thousands);
                    }
#pragma unroll
                    for (int x = 0; x < NT; ++x) o[j] = mma16<TML_TYPE_F16>(n, weight[x], o[j]);
                }
                if (G > 4 && g % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // (else registers run out)
            }
            load_v();
        }

        // ---- the waves' parts
        const float f = join_scale(wave_m, wave_l, wave, m, l);
        const float up = (peak == 0u ? 0.0f : __uint_as_float(peak) * 2.0f) * f;  // out of the weights' units
#pragma unroll
        for (int g = 0; g < G; ++g) {
            middle[g] += __shfl_xor(middle[g], 16);
            middle[g] += __shfl_xor(middle[g], 32);
        }
        if (l16 < gn) {
#pragma unroll
            for (int j = 0; j < 2 * G; ++j) {
                const float r = j % 2 ? up * 0x1p-4f : up, z = middle[j / 2] * f;
                *(floatx4 *)(wave_o + (wave * sh.heads + l16) * D + 16 * j + 4 * c4) =
                    floatx4{fmaf(o[j][0], r, z), fmaf(o[j][1], r, z), fmaf(o[j][2], r, z), fmaf(o[j][3], r, z)};
            }
        }
        store_list(a.q_type, a, sh, walk, t1, head0, gn, D, wave_m, wave_l, wave_o);
        if (!next_list(a, sh, walk, t1)) return;
    }
}

template <int QT>
Status launch_join(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    if (sh.lists == nullptr) return Status::Ok();
    paged_attention_join_kernel<QT><<<dim3((unsigned)((a.q_heads + kJoinWaves - 1) / kJoinWaves), (unsigned)a.batch), dim3(64 * kJoinWaves), 0, s>>>(a, sh);
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

constexpr int kPerCu = 2;  // workgroups
constexpr int64_t kLastLevel = (int64_t)256 << 20;  // a cache past it is read with the streaming policy

template <int G, bool WIDE, bool FORM>
void launch_kernel(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    const size_t lds = (size_t)kWaves * sh.heads * 32 * G * 4;
    const dim3 grid(1u << sh.grid_log2), block(kThreads);
    const double bytes = 40.0 * G * a.n_blocks * a.block_size * a.kv_heads;
    if (bytes > kLastLevel) paged_attention_q4_kernel<G, WIDE, FORM, true><<<grid, block, lds, s>>>(a, sh);
    else paged_attention_q4_kernel<G, WIDE, FORM, false><<<grid, block, lds, s>>>(a, sh);
}
template <int G>
void launch_groups(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    const bool form = a.cap != 0.0f || a.slopes != nullptr;
    if (a.q_type == TML_TYPE_F32) form ? launch_kernel<G, true, true>(a, sh, s) : launch_kernel<G, true, false>(a, sh, s);
    else form ? launch_kernel<G, false, true>(a, sh, s) : launch_kernel<G, false, false>(a, sh, s);
}

}  // namespace

Status check_paged_attention_q4(const PagedAttentionArgs &a) {
    PagedAttentionArgs b = a;  // as over a cache of q's type, whose rows are aligned whatever they are here
    b.cache_type = a.q_type;
    b.k_cache = a.k_cache == nullptr ? nullptr : (const void *)16;
    b.v_cache = a.v_cache == nullptr ? nullptr : (const void *)16;
    b.block_stride = b.token_stride = b.head_stride = 0;
    if (a.block_stride < 0 || a.token_stride < 0 || a.head_stride < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "paged attention: negative cache stride");
    TML_TRY(check_paged_attention(b));
    if (attn_empty(a)) return Status::Ok();
    if (a.head_dim % 32 != 0) return Status::Err(TML_ERR_INVALID_SHAPE, "4-bit paged attention: the head size must be a multiple of 32, at most 256");
    if (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)a.block_stride | (uintptr_t)a.token_stride | (uintptr_t)a.head_stride) % 4 != 0)
        return Status::Err(TML_ERR_INVALID_ARG, "4-bit paged attention: the cache's rows must start on 4-byte boundaries");
    return Status::Ok();
}

size_t paged_attention_q4_workspace_floats(const PagedAttentionArgs &a) { return attn_empty(a) ? 0 : split_floats(a, shape_of(a, kPerCu)); }

Status launch_paged_attention_q4(const PagedAttentionArgs &in, const Workspace &ws, hipStream_t s) {
    PagedAttentionArgs a = in;
    if (attn_empty(a)) return Status::Ok();
    if (a.n_blocks == 0) a.table_width = 0;  // no cache: nothing to look at
    AttnShape sh = shape_of(a, kPerCu);
    TML_TRY(split_in(a, ws, &sh));
    switch (a.head_dim / 32) {
        case 1: launch_groups<1>(a, sh, s); break;
        case 2: launch_groups<2>(a, sh, s); break;
        case 3: launch_groups<3>(a, sh, s); break;
        case 4: launch_groups<4>(a, sh, s); break;
        case 5: launch_groups<5>(a, sh, s); break;
        case 6: launch_groups<6>(a, sh, s); break;
        case 7: launch_groups<7>(a, sh, s); break;
        default: launch_groups<8>(a, sh, s); break;
    }
    TML_HIP_TRY(hipGetLastError());
    if (a.q_type == TML_TYPE_F32) return launch_join<TML_TYPE_F32>(a, sh, s);
    return a.q_type == TML_TYPE_F16 ? launch_join<TML_TYPE_F16>(a, sh, s) : launch_join<TML_TYPE_BF16>(a, sh, s);
}

}  // namespace tml
