// paged_attention_q4.hip -- attention of one new token a request over a paged cache in
// 4 bits (kv_q4.hip), split over the cache's length and joined (paged_split.hpp).
//
// With rows x = n s_g + z_g of nibbles n, step s and minimum z for each group g of 32, and
// c_g = z_g + 8 s_g,
//   q . k_t  = sum_g s_tg (q_g . n_tg) + z_tg sum(q_g)
//   out_d    = sum_t (p_t s_tg) (n_td - 8) + sum_t p_t c_tg,   g = d / 32
// so the matrix cores multiply nibbles as f16 numbers, without a conversion: or-ed into the
// lowest bits of 1024 a nibble is 1024 + n, four bits higher 1024 + 16 n, and a packed addition
// takes 1032 or 1152 away.  For keys and 16-bit outputs it is left out: a nibble alone is a
// number with no bits but the lowest, n 2^-24 in bits 0 .. 3, n 2^-20 in bits 4 .. 7, so a shift
// and four masks do for the eight of a word.  The matrix cores align such products as if they were
// 2^6 to 2^10 larger and lose bits below: f32 outputs were 2e-6 off at 448 tokens, 3e-7 with n - 8.
// The steps multiply the sums of a group (keys) or the weights (values), minima and middles
// go beside in fp32.  (Values less 8 and the middles, not nibbles and minima: the two sums
// would cancel each other, and the matrix cores round their sums towards zero.  f32 outputs
// were 5e-5 off that way at 448 tokens, f16 ones 5e-4 at 65536.)
//
// Four heads and four groups share the 16 rows or columns that a matrix instruction has, so
// that with grouped heads of four none of them, and none of the work on what comes out,
// is idle.  A tile is 32 tokens:
//   scores   S = q K^T for 16 tokens (columns): row 4 (w % 4) + i is head i, with the elements of
//            group w alone, zeros elsewhere.  The products of four groups go into one
//            accumulator, of which lane (token, c) holds group c's sums of four heads; it
//            multiplies them with the step, and two swaps of halves and rows add the groups
//            up and leave lane (token, c) the score of head c
//   weights  pass through LDS, to where lane (4 g + head, c) makes the next product's B operand:
//            p of its head times the steps of group g, for the eight tokens of its c
//   values   rows d = 16 j + lane % 16 of group j / 2, of whose output the columns of that group are
//            kept
// f32 q, and weights for f32 outputs, are two f16 terms each; q of 16 bits is exact in one, and
// so are the weights rounded once where the output is of 16 bits: that adds to an f16 output
// about what its own rounding does, to a bf16 one an eighth.
//
// Measured on MI355X (launches in a graph): bf16, 64 requests of up to 4096 tokens, 32 heads on 8
// of 128 65 us (2.3 TB/s of the cache's 5 bits; in 16 bits 112 us), two of 40k to 65k tokens,
// f16, 40 us (3.3 TB/s); one of 448 tokens, f32, 20 heads of 64, 9.3 us.  Memory does not bound it:
// a tile of 4 KB is some 360 vector instructions of a wave, of which the nibbles of values are
// 100 and the weights 60.  By the counters (64 requests, two long ones): vector instructions issue
// for 70 % of the time in which a CU has waves, but a CU has waves for 47 and 65 % of the kernel alone.  The
// rest is uneven shares: with requests of 2048 tokens each a tile takes 1.63 ns of the GPU, with lengths from
// 512 on 1.67, with the ragged ones 2.23, of which the short ones put many lists, each with its
// prologue and its joining, into one workgroup's share.  Loads two tiles ahead gained nothing (41.3 for 39
// us).  Short lists are bound by the chain of dependent loads and by the joining.
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

// Lane (l, c) of four rows of 16 lanes brings c's part of four sums; it gets sum c of the four rows'.
__device__ __forceinline__ float sum_and_share(const float (&v)[4]) {
    float two[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + 2]), false, false);
        two[i] = __uint_as_float(both[0]) + __uint_as_float(both[1]);
    }
    const auto both = __builtin_amdgcn_permlane16_swap(__float_as_uint(two[0]), __float_as_uint(two[1]), false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// N consecutive words at p, which may lie on any 4-byte boundary.
template <int N>
struct Words {
    uint32_t w[N];
};
template <int N>
__device__ __forceinline__ Words<N> load_words(const char *p) {
    Words<N> r;
    typedef srv_u32x4 x4 __attribute__((aligned(4)));
    typedef srv_u32x2 x2 __attribute__((aligned(4)));
    int i = 0;
#pragma unroll
    for (; i + 4 <= N; i += 4) {
        const x4 v = *(const x4 *)(p + 4 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[i + j] = v[j];
    }
    if (N % 4 >= 2) {
        const x2 v = *(const x2 *)(p + 4 * (N / 4 * 4));
        r.w[N / 4 * 4] = v[0];
        r.w[N / 4 * 4 + 1] = v[1];
    }
    if (N % 2 == 1) r.w[N - 1] = *(const uint32_t *)(p + 4 * (N - 1));
    return r;
}
// N consecutive bytes at p in (N + 3) / 4 words.  Past the last of a row's 16 lanes lie its
// steps and minima, 4 N bytes, so 3 bytes may be taken as 4 and 5 to 7 as 8.
template <int N>
__device__ __forceinline__ Words<(N + 3) / 4> load_bytes(const char *p) {
    Words<(N + 3) / 4> r;
    if constexpr (N == 1) {
        r.w[0] = *(const uint8_t *)p;
    } else if constexpr (N == 2) {
        r.w[0] = *(const uint16_t *)p;
    } else if constexpr (N <= 4) {
        typedef uint32_t any __attribute__((aligned(1)));
        r.w[0] = *(const any *)p;
    } else {
        const srv_u32x2_any v = *(const srv_u32x2_any *)p;
        r.w[0] = v[0];
        r.w[1] = v[1];
    }
    return r;
}

// Workgroups on a CU: three where the registers hold them, else two.  Three / two, bf16, 32 heads on 8
// of 128: 64 ragged requests of up to 4096 tokens 64 / 70 us, of up to 2048 42 / 47 us, one of 60000
// 35 / 31 us, 32 of 2048 alike 30 / 25 us (a list is half a workgroup's share there); over
// eighteen batches two took 1.02 times as long.  Four spill: 102 us for the first.  Where two spill:
// two / one, f32, 64 of 1000 tokens, 32 heads on 8 of 192, 34 / 45 us.
constexpr int per_cu(int groups, int fours, bool wide) { return wide || groups * fours > 4 || fours > 1 ? 2 : 3; }

// G: groups of a head.  HQ: heads taken at once, in fours.  WIDE: q and the output are f32.  FORM:
// the scores are capped or biased.
template <int G, int HQ, bool WIDE, bool FORM>
__global__ __launch_bounds__(kThreads, per_cu(G, HQ, WIDE)) void paged_attention_q4_kernel(PagedAttentionArgs a, AttnShape sh) {
    constexpr int D = 32 * G;
    constexpr int VW = (G + 3) / 4;   // words of a lane's values
    constexpr int GQ = (G + 3) / 4;   // groups, in fours
    constexpr int MW = (G + 1) / 2;   // steps and minima that a lane brings of a token's value
    constexpr int NT = WIDE ? 2 : 1;  // terms of q and of the weights
    // The maximum that weights are relative to may fall behind by kBehind (in powers of two)
    // before sums are scaled.  kUp: base of the weights' exponent, their terms reach down to
    // 2^-34 of the largest (f32 outputs) or 2^-23 (and the maximum behind).
    // kKeys: what a key's number is multiplied with for its nibble (less 8 where WIDE).
    constexpr float kKeys = WIDE ? 1.0f : 0x1p24f;
    constexpr float kBehind = WIDE ? 4.0f : 8.0f, kUp = WIDE ? 10.0f : 6.0f;

    __shared__ __align__(16) int64_t row_off[kWaves][kTile];
    __shared__ __align__(16) srv_f32x2 marks[kWaves][4 * GQ][kTile];  // steps and middles of values
    __shared__ __align__(16) float weights[kWaves][4 * HQ][kTile];
    __shared__ float wave_m[kWaves][16], wave_l[kWaves][16];
    TML_DYNAMIC_LDS(floatx4, dyn);
    float *const wave_o = (float *)dyn;  // [wave][head][D]
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int l16 = lane & 15, c4 = lane >> 4;
    const int hi = l16 & 3, gi = l16 >> 2;  // this lane's column: of the heads, of the groups
    const int64_t P = a.block_size;
    const uint32_t thousands = two_thousands();

    ListWalk walk;
    if (!first_list(a.q_type, a, sh, walk)) return;
    for (;;) {
        const int t1 = list_end(walk);
        const int64_t b = walk.b, unit = walk.unit;
        const Span sp = walk.sp;
        const int64_t kv = sh.parts == 1 ? unit : div_short(unit, sh.parts);
        const int g0 = (int)(unit - kv * sh.parts) * 4 * HQ, gn = min(4 * HQ, sh.group - g0);
        const int64_t head0 = kv * sh.group + g0;

        // ---- q as the scores' A operand: lane (4 (w % 4) + head, c) has d = 32 w + 8 c + e, in the
        // nibbles' order, others zeros.  Scaled by a power of two to [2^14, 2^15) at most, and the
        // odd registers by 2^-4.
        srv_u32x4 q[HQ][NT][G];
        float q_sum[HQ][4][GQ], to_score[HQ];  // sums of head 4 x + i over group 4 y + c; of head 4 x + c
#pragma unroll
        for (int x = 0; x < HQ; ++x) {
            const int64_t q_at = b * a.q_stride + (head0 + min(4 * x + hi, gn - 1)) * D;
            float v[GQ][8];  // of this lane's groups 4 y + gi
            uint32_t most = 27u << 23;
#pragma unroll
            for (int y = 0; y < GQ; ++y) {
                const int w = 4 * y + gi;
                const int64_t at = q_at + 32 * min(w, G - 1) + 8 * c4;
                if (WIDE) srv_floats<TML_TYPE_F32>(srv_load8<TML_TYPE_F32>(a.q, at), v[y]);
                else if (a.q_type == TML_TYPE_F16) srv_floats<TML_TYPE_F16>(srv_load8<TML_TYPE_F16>(a.q, at), v[y]);
                else srv_floats<TML_TYPE_BF16>(srv_load8<TML_TYPE_BF16>(a.q, at), v[y]);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (w >= G) v[y][e] = 0.0f;
                    const uint32_t bits = __float_as_uint(v[y][e]) & 0x7F800000u;
                    most = max(most, bits < 0x7F800000u ? bits : 0u);
                }
            }
#pragma unroll
            for (int o = 4; o < 64; o <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o));  // over groups and c
            const float up = __uint_as_float((268u << 23) - most);
            to_score[x] = a.scale * __uint_as_float((uint32_t)__shfl((int)most, c4) - (14u << 23)) * kKeys;
#pragma unroll
            for (int y = 0; y < GQ; ++y) {
                float sum = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[y][e] *= up;
                    sum += v[y][e];
                }
                sum += __shfl_xor(sum, 16);
                sum += __shfl_xor(sum, 32);
#pragma unroll
                for (int i = 0; i < 4; ++i) q_sum[x][i][y] = __shfl(sum, 4 * c4 + i) / kKeys;  // (of column 4 c + i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float f = r % 2 ? 0x1p-4f : 1.0f;
                    uint32_t term[2];
                    if constexpr (WIDE) two_terms(v[y][r] * f, v[y][r + 4] * f, &term[0], &term[1]);
                    else term[0] = srv_pack_f16(v[y][r] * f, v[y][r + 4] * f);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int w = 4 * y; w < min(4 * y + 4, G); ++w) q[x][n][w][r] = gi == w % 4 ? term[n] : 0u;
                }
            }
        }
        float slope[HQ], inv_cap = 0.0f;
        if constexpr (FORM) {
#pragma unroll
            for (int x = 0; x < HQ; ++x) slope[x] = a.slopes != nullptr ? a.slopes[head0 + min(4 * x + c4, gn - 1)] * kLog2E : 0.0f;
            if (a.cap != 0.0f) inv_cap = 1.0f / a.cap;
        }

        float m[HQ], l[HQ];  // of head 4 x + c4; l over the tokens of this lane alone
        uint32_t peak = 0;   // exponent of the largest step so far, of f32 bits; the weights are in units of it
        floatx4 o[HQ][2 * G];
        float middle[HQ][GQ];  // sums of p c of head 4 x + hi over the tokens of c4, group 4 y + gi
#pragma unroll
        for (int x = 0; x < HQ; ++x) {
            m[x] = -INFINITY;
            l[x] = 0.0f;
#pragma unroll
            for (int j = 0; j < 2 * G; ++j) o[x][j] = floatx4{0, 0, 0, 0};
#pragma unroll
            for (int y = 0; y < GQ; ++y) middle[x][y] = 0.0f;
        }

        // ---- the tiles: lane % 32 looks up a token's row
        auto block_of = [&](int tile) {
            const int64_t tok = sp.first + (int64_t)tile * kTile + (lane & 31);
            return a.block_table[b * a.table_stride + (uint32_t)min(tok, sp.len - 1) / (uint32_t)P];
        };
        Words<G> kr[2];             // keys of tokens 16 h + l16, the lane's words of groups 0 ..
        uint32_t km[2][GQ];         // and the steps and minima of group 4 y + c4
        Words<VW> vr[8];            // values of tokens 8 c4 + e
        uint32_t vm[MW];            // steps and minima of the value of token lane % 32: groups MW (lane / 32) ..
        auto rows_of = [&](int tile, int in_block) {
            const int64_t tok = sp.first + (int64_t)tile * kTile + (lane & 31);
            const bool live = tile < t1 && tok < sp.len && in_block >= 0 && in_block < a.n_blocks;
            // (a token no one may look at reads the cache's first row)
            const int64_t off = live ? in_block * a.block_stride + (int64_t)((uint32_t)tok % (uint32_t)P) * a.token_stride + kv * a.head_stride : 0;
            row_off[wave][lane & 31] = off;
            const char *const from = (const char *)a.v_cache + off + 16 * G;
            if constexpr (G % 2 == 0) {
                const Words<MW> w = load_words<MW>(from + (lane >> 5) * 4 * MW);
#pragma unroll
                for (int i = 0; i < MW; ++i) vm[i] = w.w[i];
            } else {
#pragma unroll
                for (int i = 0; i < MW; ++i) vm[i] = *(const uint32_t *)(from + 4 * min((lane >> 5) * MW + i, G - 1));
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            return (uint32_t)__builtin_amdgcn_ballot_w64(live);
        };
        auto load_k = [&]() {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char *const row = (const char *)a.k_cache + row_off[wave][16 * h + l16];
                kr[h] = load_words<G>(row + 4 * G * c4);
#pragma unroll
                for (int y = 0; y < GQ; ++y) km[h][y] = *(const uint32_t *)(row + 16 * G + 4 * min(4 * y + c4, G - 1));
            }
        };
        auto load_v = [&]() {
#pragma unroll
            for (int e = 0; e < 8; ++e) vr[e] = load_bytes<G>((const char *)a.v_cache + row_off[wave][8 * c4 + e] + G * l16);
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
            // ---- steps and middles of the values to LDS, the steps in units of the largest so far (a
            // step that is no number, or infinite, counts as none: its weights are what they are)
            {
                const bool mine = seen >> (lane & 31) & 1;
                float step[MW], least[MW];
                uint32_t most = 0;
#pragma unroll
                for (int i = 0; i < MW; ++i) {
                    const uint32_t d = mine ? vm[i] : 0u;
                    step[i] = tml_half_bits(d & 0xFFFFu);
                    least[i] = tml_half_bits(d >> 16);
                    const uint32_t bits = __float_as_uint(step[i]) & 0x7F800000u;
                    most = max(most, bits < 0x7F800000u ? bits : 0u);
                }
                if (__builtin_amdgcn_ballot_w64(most > peak) != 0) {
#pragma unroll
                    for (int x = 1; x < 64; x <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, x));
                    const float f = peak == 0u ? 1.0f : __uint_as_float(peak) / __uint_as_float(most);
                    peak = most;
#pragma unroll
                    for (int x = 0; x < HQ; ++x)
#pragma unroll
                        for (int j = 0; j < 2 * G; ++j) o[x][j] *= f;
                }
                // (no step yet: all of them are zero)
                const float in_units = peak == 0u ? 1.0f : __uint_as_float((253u << 23) - peak);  // 2^-1 / the largest's power of two
#pragma unroll
                for (int i = 0; i < MW; ++i) {
                    const int g = (lane >> 5) * MW + i;
                    if (G % 2 == 0 || g < G) marks[wave][g][lane & 31] = srv_f32x2{step[i] * in_units, fmaf(step[i], 8.0f, least[i])};
                }
            }
            // ---- scores: of head 4 x + c4 and tokens 16 h + l16
            float s[HQ][2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                floatx4 sum[HQ][GQ];
#pragma unroll
                for (int x = 0; x < HQ; ++x)
#pragma unroll
                    for (int y = 0; y < GQ; ++y) sum[x][y] = floatx4{0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < G; ++w) {
                    const uint32_t word = kr[h].w[w];
                    const srv_u32x4 n = WIDE ? srv_u32x4{two_nibbles<0>(word, thousands), two_nibbles<4>(word, thousands), two_nibbles<0>(word >> 8, thousands),
                                                         two_nibbles<4>(word >> 8, thousands)}
                                             : nibbles(word);
#pragma unroll
                    for (int x = 0; x < HQ; ++x)
#pragma unroll
                        for (int term = 0; term < NT; ++term) sum[x][w / 4] = mma16<TML_TYPE_F16>(q[x][term][w], n, sum[x][w / 4]);
                }
#pragma unroll
                for (int x = 0; x < HQ; ++x) {
                    float by[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int y = 0; y < GQ; ++y) {
                        const uint32_t d = G % 4 == 0 || 4 * y + c4 < G ? km[h][y] : 0u;
                        const float step = tml_half_bits(d & 0xFFFFu), least = fmaf(step, WIDE ? 8.0f : 0.0f, tml_half_bits(d >> 16));
#pragma unroll
                        for (int i = 0; i < 4; ++i) by[i] = fmaf(sum[x][y][i], step, fmaf(q_sum[x][i][y], least, by[i]));
                    }
                    s[x][h] = sum_and_share(by);
                }
            }
            bool behind = false;
#pragma unroll
            for (int x = 0; x < HQ; ++x)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    if constexpr (FORM) {
                        const float y = s[x][h] * to_score[x], from = (float)(sp.len - 1 - sp.first - ((int64_t)t * kTile + 16 * h + l16));
                        s[x][h] = fmaf(-slope[x], from, (inv_cap != 0.0f ? cap_score(y, a.cap, inv_cap) : y) * kLog2E);
                    } else {
                        s[x][h] *= to_score[x] * kLog2E;
                    }
                    s[x][h] = (seen >> (16 * h + l16) & 1) ? s[x][h] : -INFINITY;
                    behind |= s[x][h] > m[x] + kBehind;
                }
            t += kWaves;
            seen = rows_of(t, block);
            load_k();
            block = block_of(t + kWaves);

            // ---- weights
            if (__builtin_amdgcn_ballot_w64(behind) != 0) {
#pragma unroll
                for (int x = 0; x < HQ; ++x) {
                    float most = fmaxf(s[x][0], s[x][1]);
#pragma unroll
                    for (int i = 1; i < 16; i <<= 1) most = fmaxf(most, __shfl_xor(most, i));
                    const float m_new = fmaxf(m[x], most), f = rescale(m[x], m_new);
                    m[x] = m_new;
                    l[x] *= f;
                    const float column = __shfl(f, 16 * hi);
#pragma unroll
                    for (int j = 0; j < 2 * G; ++j) o[x][j] *= column;
#pragma unroll
                    for (int y = 0; y < GQ; ++y) middle[x][y] *= column;
                }
            }
#pragma unroll
            for (int x = 0; x < HQ; ++x) {
                const float base = (m[x] == -INFINITY ? 0.0f : m[x]) - kUp;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p = __builtin_amdgcn_exp2f(s[x][h] - base);
                    l[x] += p;
                    weights[wave][4 * x + c4][16 * h + l16] = p;
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
            // ---- values
            srv_u32x4 pair[2 * VW];  // 16 bits of tokens 2 i and 2 i + 1
#pragma unroll
            for (int x = 0; x < (G + 1) / 2; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    pair[x][i] = __builtin_amdgcn_perm(vr[2 * i + 1].w[x / 2], vr[2 * i].w[x / 2], x % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int y = 0; y < GQ; ++y) {
                srv_u32x4 weight[HQ][NT];
                srv_f32x2 mark[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) mark[e] = marks[wave][4 * y + gi][8 * c4 + e];
#pragma unroll
                for (int x = 0; x < HQ; ++x) {
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = weights[wave][4 * x + hi][8 * c4 + e];
                        middle[x][y] = fmaf(p[e], mark[e][1], middle[x][y]);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float u = p[2 * i] * mark[2 * i][0], v = p[2 * i + 1] * mark[2 * i + 1][0];
                        uint32_t term[2];
                        if constexpr (WIDE) two_terms(u, v, &term[0], &term[1]);
                        else term[0] = srv_pack_f16(u, v);
#pragma unroll
                        for (int n = 0; n < NT; ++n) weight[x][n][i] = term[n];
                    }
                }
#pragma unroll
                for (int j = 8 * y; j < min(8 * y + 8, 2 * G); ++j) {
                    srv_u32x4 n;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint32_t two = j % 4 >= 2 ? pair[j / 4][i] >> 8 : pair[j / 4][i];
                        n[i] = j % 2 ? two_nibbles<4>(two, thousands) : two_nibbles<0>(two, thousands);
                    }
#pragma unroll
                    for (int x = 0; x < HQ; ++x)
#pragma unroll
                        for (int term = 0; term < NT; ++term) o[x][j] = mma16<TML_TYPE_F16>(n, weight[x][term], o[x][j]);
                }
            }
            load_v();
        }

        // ---- the waves' parts
#pragma unroll
        for (int x = 0; x < HQ; ++x) {
#pragma unroll
            for (int i = 1; i < 16; i <<= 1) l[x] += __shfl_xor(l[x], i);
            if (l16 == 0) {
                wave_m[wave][4 * x + c4] = m[x];
                wave_l[wave][4 * x + c4] = l[x];
            }
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < HQ; ++x) {
            const int head = 4 * x + hi;
            float top = wave_m[0][head];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, wave_m[w][head]);
            const float f = rescale(wave_m[wave][head], top);
            const float up = (peak == 0u ? 0.0f : __uint_as_float(peak) * 2.0f) * f;  // out of the weights' units
#pragma unroll
            for (int y = 0; y < GQ; ++y) {
                float z = middle[x][y];
                z += __shfl_xor(z, 16);
                z += __shfl_xor(z, 32);
                z *= f;
#pragma unroll
                for (int j = 8 * y; j < min(8 * y + 8, 2 * G); ++j) {
                    const float r = j % 2 ? up * 0x1p-4f : up;
                    if (head < gn && gi == j / 2 % 4)
                        *(floatx4 *)(wave_o + (wave * sh.heads + head) * D + 16 * j + 4 * c4) =
                            floatx4{fmaf(o[x][j][0], r, z), fmaf(o[x][j][1], r, z), fmaf(o[x][j][2], r, z), fmaf(o[x][j][3], r, z)};
                }
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

// Query heads taken at once: four, or eight where a group has more and the registers hold two
// workgroups a CU.  32 requests of 2048 tokens, 64 heads on 8, eight / four at once: bf16, dim 128
// 34.5 / 44.4 us, dim 64 27 / 34 us; f32 q, dim 64 30 / 31 us, dim 128 (one workgroup a CU) 44.8 /
// 41.2 us.
constexpr bool eights_fit(int groups, bool wide) { return groups <= (wide ? 2 : 4); }
int heads_at_once(const PagedAttentionArgs &a) {
    return a.q_heads / a.kv_heads > 4 && eights_fit((int)a.head_dim / 32, a.q_type == TML_TYPE_F32) ? 8 : 4;
}
AttnShape shape_of(const PagedAttentionArgs &a) {
    const int heads = heads_at_once(a);
    return shape_of(a, per_cu((int)a.head_dim / 32, heads / 4, a.q_type == TML_TYPE_F32), heads);
}

template <int G, int HQ, bool WIDE, bool FORM>
void launch_kernel(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    const size_t lds = (size_t)kWaves * sh.heads * 32 * G * 4;
    const dim3 grid(sh.grid), block(kThreads);
    paged_attention_q4_kernel<G, HQ, WIDE, FORM><<<grid, block, lds, s>>>(a, sh);
}
template <int G, int HQ>
void launch_form(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    const bool form = a.cap != 0.0f || a.slopes != nullptr;
    if (a.q_type == TML_TYPE_F32) {
        if constexpr (HQ == 1 || eights_fit(G, true)) form ? launch_kernel<G, HQ, true, true>(a, sh, s) : launch_kernel<G, HQ, true, false>(a, sh, s);
    } else form ? launch_kernel<G, HQ, false, true>(a, sh, s) : launch_kernel<G, HQ, false, false>(a, sh, s);
}
template <int G>
void launch_groups(const PagedAttentionArgs &a, const AttnShape &sh, hipStream_t s) {
    if constexpr (eights_fit(G, false)) {
        if (sh.at_once == 8) return launch_form<G, 2>(a, sh, s);
    }
    launch_form<G, 1>(a, sh, s);
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

size_t paged_attention_q4_workspace_floats(const PagedAttentionArgs &a) { return attn_empty(a) ? 0 : split_floats(a, shape_of(a)); }

Status launch_paged_attention_q4(const PagedAttentionArgs &in, const Workspace &ws, hipStream_t s) {
    PagedAttentionArgs a = in;
    if (attn_empty(a)) return Status::Ok();
    if (a.n_blocks == 0) a.table_width = 0;  // no cache: nothing to look at
    AttnShape sh = shape_of(a);
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
