// prompt_attention.hip -- attention of prompts: any number of new tokens a request over
// its paged key-value cache, under causal, windowed and prefix masks, with scores capped
// by a tanh or biased by distance.
//
//   s_t = cap tanh(scale q . k_t / cap) - slope_h |pos - t|
//   out = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m),   m = max_t s_t
//
// over the t that the query at position pos sees: t < len, t <= pos or t < prefix, t >
// pos - window.  4 dim operations a pair seen, so the matrix cores bound all but the
// shortest prompts, and beside them the exponentials.
//
// A workgroup takes 128 rows of a request and a key-value head, a row being a query head
// of the group at a token: row r is token r / group, head r % group, so short prompts
// with grouped heads fill the matrix instructions and share each key.  Its four waves
// have 32 rows each and go through the tiles of tokens that any of the rows sees, with a
// running maximum and sum; keys and values of a tile are in LDS, those of the next on
// their way to registers.
//   scores   S^T = K Q^T, 32 tokens x 32 rows: a lane holds sixteen tokens of one row, so a
//            row's maximum and sum need one exchange between two lanes
//   weights  are the B operand of the next product as they lie if its k slots are numbered
//            as the lane's tokens are: 8 j + 4 (lane / 32) + i
//   values   O^T += V^T P^T: V goes to LDS transposed, its tokens in that order
// 16-byte pieces of a row in LDS are exchanged by the row's number, so that lanes that
// read the same piece of different rows use all banks.
//
// Precision: sums, maxima and the scores are fp32.  f32 queries go in as terms of the
// cache's type (two of f16, scaled by a power of two, three of bf16), and so do the
// weights where the output is f32; where it has 16 bits the weights are rounded to them
// once, which adds to an output about what its own rounding does (2^-8 of bf16, 2^-11 of f16,
// at most).
// An f32 cache runs on the fp32 matrix cores.
#include "terms.hpp"

#include <algorithm>

namespace tml {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4, kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // of a workgroup

struct PromptShape {
    int group;          // query heads of a key-value head
    int64_t positions;  // of a table row
    unsigned tiles;     // of rows, at most, over the batch
};

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// 32 rows, 32 columns, k of 16.
template <int CT>
__device__ __forceinline__ floatx16 mma32(const srv_u32x4 &x, const srv_u32x4 &y, floatx16 c) {
    if constexpr (CT == TML_TYPE_F16)
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(halfx8, x), __builtin_bit_cast(halfx8, y), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0, 0);
}

// New tokens of request r: their first row of q, and how many (not past q's end).
struct Request {
    int first, count;
};
__device__ __forceinline__ Request request_at(const PromptAttentionArgs &a, int64_t r) {
    const int first = max(a.query_start[r], 0);
    return {first, (int)max(min((int64_t)a.query_start[r + 1], a.tokens) - first, (int64_t)0)};
}
__device__ __forceinline__ int64_t tiles_of(const PromptShape &sh, int count) { return ((int64_t)count * sh.group + kRows - 1) / kRows; }

// Where piece `piece` of row `row` lies among the row's N pieces of 16 bytes (N a power of
// two): 16 rows of neighbouring lanes meet each bank once.
template <int N>
__device__ __forceinline__ int placed(int row, int piece) {
    if constexpr (N >= 16) return piece ^ (row & 15);
    else if constexpr (N == 8) return piece ^ ((row ^ row >> 3) & 7);
    else return piece ^ (row >> 2 & 3);
}

// CT: the cache's type.  QT: q's and the output's (CT or f32).  DP: the head size rounded
// up to 64, 128 or 256.  FORM: the scores are capped or biased.
template <int CT, int QT, int DP, bool FORM>
struct Prompt {
    static constexpr bool kF32 = CT == TML_TYPE_F32;
    static constexpr int kBytes = kF32 ? 4 : 2;
    static constexpr int E = 16 / kBytes;                       // elements of a piece
    static constexpr int NQ = QT == CT ? 1 : CT == TML_TYPE_F16 ? 2 : 3;
    static constexpr int NP = QT == CT ? 1 : CT == TML_TYPE_F16 ? 2 : 3;
    static constexpr int BN = kF32 || DP == 256 ? 32 : 64;       // tokens of a tile
    static constexpr int KP = DP / E, VP = BN / E;               // pieces of a row of K, of V^T
    static constexpr int kLoadsK = BN * KP / kThreads;           // pieces a thread moves
    static constexpr int kItems = BN / 4 * KP;                   // V: four tokens of a piece each
    static constexpr int kLoadsV = (kItems + kThreads - 1) / kThreads;
    static constexpr int kQ = kF32 ? DP / 8 : DP / 16;           // 16 bytes of q a lane, each term
    // registers of a lane: q, output, scores, tiles under way; two workgroups a CU where they fit half
    static constexpr int kRegs = 4 * kQ * NQ + DP / 2 + BN / 2 + 4 * kLoadsK + 16 * kLoadsV + 16 * NP;
    static constexpr int kPerCu = kRegs > 190 ? 1 : 2;
};

template <int CT, int QT, int DP, bool FORM>
__global__ __launch_bounds__(kThreads, (Prompt<CT, QT, DP, FORM>::kPerCu)) void prompt_attention_kernel(PromptAttentionArgs a, PromptShape sh) {
    using C = Prompt<CT, QT, DP, FORM>;
    constexpr bool kF32 = C::kF32;
    constexpr int kBytes = C::kBytes, E = C::E, NQ = C::NQ, NP = C::NP, BN = C::BN, KP = C::KP, VP = C::VP, kQ = C::kQ;
    // base of the weights' exponent: f16 terms of e^(s - m) reach down to 2^-39 of the largest
    constexpr float kUp = CT == TML_TYPE_F16 ? 14.0f : 0.0f;

    __shared__ srv_u32x4 lds_k[BN * KP], lds_v[DP * VP];
    __shared__ int64_t row_off[kWaves][BN];
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int l32 = lane & 31, half = lane >> 5;
    const int D = (int)a.head_dim;
    const int64_t P = a.block_size;

    // ---- which rows: the key-value head first, so that the workgroups of one are on one
    // XCD; the batch's last tiles, which see the most, first
    const unsigned kv = blockIdx.x % (unsigned)a.kv_heads, index = blockIdx.x / (unsigned)a.kv_heads;
    const int64_t strip = (a.requests + 63) / 64;
    int64_t upto = 0;
    for (int64_t r = lane * strip; r < min((lane + 1) * strip, a.requests); ++r) upto += tiles_of(sh, request_at(a, r).count);
    const int64_t own = upto;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int lo = __shfl_up((int)(uint32_t)upto, o), hi = __shfl_up((int)(upto >> 32), o);
        if (lane >= o) upto += (int64_t)(((uint64_t)(uint32_t)hi << 32) | (uint32_t)lo);
    }
    // (requests that overlap could have more tiles than the grid)
    const int total = uniform(__shfl((int)min(upto, (int64_t)sh.tiles), 63));
    if (index >= (unsigned)total) return;
    int rem = total - 1 - (int)index;
    const int at_lane = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > rem));
    rem -= uniform(__shfl((int)(upto - own), at_lane));
    int64_t b = at_lane * strip;
    Request request = request_at(a, b);
    while (rem >= tiles_of(sh, request.count)) {
        rem -= (int)tiles_of(sh, request.count);
        request = request_at(a, ++b);
    }
    const int first = uniform(request.first), count = uniform(request.count);
    const int64_t row0 = (int64_t)uniform(rem) * kRows, rows = (int64_t)count * sh.group;
    const int64_t len = min((int64_t)max(uniform(a.seq_len[b]), 0), sh.positions);
    const int64_t prefix = a.prefix_len != nullptr ? min((int64_t)max(uniform(a.prefix_len[b]), 0), len) : 0;
    const int64_t ctx = len - count;  // position of the first new token
    // what a row sees: [low, high)
    auto low_of = [&](int64_t pos) { return a.window > 0 ? max(pos - a.window + 1, (int64_t)0) : (int64_t)0; };
    auto high_of = [&](int64_t pos) { return min(max(pos + 1, prefix), len); };
    const unsigned group = (unsigned)sh.group;
    auto token_of = [&](int64_t row) { return rows >> 32 == 0 ? (int64_t)((uint32_t)row / group) : row / group; };
    const int64_t block_first = ctx + token_of(row0), block_last = ctx + token_of(min(row0 + kRows, rows) - 1);
    const int64_t begin = low_of(block_first), end = high_of(block_last);
    // this wave's rows, and this lane's (past the last: it again)
    const int64_t wave0 = min(row0 + 32 * wave, rows - 1);
    const int64_t wave_first = ctx + token_of(wave0), wave_last = ctx + token_of(min(wave0 + 31, rows - 1));
    const int64_t row = min(row0 + 32 * wave + l32, rows - 1);
    const int64_t token = token_of(row), head = (int64_t)kv * sh.group + (row - token * sh.group);
    const int64_t pos = ctx + token, low = low_of(pos), high = high_of(pos);

    // ---- q: lane (row, half) has the k of its half
    srv_u32x4 q[NQ][kQ];
    float to_score = a.scale;
    {
        const int64_t at = (first + token) * a.q_stride + head * D;
        if constexpr (kF32) {
#pragma unroll
            for (int c = 0; c < kQ; ++c) {
                const int d = 8 * c + 4 * half;
                q[0][c] = srv_u32x4{0, 0, 0, 0};
                if (d < D) q[0][c] = *(const srv_u32x4_any *)((const float *)a.q + at + d);
            }
        } else if constexpr (NQ == 1) {
#pragma unroll
            for (int c = 0; c < kQ; ++c) {
                const int d = 16 * c + 8 * half;
                q[0][c] = srv_u32x4{0, 0, 0, 0};
                if (d < D) q[0][c] = srv_load8<CT>(a.q, at + d).d[0];
            }
        } else {
            float up = 1.0f;
            if constexpr (CT == TML_TYPE_F16) {  // f16's range is short: the largest goes to [2^14, 2^15)
                uint32_t most = 27u << 23;
#pragma unroll
                for (int c = 0; c < kQ; ++c) {
                    const int d = 16 * c + 8 * half;
                    float v[8] = {};
                    if (d < D) srv_floats<QT>(srv_load8<QT>(a.q, at + d), v);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint32_t x = __float_as_uint(v[e]) & 0x7F800000u;
                        most = max(most, x < 0x7F800000u ? x : 0u);
                    }
                }
                most = max(most, (uint32_t)__shfl_xor((int)most, 32));
                up = __uint_as_float((268u << 23) - most);
                to_score *= __uint_as_float(most - (14u << 23));
            }
#pragma unroll
            for (int c = 0; c < kQ; ++c) {
                const int d = 16 * c + 8 * half;
                float v[8] = {};
                if (d < D) srv_floats<QT>(srv_load8<QT>(a.q, at + d), v);
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] *= up;
                srv_u32x4 t[NQ];
                to_terms<CT, NQ>(v, t);
#pragma unroll
                for (int n = 0; n < NQ; ++n) q[n][c] = t[n];
            }
        }
    }
    const float to_log2 = to_score * kLog2E;
    float slope = 0.0f, inv_cap = 0.0f;
    if constexpr (FORM) {
        if (a.slopes != nullptr) slope = a.slopes[head] * kLog2E;
        if (a.cap != 0.0f) inv_cap = 1.0f / a.cap;
    }

    float m = -INFINITY, l = 0.0f;  // of this lane's row; l over this lane's tokens alone
    floatx16 o[DP / 32];            // lane (row, half): d = 32 t + 8 j + 4 half + i
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

    // ---- the tiles' rows: lane % BN looks up a token's
    auto block_of = [&](int64_t k0) {
        const int64_t tok = k0 + lane % BN;
        return a.block_table[b * a.table_stride + (uint32_t)min(tok, len - 1) / (uint32_t)P];
    };
    auto rows_of = [&](int64_t k0, int in_block) {
        const int64_t tok = k0 + lane % BN;
        const bool live = tok < end && in_block >= 0 && in_block < a.n_blocks;
        // (a token no one may look at reads the cache's first row)
        const int64_t off = live ? (in_block * a.block_stride + (int64_t)((uint32_t)tok % (uint32_t)P) * a.token_stride + kv * a.head_stride) * kBytes : 0;
        row_off[wave][lane % BN] = off;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        return __builtin_amdgcn_ballot_w64(live);
    };
    srv_u32x4 kr[C::kLoadsK], vr[C::kLoadsV][4];
    auto load_tile = [&]() {
#pragma unroll
        for (int i = 0; i < C::kLoadsK; ++i) {
            const int at = i * kThreads + (int)threadIdx.x, tok = at / KP, d = at % KP * E;
            kr[i] = *(const srv_u32x4 *)((const char *)a.k_cache + row_off[wave][tok] + (d < D ? d : 0) * kBytes);
        }
#pragma unroll
        for (int i = 0; i < C::kLoadsV; ++i) {
            const int at = min(i * kThreads + (int)threadIdx.x, C::kItems - 1), d = at % KP * E;
#pragma unroll
            for (int j = 0; j < 4; ++j) vr[i][j] = *(const srv_u32x4 *)((const char *)a.v_cache + row_off[wave][at / KP * 4 + j] + (d < D ? d : 0) * kBytes);
        }
    };
    // To LDS: past the head size zeros (what is there may be infinite), and zeros for values no one may look at.
    auto store_tile = [&](uint64_t live) {
#pragma unroll
        for (int i = 0; i < C::kLoadsK; ++i) {
            const int at = i * kThreads + (int)threadIdx.x, tok = at / KP, piece = at % KP;
            if (D < DP && piece * E >= D) kr[i] = srv_u32x4{0, 0, 0, 0};
            lds_k[tok * KP + placed<KP>(tok, piece)] = kr[i];
        }
#pragma unroll
        for (int i = 0; i < C::kLoadsV; ++i) {
            const int at = i * kThreads + (int)threadIdx.x, quad = at / KP, d0 = at % KP * E;
            if (C::kItems % kThreads != 0 && at >= C::kItems) break;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if ((live >> (4 * quad + j) & 1) == 0) vr[i][j] = srv_u32x4{0, 0, 0, 0};
            if constexpr (kF32) {  // a piece is four tokens
#pragma unroll
                for (int e = 0; e < 4; ++e) lds_v[(d0 + e) * VP + placed<VP>(d0 + e, quad)] = srv_u32x4{vr[i][0][e], vr[i][1][e], vr[i][2][e], vr[i][3][e]};
            } else {  // a piece is four tokens and the four eight further on: quads 0 2 1 3 of sixteen tokens
                const int spot = (quad & ~3) + ((quad & 1) << 1 | (quad >> 1 & 1));
                srv_u32x2 *const to = (srv_u32x2 *)lds_v + (spot & 1);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t sel = e % 2 ? 0x07060302u : 0x05040100u;
                    to[2 * ((d0 + e) * VP + placed<VP>(d0 + e, spot >> 1))] =
                        srv_u32x2{__builtin_amdgcn_perm(vr[i][1][e / 2], vr[i][0][e / 2], sel), __builtin_amdgcn_perm(vr[i][3][e / 2], vr[i][2][e / 2], sel)};
                }
            }
        }
    };

    if (begin < end) {
        uint64_t live = rows_of(begin, block_of(begin));
        load_tile();
        int next_block = block_of(begin + BN);
        for (int64_t k0 = begin; k0 < end; k0 += BN) {
            __syncthreads();  // the last tile was read
            store_tile(live);
            const uint64_t live_now = live;
            __syncthreads();
            if (k0 + BN < end) {
                live = rows_of(k0 + BN, next_block);
                load_tile();
                next_block = block_of(k0 + 2 * BN);
            }
            // rows of this wave that see none of the tile, or all of it
            if (k0 >= high_of(wave_last) || k0 + BN <= low_of(wave_first)) continue;
            const bool whole = k0 + BN <= high_of(wave_first) && k0 >= low_of(wave_last) && (live_now & (~0ull >> (64 - BN))) == ~0ull >> (64 - BN);

            // ---- scores
            float s[BN / 2];
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                floatx16 sum;
#pragma unroll
                for (int i = 0; i < 16; ++i) sum[i] = 0.0f;
#pragma unroll
                for (int c = 0; c < kQ; ++c) {
                    const int tok = 32 * u + l32;
                    const srv_u32x4 k = lds_k[tok * KP + placed<KP>(tok, 2 * c + half)];
                    if constexpr (kF32) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) sum = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[e]), __uint_as_float(q[0][c][e]), sum, 0, 0, 0);
                    } else {
#pragma unroll
                        for (int n = 0; n < NQ; ++n) sum = mma32<CT>(k, q[n][c], sum);
                    }
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if constexpr (FORM) {
                        const float x = sum[i] * to_score;
                        const int64_t away = pos - (k0 + 32 * u + 8 * (i / 4) + 4 * half + i % 4);
                        s[16 * u + i] = (inv_cap != 0.0f ? cap_score(x, a.cap, inv_cap) : x) * kLog2E - slope * fabsf((float)away);
                    } else {
                        s[16 * u + i] = sum[i] * to_log2;
                    }
                }
            }
            if (!whole) {
                const int from = (int)max(min(low - k0, (int64_t)BN), (int64_t)0), to = (int)max(min(high - k0, (int64_t)BN), (int64_t)0);
#pragma unroll
                for (int i = 0; i < BN / 2; ++i) {
                    const int t = 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * half + i % 4;
                    if (t < from || t >= to || (live_now >> t & 1) == 0) s[i] = -INFINITY;
                }
            }
            // ---- weights
            float most = s[0];
#pragma unroll
            for (int i = 1; i < BN / 2; ++i) most = fmaxf(most, s[i]);
            most = fmaxf(most, __shfl_xor(most, 32));
            if (__builtin_amdgcn_ballot_w64(most > m) != 0) {
                const float m_new = fmaxf(m, most);
                const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
                m = m_new;
                l *= f;
#pragma unroll
                for (int t = 0; t < DP / 32; ++t)
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[t][i] *= f;
            }
            const float base = (m == -INFINITY ? 0.0f : m) - kUp;
#pragma unroll
            for (int i = 0; i < BN / 2; ++i) {
                s[i] = __builtin_amdgcn_exp2f(s[i] - base);
                l += s[i];
            }
            // ---- values
            if constexpr (kF32) {
#pragma unroll
                for (int j = 0; j < BN / 8; ++j)
#pragma unroll
                    for (int t = 0; t < DP / 32; ++t) {
                        const int d = 32 * t + l32;
                        const srv_u32x4 v = lds_v[d * VP + placed<VP>(d, 2 * j + half)];
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v[i]), s[4 * j + i], o[t], 0, 0, 0);
                    }
            } else {
#pragma unroll
                for (int j = 0; j < BN / 16; ++j) {
                    float p[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) p[e] = s[8 * j + e];
                    srv_u32x4 w[NP];
                    to_terms<CT, NP>(p, w);
#pragma unroll
                    for (int t = 0; t < DP / 32; ++t) {
                        const int d = 32 * t + l32;
                        const srv_u32x4 v = lds_v[d * VP + placed<VP>(d, 2 * j + half)];
#pragma unroll
                        for (int n = 0; n < NP; ++n) o[t] = mma32<CT>(v, w[n], o[t]);
                    }
                }
            }
        }
    }

    l += __shfl_xor(l, 32);
    if (row0 + 32 * wave + l32 >= rows) return;
    const float r = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t at = (first + token) * a.out_stride + head * D;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * t + 8 * j + 4 * half;
            if (d >= D) continue;
            const float x0 = o[t][4 * j] * r, x1 = o[t][4 * j + 1] * r, x2 = o[t][4 * j + 2] * r, x3 = o[t][4 * j + 3] * r;
            if constexpr (QT == TML_TYPE_F32) {
                *(srv_u32x4_any *)((float *)a.out + at + d) = srv_u32x4{__float_as_uint(x0), __float_as_uint(x1), __float_as_uint(x2), __float_as_uint(x3)};
            } else {
                *(srv_u32x2_any *)((uint16_t *)a.out + at + d) =
                    QT == TML_TYPE_F16 ? srv_u32x2{srv_pack_f16(x0, x1), srv_pack_f16(x2, x3)} : srv_u32x2{srv_pack_bf16(x0, x1), srv_pack_bf16(x2, x3)};
            }
        }
}

template <int CT, int QT, bool FORM>
void launch_dim(const PromptAttentionArgs &a, const PromptShape &sh, hipStream_t s) {
    const dim3 grid((unsigned)(sh.tiles * (unsigned)a.kv_heads)), block(kThreads);
    if (a.head_dim <= 64) prompt_attention_kernel<CT, QT, 64, FORM><<<grid, block, 0, s>>>(a, sh);
    else if (a.head_dim <= 128) prompt_attention_kernel<CT, QT, 128, FORM><<<grid, block, 0, s>>>(a, sh);
    else prompt_attention_kernel<CT, QT, 256, FORM><<<grid, block, 0, s>>>(a, sh);
}
template <int CT, int QT>
void launch_form(const PromptAttentionArgs &a, const PromptShape &sh, hipStream_t s) {
    if (a.cap != 0.0f || a.slopes != nullptr) launch_dim<CT, QT, true>(a, sh, s);
    else launch_dim<CT, QT, false>(a, sh, s);
}

}  // namespace

Status launch_prompt_attention(const PromptAttentionArgs &in, hipStream_t s) {
    PromptAttentionArgs a = in;
    if (!float_type(a.cache_type) || (a.q_type != a.cache_type && a.q_type != TML_TYPE_F32))
        return Status::Err(TML_ERR_INVALID_FORMAT, "prompt attention: the cache is f32, f16 or bf16, q the same or f32");
    if (a.tokens < 0 || a.requests < 0 || a.q_heads < 0 || a.kv_heads < 0 || a.head_dim < 0 || a.n_blocks < 0 || a.table_width < 0 || a.window < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: negative size");
    if (a.block_size < 1) return Status::Err(TML_ERR_INVALID_ARG, "prompt attention: the block size must be positive");
    if (!valid_cap(a.cap)) return Status::Err(TML_ERR_INVALID_ARG, "prompt attention: the cap must be 0 or from 2^-100 to 2^100");
    if (a.tokens == 0 || a.requests == 0 || a.q_heads == 0 || a.kv_heads == 0 || a.head_dim == 0) return Status::Ok();
    if (a.q_heads % a.kv_heads != 0)
        return Status::Err(TML_ERR_SHAPE_MISMATCH, "prompt attention: query heads are no multiple of key-value heads");
    if (a.head_dim % 8 != 0 || a.head_dim > 256)
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: the head size must be a multiple of 8, at most 256");
    const int64_t most = (int64_t)1 << 31;
    if (a.n_blocks >= most || a.block_size >= most || a.requests >= (1 << 16) || a.q_heads >= (1 << 16) || a.tokens >= (1 << 24) ||
        a.table_width >= most || a.table_width * a.block_size > most)
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: requests and heads must be below 2^16, tokens below 2^24, a table's positions at most 2^31");
    if (a.q == nullptr || a.out == nullptr || a.query_start == nullptr || a.seq_len == nullptr ||
        (a.n_blocks > 0 && (a.k_cache == nullptr || a.v_cache == nullptr)) || (a.table_width > 0 && a.block_table == nullptr))
        return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    if (a.tokens > 1 && (a.q_stride < a.q_heads * a.head_dim || a.out_stride < a.q_heads * a.head_dim))
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: a row stride is shorter than the row");
    if (a.requests > 1 && a.table_stride < a.table_width)
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: a row stride is shorter than the row");
    if (a.block_stride < 0 || a.token_stride < 0 || a.head_stride < 0)
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: negative cache stride");
    const int64_t bytes = type_bytes(a.cache_type);
    if (((uintptr_t)a.k_cache | (uintptr_t)a.v_cache | (uintptr_t)(a.block_stride * bytes) | (uintptr_t)(a.token_stride * bytes) |
         (uintptr_t)(a.head_stride * bytes)) % 16 != 0)
        return Status::Err(TML_ERR_INVALID_ARG, "prompt attention: the cache's rows must start on 16-byte boundaries");
    if (a.n_blocks == 0) a.table_width = 0;  // no cache: nothing to look at
    PromptShape sh;
    sh.group = (int)(a.q_heads / a.kv_heads);
    sh.positions = a.table_width * a.block_size;
    const int64_t tiles = a.tokens * sh.group / kRows + std::min(a.requests, a.tokens);
    if (tiles * a.kv_heads > (1 << 23))
        return Status::Err(TML_ERR_INVALID_SHAPE, "prompt attention: tokens * heads / 128 + requests * key-value heads must be at most 2^23");
    sh.tiles = (unsigned)tiles;
    if (a.cache_type == TML_TYPE_F32) launch_form<TML_TYPE_F32, TML_TYPE_F32>(a, sh, s);
    else if (a.cache_type == TML_TYPE_F16) a.q_type == TML_TYPE_F32 ? launch_form<TML_TYPE_F16, TML_TYPE_F32>(a, sh, s) : launch_form<TML_TYPE_F16, TML_TYPE_F16>(a, sh, s);
    else a.q_type == TML_TYPE_F32 ? launch_form<TML_TYPE_BF16, TML_TYPE_F32>(a, sh, s) : launch_form<TML_TYPE_BF16, TML_TYPE_BF16>(a, sh, s);
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

}  // namespace tml
