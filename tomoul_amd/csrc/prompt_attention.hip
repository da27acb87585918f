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
// running maximum and sum.  Keys and values are copied straight to LDS, the next tile's
// while this one is multiplied; one barrier a tile.
//   scores   S^T = K Q^T, 32 tokens x 32 rows: a lane holds sixteen tokens of one row, so a
//            row's maximum and sum need one exchange between two lanes
//   weights  are the B operand of the next product as they lie if its k slots are numbered
//            as the lane's tokens are: 8 j + 4 (lane / 32) + i
//   values   O^T += V^T P^T: the LDS reads that transpose 4 x 16 blocks give a lane four
//            tokens of its d
// 16-byte pieces of a row in LDS are exchanged by the token's number, so that neither the
// reads of one piece of 16 rows (keys) nor those of 64 bytes of four rows (values) meet in a
// bank.
// Precision: sums, maxima and the scores are fp32.  f32 queries go in as terms of the
// cache's type (two of f16, scaled by a power of two, three of bf16; see to_query_terms), and so do the
// weights where the output is f32; where it has 16 bits the weights are rounded to them
// once, which adds to an output about what its own rounding does (2^-8 of bf16, 2^-11 of f16,
// at most).
// An f32 cache runs on the fp32 matrix cores.
//
// Measured on MI355X (launches in a graph): bf16, two causal prompts of 6000 to 8192 tokens, 32
// heads on 8 of 128, 0.94 ms, 867 TFLOP/s of the pairs seen (a library product reaches 1130);
// 1500 frames, 20 heads of 64, f16, 28 to 32 us; sixteen chunks of 1 to 256 tokens over contexts to 4096,
// capped, 160 to 165 us.  The first is bound by issue: without the exponentials it took 918, without the
// second product 722, without the copies 713 of then 970 us, so a SIMD's two waves hardly overlap
// their products with each other's exponentials.  The others are bound by their longest workgroups (66 tiles of
// 2.5 us): a request's tokens are not split.
#include "terms.hpp"

#include <algorithm>

namespace tml {
namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4;           // of a team: 32 rows each
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

typedef short shortx4 __attribute__((ext_vector_type(4)));
#define TML_GPTR(p) ((__attribute__((address_space(1))) void *)(p))
#define TML_LPTR(p) ((__attribute__((address_space(3))) void *)(p))
// Lane i of a group of 16 reads four numbers, row i / 4 and columns 4 (i % 4) and on of a block
// of 4 x 16; it gets the four rows of column i.
__device__ __forceinline__ shortx4 read_turned(const shortx4 *p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) shortx4 *)p);
}

// A value that the compiler takes to be new here: what is made of it is made anew in every
// tile instead of being kept in registers.
__device__ __forceinline__ int anew(int v) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("" : "+v"(v));
#endif
    return v;
}

// The larger of a lane's and the lane's 32 away.
__device__ __forceinline__ float max_of_halves(float v) {
    const auto two = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(two[0]), __uint_as_float(two[1]));
}

// f32 elements of q (f16: below 2^15) in N terms of type CT.  All but the last are cut off strictly
// below what is left, so each term of an element that is not 0 has its sign and is not 0 itself:
// an infinite key is infinite with all of them alike, where a later term of 0 or of the other sign
// would make a NaN of the sum.  The terms are off by 2^-22 of the element and 2^-22 (two of f16), or by
// 2^-100 (three of bf16: 8 bits, the next 8, and 1 to 256 units of the last place).
template <int CT, int N>
__device__ __forceinline__ void to_query_terms(const float (&v)[8], srv_u32x4 (&t)[N]) {
    constexpr bool kF16 = CT == TML_TYPE_F16;
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        float terms[2][N];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float x = v[e + i];
            const bool itself = __builtin_isfpclass(x, 0x267);  // zeros, infinities, NaNs
            float left = __builtin_copysignf(fmaxf(fabsf(x), kF16 ? 0x1p-23f : 0x1p-100f), x);
#pragma unroll
            for (int n = 0; n < N; ++n) {
                float term = left;
                if (n + 1 < N) term = __uint_as_float((__float_as_uint(left) - 1) & (kF16 ? 0xFFFFE000u : 0xFFFF0000u));
                else if (kF16) term = __builtin_copysignf(fmaxf(fabsf(left), 0x1p-24f), x);
                terms[i][n] = itself ? x : term;
                left -= term;
            }
        }
#pragma unroll
        for (int n = 0; n < N; ++n) t[n][e / 2] = kF16 ? srv_pack_f16(terms[0][n], terms[1][n]) : srv_pack_bf16(terms[0][n], terms[1][n]);
    }
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

// What a token's pieces of 16 bytes are exchanged by in LDS, N of them a row: piece p is in
// place p ^ this.
template <int N>
__device__ __forceinline__ int turn_of(int token) {
    return N >= 16 ? (token & 3) << 2 | (token >> 2 & 3) : (token >> 1 & 1) << 2 | (token >> 2 & 3);
}

// Where a token's key and value are.
struct alignas(16) RowAt {
    const char *k, *v;
};

// Read in the place of what no one may look at, and of what is past the head size.
__device__ srv_u32x4 zero_row[64];

// CT: the cache's type.  QT: q's and the output's (CT or f32).  DP: the head size rounded
// up to 64, 128 or 256.  FORM: the scores are capped or biased.
template <int CT, int QT, int DP, bool FORM>
struct Prompt {
    static constexpr bool kF32 = CT == TML_TYPE_F32;
    static constexpr int kBytes = kF32 ? 4 : 2;
    static constexpr int NQ = QT == CT ? 1 : CT == TML_TYPE_F16 ? 2 : 3;
    static constexpr int NP = QT == CT ? 1 : CT == TML_TYPE_F16 ? 2 : 3;
    static constexpr int BN = kF32 || DP == 256 ? 32 : 64;  // tokens of a tile
    static constexpr int KP = DP * kBytes / 16;              // pieces of a token's row
    static constexpr int kOwn = BN / kWaves;                 // tokens that a wave copies
    static constexpr int kCopies = kOwn * KP / 64;
    static constexpr int kQ = kF32 ? DP / 8 : DP / 16;       // 16 bytes of q a lane, each term
    // Two workgroups a CU, two waves of a SIMD, or one with all of the registers.  Two / one, two causal
    // prompts of 4096 tokens: bf16, 32 heads on 8 of 128 399 / 539 us; f32 q on f16 597 / 834, on
    // bf16 840 / 971; 16 heads on 8 of 256, bf16 653 / 504; f32 cache, 2048 tokens, 16 on 8 of 128
    // 657 / 448, 20 of 64 335 / 322.
    static constexpr bool kTwo = !kF32 && DP <= 128;
    static constexpr int kTile = BN * KP;                    // pieces of a tile's keys
};

// Until at most N of this wave's copies are under way.
template <int N>
__device__ __forceinline__ void wait_copies() {
    __builtin_amdgcn_s_waitcnt((N & 0xF) | ((N >> 4) << 14) | 0x7 << 4 | 0xF << 8);
}

// TEAMS: of four waves with the same rows each, which share the tiles.
template <int CT, int QT, int DP, bool FORM, int TEAMS>
__global__ __launch_bounds__(64 * kWaves * TEAMS, (Prompt<CT, QT, DP, FORM>::kTwo && TEAMS == 1 ? 2 : 1)) void prompt_attention_kernel(PromptAttentionArgs a, PromptShape sh) {
    using C = Prompt<CT, QT, DP, FORM>;
    constexpr bool kF32 = C::kF32;
    constexpr int kBytes = C::kBytes, NQ = C::NQ, NP = C::NP, BN = C::BN, KP = C::KP, kQ = C::kQ, kOwn = C::kOwn;
    // The maximum that weights are relative to may fall behind the row's by kBehind (in
    // powers of two) before sums are scaled: with 32 rows one of them rises in most tiles.
    // kUp: base of the weights' exponent, for f16's range; terms of them reach down to 2^-39
    // (f32 outputs) or 2^-24 (one term, and the maximum behind) of the largest.
    constexpr float kBehind = QT == TML_TYPE_F32 ? 0.0f : 8.0f;
    constexpr float kUp = CT != TML_TYPE_F16 ? 0.0f : QT == TML_TYPE_F32 ? 14.0f : 7.0f;
    // A cap as cap - 2 cap / (1 + e^(2 x / cap)) is up to 12 2^-24 of the CAP off, whatever x is, and
    // as much of a weight.  It is for 16-bit weights and caps up to this, where that is a tenth of what
    // the weights' rounding is off; past it the cap is cap_score's (two f16 prompts of 4096 tokens, 32 heads
    // on 8 of 128: 439 us up to this, 530 past it).
    constexpr float kShortCap = QT == TML_TYPE_F32 ? 0.0f : QT == TML_TYPE_F16 ? 64.0f : 512.0f;

    // (arrays of their own: the compiler waits for copies to the array that it reads)
    __shared__ srv_u32x4 lds_k0[TEAMS * C::kTile], lds_k1[TEAMS * C::kTile], lds_v0[TEAMS * C::kTile], lds_v1[TEAMS * C::kTile];
    __shared__ RowAt row_at[2][TEAMS * kWaves][kOwn];
    __shared__ uint64_t lds_live[2][TEAMS];  // of a tile's tokens
    __shared__ int lds_odd;                  // infinities or NaNs were cleared
    const int lane = threadIdx.x & 63, any_wave = uniform((int)(threadIdx.x >> 6)), wave = any_wave % kWaves, team = any_wave / kWaves;
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
    const int pos = (int)(ctx + token);
    const uint32_t low = (uint32_t)low_of(pos), high = (uint32_t)max(high_of(pos), (int64_t)0);  // (at most 2^31)

    // ---- q: lane (row, half) has the k of its half
    // (with the scale's sign, for maxima to be taken before the scale; a scale of 0 is a q of 0)
    srv_u32x4 q[NQ][kQ];
    float to_score = a.scale == 0.0f ? 1.0f : fabsf(a.scale);
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
                to_query_terms<CT, NQ>(v, t);
#pragma unroll
                for (int n = 0; n < NQ; ++n) q[n][c] = t[n];
            }
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int c = 0; c < kQ; ++c) {
            if (a.scale < 0.0f) q[n][c] ^= kF32 ? 0x80000000u : 0x80008000u;
            if (a.scale == 0.0f) q[n][c] = srv_u32x4{0, 0, 0, 0};
        }
    const float to_log2 = to_score * kLog2E;
    float slope = 0.0f, inv_cap = 0.0f, short_cap = 0.0f;
    if constexpr (FORM) {
        if (a.slopes != nullptr) slope = a.slopes[head] * kLog2E;
        if (a.cap != 0.0f) inv_cap = 1.0f / a.cap;
        if (a.cap <= kShortCap) short_cap = 2.0f * to_log2 * inv_cap;  // (16 bits: of the scale and the cap alone)
    }

    float m = -INFINITY, l = 0.0f;  // of this lane's row; l over this lane's tokens alone
    floatx16 o[DP / 32];            // lane (row, half): d = 32 t + 8 j + 4 half + i
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;

    const char *const zeros_at = (const char *)zero_row;
    // ---- the team's tile `it` is tokens tile_at(it) and on
    const int steps = (int)((max(end - begin, (int64_t)0) + BN * TEAMS - 1) / (BN * TEAMS));
    auto tile_at = [&](int it) { return begin + (int64_t)(TEAMS * it + team) * BN; };
    // copies: a wave's tokens are its share of the tile, lane % kOwn looks one up
    auto block_of = [&](int it) {
        const int64_t tok = tile_at(it) + wave * kOwn + lane % kOwn;
        return a.block_table[b * a.table_stride + (uint32_t)min(tok, len - 1) / (uint32_t)P];
    };
    auto find_rows = [&](int it, int in_block) __attribute__((always_inline)) {
        const int64_t tok = tile_at(it) + wave * kOwn + lane % kOwn;
        const bool live = tok < end && in_block >= 0 && in_block < a.n_blocks;
        const int64_t off = (in_block * a.block_stride + (int64_t)((uint32_t)tok % (uint32_t)P) * a.token_stride + kv * a.head_stride) * kBytes;
        row_at[it & 1][any_wave][lane % kOwn] =
            live ? RowAt{(const char *)a.k_cache + off, (const char *)a.v_cache + off} : RowAt{zeros_at, zeros_at};
        const uint64_t all = __builtin_amdgcn_ballot_w64(live);
        if (lane == 0) {
            if constexpr (kOwn == 16) ((uint16_t *)&lds_live[it & 1][team])[wave] = (uint16_t)all;
            else ((uint8_t *)&lds_live[it & 1][team])[wave] = (uint8_t)all;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    };
    // Copy i is of 64 / KP tokens, a lane a piece: the turn of a token's number is that of its bits
    // one by one, so the pieces of copy i are those of copy 0 turned on.
    constexpr int kAtOnce = 64 / KP;
    const uint32_t first_piece = ((uint32_t)lane % KP ^ turn_of<KP>((uint32_t)lane / KP)) * 16;
    struct Sources {
        const char *at[C::kCopies];
    };
    auto sources_of = [&](const RowAt (&rows_here)[kOwn], bool values) __attribute__((always_inline)) {
        Sources from;
#pragma unroll
        for (int i = 0; i < C::kCopies; ++i) {
            const RowAt &row_here = rows_here[i * kAtOnce + (uint32_t)lane / KP];
            from.at[i] = values ? row_here.v : row_here.k;
        }
        return from;
    };
    auto copy_rows = [&](srv_u32x4 *to, const Sources &from) __attribute__((always_inline)) {
        const uint32_t here = (uint32_t)anew((int)first_piece);
#pragma unroll
        for (int i = 0; i < C::kCopies; ++i) {
            const uint32_t turned = (uint32_t)turn_of<KP>(wave * kOwn + i * kAtOnce) * 16;
            const char *const piece = D == DP || (int)(first_piece ^ turned) < D * kBytes ? from.at[i] + (here ^ turned) : zeros_at;
            __builtin_amdgcn_global_load_lds(TML_GPTR(piece), TML_LPTR(to + any_wave * kOwn * KP + i * 64), 16, 0, 0);
        }
    };

    float s[BN / 2];  // scores, then weights
    srv_u32x4 weights[kF32 ? 1 : BN / 16][NP];
#pragma unroll
    for (int i = 0; i < BN / 2; ++i) s[i] = 0.0f;
#pragma unroll
    for (int j = 0; j < (kF32 ? 1 : BN / 16); ++j)
#pragma unroll
        for (int n = 0; n < NP; ++n) weights[j][n] = srv_u32x4{0, 0, 0, 0};

    // ---- scores of a tile, before the scale
    auto multiply_keys = [&](const srv_u32x4 *tile_k, floatx16 (&sum)[BN / 32]) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < BN / 32; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) sum[u][i] = 0.0f;
        const int k_row = anew(l32);
#pragma unroll
        for (int c = 0; c < kQ; ++c)
#pragma unroll
            for (int u = 0; u < BN / 32; ++u) {
                const srv_u32x4 k = tile_k[team * C::kTile + (32 * u + k_row) * KP + ((2 * c + half) ^ turn_of<KP>(k_row))];
                if constexpr (kF32) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum[u] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(k[e]), __uint_as_float(q[0][c][e]), sum[u], 0, 0, 0);
                } else {
#pragma unroll
                    for (int n = 0; n < NQ; ++n) sum[u] = mma32<CT>(k, q[n][c], sum[u]);
                }
            }
    };
    auto take_scores = [&](const floatx16 (&sum)[BN / 32]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < BN / 2; ++i) s[i] = sum[i / 16][i % 16];
    };
    // Values: eight tokens of 16 j and on of this lane's d of 32 t and on (f32: the one of token j).
    // (few steps from the array on: through a longer way the compiler loses which array is read,
    // and waits for the copies to all)
    struct Places {
        int lane;
        uint32_t at[DP / 32][2];  // bytes, of the first 16 tokens' two fours
    };
    auto places = [&]() __attribute__((always_inline)) {
        Places p;
        const int v_lane = p.lane = anew(lane);
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                // four tokens a read, of 16 d a group of 16 lanes
                const int tok = 8 * r + 4 * (v_lane >> 5) + (v_lane & 15) / 4, piece = 4 * t + (v_lane >> 4 & 1) * 2 + (v_lane >> 1 & 1);
                p.at[t][r] = (uint32_t)((team * C::kTile + tok * KP + (piece ^ turn_of<KP>(tok))) * 16 + 8 * (v_lane & 1));
            }
        return p;
    };
    auto value_at = [&](const srv_u32x4 *tile_v, const Places &p, int j, int t) __attribute__((always_inline)) {
        if constexpr (kF32) {
            const int tok = 8 * (j / 4) + 4 * (p.lane >> 5) + j % 4, d = 32 * t + (p.lane & 31);
            return ((const float *)tile_v)[4 * (team * C::kTile + tok * KP + ((d / 4) ^ turn_of<KP>(tok))) + d % 4];
        } else {
            srv_u32x4 v;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const shortx4 four = read_turned((const shortx4 *)((const char *)tile_v + p.at[t][r]) + 32 * j * KP);
                const srv_u32x2 two = __builtin_bit_cast(srv_u32x2, four);
                v[2 * r] = two[0];
                v[2 * r + 1] = two[1];
            }
            return v;
        }
    };
    constexpr int kJ = kF32 ? BN / 2 : BN / 16;
    auto multiply_value = [&](auto v, int j, floatx16 sum) __attribute__((always_inline)) {
        if constexpr (kF32) {
            return __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[j], sum, 0, 0, 0);
        } else {
#pragma unroll
            for (int n = 0; n < NP; ++n) sum = mma32<CT>(v, weights[j][n], sum);
            return sum;
        }
    };
    auto multiply_values = [&](const srv_u32x4 *tile_v) __attribute__((always_inline)) {
        const Places p = places();
#pragma unroll
        for (int j = 0; j < kJ; ++j)
#pragma unroll
            for (int t = 0; t < DP / 32; ++t) o[t] = multiply_value(value_at(tile_v, p, j, t), j, o[t]);
    };
    struct Moved {
        bool any;
        float by, unit;  // what the output is multiplied with; of the scores
    };
    // ---- weights of tile `it`
    // (the maximum moves, and the output waits for that until the products under way are in it)
    auto new_maximum = [&](int it) __attribute__((always_inline)) {
        const int64_t k0 = tile_at(it);
        const uint64_t live = lds_live[it & 1][team];
        const bool whole = k0 + BN <= high_of(wave_first) && k0 >= low_of(wave_last) && (live & (~0ull >> (64 - BN))) == ~0ull >> (64 - BN);
        if constexpr (FORM) {
            if (QT != TML_TYPE_F32 && short_cap > 0.0f && short_cap < INFINITY) {
#pragma unroll
                for (int i = 0; i < BN / 2; ++i) {
                    const float e = __builtin_amdgcn_exp2f(s[i] * short_cap);
                    s[i] = fmaf(__builtin_amdgcn_rcpf(1.0f + e), -2.0f * kLog2E * a.cap, kLog2E * a.cap);
                }
            } else if (inv_cap != 0.0f) {
#pragma unroll
                for (int i = 0; i < BN / 2; ++i) s[i] = cap_score(s[i] * to_score, a.cap, inv_cap) * kLog2E;
            } else {
#pragma unroll
                for (int i = 0; i < BN / 2; ++i) s[i] *= to_log2;
            }
            if (a.slopes != nullptr) {
                const float from = (float)((int64_t)pos - k0 - 4 * half);
#pragma unroll
                for (int i = 0; i < BN / 2; ++i) s[i] = fmaf(-slope, fabsf(from - (float)(32 * (i / 16) + 8 * (i % 16 / 4) + i % 4)), s[i]);
            }
        }
        const float unit = FORM ? 1.0f : to_log2;  // of the scores
        if (!whole) {
            const uint32_t k = (uint32_t)k0;
            const int from = (low > k ? (int)min(low - k, (uint32_t)BN) : 0) - 4 * half, to = (high > k ? (int)min(high - k, (uint32_t)BN) : 0) - 4 * half;
            const uint32_t there[2] = {(uint32_t)live >> 4 * half, (uint32_t)(live >> 32) >> 4 * half};
#pragma unroll
            for (int i = 0; i < BN / 2; ++i) {
                const int t = 32 * (i / 16) + 8 * (i % 16 / 4) + i % 4;  // (+ 4 half)
                if (t < from || t >= to || (there[i / 16] >> t % 32 & 1) == 0) s[i] = -INFINITY;
            }
        }
        float most = s[0];
#pragma unroll
        for (int i = 1; i < BN / 2; ++i) most = fmaxf(most, s[i]);
        most = max_of_halves(most) * unit;
        const bool moves = __builtin_amdgcn_ballot_w64(most > m + kBehind) != 0;
        const float m_new = moves ? fmaxf(m, most) : m, f = m == m_new || m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
        m = m_new;
        l *= f;
        return Moved{moves, f, unit};
    };
    auto new_weights = [&](float unit, srv_u32x4 (&to)[kF32 ? 1 : BN / 16][NP]) __attribute__((always_inline)) {
        const float base = kUp - (m == -INFINITY ? 0.0f : m);
#pragma unroll
        for (int i = 0; i < BN / 2; ++i) {
            s[i] = __builtin_amdgcn_exp2f(fmaf(s[i], unit, base));
            l += s[i];
        }
        if constexpr (!kF32) {
#pragma unroll
            for (int j = 0; j < BN / 16; ++j) {
                float p[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) p[e] = s[8 * j + e];
                to_terms<CT, NP>(p, to[j]);
            }
        }
    };

    // What some rows of the workgroup do not see of a tile weighs nothing for them, but zero times
    // an infinity or a NaN is a NaN.  Such a tile's infinities and NaNs are cleared before anyone
    // multiplies it, by the wave that copied them, and go to those who see them in the end.  With one
    // of them near the ends of two bf16 prompts of 4096 tokens, 32 heads on 8 of 128, 381 to 423 us, without
    // 359 to 394 (taking the workgroup's rows again one by one: 101 ms).
    constexpr uint32_t kExponent = kF32 ? 0x7F800000u : CT == TML_TYPE_F16 ? 0x7C00u : 0x7F80u;
    // (bits of a word that hold its infinities and NaNs)
    auto odd_bits = [](uint32_t w) __attribute__((always_inline)) {
        if constexpr (kF32) return (w & kExponent) == kExponent ? ~0u : 0u;
        return ((w & kExponent) == kExponent ? 0xFFFFu : 0u) | ((w >> 16 & kExponent) == kExponent ? 0xFFFF0000u : 0u);
    };
    const int64_t all_from = low_of(block_last), all_to = high_of(block_first);
    auto seen_by_all = [&](int64_t k0) { return min(k0 + BN, end) <= all_to && k0 >= all_from; };
    // (the tiles from .. to .. are seen by all; where all see the end, the last may be too)
    const int whole_from = uniform((int)((max(all_from - begin, (int64_t)0) + BN - 1) / BN)), whole_to = uniform((int)(max(all_to - begin, (int64_t)0) / BN));
    auto clear_odd = [&](srv_u32x4 *tile_v, int it) __attribute__((always_inline)) {
        const int tile = TEAMS * it + team;
        if (__builtin_expect(tile < 0 || (tile >= whole_from && tile < whole_to), 1)) return;  // (before the first tile: zeros that other waves write)
        if (seen_by_all(tile_at(it))) return;
        srv_u32x4 *const mine = tile_v + any_wave * kOwn * KP + lane;
#pragma unroll
        for (int i = 0; i < C::kCopies; ++i) {
            srv_u32x4 v = mine[64 * i];
            uint32_t odd = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const uint32_t bits = odd_bits(v[x]);
                odd |= bits;
                v[x] &= ~bits;
            }
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd != 0) == 0, 1)) continue;
            mine[64 * i] = v;
            lds_odd = 1;
        }
    };

    // ---- A turn a tile: the scores' product, then the weights beside the product of the tile
    // before.  Keys are copied one tile ahead, values with their weights' turn.
    if (steps > 0) {
        // (the first turn multiplies the values of lds_v1 by no weights)
#pragma unroll 1
        for (int i = threadIdx.x; i < TEAMS * C::kTile; i += 64 * kWaves * TEAMS) lds_v1[i] = srv_u32x4{0, 0, 0, 0};
        if (threadIdx.x == 0) lds_odd = 0;
        find_rows(0, block_of(0));
        copy_rows(lds_k0, sources_of(row_at[0][any_wave], false));
        int next_block = block_of(1);
        auto turn = [&](int it, srv_u32x4 *k_now, srv_u32x4 *k_next, srv_u32x4 *v_now, srv_u32x4 *v_before) __attribute__((always_inline)) {
            // (no branch around the copies, or a wait for one would be a wait for all: past the last tile
            // they copy zeros)
            const Sources values = sources_of(row_at[it & 1][any_wave], true);
            wait_copies<0>();
            clear_odd(v_before, it - 1);
            __syncthreads();  // this tile's keys and the values before are there, the tile before was read
            find_rows(it + 1, next_block);
            const Sources keys = sources_of(row_at[(it + 1) & 1][any_wave], false);
            copy_rows(k_next, keys);
            copy_rows(v_now, values);
            next_block = block_of(it + 2);
            floatx16 sum[BN / 32];
            if constexpr (kF32) {  // (the weights are the scores' registers)
                multiply_values(v_before);
                multiply_keys(k_now, sum);
                constexpr int kAhead = 8, kReads = kJ * (DP / 32);  // reads ahead of the products
                __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
                for (int i = kAhead; i < kReads; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
#pragma unroll
                for (int i = 2; i < kQ; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 8, 0);
                take_scores(sum);
                const Moved moved = new_maximum(it);
                new_weights(moved.unit, weights);
                if (moved.any)
#pragma unroll
                    for (int t = 0; t < DP / 32; ++t) o[t] *= moved.by;
            } else {
                multiply_keys(k_now, sum);
                constexpr int kReads = kQ * (BN / 32);  // four ahead of the products
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
                for (int i = 4; i < kReads; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, NQ, 0);
                    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 4 * NQ, 0);
                take_scores(sum);
                const Moved moved = new_maximum(it);
                srv_u32x4 next[BN / 16][NP];
                multiply_values(v_before);
                new_weights(moved.unit, next);
                constexpr int kProducts = BN / 16 * (DP / 32);
                __builtin_amdgcn_sched_group_barrier(0x100, 4, 1);
#pragma unroll
                for (int i = 2; i < kProducts; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, NP, 1);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2, 1);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, 2 * NP, 1);
                if (moved.any)
#pragma unroll
                    for (int t = 0; t < DP / 32; ++t) o[t] *= moved.by;
#pragma unroll
                for (int j = 0; j < BN / 16; ++j)
#pragma unroll
                    for (int n = 0; n < NP; ++n) weights[j][n] = next[j][n];
            }
        };
        for (int it = 0; it < steps; it += 2) {
            turn(it, lds_k0, lds_k1, lds_v0, lds_v1);
            turn(it + 1, lds_k1, lds_k0, lds_v1, lds_v0);
        }
        wait_copies<0>();
        clear_odd(lds_v1, (steps - 1) | 1);
        __syncthreads();
        multiply_values(lds_v1);
    }

    l += __shfl_xor(l, 32);
    if constexpr (TEAMS == 2) {  // the second team's part joins the first's
        // (in the tiles' LDS: 16 bytes of each lane follow each other, DP / 8 times, half of them in
        // the keys' array)
        __syncthreads();
        constexpr int kHalf = DP / 16;
        static_assert(TEAMS == 1 || kHalf * 256 <= TEAMS * C::kTile, "the output fits the tiles");
        const int at = wave * 64 + lane;
        if (team == 1) {
#pragma unroll
            for (int x = 0; x < DP / 8; ++x)
                (x < kHalf ? lds_k0 : lds_v0)[x % kHalf * 256 + at] =
                    srv_u32x4{__float_as_uint(o[x / 4][4 * (x % 4)]), __float_as_uint(o[x / 4][4 * (x % 4) + 1]), __float_as_uint(o[x / 4][4 * (x % 4) + 2]),
                              __float_as_uint(o[x / 4][4 * (x % 4) + 3])};
            ((srv_f32x2 *)lds_k1)[at] = srv_f32x2{m, l};
        }
        __syncthreads();
        if (team == 1) return;
        const srv_f32x2 other = ((const srv_f32x2 *)lds_k1)[at];
        const float top = fmaxf(m, other[0]);
        const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - top), g = other[0] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(other[0] - top);
        l = l * f + other[1] * g;
#pragma unroll
        for (int x = 0; x < DP / 8; ++x) {
            const srv_u32x4 four = (x < kHalf ? lds_k0 : lds_v0)[x % kHalf * 256 + at];
#pragma unroll
            for (int i = 0; i < 4; ++i) o[x / 4][4 * (x % 4) + i] = fmaf(o[x / 4][4 * (x % 4) + i], f, __uint_as_float(four[i]) * g);
        }
    }
    const bool mine = row0 + 32 * wave + l32 < rows;
    const bool none = l == 0.0f;  // nothing weighs: zeros, also where a value is infinite or NaN
    const float r = none ? 0.0f : 1.0f / l;
    if (__builtin_amdgcn_ballot_w64(none) != 0)
#pragma unroll
        for (int t = 0; t < DP / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = none ? 0.0f : o[t][i];
    const int64_t to = (first + token) * a.out_stride + head * D;
#pragma unroll
    for (int t = 0; t < DP / 32; ++t)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int d = 32 * t + 8 * j + 4 * half;
            if (!mine || d >= D) continue;
            const float x0 = o[t][4 * j] * r, x1 = o[t][4 * j + 1] * r, x2 = o[t][4 * j + 2] * r, x3 = o[t][4 * j + 3] * r;
            if constexpr (QT == TML_TYPE_F32) {
                *(srv_u32x4_any *)((float *)a.out + to + d) = srv_u32x4{__float_as_uint(x0), __float_as_uint(x1), __float_as_uint(x2), __float_as_uint(x3)};
            } else {
                *(srv_u32x2_any *)((uint16_t *)a.out + to + d) =
                    QT == TML_TYPE_F16 ? srv_u32x2{srv_pack_f16(x0, x1), srv_pack_f16(x2, x3)} : srv_u32x2{srv_pack_bf16(x0, x1), srv_pack_bf16(x2, x3)};
            }
        }
    if (__builtin_expect(steps > 0 && lds_odd != 0, 0)) {  // (set before the last barrier)
        // A lane a token finds the ones that were cleared; their rows' lanes then take them one by one.
        // The tiles that all see, in the middle, are left out.
        for (int64_t k0 = begin; k0 < end; k0 += BN) {
            if (seen_by_all(k0)) {
                if (end <= all_to) break;
                k0 = begin + (whole_to - 1) * (int64_t)BN;
                continue;
            }
            const int64_t tok = k0 + lane % BN;
            int64_t off = -1;
            if (tok < end) {
                const int block = a.block_table[b * a.table_stride + (uint32_t)tok / (uint32_t)P];
                if (block >= 0 && block < a.n_blocks) off = (block * a.block_stride + (int64_t)((uint32_t)tok % (uint32_t)P) * a.token_stride + kv * a.head_stride) * kBytes;
            }
            uint32_t odd = 0;
            if (off >= 0)
                for (int x = 0; x < D * kBytes / 16; ++x) {
                    const srv_u32x4 v = *(const srv_u32x4 *)((const char *)a.v_cache + off + 16 * x);
                    odd |= odd_bits(v[0]) | odd_bits(v[1]) | odd_bits(v[2]) | odd_bits(v[3]);
                }
            uint64_t todo = __builtin_amdgcn_ballot_w64(odd != 0) & (~0ull >> (64 - BN));
            while (todo != 0) {
                const int from = __builtin_ctzll(todo);
                todo &= todo - 1;
                const int64_t at = (int64_t)(((uint64_t)(uint32_t)__shfl((int)(off >> 32), from) << 32) | (uint32_t)__shfl((int)(uint32_t)off, from));
                const bool sees = mine && k0 + from >= low && k0 + from < high && !none;
                for (int i = 0; i < D / 2; ++i) {
                    const int d = 8 * (i / 4) + 4 * half + i % 4;
                    const float x = srv_load1(CT, (const char *)a.v_cache + at, d);
                    if (sees && !(fabsf(x) < INFINITY)) srv_store1(QT, a.out, to + d, srv_load1(QT, a.out, to + d) + x);
                }
            }
        }
    }
}

// Two teams halve a workgroup's way through its tiles and fill the SIMDs where there are few
// workgroups, for the joining of their parts; where two workgroups of one team share a CU they go their ways
// apart, which eight waves behind one barrier do not.  Measured, one / two teams: 1500 frames, 20 heads
// of 64 (240 workgroups) 37.8 / 32.7 us; two prompts of 6000 to 8192 tokens (3500) 978 / 1129; 16 heads on
// 8 of 128, f16, 448 new tokens 23.1 / 21.9, 128 over 966 39.3 / 36.1, 64 13.4 / 16.9 (a tile a team, and the
// joining).  Capped or biased scores and f32 q have one team whatever the grid: the same three 28.0 / 25.3,
// 50.5 / 44.8 and 14.8 / 18.7 capped, 33.6 / 36.1, 55.9 / 57.5 and 20.2 / 27.8 with f32 q on f16.
template <int CT, int QT, int DP, bool FORM>
void launch_teams(const PromptAttentionArgs &a, const PromptShape &sh, hipStream_t s) {
    const dim3 grid(sh.tiles * (unsigned)a.kv_heads);
    if constexpr (Prompt<CT, QT, DP, FORM>::kTwo && CT == QT && CT != TML_TYPE_F32 && !FORM) {
        if (grid.x <= (unsigned)device_cus()) {
            prompt_attention_kernel<CT, QT, DP, FORM, 2><<<grid, dim3(128 * kWaves), 0, s>>>(a, sh);
            return;
        }
    }
    prompt_attention_kernel<CT, QT, DP, FORM, 1><<<grid, dim3(64 * kWaves), 0, s>>>(a, sh);
}
template <int CT, int QT, bool FORM>
void launch_dim(const PromptAttentionArgs &a, const PromptShape &sh, hipStream_t s) {
    if (a.head_dim <= 64) launch_teams<CT, QT, 64, FORM>(a, sh, s);
    else if (a.head_dim <= 128) launch_teams<CT, QT, 128, FORM>(a, sh, s);
    else launch_teams<CT, QT, 256, FORM>(a, sh, s);
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
    if (a.window >= sh.positions) a.window = 0;  // (all of the cache; and pos - window stays a number)
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
