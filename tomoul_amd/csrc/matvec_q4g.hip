// matvec_q4g.hip -- a few rows times a 4-bit weight with a scale for each
// group of K, and the quantizer of such weights.
//
//   y[m,n] = sum_g s[n,g] * ( sum_{k in g} q[n,k] * x[m,k] ) + bias[n]
//
// Row n of the weight is K-contiguous (even k in the low nibble, two's
// complement) and has ceil(K / group) fp32 scales.  x is f32, f16, bf16, or 8
// bits with a scale a row or a group.  What it has to read is the weight,
// K / 2 + 4 K / group bytes a column, so the kernel is built to stream it.
//
// Products on the matrix cores.  A lane loads 16 bytes of one column: 32
// consecutive k, all of one group.  Lanes (n, c) of a wave hold column n = lane
// % 16 and the four 32-k chunks c = lane / 16 of a 128-k run, which as the
// MFMA's B operand would add up k of four groups.  So x goes into the A operand
// four times apart: A row 4 c + i has row i of x where the k slot belongs to
// chunk c, and zeros elsewhere.  The result's row 4 c + i, which lane (n, c)
// holds, is then the sum over chunk c alone, and a multiply-add with that lane's
// own scale finishes it.  Rows that a matrix-vector product leaves empty pay
// for it; any group of whole 32s costs the same.
//
// x as terms, so that f32 x keeps its precision: each 32-k chunk of x is scaled
// by a power of two (largest finite magnitude to [2^14, 2^15)) and split into
// two f16 terms, |x - hi - lo| <= 2^-23 |x| + 2^-39 max|x|, which are two rows of
// A; bf16 x is exact in one term but for the same 2^-39 of the chunk's maximum,
// f16 x is itself.  4-bit weights are exact in f16; sums are fp32.  8-bit x runs
// on the int8 matrix cores, exact up to the scales.  An infinity leaves
// hi = +-65504 and lo = itself, so it and a NaN give what fp32 gives.
//
// A workgroup's waves share x, split to terms once into LDS; `ks` of them share a
// 16-column tile and add up through LDS in wave order (no atomics: the same bits
// every time), the others take other tiles.  The scales go through LDS too, a
// stretch's at a time: loaded one by one they touch as many cache lines as the
// weights (65536 x 4096: 43 us so, 32 us through LDS).
//
// Measured on MI355X (launches in a graph, three weights in turn; an empty launch
// there is 1.8 us): f32 x, 1 row, 1280 x 5120, groups of 32 6.8 us; 8-bit x, 8 rows,
// 14336 x 4096, groups of 128 12.0 us (2.6 TB/s); bf16 x, 4 rows, 51866 x 1280 10.7 us
// (3.6 TB/s); 65536 x 4096, 1 row 33 us (4.3 TB/s).  Small products are bound by the
// chain of one launch: x and the first weights from memory, x to LDS, a few runs of
// dependent matrix instructions, the waves' sum.
#include "serving.hpp"

#include <algorithm>

namespace tml {
namespace {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef int intx4 __attribute__((ext_vector_type(4)));
typedef _Float16 halfx8 __attribute__((ext_vector_type(8)));

// How x comes: f32, f16, bf16, 8 bits with row scales, 8 bits with group scales.
enum { MV_F32, MV_F16, MV_BF16, MV_I8, MV_I8G };
constexpr bool mv_int(int kind) { return kind >= MV_I8; }
constexpr bool mv_chunk_scales(int kind) { return kind == MV_F32 || kind == MV_BF16 || kind == MV_I8G; }
constexpr int mv_terms(int kind) { return kind == MV_F32 ? 2 : 1; }
// Bytes of an LDS row of kp elements: 16 past its end turn the four rows of a
// set away from each other's banks.
constexpr int mv_row_bytes(int kind, int kp) { return kp * (mv_int(kind) ? 1 : 2) + 16; }

// 128-k runs a wave has under way ahead of the one it works on: a stretch.  Two and
// not more: the loop is unrolled over them, and the kernel's code, which every launch
// fetches anew, costs a small product more than the loads in flight give a large one
// (1280 x 5120 with f32 x: 6.7, 7.1, 11.8 us for two, four, eight).
constexpr int kAhead = 2;
constexpr int kScaleRow = 4 * kAhead + 4;  // floats of a column's scales in LDS: a stretch's, on banks of their own
constexpr int kLdsHead = 128;  // zeros, and the scales of 8-bit rows of x
constexpr int mv_items(int kind) { return mv_chunk_scales(kind) && !mv_int(kind) ? 2 : 4; }  // eights of x a thread has under way

struct MvShape {
    int runs;       // 128-k runs of K
    int chunks;     // 32-k chunks of K
    int phase_runs;  // runs of x in LDS at a time
    int ks_log2;    // 2^ks_log2 waves share a tile, 2^tiles_log2 tiles a workgroup
    int tiles_log2;
    unsigned eights_magic;  // 2^32 / (eights of a phase's row of x), rounded up
    unsigned group_magic, group_one;  // 2^32 / (chunks of a group), rounded up, and 0; of one chunk: 0, and ~0
    int groups;     // scales of a column
    int row_bytes;   // of a column's nibbles
    int x_group, x_groups;  // columns of a scale of 8-bit x, scales of a row
    int lds_scales, lds_red, lds_cols;  // byte offsets in LDS
    unsigned scale_bytes;  // of all scales of the weight (not for rows on any address)
};

template <bool WIDE>
__device__ __forceinline__ srv_u32x4 mv_weights(const uint8_t *row, int chunk, int row_bytes) {
    if constexpr (WIDE) return *(const srv_u32x4 *)(row + chunk * 16);
    if (chunk * 16 + 16 <= row_bytes) return *(const srv_u32x4_any *)(row + chunk * 16);
    srv_u32x4 v = {0, 0, 0, 0};
#pragma unroll
    for (int b = 0; b < 16; ++b)
        if (chunk * 16 + b < row_bytes) v[b / 4] |= (uint32_t)row[chunk * 16 + b] << (8 * (b % 4));
    return v;
}

// The eight nibbles of d as f16 in the order 0 4 1 5 2 6 3 7.  A nibble with its
// sign bit turned is u = q + 8; in the low bits of f16 1024 it makes 1024 + u
// (1024 + 16 u for the upper one of a byte), from which one exact operation makes
// q.  Turning the bit and setting 1024 is one xor; `one` and `sixteen` hold its
// constants in vector registers, where one instruction can take them with the mask.
struct MvMagic {
    uint32_t one, sixteen;
};
__device__ __forceinline__ MvMagic mv_magic() {
    MvMagic m = {0x64086408u, 0x64806480u};
#ifdef __HIP_DEVICE_COMPILE__
    asm("" : "+v"(m.one), "+v"(m.sixteen));
#endif
    return m;
}
__device__ __forceinline__ halfx8 mv_halves(uint32_t d, const MvMagic &m) {
    const srv_f16x2 lo_bias = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    const srv_f16x2 hi_mul = {(_Float16)0.0625f, (_Float16)0.0625f}, hi_bias = {(_Float16)-72.0f, (_Float16)-72.0f};
    const uint32_t v = d >> 8;
    const srv_f16x2 a = __builtin_bit_cast(srv_f16x2, (d & 0x000F000Fu) ^ m.one) + lo_bias;
    const srv_f16x2 b = __builtin_bit_cast(srv_f16x2, (d & 0x00F000F0u) ^ m.sixteen) * hi_mul + hi_bias;
    const srv_f16x2 c = __builtin_bit_cast(srv_f16x2, (v & 0x000F000Fu) ^ m.one) + lo_bias;
    const srv_f16x2 e = __builtin_bit_cast(srv_f16x2, (v & 0x00F000F0u) ^ m.sixteen) * hi_mul + hi_bias;
    return halfx8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

// Eight elements of x in the order of mv_halves, as four packed pairs.
__device__ __forceinline__ srv_u32x4 mv_pairs(const float (&v)[8]) {
    return srv_u32x4{srv_pack_f16(v[0], v[4]), srv_pack_f16(v[1], v[5]), srv_pack_f16(v[2], v[6]), srv_pack_f16(v[3], v[7])};
}

// Eight consecutive elements of x as loaded.
template <int KIND>
struct MvRaw {
    srv_u32x4 d[KIND == MV_F32 ? 2 : 1];  // (8 bits: the first two dwords)
};
template <int KIND>
__device__ __forceinline__ MvRaw<KIND> mv_load_x(const void *x, int64_t i) {
    MvRaw<KIND> r;
    if constexpr (mv_int(KIND)) {
        const srv_u32x2 v = *(const srv_u32x2_any *)((const int8_t *)x + i);
        r.d[0] = srv_u32x4{v[0], v[1], 0, 0};
    } else {
        const auto v = srv_load8<KIND == MV_F32 ? TML_TYPE_F32 : TML_TYPE_F16>(x, i);
#pragma unroll
        for (int j = 0; j < (KIND == MV_F32 ? 2 : 1); ++j) r.d[j] = v.d[j];
    }
    return r;
}
// `live` of them from element i, the others zero.  (The last one again in their
// place: eight loads without a branch are one wait.)
template <int KIND>
__device__ __forceinline__ MvRaw<KIND> mv_load_few(const void *x, int64_t i, int live) {
    uint32_t v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (live > 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int64_t at = i + min(e, live - 1);
            v[e] = mv_int(KIND) ? ((const uint8_t *)x)[at] : KIND == MV_F32 ? ((const uint32_t *)x)[at] : ((const uint16_t *)x)[at];
        }
    }
    MvRaw<KIND> r;
#pragma unroll
    for (int j = 0; j < (KIND == MV_F32 ? 2 : 1); ++j) r.d[j] = srv_u32x4{0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t u = e < live ? v[e] : 0u;
        if constexpr (mv_int(KIND)) r.d[0][e / 4] |= u << (8 * (e % 4));
        else if constexpr (KIND == MV_F32) r.d[e / 4][e % 4] = u;
        else r.d[0][e / 2] |= u << (16 * (e % 2));
    }
    return r;
}

// One eight of x to LDS row `to` (and the next, for a second term); `scale`, where
// this kind has them: the chunk's, written by the first of its four eights.
template <int KIND>
__device__ __forceinline__ void mv_put(const MvRaw<KIND> &raw, char *to, int row_bytes, int e8, float *scale) {
    if constexpr (mv_int(KIND)) {
        // even k of the eight, then odd ones, as the weight's nibbles come apart
        const uint32_t p = raw.d[0][0], q = raw.d[0][1];
        *(srv_u32x2 *)(to + e8 * 8) = srv_u32x2{__builtin_amdgcn_perm(q, p, 0x06040200u), __builtin_amdgcn_perm(q, p, 0x07050301u)};
    } else {
        constexpr int kType = KIND == MV_F32 ? TML_TYPE_F32 : KIND == MV_F16 ? TML_TYPE_F16 : TML_TYPE_BF16;
        SrvRaw<kType> r;
#pragma unroll
        for (int j = 0; j < (KIND == MV_F32 ? 2 : 1); ++j) r.d[j] = raw.d[j];
        float v[8];
        srv_floats<kType>(r, v);
        if constexpr (KIND != MV_F16) {
            uint32_t most = 0;  // exponent of the chunk's largest finite magnitude
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t g = __float_as_uint(v[e]) & 0x7F800000u;
                most = max(most, g < 0x7F800000u ? g : 0u);
            }
            most = max(most, (uint32_t)__shfl_xor((int)most, 1));
            most = max(most, (uint32_t)__shfl_xor((int)most, 2));
            most = max(most, 27u << 23);  // (both powers below stay normal numbers)
            const float up = __uint_as_float((268u << 23) - most);  // 2^14 / 2^exponent
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= up;
            if (e8 % 4 == 0) {
                scale[0] = __uint_as_float(most - (14u << 23));
                if constexpr (KIND == MV_F32) scale[1] = __uint_as_float(most - (14u << 23));
            }
        }
        if constexpr (KIND == MV_F32) {
            float hi[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                hi[e] = (float)(_Float16)__builtin_amdgcn_fmed3f(v[e], -65504.0f, 65504.0f);
                v[e] -= hi[e];
            }
            *(srv_u32x4 *)(to + e8 * 16) = mv_pairs(hi);
            *(srv_u32x4 *)(to + row_bytes + e8 * 16) = mv_pairs(v);
        } else {
            *(srv_u32x4 *)(to + e8 * 16) = mv_pairs(v);
        }
    }
}

// ANY: weight rows on any address, and x in as many fills of LDS as it takes.
template <int KIND, int SETS, bool ANY>
__global__ __launch_bounds__(SETS > 2 ? 512 : 1024) void matvec_q4g_kernel(Matvec4Args a, MvShape sh) {
    constexpr int kTerms = mv_terms(KIND), kRows = SETS * 4 / kTerms, kItems = mv_items(KIND);
    TML_DYNAMIC_LDS(srv_u32x4, dyn);
    char *const lds = (char *)dyn;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n16 = lane & 15, c4 = lane >> 4;
    const int ks = 1 << sh.ks_log2, tslot = wave >> sh.ks_log2, kslot = wave & (ks - 1);
    const int64_t m0 = (int64_t)blockIdx.y * kRows;
    const int64_t n_wg = ((int64_t)blockIdx.x << sh.tiles_log2) * 16, n_first = n_wg + tslot * 16;
    const int row_bytes = mv_row_bytes(KIND, sh.phase_runs * 128);
    float *lds_scales = (float *)(lds + sh.lds_scales);
    // this lane's column, and its row of the A operand: x row lane % 4 of each set, if its k slots belong to the row's chunk
    const int64_t n = min(n_first + n16, a.N - 1);
    const uint8_t *w_row = a.w + n * a.w_stride;
    const float *s_row = a.w_scales + n * sh.groups;
    const __amdgpu_buffer_rsrc_t s_all = __builtin_amdgcn_make_buffer_rsrc((void *)a.w_scales, (short)0, (int)(ANY ? 0u : sh.scale_bytes), 0x00020000);
    const unsigned s_off = (unsigned)(n * sh.groups + kAhead * c4) * 4u;
    float *const s_lds = (float *)(lds + sh.lds_cols) + wave * 16 * kScaleRow;
    // an output of this thread's in the end has this column
    const int col = threadIdx.x & ((16 << sh.tiles_log2) - 1);
    const int64_t out_col = ks == 1 ? n_first + n16 : n_wg + col;
    const float bias = a.bias != nullptr ? a.bias[min(out_col, a.N - 1)] : 0.0f;
    const bool has_x = (n16 >> 2) == c4;
    // (lanes whose row has no x read 64 bytes of zeros at the start of LDS)
    constexpr int kRun = mv_int(KIND) ? 128 : 256;  // bytes of a run of x
    int x_at[SETS];
#pragma unroll
    for (int t = 0; t < SETS; ++t) x_at[t] = has_x ? kLdsHead + (t * 4 + (lane & 3)) * row_bytes + c4 * (kRun / 4) : 0;
    const int x_step = has_x ? kRun : 0;
    if (threadIdx.x < 16) ((uint32_t *)lds)[threadIdx.x] = 0;
    float *const x_row_scales = (float *)(lds + 64);
    if (KIND == MV_I8 && threadIdx.x < kRows) x_row_scales[threadIdx.x] = m0 + threadIdx.x < a.M ? 0.0625f * a.x_scales[m0 + threadIdx.x] : 0.0f;
    const MvMagic magic = mv_magic();

    floatx4 acc[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) acc[s] = floatx4{0, 0, 0, 0};
    for (int run0 = 0; run0 < sh.runs; run0 += sh.phase_runs) {
        const int nruns = ANY ? min(sh.phase_runs, sh.runs - run0) : sh.runs;
        const int c0 = nruns * kslot >> sh.ks_log2, c1 = n_first < a.N ? nruns * (kslot + 1) >> sh.ks_log2 : 0;
        auto group_of = [&](int chunk) {
            return (int)((unsigned)(((uint64_t)(unsigned)chunk * sh.group_magic) >> 32) + ((unsigned)chunk & sh.group_one));
        };
        auto load = [&](int run) { return mv_weights<!ANY>(w_row, min((run0 + run) * 4 + c4, sh.chunks - 1), sh.row_bytes); };
        // the scales of the stretch that begins at `run`: its 4 kAhead chunks are of at most as many groups, kAhead a lane
        srv_u32x2 ws[kAhead / 2];
        auto load_scales = [&](int run) {
            if constexpr (!ANY) {
#pragma unroll
                for (int i = 0; i < kAhead / 2; ++i)
                    ws[i] = __builtin_amdgcn_raw_buffer_load_b64(s_all, s_off + group_of((run0 + run) * 4) * 4u + 8 * i, 0, 0);
            }
        };
        // weights are under way before x is made ready
        srv_u32x4 w[kAhead];
        load_scales(max(min(c0, c1 - 1), 0));
#pragma unroll
        for (int u = 0; u < kAhead; ++u) w[u] = load(max(min(c0 + u, c1 - 1), 0));

        // ---- x, runs [run0, run0 + nruns): term t of row r is LDS row r * kTerms + t, zeros past M and K
        if (ANY && run0 > 0) __syncthreads();
        const int eights = nruns * 16, items = kRows * eights;
        for (int i0 = threadIdx.x; i0 < items; i0 += kItems * blockDim.x) {
            MvRaw<KIND> raw[kItems];
            int row[kItems], e8[kItems], live[kItems];
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                const int i = min(i0 + j * (int)blockDim.x, items - 1);
                row[j] = ANY ? i / eights : kRows == 1 ? 0 : (int)(((uint64_t)(unsigned)i * sh.eights_magic) >> 32);
                e8[j] = i - row[j] * eights;
                const int64_t k = (int64_t)run0 * 128 + e8[j] * 8;
                live[j] = m0 + row[j] < a.M && k < a.K ? (int)min((int64_t)8, a.K - k) : 0;
                const int64_t at = (m0 + row[j]) * a.x_stride + k;
                if (a.K < 8) raw[j] = mv_load_few<KIND>(a.x, at, live[j]);
                else raw[j] = mv_load_x<KIND>(a.x, live[j] == 8 ? at : 0);
            }
#pragma unroll
            for (int j = 0; j < kItems; ++j) {
                if (i0 + j * (int)blockDim.x >= items) break;
                if (live[j] < 8) raw[j] = mv_load_few<KIND>(a.x, (m0 + row[j]) * a.x_stride + (int64_t)run0 * 128 + e8[j] * 8, live[j]);
                float *scale = lds_scales + (e8[j] / 4) * SETS * 4 + row[j] * kTerms;
                if constexpr (KIND == MV_I8G)  // (1 / 16: the weight's nibbles are used as 16 q)
                    if (e8[j] % 4 == 0)
                        *scale = live[j] > 0 ? 0.0625f * a.x_scales[(m0 + row[j]) * sh.x_groups + (run0 * 128 + e8[j] * 8) / sh.x_group] : 0.0f;
                mv_put<KIND>(raw[j], lds + kLdsHead + row[j] * kTerms * row_bytes, row_bytes, e8[j], scale);
            }
        }
        __syncthreads();

        for (int c = c0; c < c1; c += kAhead) {
            float cs[kAhead];
            if constexpr (!ANY) {
#pragma unroll
                for (int i = 0; i < kAhead / 2; ++i) *(srv_u32x2 *)(s_lds + n16 * kScaleRow + c4 * kAhead + 2 * i) = ws[i];
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
                load_scales(min(c + kAhead, c1 - 1));
            }
            const int first_group = group_of((run0 + c) * 4);
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int chunk = (run0 + min(c + u, c1 - 1)) * 4 + c4, g = group_of(min(chunk, sh.chunks - 1));
                if constexpr (ANY) cs[u] = s_row[g];
                else cs[u] = s_lds[n16 * kScaleRow + g - first_group];
                if (chunk >= sh.chunks) cs[u] = 0.0f;  // (past K there is nothing, whatever the last group's scale is)
            }
            if constexpr (!ANY) {
                __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                __builtin_amdgcn_wave_barrier();
            }
#pragma unroll
            for (int u = 0; u < kAhead; ++u) {
                const int run = c + u;
                const srv_u32x4 d = w[u];
                const float s = cs[u];
                w[u] = load(min(run + kAhead, c1 - 1));
                if (u > 0 && run >= c1) continue;
                floatx4 xs[SETS];
                if constexpr (mv_chunk_scales(KIND)) {
#pragma unroll
                    for (int t = 0; t < SETS; ++t) xs[t] = *(const floatx4 *)(lds_scales + ((run * 4 + c4) * SETS + t) * 4);
                }
                if constexpr (mv_int(KIND)) {
                    intx4 x[2][SETS], part[SETS];
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int t = 0; t < SETS; ++t) x[j][t] = *(const intx4 *)(lds + x_at[t] + run * x_step + j * 16);
#pragma unroll
                    for (int t = 0; t < SETS; ++t) part[t] = intx4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const intx4 b = {(int)(d[2 * j] << 4 & 0xF0F0F0F0u), (int)(d[2 * j] & 0xF0F0F0F0u),
                                         (int)(d[2 * j + 1] << 4 & 0xF0F0F0F0u), (int)(d[2 * j + 1] & 0xF0F0F0F0u)};
#pragma unroll
                        for (int t = 0; t < SETS; ++t) part[t] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x[j][t], b, part[t], 0, 0, 0);
                    }
#pragma unroll
                    for (int t = 0; t < SETS; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][i] += (KIND == MV_I8G ? s * xs[t][i] : s) * (float)part[t][i];
                } else {
                    floatx4 part[SETS];
#pragma unroll
                    for (int t = 0; t < SETS; ++t) part[t] = floatx4{0, 0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const halfx8 b = mv_halves(d[j], magic);
#pragma unroll
                        for (int t = 0; t < SETS; ++t) {
                            const halfx8 x = *(const halfx8 *)(lds + x_at[t] + run * x_step + j * 16);
                            part[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, b, part[t], 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < SETS; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[t][i] += (mv_chunk_scales(KIND) ? s * xs[t][i] : s) * part[t][i];
                }
            }
        }
    }

    if (sh.runs == 0) __syncthreads();  // (the loop's barriers stand for it otherwise)

    // the four chunks of a run, then the waves that share the tile, in their order
#pragma unroll
    for (int t = 0; t < SETS; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[t][i] += __shfl_xor(acc[t][i], 16);
            acc[t][i] += __shfl_xor(acc[t][i], 32);
        }
    auto finish = [&](int r, float v) {  // y[m0 + r, out_col]
        if (out_col >= a.N || m0 + r >= a.M) return;
        if constexpr (KIND == MV_I8) v *= x_row_scales[r];
        srv_store1(a.y_type, a.y, (m0 + r) * a.y_stride + out_col, v + bias);
    };
    float sum[kRows];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        sum[r] = acc[r * kTerms / 4][r * kTerms % 4];
        if constexpr (kTerms == 2) sum[r] += acc[r * kTerms / 4][r * kTerms % 4 + 1];
    }
    if (ks == 1) {
#pragma unroll
        for (int r = 0; r < kRows; ++r)
            if (r % 4 == c4) finish(r, sum[r]);
        return;
    }
    float *red = (float *)(lds + sh.lds_red);
    if (c4 == 0) {
#pragma unroll
        for (int r = 0; r < kRows; ++r) red[(wave * kRows + r) * 16 + n16] = sum[r];
    }
    __syncthreads();
    for (int r = threadIdx.x >> (4 + sh.tiles_log2); r < kRows; r += 4 * ks) {
        float v = 0.0f;
        for (int k = 0; k < ks; ++k) v += red[(((col >> 4 << sh.ks_log2) + k) * kRows + r) * 16 + (col & 15)];
        finish(r, v);
    }
}

// One wave a group: the per-tensor int4 quantizer of quantize.hip on the group alone.
__global__ __launch_bounds__(256) void quantize_groups_kernel(int64_t N, int64_t K, int64_t group, const float *w, int64_t w_stride,
                                                              uint8_t *q, int64_t q_stride, float *scales) {
    const int64_t groups = (K + group - 1) / group, total = N * groups;
    const int lane = threadIdx.x & 63;
    for (int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); i < total; i += (int64_t)gridDim.x * 4) {
        const int64_t n = i / groups, g = i - n * groups, k0 = g * group, k1 = min(k0 + group, K);
        const float *row = w + n * w_stride;
        float m = 0.0f;
        for (int64_t k = k0 + lane; k < k1; k += 64) {
            const float v = fabsf(row[k]);
            m = v > m ? v : m;  // a NaN never wins
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        const bool zero = m == 0.0f;
        const float inv = zero ? 0.0f : 7.0f / m;
        if (lane == 0) scales[i] = zero ? 1.0f : m / 7.0f;
        auto nibble = [&](float v) {
            const float r = zero ? 0.0f : roundf(v * inv);
            return (uint32_t)(int)(r < -7.0f ? -7.0f : (r > 7.0f ? 7.0f : r)) & 0xFu;
        };
        for (int64_t k = k0 + 2 * lane; k < k1; k += 128) {
            uint32_t b = nibble(row[k]);
            if (k + 1 < k1) b |= nibble(row[k + 1]) << 4;
            q[n * q_stride + k / 2] = (uint8_t)b;
        }
    }
}

constexpr int kLdsMost = 150 * 1024;

template <int KIND, int SETS>
Status launch_sets(const Matvec4Args &a, MvShape sh, bool wide, hipStream_t s) {
    constexpr int kRows = SETS * 4 / mv_terms(KIND);
    const int cus = device_cus();
    const int64_t tiles = (a.N + 15) / 16, gy = (a.M + kRows - 1) / kRows;
    // One workgroup a CU, of as many waves as that leaves work: 16 (which share one
    // copy of x) from two tiles a CU on, 8 below, splitting K between the waves of a
    // tile up to where the workgroups would no longer all run at once.  Measured,
    // 16 / 8 waves: 8-bit x, 8 rows, 14336 x 4096 12.0 / 13.1 us; bf16, 4 rows, 51866 x
    // 1280 10.6 / 11.5; f32, 1 row, 1280 x 5120 7.2 / 6.7; splits one power of two more
    // or less there 16.5, 16.8 (of 12.0), 8.1 (of 6.7).
    const int nw = tiles * gy >= 2 * cus && SETS < 3 ? 16 : 8;
    int ks = 1;
    while (ks < nw && tiles * gy * ks * 2 <= (int64_t)cus * nw && ks * 2 <= sh.runs) ks *= 2;
    const int tiles_wg = nw / ks;
    sh.ks_log2 = __builtin_ctz(ks);
    sh.tiles_log2 = __builtin_ctz(tiles_wg);
    const int red = nw * kRows * 16 * 4, cols = nw * 16 * kScaleRow * 4;
    const int scale_bytes = mv_chunk_scales(KIND) ? 4 * SETS * 16 : 0;  // a run
    auto need = [&](int runs) { return kLdsHead + SETS * 4 * mv_row_bytes(KIND, runs * 128) + runs * scale_bytes + red + cols; };
    sh.phase_runs = std::max(sh.runs, 1);
    if (need(sh.phase_runs) > kLdsMost) {
        const int per_run = need(2) - need(1);
        sh.phase_runs = std::max(1, (kLdsMost - (need(1) - per_run)) / per_run);
    }
    // (one variant for rows on any address, x in several fills of LDS and scales past 4
    // GiB; it reads scales one by one.  f32 x, 65536 x 4096, 1 row: rows of 2048 bytes 36 us,
    // of 2049 78; 4096 outputs, 8 rows, K = 4096 in one fill 11.3, 4224 in two 13.5)
    const int64_t bytes = a.N * sh.groups * 4;
    const bool any = !wide || sh.phase_runs < sh.runs || bytes >= (int64_t)1 << 32;
    sh.scale_bytes = any ? 0 : (unsigned)bytes;
    sh.lds_scales = kLdsHead + SETS * 4 * mv_row_bytes(KIND, sh.phase_runs * 128);
    sh.lds_red = sh.lds_scales + sh.phase_runs * scale_bytes;
    sh.lds_cols = sh.lds_red + red;
    sh.eights_magic = (unsigned)((((uint64_t)1 << 32) + sh.phase_runs * 16 - 1) / (sh.phase_runs * 16));
    const dim3 grid((unsigned)((tiles + tiles_wg - 1) / tiles_wg), (unsigned)gy), block(nw * 64);
    const size_t lds = (size_t)need(sh.phase_runs);
    auto *k = any ? matvec_q4g_kernel<KIND, SETS, true> : matvec_q4g_kernel<KIND, SETS, false>;
    k<<<grid, block, lds, s>>>(a, sh);
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

template <int KIND>
Status launch_kind(const Matvec4Args &a, const MvShape &sh, bool wide, hipStream_t s) {
    const int64_t rows = a.M * mv_terms(KIND);
    if (rows <= 4) return launch_sets<KIND, 1>(a, sh, wide, s);
    if (rows <= 8) return launch_sets<KIND, 2>(a, sh, wide, s);
    if (rows <= 12) return launch_sets<KIND, 3>(a, sh, wide, s);  // (5 rows of f32 x, 3091 x 4950: 18.2 us as four sets, 10.4)
    return launch_sets<KIND, 4>(a, sh, wide, s);
}

constexpr int64_t kMostK = (int64_t)1 << 20;
// Columns of a launch: four threads each, and a grid has fewer than 2^32 (a larger one
// is cut without an error).
constexpr int64_t kMostN = (int64_t)1 << 29;

}  // namespace

Status launch_matvec_q4g(const Matvec4Args &in, hipStream_t s) {
    Matvec4Args a = in;
    if (!float_type(a.x_type) && a.x_type != TML_TYPE_I8)
        return Status::Err(TML_ERR_INVALID_FORMAT, "matvec_q4g: x must be f32, f16, bf16 or 8 bits");
    if (!float_type(a.y_type)) return Status::Err(TML_ERR_INVALID_FORMAT, "matvec_q4g: y must be f32, f16 or bf16");
    if (a.M < 0 || a.N < 0 || a.K < 0) return Status::Err(TML_ERR_INVALID_SHAPE, "negative matrix dimension");
    if (a.group <= 0 || a.x_group < 0) return Status::Err(TML_ERR_INVALID_ARG, "matvec_q4g: the group must be positive");
    if (a.M == 0 || a.N == 0) return Status::Ok();
    if (a.K > kMostK || a.N > 0x7FFFFFFF || a.M > 65535 * 2)
        return Status::Err(TML_ERR_INVALID_SHAPE, "matvec_q4g: at most 2^20 columns of x, 2^31 - 1 outputs and 131070 rows");
    if (a.group % 32 != 0 && a.group < a.K)
        return Status::Err(TML_ERR_INVALID_SHAPE, "matvec_q4g: a weight group must be a multiple of 32");
    const bool i8 = a.x_type == TML_TYPE_I8;
    if (i8 && a.x_group % 32 != 0 && a.x_group < a.K)
        return Status::Err(TML_ERR_INVALID_SHAPE, "matvec_q4g: a group of x must be a multiple of 32");
    if (a.y == nullptr || (a.K > 0 && (a.x == nullptr || a.w == nullptr || a.w_scales == nullptr)) ||
        (i8 && a.x_scales == nullptr))
        return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    const int64_t row = (a.K + 1) / 2;
    if ((a.M > 1 && (a.x_stride < a.K || a.y_stride < a.N)) || (a.N > 1 && a.w_stride < row))
        return Status::Err(TML_ERR_INVALID_SHAPE, "matvec_q4g: a row stride is shorter than the row");
    a.group = std::min(a.group, std::max<int64_t>(a.K, 1));
    if (a.N > kMostN) {  // the last columns in a launch of their own
        a.N = kMostN;
        Status first = launch_matvec_q4g(a, s);
        if (!first.ok()) return first;
        a.N = in.N - kMostN;
        if (a.K > 0) {
            a.w += kMostN * a.w_stride;
            a.w_scales += kMostN * ((a.K + a.group - 1) / a.group);
        }
        if (a.bias != nullptr) a.bias += kMostN;
        a.y = (char *)a.y + kMostN * type_bytes(a.y_type);
        return launch_matvec_q4g(a, s);
    }
    MvShape sh{};
    sh.chunks = (int)((a.K + 31) / 32);
    sh.runs = (sh.chunks + 3) / 4;
    sh.groups = (int)((a.K + a.group - 1) / a.group);
    const int64_t group32 = (a.group + 31) / 32;
    sh.group_magic = group32 > 1 ? (unsigned)((((uint64_t)1 << 32) + group32 - 1) / group32) : 0;
    sh.group_one = group32 > 1 ? 0 : ~0u;
    sh.row_bytes = (int)row;
    // whole aligned 16-byte loads, all inside the rows' own bytes
    const bool wide = ((uintptr_t)a.w | (uintptr_t)a.w_stride) % 16 == 0 && a.w_stride >= (int64_t)sh.chunks * 16;
    if (i8) {
        if (a.x_group == 0 || a.x_group >= a.K) {
            a.x_group = std::max<int64_t>(a.K, 1);
            return launch_kind<MV_I8>(a, sh, wide, s);
        }
        sh.x_group = (int)a.x_group;
        sh.x_groups = (int)((a.K + a.x_group - 1) / a.x_group);
        return launch_kind<MV_I8G>(a, sh, wide, s);
    }
    if (a.x_type == TML_TYPE_F32) return launch_kind<MV_F32>(a, sh, wide, s);
    if (a.x_type == TML_TYPE_F16) return launch_kind<MV_F16>(a, sh, wide, s);
    return launch_kind<MV_BF16>(a, sh, wide, s);
}

Status launch_quantize_groups(int64_t N, int64_t K, int64_t group, const float *w, int64_t w_stride, uint8_t *q, int64_t q_stride,
                              float *scales, hipStream_t s) {
    if (N < 0 || K < 0) return Status::Err(TML_ERR_INVALID_SHAPE, "negative matrix dimension");
    if (group <= 0) return Status::Err(TML_ERR_INVALID_ARG, "group quantizer: the group must be positive");
    if (group % 2 != 0 && group < K) return Status::Err(TML_ERR_INVALID_SHAPE, "group quantizer: the group must be even");
    if (N == 0 || K == 0) return Status::Ok();
    group = std::min(group, K);
    if (w == nullptr || q == nullptr || scales == nullptr) return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    if (N > 1 && (w_stride < K || q_stride < (K + 1) / 2))
        return Status::Err(TML_ERR_INVALID_SHAPE, "group quantizer: a row stride is shorter than the row");
    const int64_t total = N * ((K + group - 1) / group);
    quantize_groups_kernel<<<dim3((unsigned)std::min<int64_t>((total + 3) / 4, 1 << 16)), dim3(256), 0, s>>>(
        N, K, group, w, w_stride, q, q_stride, scales);
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

}  // namespace tml
