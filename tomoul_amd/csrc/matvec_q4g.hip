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
// every time), the others take other tiles.
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

constexpr int kBatch = 4;  // 128-k runs a wave has under way ahead of the ones it works on

struct MvShape {
    int runs;       // 128-k runs of K
    int chunks;     // 32-k chunks of K
    int phase_runs;  // runs of x in LDS at a time
    int ks;         // waves that share a tile
    int tiles;      // 16-column tiles
    int group32;    // chunks of a group, and 2^32 / group32 rounded up
    unsigned group_magic;
    int64_t groups;  // scales of a column
    int row_bytes;   // of a column's nibbles
    int x_group, x_groups;  // columns of a scale of 8-bit x, scales of a row
    int lds_scales, lds_red;  // byte offsets in LDS
};

struct MvItem {
    srv_u32x4 w;
    float s;
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

// The eight nibbles of d as f16 in the order 0 4 1 5 2 6 3 7: a nibble's place
// in a half of 1024 makes 1024 + u (1024 + 16 u for the upper ones of a byte),
// u = q + 8, from which one exact operation makes q.
__device__ __forceinline__ halfx8 mv_halves(uint32_t d) {
    const uint32_t u = d ^ 0x88888888u, v = u >> 8;
    const srv_f16x2 lo_bias = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    const srv_f16x2 hi_mul = {(_Float16)0.0625f, (_Float16)0.0625f}, hi_bias = {(_Float16)-72.0f, (_Float16)-72.0f};
    const srv_f16x2 a = __builtin_bit_cast(srv_f16x2, (u & 0x000F000Fu) | 0x64006400u) + lo_bias;
    const srv_f16x2 b = __builtin_bit_cast(srv_f16x2, (u & 0x00F000F0u) | 0x64006400u) * hi_mul + hi_bias;
    const srv_f16x2 c = __builtin_bit_cast(srv_f16x2, (v & 0x000F000Fu) | 0x64006400u) + lo_bias;
    const srv_f16x2 e = __builtin_bit_cast(srv_f16x2, (v & 0x00F000F0u) | 0x64006400u) * hi_mul + hi_bias;
    return halfx8{a[0], a[1], b[0], b[1], c[0], c[1], e[0], e[1]};
}

// Eight elements of x in the order of mv_halves, as four packed pairs.
__device__ __forceinline__ srv_u32x4 mv_pairs(const float (&v)[8]) {
    return srv_u32x4{srv_pack_f16(v[0], v[4]), srv_pack_f16(v[1], v[5]), srv_pack_f16(v[2], v[6]), srv_pack_f16(v[3], v[7])};
}

// Rows m0 .. of x, runs [run0, run0 + nruns) of K, to LDS: term t of row r is
// LDS row r * terms + t, zeros past M and K.
template <int KIND, int SETS>
__device__ __forceinline__ void mv_stage(const Matvec4Args &a, const MvShape &sh, char *lds, int64_t m0, int run0, int nruns) {
    constexpr int kTerms = mv_terms(KIND), kRows = SETS * 4 / kTerms;
    const int eights = nruns * 16, row_bytes = mv_row_bytes(KIND, sh.phase_runs * 128);
    float *scales = (float *)(lds + sh.lds_scales);
    for (int i = threadIdx.x; i < kRows * eights; i += blockDim.x) {
        const int r = i / eights, e8 = i - r * eights;
        const int64_t m = m0 + r, k = (int64_t)run0 * 128 + e8 * 8;
        const int live = m < a.M && k < a.K ? (int)min((int64_t)8, a.K - k) : 0;
        char *to = lds + r * kTerms * row_bytes;
        if constexpr (mv_int(KIND)) {
            const int8_t *x = (const int8_t *)a.x + m * a.x_stride + k;
            srv_u32x2 d = {0, 0};
            if (live == 8) d = *(const srv_u32x2_any *)x;
            else
                for (int e = 0; e < live; ++e) d[e / 4] |= (uint32_t)(uint8_t)x[e] << (8 * (e % 4));
            // even k of the eight, then odd ones, as the weight's nibbles come apart
            const uint32_t p = d[0], q = d[1];
            *(srv_u32x2 *)(to + e8 * 8) =
                srv_u32x2{(p & 0xFFu) | (p >> 8 & 0xFF00u) | (q & 0xFFu) << 16 | (q << 8 & 0xFF000000u),
                          (p >> 8 & 0xFFu) | (p >> 16 & 0xFF00u) | (q << 8 & 0xFF0000u) | (q & 0xFF000000u)};
            if constexpr (KIND == MV_I8G) {
                // (1 / 16: the weight's nibbles are used as 16 q)
                if (e8 % 4 == 0)
                    scales[(e8 / 4) * SETS * 4 + r] =
                        live > 0 ? 0.0625f * a.x_scales[m * sh.x_groups + (int)k / sh.x_group] : 0.0f;
            }
        } else {
            constexpr int kType = KIND == MV_F32 ? TML_TYPE_F32 : KIND == MV_F16 ? TML_TYPE_F16 : TML_TYPE_BF16;
            float v[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (live == 8) srv_floats<kType>(srv_load8<kType>(a.x, m * a.x_stride + k), v);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e < live) v[e] = srv_load1(kType, a.x, m * a.x_stride + k + e);
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
                if (e8 % 4 == 0)
#pragma unroll
                    for (int t = 0; t < kTerms; ++t)
                        scales[(e8 / 4) * SETS * 4 + r * kTerms + t] = __uint_as_float(most - (14u << 23));
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
}

template <int KIND, int SETS, bool WIDE>
__global__ __launch_bounds__(1024) void matvec_q4g_kernel(Matvec4Args a, MvShape sh) {
    constexpr int kTerms = mv_terms(KIND), kRows = SETS * 4 / kTerms;
    TML_DYNAMIC_LDS(srv_u32x4, dyn);
    char *const lds = (char *)dyn;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, nw = blockDim.x >> 6;
    const int n16 = lane & 15, c4 = lane >> 4;
    const int kslot = wave % sh.ks, tslot = wave / sh.ks, tiles_wg = nw / sh.ks;
    const int64_t m0 = (int64_t)blockIdx.y * kRows;
    const int row_bytes = mv_row_bytes(KIND, sh.phase_runs * 128);
    const float *lds_scales = (const float *)(lds + sh.lds_scales);
    float *red = (float *)(lds + sh.lds_red);
    // this lane's row of the A operand: x row lane % 4 of each set, if its k slots belong to the row's chunk
    const bool has_x = (n16 >> 2) == c4;
    const char *xrow = lds + (lane & 3) * row_bytes + c4 * 32 * (mv_int(KIND) ? 1 : 2);
    const bool one_phase = sh.phase_runs >= sh.runs;

    // runs [c0, c1) of a phase of `nruns` belong to this wave
    auto first_run = [&](int nruns, int slot) { return (int)((int64_t)nruns * slot / sh.ks); };
    auto load = [&](int tile, int run) {  // (run counted from K's start)
        const int64_t n = min((int64_t)tile * 16 + n16, a.N - 1);
        const int chunk = run * 4 + c4, at = min(chunk, sh.chunks - 1);
        const int g = sh.group32 == 1 ? at : (int)(((uint64_t)(unsigned)at * sh.group_magic) >> 32);
        MvItem it;
        it.w = mv_weights<WIDE>(a.w + n * a.w_stride, at, sh.row_bytes);
        it.s = chunk < sh.chunks ? a.w_scales[n * sh.groups + g] : 0.0f;
        return it;
    };

    MvItem cur[kBatch], nxt[kBatch];
    const int c0_first = first_run(min(sh.phase_runs, sh.runs), kslot), c1_first = first_run(min(sh.phase_runs, sh.runs), kslot + 1);
    int tile = blockIdx.x * tiles_wg + tslot;
    const int tile_step = gridDim.x * tiles_wg;
    auto load_batch = [&](MvItem(&b)[kBatch], int t, int run, int end, int run0) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u)
            if (run + u < end) b[u] = load(t, run0 + run + u);
    };
    // weights are under way before x is made ready
    if (tile < sh.tiles) load_batch(cur, tile, c0_first, c1_first, 0);
    if (one_phase) {
        mv_stage<KIND, SETS>(a, sh, lds, m0, 0, sh.runs);
        __syncthreads();
    }
    // every wave of a workgroup goes through the loop equally often: it holds barriers
    for (int it = blockIdx.x * tiles_wg; it < sh.tiles; it += tile_step, tile += tile_step) {
        floatx4 acc[SETS];
#pragma unroll
        for (int s = 0; s < SETS; ++s) acc[s] = floatx4{0, 0, 0, 0};
        for (int run0 = 0; run0 < sh.runs; run0 += sh.phase_runs) {
            const int nruns = min(sh.phase_runs, sh.runs - run0);
            const int c0 = first_run(nruns, kslot), c1 = first_run(nruns, kslot + 1);
            if (!one_phase) {
                __syncthreads();
                mv_stage<KIND, SETS>(a, sh, lds, m0, run0, nruns);
                __syncthreads();
            }
            if (tile >= sh.tiles) continue;
            for (int c = c0; c < c1; c += kBatch) {
                if (c + kBatch < c1) load_batch(nxt, tile, c + kBatch, c1, run0);
                else if (run0 + nruns < sh.runs) {
                    const int left = min(sh.phase_runs, sh.runs - run0 - nruns);
                    load_batch(nxt, tile, first_run(left, kslot), first_run(left, kslot + 1), run0 + nruns);
                } else if (tile + tile_step < sh.tiles) {
                    load_batch(nxt, tile + tile_step, c0_first, c1_first, 0);
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) {
                    if (c + u >= c1) break;
                    const int run = c + u;
                    floatx4 xs[SETS];
                    if constexpr (mv_chunk_scales(KIND)) {
#pragma unroll
                        for (int s = 0; s < SETS; ++s) xs[s] = *(const floatx4 *)(lds_scales + ((run * 4 + c4) * SETS + s) * 4);
                    }
                    if constexpr (mv_int(KIND)) {
                        intx4 part[SETS];
#pragma unroll
                        for (int s = 0; s < SETS; ++s) part[s] = intx4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint32_t d0 = cur[u].w[2 * j], d1 = cur[u].w[2 * j + 1];
                            const intx4 b = {(int)(d0 << 4 & 0xF0F0F0F0u), (int)(d0 & 0xF0F0F0F0u), (int)(d1 << 4 & 0xF0F0F0F0u),
                                             (int)(d1 & 0xF0F0F0F0u)};
#pragma unroll
                            for (int s = 0; s < SETS; ++s) {
                                intx4 x = {0, 0, 0, 0};
                                if (has_x) x = *(const intx4 *)(xrow + s * 4 * row_bytes + run * 128 + j * 16);
                                part[s] = __builtin_amdgcn_mfma_i32_16x16x64_i8(x, b, part[s], 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int s = 0; s < SETS; ++s)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const float p = (float)part[s][i];
                                acc[s][i] += (KIND == MV_I8G ? cur[u].s * xs[s][i] : cur[u].s) * p;
                            }
                    } else {
                        floatx4 part[SETS];
#pragma unroll
                        for (int s = 0; s < SETS; ++s) part[s] = floatx4{0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const halfx8 b = mv_halves(cur[u].w[j]);
#pragma unroll
                            for (int s = 0; s < SETS; ++s) {
                                srv_u32x4 x = {0, 0, 0, 0};
                                if (has_x) x = *(const srv_u32x4 *)(xrow + s * 4 * row_bytes + run * 256 + j * 16);
                                part[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(halfx8, x), b, part[s], 0, 0, 0);
                            }
                        }
#pragma unroll
                        for (int s = 0; s < SETS; ++s)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                acc[s][i] += (mv_chunk_scales(KIND) ? cur[u].s * xs[s][i] : cur[u].s) * part[s][i];
                    }
                }
#pragma unroll
                for (int u = 0; u < kBatch; ++u) cur[u] = nxt[u];
            }
            // a wave without runs in this phase still needs its first ones of the next phase or tile
            if (c0 >= c1) {
                const int left = min(sh.phase_runs, sh.runs - run0 - nruns);
                if (left > 0) load_batch(cur, tile, first_run(left, kslot), first_run(left, kslot + 1), run0 + nruns);
                else if (tile + tile_step < sh.tiles) load_batch(cur, tile + tile_step, c0_first, c1_first, 0);
            }
        }
        // the four chunks of a run, then the waves that share the tile
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                acc[s][i] += __shfl_xor(acc[s][i], 16);
                acc[s][i] += __shfl_xor(acc[s][i], 32);
            }
        auto finish = [&](int64_t n, int r, float v) {  // y[m0 + r, n]
            if (n >= a.N || m0 + r >= a.M) return;
            if constexpr (KIND == MV_I8) v *= 0.0625f * a.x_scales[m0 + r];
            if (a.bias != nullptr) v += a.bias[n];
            srv_store1(a.y_type, a.y, (m0 + r) * a.y_stride + n, v);
        };
        if (sh.ks == 1) {
            if (tile < sh.tiles) {
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    float v = 0.0f;
#pragma unroll
                    for (int t = 0; t < kTerms; ++t) v += acc[(r * kTerms + t) / 4][(r * kTerms + t) % 4];
                    if (r % 4 == c4) finish((int64_t)tile * 16 + n16, r, v);
                }
            }
            continue;
        }
        __syncthreads();  // the last tile's sums have been read
        if (c4 == 0) {
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                float v = 0.0f;
#pragma unroll
                for (int t = 0; t < kTerms; ++t) v += acc[(r * kTerms + t) / 4][(r * kTerms + t) % 4];
                red[(wave * kRows + r) * 16 + n16] = v;
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < tiles_wg * kRows * 16; i += blockDim.x) {
            const int ts = i / (kRows * 16), r = i / 16 % kRows, n = i % 16;
            float v = 0.0f;
            for (int w = 0; w < sh.ks; ++w) v += red[((ts * sh.ks + w) * kRows + r) * 16 + n];
            if (it + ts < sh.tiles) finish((int64_t)(it + ts) * 16 + n, r, v);
        }
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
    // Enough waves for the memory's latency: 16 a CU, sharing tiles where the
    // tiles alone are fewer, but no wave without a run of its own.
    const int cus = device_cus();
    int nw = 16;
    sh.ks = 1;
    while (sh.ks < nw && (int64_t)sh.tiles * sh.ks < (int64_t)cus * nw && sh.ks < sh.runs) sh.ks *= 2;
    if (sh.ks <= 4 && (int64_t)sh.tiles * sh.ks < (int64_t)cus * nw) nw = 8;
    const int red = nw * kRows * 16 * 4;
    const int scale_bytes = mv_chunk_scales(KIND) ? 4 * SETS * 16 : 0;  // a run
    auto need = [&](int runs) { return SETS * 4 * mv_row_bytes(KIND, runs * 128) + runs * scale_bytes + red; };
    sh.phase_runs = sh.runs;
    if (need(sh.runs) > kLdsMost) {
        const int per_run = need(2) - need(1);
        sh.phase_runs = std::max(1, (kLdsMost - (need(1) - per_run)) / per_run);
    }
    sh.lds_scales = SETS * 4 * mv_row_bytes(KIND, sh.phase_runs * 128);
    sh.lds_red = sh.lds_scales + sh.phase_runs * scale_bytes;
    const int tiles_wg = nw / sh.ks;
    int64_t gx = (sh.tiles + tiles_wg - 1) / tiles_wg;
    const int64_t gy = (a.M + kRows - 1) / kRows;
    gx = std::min<int64_t>(gx, std::max<int64_t>(1, 2 * cus / gy));
    const dim3 grid((unsigned)gx, (unsigned)gy), block(nw * 64);
    const size_t lds = (size_t)need(sh.phase_runs);
    auto *k = wide ? matvec_q4g_kernel<KIND, SETS, true> : matvec_q4g_kernel<KIND, SETS, false>;
    k<<<grid, block, lds, s>>>(a, sh);
    TML_HIP_TRY(hipGetLastError());
    return Status::Ok();
}

template <int KIND>
Status launch_kind(const Matvec4Args &a, const MvShape &sh, bool wide, hipStream_t s) {
    const int64_t rows = a.M * mv_terms(KIND);
    if (rows <= 4) return launch_sets<KIND, 1>(a, sh, wide, s);
    if (rows <= 8) return launch_sets<KIND, 2>(a, sh, wide, s);
    return launch_sets<KIND, 4>(a, sh, wide, s);
}

constexpr int64_t kMostK = (int64_t)1 << 20;

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
    MvShape sh{};
    sh.chunks = (int)((a.K + 31) / 32);
    sh.runs = (sh.chunks + 3) / 4;
    sh.tiles = (int)((a.N + 15) / 16);
    sh.groups = (a.K + a.group - 1) / a.group;
    sh.group32 = (int)((a.group + 31) / 32);
    sh.group_magic = sh.group32 > 1 ? (unsigned)((((uint64_t)1 << 32) + sh.group32 - 1) / sh.group32) : 0;
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
