// rmsnorm.hip -- root-mean-square norm with the residual's addition, its
// output as floats or in 8 bits with scales.
//
//   h = x + residual                          (32 bits; `sum` gets it rounded)
//   y = h / sqrt(mean(h^2) + eps) * weight    (from the unrounded h)
//   8 bits: scale = max|y| / 127 over the row or each `group` columns,
//           q = rint(y / scale)
//
// One pass: a row's h stays in registers between its sum of squares and the
// output, so x and the residual are read once and sum and y written once.
// Bound by memory past a few hundred rows, by latency below: 8192 x 5120 bf16 to 8
// bits 53.4 us on MI355X (294 MB, 5.5 TB/s), one row of 1280 f32 2.8 us.  A lane holds
// runs of eight columns (16-byte accesses of 16-bit types), NV of them; a row
// belongs to one wave (no barrier, four rows a workgroup) or to a workgroup.
// A row's last run is moved back to end with the row: the columns it shares
// with the run before are counted once and written twice with the same value,
// so odd lengths take no scalar tail.
#include "serving.hpp"

#include <algorithm>

namespace tml {
namespace {

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
// Maxima of magnitudes go as the bits of non-negative floats: these compare
// like the floats, and a NaN above an infinity, so it is not lost.
__device__ __forceinline__ uint32_t mag(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t wave_max(uint32_t v, int width) {
    for (int o = width / 2; o > 0; o >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, o));
    return v;
}

// scale of a group whose largest magnitude has the bits `most`.  A group of (nearly)
// zeros has scale 1; one that holds an infinity or a NaN has that as its scale.
constexpr uint32_t kLeast = (127u - 118u) << 23;  // 2^-118: m / 127 and 127 / m are normal numbers from it on
__device__ __forceinline__ float group_scale(uint32_t most) {
    const float m = __uint_as_float(most);
    return most >= 0x7F800000u ? m : most < kLeast ? 1.0f : m / 127.0f;
}
// rint(y / scale), and 0 where the scale is no number.
__device__ __forceinline__ int quantum(float y, float scale) {
    const float q = y / scale;
    return scale < INFINITY ? (int)__builtin_rintf(q) : 0;
}
// The same for eight columns of one group, whose largest magnitude is `most`.  A
// product with 127 / most, off by less than 2^-22 of 127, goes the other way at some of
// the halves between two integers: a wave that has a product so near to one divides
// (8192 x 5120 bf16, groups of 128: divisions alone 65 us, this 61, products alone 60).
__device__ __forceinline__ srv_u32x2 quanta(const float (&y)[8], uint32_t most, float scale) {
    const float inv = most < 0x7F800000u && most >= kLeast ? 127.0f / __uint_as_float(most) : 0.0f;
    int n[8];
    float off = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float q = inv == 0.0f ? 0.0f : y[e] * inv, r = __builtin_rintf(q);
        off = fmaxf(off, fabsf(q - r));
        n[e] = (int)r;
    }
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(off > 0.5f - 0x1p-14f) != 0, 0)) {
#pragma unroll
        for (int e = 0; e < 8; ++e) n[e] = quantum(y[e], scale);
    }
    srv_u32x2 d = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e) d[e / 4] |= (uint32_t)(n[e] & 0xFF) << (8 * (e % 4));
    return d;
}

// TPR threads a row, NV runs of eight columns a thread.
template <int T, int TPR, int NV>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rmsnorm_kernel(RmsNormArgs a) {
    constexpr int kRows = TPR < 256 ? 256 / TPR : 1, kWaves = TPR / 64;
    const int t = threadIdx.x & (TPR - 1);
    const int64_t row = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR;
    if (kRows > 1 && row >= a.rows) return;  // whole waves, and no barrier follows
    const int cols = (int)a.cols;
    int off[NV], skip[NV];  // a run's first column, and how many of its eight are counted elsewhere
    SrvRaw<T> rx[NV], rr[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        const int c = (v * TPR + t) * 8;
        off[v] = min(c, cols - 8);
        skip[v] = c - off[v];
        rx[v] = srv_load8<T>(a.x, row * a.x_stride + off[v]);
    }
    if (a.residual != nullptr) {
#pragma unroll
        for (int v = 0; v < NV; ++v) rr[v] = srv_load8<T>(a.residual, row * a.residual_stride + off[v]);
    }
    SrvRaw<TML_TYPE_F32> rw[NV];
    if (a.weight != nullptr) {
#pragma unroll
        for (int v = 0; v < NV; ++v) rw[v] = srv_load8<TML_TYPE_F32>(a.weight, off[v]);
    }
    float h[NV][8], ss = 0.0f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        srv_floats<T>(rx[v], h[v]);
        if (a.residual != nullptr) {
            float r[8];
            srv_floats<T>(rr[v], r);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[v][e] += r[e];
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += e >= skip[v] ? h[v][e] * h[v][e] : 0.0f;
    }
    ss = wave_sum(ss);
    if constexpr (kWaves > 1) {
        __shared__ float part[kWaves];
        if ((t & 63) == 0) part[t >> 6] = ss;
        __syncthreads();
        ss = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) ss += part[w];
    }
    // after every thread of the row has read it: sum may be x or the residual
    __builtin_amdgcn_sched_barrier(0);
    if (a.sum != nullptr) {
#pragma unroll
        for (int v = 0; v < NV; ++v)
            if (skip[v] < 8) srv_store8<T>(a.sum, row * a.sum_stride + off[v], h[v]);
    }
    const float root = 1.0f / sqrtf(ss / (float)cols + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        float w[8];
        if (a.weight != nullptr) srv_floats<TML_TYPE_F32>(rw[v], w);
#pragma unroll
        for (int e = 0; e < 8; ++e) h[v][e] = a.weight != nullptr ? h[v][e] * root * w[e] : h[v][e] * root;
    }
    if (a.out_type != TML_TYPE_I8) {
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            if (skip[v] >= 8) continue;
            const int64_t at = row * a.out_stride + off[v];
            if (a.out_type == TML_TYPE_F32) srv_store8<TML_TYPE_F32>(a.out, at, h[v]);
            else if (a.out_type == TML_TYPE_F16) srv_store8<TML_TYPE_F16>(a.out, at, h[v]);
            else srv_store8<TML_TYPE_BF16>(a.out, at, h[v]);
        }
        return;
    }
    const int group = (int)a.group, ngroups = (cols + group - 1) / group;
    uint32_t most[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        most[v] = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) most[v] = e >= skip[v] ? max(most[v], mag(h[v][e])) : most[v];
    }
    if (group >= cols) {  // one scale a row
        uint32_t m = 0;
#pragma unroll
        for (int v = 0; v < NV; ++v) m = max(m, most[v]);
        m = wave_max(m, 64);
        if constexpr (kWaves > 1) {
            __shared__ uint32_t part_m[kWaves];
            if ((t & 63) == 0) part_m[t >> 6] = m;
            __syncthreads();
            m = 0;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) m = max(m, part_m[w]);
        }
        const float s = group_scale(m);
        if (t == 0) a.scales[row] = s;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const srv_u32x2 d = quanta(h[v], m, s);
            if (skip[v] < 8) *(srv_u32x2_any *)((int8_t *)a.out + row * a.out_stride + off[v]) = d;
        }
        return;
    }
    // Groups of 8, 16, .. 512 columns in a row of whole runs are a power of two
    // of neighbouring lanes; any other goes through LDS, the maxima of integers
    // that its atomics take not depending on their order (8192 rows of bf16 in launches of
    // a graph: 5120 columns, groups of 128 61 us; 4992 columns, groups of 96 91).
    const bool by_lanes = cols % 8 == 0 && group >= 8 && group <= 512 && (group & (group - 1)) == 0;
    TML_DYNAMIC_LDS(uint32_t, all_most);
    uint32_t *lds_most = all_most + (threadIdx.x / TPR) * ngroups;
    if (!by_lanes) {
        for (int i = t; i < ngroups; i += TPR) lds_most[i] = 0;
        if constexpr (kWaves > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
        for (int v = 0; v < NV; ++v)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e >= skip[v]) atomicMax(&lds_most[(off[v] + e) / group], mag(h[v][e]));
        if constexpr (kWaves > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int i = t; i < ngroups; i += TPR) {
            const float s = group_scale(lds_most[i]);
            a.scales[row * ngroups + i] = s;
            lds_most[i] = __float_as_uint(s);
        }
        if constexpr (kWaves > 1) __syncthreads();
        else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
        srv_u32x2 d = {0, 0};
        if (by_lanes) {
            const uint32_t m = wave_max(most[v], group / 8);
            const float s = group_scale(m);
            if (off[v] % group == 0 && skip[v] == 0) a.scales[row * ngroups + off[v] / group] = s;
            d = quanta(h[v], m, s);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                d[e / 4] |= (uint32_t)(quantum(h[v][e], __uint_as_float(lds_most[(off[v] + e) / group])) & 0xFF) << (8 * (e % 4));
        }
        if (skip[v] < 8) *(srv_u32x2_any *)((int8_t *)a.out + row * a.out_stride + off[v]) = d;
    }
}

// Rows under eight columns, or too long for registers (256 rows of f32: 32768 columns 32
// us in registers, 14 of them of a lane in scratch; 40000 this way 79): the row is read once
// for its sum of squares, once more for the maxima of 8-bit outputs, and a last
// time to write, column by column.  Nothing is written before that last time,
// and a thread writes the columns it reads, so sum may be x or the residual.
__global__ __launch_bounds__(1024) void rmsnorm_any_kernel(RmsNormArgs a) {
    __shared__ float part[16];
    TML_DYNAMIC_LDS(uint32_t, lds_most);
    const int t = threadIdx.x;
    const int64_t row = blockIdx.x;
    const bool i8 = a.out_type == TML_TYPE_I8;
    const int ngroups = i8 ? (int)((a.cols + a.group - 1) / a.group) : 0;
    auto sum_at = [&](int64_t c) {
        float h = srv_load1(a.type, a.x, row * a.x_stride + c);
        if (a.residual != nullptr) h += srv_load1(a.type, a.residual, row * a.residual_stride + c);
        return h;
    };
    for (int i = t; i < ngroups; i += 1024) lds_most[i] = 0;
    float ss = 0.0f;
    for (int64_t c = t; c < a.cols; c += 1024) {
        const float h = sum_at(c);
        ss += h * h;
    }
    ss = wave_sum(ss);
    if ((t & 63) == 0) part[t >> 6] = ss;
    __syncthreads();
    ss = 0.0f;
    for (int w = 0; w < 16; ++w) ss += part[w];
    const float root = 1.0f / sqrtf(ss / (float)a.cols + a.eps);
    auto norm_at = [&](int64_t c, float h) { return a.weight != nullptr ? h * root * a.weight[c] : h * root; };
    if (i8) {
        for (int64_t c = t; c < a.cols; c += 1024) atomicMax(&lds_most[c / a.group], mag(norm_at(c, sum_at(c))));
        __syncthreads();
        for (int i = t; i < ngroups; i += 1024) {
            const float s = group_scale(lds_most[i]);
            a.scales[row * ngroups + i] = s;
            lds_most[i] = __float_as_uint(s);
        }
        __syncthreads();
    }
    for (int64_t c = t; c < a.cols; c += 1024) {
        const float h = sum_at(c), y = norm_at(c, h);
        if (a.sum != nullptr) srv_store1(a.type, a.sum, row * a.sum_stride + c, h);
        if (i8) {
            ((int8_t *)a.out)[row * a.out_stride + c] = (int8_t)quantum(y, __uint_as_float(lds_most[c / a.group]));
        } else {
            srv_store1(a.out_type, a.out, row * a.out_stride + c, y);
        }
    }
}

constexpr int64_t kMaxGroups = 16384;  // maxima in LDS, 64 KiB

// Rows of one launch, of workgroups of `threads` that take rows_wg rows each: a
// grid has fewer than 2^32 threads (a larger one is cut without an error).
int64_t launch_rows(int threads, int rows_wg) { return (int64_t)(0xFFFFFFFFu / (unsigned)threads) * rows_wg; }

RmsNormArgs rows_from(const RmsNormArgs &a, int64_t r0, int64_t rows) {
    RmsNormArgs p = a;
    const int64_t size = type_bytes(a.type), groups = a.out_type == TML_TYPE_I8 ? (a.cols + a.group - 1) / a.group : 0;
    p.rows = rows;
    p.x = (const char *)a.x + r0 * a.x_stride * size;
    if (a.residual != nullptr) p.residual = (const char *)a.residual + r0 * a.residual_stride * size;
    if (a.sum != nullptr) p.sum = (char *)a.sum + r0 * a.sum_stride * size;
    p.out = (char *)a.out + r0 * a.out_stride * type_bytes(a.out_type);
    if (groups > 0) p.scales = a.scales + r0 * groups;
    return p;
}

template <int T>
Status launch_type(const RmsNormArgs &all, hipStream_t s) {
    const int64_t groups = all.out_type == TML_TYPE_I8 ? (all.cols + all.group - 1) / all.group : 0;
    const int64_t runs = (all.cols + 7) / 8;
    const bool any = all.cols < 8 || runs > 4 * 1024;
    // A wave a row where that leaves enough waves to fill the GPU; otherwise a
    // workgroup a row, whose four waves share its latency.
    const bool wave = runs <= 64 || (runs <= 256 && all.rows >= 4 * (int64_t)device_cus());
    const int tpr = any ? 1024 : wave ? 64 : runs <= 1024 ? 256 : 1024;
    const int nv = (int)((runs + tpr - 1) / tpr), rows_wg = tpr == 64 ? 4 : 1;
    const dim3 block(tpr < 256 ? 256 : tpr);
    const size_t lds = any || groups > 1 ? (size_t)groups * rows_wg * 4 : 0;
    const int64_t most = launch_rows((int)block.x, rows_wg);
    for (int64_t r0 = 0; r0 < all.rows; r0 += most) {
        const RmsNormArgs a = rows_from(all, r0, std::min(most, all.rows - r0));
        const dim3 grid((unsigned)((a.rows + rows_wg - 1) / rows_wg));
#define TML_NORM(TPR, NV) rmsnorm_kernel<T, TPR, NV><<<grid, block, lds, s>>>(a)
        if (any) {
            rmsnorm_any_kernel<<<grid, block, lds, s>>>(a);
        } else if (tpr == 64) {
            if (nv == 1) TML_NORM(64, 1);
            else if (nv == 2) TML_NORM(64, 2);
            else if (nv == 3) TML_NORM(64, 3);
            else TML_NORM(64, 4);
        } else if (tpr == 256) {
            if (nv == 1) TML_NORM(256, 1);
            else if (nv == 2) TML_NORM(256, 2);
            else if (nv == 3) TML_NORM(256, 3);
            else TML_NORM(256, 4);
        } else {
            if (nv <= 2) TML_NORM(1024, 2);
            else TML_NORM(1024, 4);
        }
#undef TML_NORM
        TML_HIP_TRY(hipGetLastError());
    }
    return Status::Ok();
}

}  // namespace

Status launch_rmsnorm(const RmsNormArgs &in, hipStream_t s) {
    RmsNormArgs a = in;
    if (!float_type(a.type)) return Status::Err(TML_ERR_INVALID_FORMAT, "rmsnorm: x must be f32, f16 or bf16");
    if (!float_type(a.out_type) && a.out_type != TML_TYPE_I8)
        return Status::Err(TML_ERR_INVALID_FORMAT, "rmsnorm: the output must be f32, f16, bf16 or 8 bits");
    if (a.rows < 0 || a.cols < 0) return Status::Err(TML_ERR_INVALID_SHAPE, "negative matrix dimension");
    if (a.rows == 0 || a.cols == 0) return Status::Ok();
    if (a.rows > 0x7FFFFFFF || a.cols > 0x7FFFFFFF)
        return Status::Err(TML_ERR_INVALID_SHAPE, "rmsnorm: rows and columns must be below 2^31");
    if (a.x == nullptr || a.out == nullptr) return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    const int64_t m = a.rows > 1 ? a.cols : 0;  // strides of a single row are not used
    if (a.x_stride < m || a.out_stride < m || (a.residual != nullptr && a.residual_stride < m) ||
        (a.sum != nullptr && a.sum_stride < m))
        return Status::Err(TML_ERR_INVALID_SHAPE, "rmsnorm: a row stride is shorter than the row");
    if (a.out_type == TML_TYPE_I8) {
        if (a.scales == nullptr) return Status::Err(TML_ERR_INVALID_ARG, "rmsnorm: 8-bit output needs scales");
        if (a.group < 0) return Status::Err(TML_ERR_INVALID_SHAPE, "rmsnorm: negative group");
        if (a.group == 0 || a.group > a.cols) a.group = a.cols;
        if ((a.cols + a.group - 1) / a.group > kMaxGroups)
            return Status::Err(TML_ERR_INVALID_SHAPE, "rmsnorm: more than 16384 groups a row");
    }
    if (a.type == TML_TYPE_F32) return launch_type<TML_TYPE_F32>(a, s);
    if (a.type == TML_TYPE_F16) return launch_type<TML_TYPE_F16>(a, s);
    return launch_type<TML_TYPE_BF16>(a, s);
}

}  // namespace tml
