// logprobs.hip -- what logits say of tokens: log probabilities of given ones, the
// entropy, the most likely ones.
//
//   m = max x,  S = sum e^(x - m),  T = sum e^(x - m) (x - m)
//   log p = (x - m) - log S,  entropy = log S - T / S
//
// A workgroup takes a row.  One pass keeps m, S and T in every lane (a lane's own
// maximum: it rises a few times a row) and joins them at the end.  2048 rows of 51866 bf16
// logits take 42 us, 5.1 TB/s: bound by memory.  Four f32 rows with the five best take 12 us,
// most of it the instructions of one CU a row (some nine an element); a row on more CUs would
// take a second launch and a workspace to save about a third of that.
//
// The `top` best, by value and then by the lower index, from the lanes' own best: in each
// of w waves at least n / w elements reach the (n / w)-th largest of them, so n of the row
// reach the least of the waves' such values, T, and a second pass over the row (out of the
// caches) collects the few that do.  Each of them then counts those before it, which is its
// place.  Where they are more than LDS holds, the n-th of those held is the next T.
#include "serving.hpp"

#include <algorithm>

namespace tml {
namespace {

constexpr int kHeld = 1024;  // candidates in LDS
constexpr float kLowest = -0x1.fffffep127f;
// A distance of logits past which e^ of it is zero, short of what a sum times it overflows at.
constexpr float kFar = -1e20f;

// The order of a value and its index as one number: larger first, equal values by index.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t index) {
    const uint32_t u = __float_as_uint(x + 0.0f);  // (zeros alike)
    return (uint64_t)(u ^ ((u >> 31) != 0u ? 0xFFFFFFFFu : 0x80000000u)) << 32 | (0xFFFFFFFFu - index);
}
__device__ __forceinline__ float value_of(uint64_t key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u ^ ((u >> 31) != 0u ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint32_t index_of(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

struct Sums {
    float m, s, t;
};
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    const float m = fmaxf(a.m, b.m), da = a.m - m, db = b.m - m;
    const float fa = __builtin_amdgcn_exp2f(da * kLog2E), fb = __builtin_amdgcn_exp2f(db * kLog2E);
    return {m, a.s * fa + b.s * fb, (a.t + a.s * fmaxf(da, kFar)) * fa + (b.t + b.s * fmaxf(db, kFar)) * fb};
}

template <int T, int WAVES, bool TOP>
__global__ __launch_bounds__(64 * WAVES) void logprobs_kernel(LogprobsArgs a) {
    constexpr int kThreads = 64 * WAVES, kAhead = 4;
    __shared__ Sums wave_sums[WAVES];
    __shared__ uint64_t wave_key[WAVES];
    __shared__ uint64_t held[TOP ? kHeld : 1];
    __shared__ int count;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = blockIdx.x, at = row * a.stride;
    const unsigned cols = (unsigned)a.cols, chunks = cols / 8, rest = cols % 8;

    Sums sum{kLowest, 0.0f, 0.0f};
    float best = -INFINITY;  // of this lane, NaN aside
    auto take = [&](const auto &v) {
        constexpr int N = sizeof v / sizeof(float);
        float most = v[0];
#pragma unroll
        for (int e = 1; e < N; ++e) most = fmaxf(most, v[e]);
        if (most > sum.m) {
            const float d = sum.m - most, f = __builtin_amdgcn_exp2f(d * kLog2E);
            sum = {most, sum.s * f, (sum.t + sum.s * fmaxf(d, kFar)) * f};
        }
        if (TOP) best = fmaxf(best, most);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const float y = v[e] - sum.m, p = __builtin_amdgcn_exp2f(y * kLog2E);
            sum.s += p;
            sum.t = fmaf(p, fmaxf(y, kFar), sum.t);
        }
    };
    for (unsigned c = threadIdx.x; c < chunks; c += kAhead * kThreads) {
        SrvRaw<T> raw[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) raw[u] = srv_load8<T>(a.logits, at + 8 * (int64_t)min(c + u * kThreads, chunks - 1));
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            if (c + u * kThreads < chunks) {
                float v[8];
                srv_floats<T>(raw[u], v);
                take(v);
            }
    }
    if (threadIdx.x < rest) {  // the odd end, an element a lane
        const float v[1] = {srv_load1(T, a.logits, at + 8 * (int64_t)chunks + threadIdx.x)};
        take(v);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) sum = join(sum, {__shfl_xor(sum.m, o), __shfl_xor(sum.s, o), __shfl_xor(sum.t, o)});
    if (lane == 0) wave_sums[wave] = sum;
    if constexpr (TOP) {
        // the k-th largest of the lanes' best, bit by bit (that of a lane without elements is -inf)
        const uint32_t key = (uint32_t)(key_of(best, 0) >> 32);
        const int k = ((int)a.top + WAVES - 1) / WAVES;
        uint32_t kth = 0;
#pragma unroll
        for (uint32_t bit = 1u << 31; bit != 0; bit >>= 1)
            if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(key >= (kth | bit))) >= k) kth |= bit;
        if (lane == 0) wave_key[wave] = (uint64_t)kth << 32;
        if (threadIdx.x == 0) count = 0;
    }
    __syncthreads();
    sum = wave_sums[lane % WAVES];
#pragma unroll
    for (int o = 1; o < WAVES; o <<= 1) sum = join(sum, {__shfl_xor(sum.m, o), __shfl_xor(sum.s, o), __shfl_xor(sum.t, o)});
    const float log_s = logf(sum.s);
    const bool none = sum.s == 0.0f;  // no logit but -inf
    if (threadIdx.x == 0) {
        if (a.tokens != nullptr && a.logprobs != nullptr) {
            const int token = a.tokens[row];
            float r = 0.0f;
            if (token >= 0 && (unsigned)token < cols) r = none ? -INFINITY : srv_load1(T, a.logits, at + token) - sum.m - log_s;
            a.logprobs[row] = r;
        }
        if (a.entropy != nullptr) a.entropy[row] = none ? 0.0f : fmaxf(log_s - sum.t / sum.s, 0.0f) + (sum.s - sum.s);
    }
    if constexpr (TOP) {
        uint64_t least = wave_key[0];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) least = min(least, wave_key[w]);
        const int n = (int)a.top;
        int found;
        for (;;) {
            const float least_x = value_of(least);
            auto offer = [&](float x, unsigned index) {
                if (x >= least_x) {
                    const uint64_t key = key_of(x, index);
                    if (key >= least) {
                        const int to = __hip_atomic_fetch_add(&count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
                        if (to < kHeld) held[to] = key;
                    }
                }
            };
            for (unsigned c = threadIdx.x; c < chunks; c += kThreads) {
                float v[8];
                srv_floats<T>(srv_load8<T>(a.logits, at + 8 * (int64_t)c), v);
                float most = v[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) most = fmaxf(most, v[e]);
                if (most >= least_x)
#pragma unroll
                    for (int e = 0; e < 8; ++e) offer(v[e], 8 * c + e);
            }
            if (threadIdx.x < rest) offer(srv_load1(T, a.logits, at + 8 * (int64_t)chunks + threadIdx.x), 8 * chunks + threadIdx.x);
            __syncthreads();
            found = count;
            if (found <= kHeld) break;
            // too many: the n-th of those held
            __syncthreads();
            for (int i = threadIdx.x; i < kHeld; i += kThreads) {
                const uint64_t key = held[i];
                int before = 0;
                for (int j = 0; j < kHeld; ++j) before += held[j] > key;
                if (before == n - 1) wave_key[0] = key;
            }
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
            least = wave_key[0];
        }
        for (int i = threadIdx.x; i < found; i += kThreads) {
            const uint64_t key = held[i];
            int before = 0;
            for (int j = 0; j < found; ++j) before += held[j] > key;
            if (before < n) {
                if (a.top_ids != nullptr) a.top_ids[row * n + before] = (int)index_of(key);
                if (a.top_logprobs != nullptr) a.top_logprobs[row * n + before] = none ? -INFINITY : value_of(key) - sum.m - log_s;
            }
        }
        for (int i = found + threadIdx.x; i < n; i += kThreads) {
            if (a.top_ids != nullptr) a.top_ids[row * n + i] = -1;
            if (a.top_logprobs != nullptr) a.top_logprobs[row * n + i] = -INFINITY;
        }
    }
}

template <int T, int WAVES>
void launch_rows(const LogprobsArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.rows), block(64 * WAVES);
    if (a.top > 0) logprobs_kernel<T, WAVES, true><<<grid, block, 0, s>>>(a);
    else logprobs_kernel<T, WAVES, false><<<grid, block, 0, s>>>(a);
}

// Waves of a row: as many as have elements for every lane (else the best of a lane say little:
// 2048 columns, top 20, 16 waves 27 us), and sixteen only where rows leave CUs empty.  Measured,
// bf16, top 20, in us with 1 / 4 / 16 waves:
//                 4 rows               4096 rows
//   2048 columns  7.5 /  5.4 / 27      12 / 15 / 288
//   8192          14  /  7.3 /  7.6    28 / 26 /  66
//   32768         34  / 13   / 10      84 / 81 / 105
// and for 512 rows of 32768 38 / 18.1 / 17.2.  f32 is within a tenth of that where memory does not bound it
// (2048 rows of 32768, top 20, 89 / 85 / 82).  Without alternatives the same rule is right by smaller
// steps: 4 rows 3.7 / 4.1, 6.1 / 5.0 / 4.3 and 16.2 / 6.3 / 5.9; 2048 rows 4.9 / 6.2, 10.2 / 10.7 / 17.9 and 27.7 / 26.3 / 29.7.
template <int T>
void launch_waves(const LogprobsArgs &a, hipStream_t s) {
    if (a.cols <= 2048) launch_rows<T, 1>(a, s);
    else if (a.cols <= 8192 || a.rows >= 2 * device_cus()) launch_rows<T, 4>(a, s);
    else launch_rows<T, 16>(a, s);
}

}  // namespace

Status launch_token_logprobs(const LogprobsArgs &in, hipStream_t s) {
    if (!float_type(in.type)) return Status::Err(TML_ERR_INVALID_FORMAT, "token logprobs: logits must be f32, f16 or bf16");
    if (in.rows < 0 || in.cols < 0 || in.top < 0) return Status::Err(TML_ERR_INVALID_SHAPE, "token logprobs: negative size");
    if (in.top > 64) return Status::Err(TML_ERR_INVALID_SHAPE, "token logprobs: at most 64 alternatives");
    if (in.cols >= (int64_t)1 << 31) return Status::Err(TML_ERR_INVALID_SHAPE, "token logprobs: columns must be below 2^31");
    if (in.rows == 0) return Status::Ok();
    if (in.cols > 0 && in.logits == nullptr) return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    if ((in.tokens == nullptr) != (in.logprobs == nullptr)) return Status::Err(TML_ERR_INVALID_ARG, "token logprobs: tokens and logprobs go together");
    if (in.top > 0 && in.top_ids == nullptr && in.top_logprobs == nullptr) return Status::Err(TML_ERR_INVALID_ARG, "null pointer");
    if (in.rows > 1 && in.stride < in.cols) return Status::Err(TML_ERR_INVALID_SHAPE, "token logprobs: a row stride is shorter than the row");
    const int64_t most = (int64_t)1 << 21;  // rows of a launch: fewer than 2^32 threads
    for (int64_t r = 0; r < in.rows; r += most) {
        LogprobsArgs a = in;
        a.rows = std::min(most, in.rows - r);
        a.logits = (const char *)in.logits + r * in.stride * type_bytes(in.type);
        if (in.tokens != nullptr) {
            a.tokens += r;
            a.logprobs += r;
        }
        if (in.entropy != nullptr) a.entropy += r;
        if (in.top_ids != nullptr) a.top_ids += r * in.top;
        if (in.top_logprobs != nullptr) a.top_logprobs += r * in.top;
        if (a.type == TML_TYPE_F32) launch_waves<TML_TYPE_F32>(a, s);
        else if (a.type == TML_TYPE_F16) launch_waves<TML_TYPE_F16>(a, s);
        else launch_waves<TML_TYPE_BF16>(a, s);
        TML_HIP_TRY(hipGetLastError());
    }
    return Status::Ok();
}

}  // namespace tml
