// CPU emulation of a workgroup's lanes -- test infrastructure for the serving
// operators, whose control flow goes through shuffles, votes and LDS.
//
// The runtime API, the buffer resources and the allocations are those of
// ../../hip/hip_runtime.h.  What differs: every thread of a workgroup runs on a
// stack of its own and stops where it meets others,
//   __syncthreads                       until every thread that is left has come
//   shuffles, votes, readlane,          until every lane of the wave that is still on
//   matrix instructions, wave           its way to the same place has come; the data
//   fences and barriers                 is then that of the lanes that did come
// so shuffles, votes and matrix products give what the GPU gives (products are
// summed in fp32, one after another), results mean something, and address
// arithmetic that depends on data is the real one.  A shuffle or readlane
// that asks a lane that is not there gets a pattern that is no number.
//
// LDS arrays keep what the workgroup before left in them, and a launch's dynamic
// LDS starts as that pattern.  With EMU_REVERSE=1 the blocks of a grid run from the
// last to the first and so do the waves of a block.  Launches that HIP refuses or cuts
// (2^32 work items or more in a dimension, over 1024 threads a block, over 160 KiB of
// dynamic LDS) do not run and are reported by hipGetLastError.
//
// NOT emulated: the memory model.  A thread sees what others wrote before it ran on,
// so a missing barrier shows only where the order of waves or blocks makes it.
#pragma once

#define __shfl_xor tml_emu_plain_shfl_xor
#define __shfl_up tml_emu_plain_shfl_up
#define __shfl tml_emu_plain_shfl
#define __syncthreads tml_emu_plain_syncthreads
#define __any tml_emu_plain_any
#define __builtin_amdgcn_ballot_w64 tml_emu_plain_ballot
#define __builtin_amdgcn_readfirstlane tml_emu_plain_readfirstlane
#define __builtin_amdgcn_readlane tml_emu_plain_readlane
#define __builtin_amdgcn_wave_barrier tml_emu_plain_wave_barrier
#define __builtin_amdgcn_fence tml_emu_plain_fence
#define __builtin_amdgcn_mfma_f32_16x16x4f32 tml_emu_plain_mfma_f32
#define __builtin_amdgcn_mfma_f32_16x16x32_bf16 tml_emu_plain_mfma_bf16
#define __builtin_amdgcn_mfma_f32_16x16x32_f16 tml_emu_plain_mfma_f16
#define __builtin_amdgcn_mfma_f32_32x32x2f32 tml_emu_plain_mfma_f32_32
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16 tml_emu_plain_mfma_bf16_32
#define __builtin_amdgcn_mfma_f32_32x32x16_f16 tml_emu_plain_mfma_f16_32
#define __builtin_amdgcn_ds_read_tr16_b64_v4i16 tml_emu_plain_read_tr
#define __builtin_amdgcn_permlane32_swap tml_emu_plain_permlane32_swap
#define __builtin_amdgcn_permlane16_swap tml_emu_plain_permlane16_swap
#define __builtin_amdgcn_mfma_i32_16x16x64_i8 tml_emu_plain_mfma_i8
#define tml_emu_launcher tml_emu_plain_launcher
#define tml_emu_launch tml_emu_plain_launch
#define hipGetLastError tml_emu_plain_hipGetLastError
#include "../../hip/hip_runtime.h"
#undef __shfl_xor
#undef __shfl_up
#undef __shfl
#undef __syncthreads
#undef __any
#undef __builtin_amdgcn_ballot_w64
#undef __builtin_amdgcn_readfirstlane
#undef __builtin_amdgcn_readlane
#undef __builtin_amdgcn_wave_barrier
#undef __builtin_amdgcn_fence
#undef __builtin_amdgcn_mfma_f32_16x16x4f32
#undef __builtin_amdgcn_mfma_f32_16x16x32_bf16
#undef __builtin_amdgcn_mfma_f32_16x16x32_f16
#undef __builtin_amdgcn_mfma_f32_32x32x2f32
#undef __builtin_amdgcn_mfma_f32_32x32x16_bf16
#undef __builtin_amdgcn_mfma_f32_32x32x16_f16
#undef __builtin_amdgcn_ds_read_tr16_b64_v4i16
#undef __builtin_amdgcn_permlane32_swap
#undef __builtin_amdgcn_permlane16_swap
#undef __builtin_amdgcn_mfma_i32_16x16x64_i8
#undef tml_emu_launcher
#undef tml_emu_launch
#undef hipGetLastError

#include <functional>

// ------------------------------------------------------ lanes (lanes_main.cpp)
// What the lanes of a wave that met at one place brought there.
struct tml_lane_meeting {
    uint64_t here = 0;            // the lanes that came
    unsigned char data[64][32];  // what each brought
};
// Stops until the wave's lanes have met here; `data` is copied.
const tml_lane_meeting &tml_lane_meet(const void *place, const void *data, size_t bytes);
void tml_lane_block_barrier();
bool tml_lane_run(dim3 grid, dim3 block, size_t lds, const std::function<void()> &body);

inline hipError_t &tml_lane_error() {
    static hipError_t e = hipSuccess;
    return e;
}
inline hipError_t tml_lane_last_error() {
    const hipError_t e = tml_lane_error();
    tml_lane_error() = hipSuccess;
    return e;
}
#define hipGetLastError tml_lane_last_error

template <typename... P>
struct tml_lane_launcher {
    void (*k)(P...);
    dim3 g, b;
    size_t shmem;
    template <typename... A>
    void operator()(A &&...args) const {
        ++tml_emu_launches;
        if (!tml_lane_run(g, b, shmem, [&] { k(args...); })) tml_lane_error() = hipErrorInvalidValue;
    }
};
template <typename... P>
tml_lane_launcher<P...> tml_emu_launch(void (*k)(P...), dim3 g, dim3 b, size_t shmem = 0, hipStream_t = nullptr) {
    return {k, g, b, shmem};
}

// One copy of each call in the program, so that lanes meet by its address.
#define TML_LANE_OP __attribute__((noinline, noduplicate))

inline void __syncthreads() { tml_lane_block_barrier(); }

template <typename T>
inline T tml_lane_from(const tml_lane_meeting &m, unsigned lane) {
    static_assert(sizeof(T) <= 32, "a lane brings at most 32 bytes");
    T v;
    if (lane < 64 && (m.here >> lane & 1)) std::memcpy(&v, m.data[lane], sizeof v);
    else std::memset(&v, 0xFF, sizeof v);
    return v;
}
template <typename T>
TML_LANE_OP T __shfl_xor(T v, int mask, int = 64) {
    const unsigned lane = tml_emu_lane();
    return tml_lane_from<T>(tml_lane_meet(__builtin_return_address(0), &v, sizeof v), lane ^ (unsigned)mask);
}
template <typename T>
TML_LANE_OP T __shfl_up(T v, int by, int = 64) {
    const unsigned lane = tml_emu_lane();
    const tml_lane_meeting &m = tml_lane_meet(__builtin_return_address(0), &v, sizeof v);
    return (int)lane < by ? v : tml_lane_from<T>(m, lane - (unsigned)by);
}
template <typename T>
TML_LANE_OP T __shfl(T v, int from, int = 64) {
    return tml_lane_from<T>(tml_lane_meet(__builtin_return_address(0), &v, sizeof v), (unsigned)from & 63u);
}
TML_LANE_OP inline uint64_t __builtin_amdgcn_ballot_w64(bool v) {
    const tml_lane_meeting &m = tml_lane_meet(__builtin_return_address(0), &v, sizeof v);
    uint64_t all = 0;
    for (unsigned l = 0; l < 64; ++l)
        if (m.here >> l & 1) all |= (uint64_t)(m.data[l][0] & 1) << l;
    return all;
}
template <typename T>
TML_LANE_OP T __builtin_amdgcn_readfirstlane(T v) {
    const tml_lane_meeting &m = tml_lane_meet(__builtin_return_address(0), &v, sizeof v);
    return tml_lane_from<T>(m, (unsigned)__builtin_ctzll(m.here));
}
template <typename T>
TML_LANE_OP T __builtin_amdgcn_readlane(T v, int from) {
    return tml_lane_from<T>(tml_lane_meet(__builtin_return_address(0), &v, sizeof v), (unsigned)from);
}
TML_LANE_OP inline void __builtin_amdgcn_wave_barrier() {
    ++tml_emu_wave_barriers;
    tml_lane_meet(__builtin_return_address(0), nullptr, 0);
}
TML_LANE_OP inline void __builtin_amdgcn_fence(int, const char *) { tml_lane_meet(__builtin_return_address(0), nullptr, 0); }

// Matrix instructions: lane l brings A row l % 16 and B column l % 16, the k of its
// group l / 16, and gets rows 4 (l / 16) + i of column l % 16.
inline void tml_lane_whole_wave(const tml_lane_meeting &m) {
    if (m.here != ~0ull) {
        std::fprintf(stderr, "EMU ERROR: a matrix instruction with lanes missing (%016llx)\n", (unsigned long long)m.here);
        std::abort();
    }
}
template <typename E, typename ACC, int N>
inline ACC tml_lane_product(const tml_lane_meeting &m, ACC c) {
    tml_lane_whole_wave(m);
    const unsigned lane = tml_emu_lane();
    for (unsigned i = 0; i < 4; ++i)
        for (unsigned g = 0; g < 4; ++g) {
            E a[N], b[N];
            std::memcpy(a, m.data[16 * g + 4 * (lane / 16) + i], sizeof a);
            std::memcpy(b, m.data[16 * g + lane % 16] + sizeof a, sizeof b);
            for (int k = 0; k < N; ++k) {
                if constexpr (sizeof(E) == 1) c[i] += (int)a[k] * (int)b[k];
                else c[i] += (float)a[k] * (float)b[k];
            }
        }
    return c;
}
template <typename V>
struct tml_lane_pair {
    V a, b;
};
TML_LANE_OP inline tml_emu_f32x4 __builtin_amdgcn_mfma_f32_16x16x4f32(float a, float b, tml_emu_f32x4 c, int, int, int) {
    const tml_lane_pair<float> ab{a, b};
    return tml_lane_product<float, tml_emu_f32x4, 1>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
TML_LANE_OP inline tml_emu_f32x4 __builtin_amdgcn_mfma_f32_16x16x32_bf16(tml_emu_bf16x8 a, tml_emu_bf16x8 b, tml_emu_f32x4 c, int, int, int) {
    const tml_lane_pair<tml_emu_bf16x8> ab{a, b};
    return tml_lane_product<__bf16, tml_emu_f32x4, 8>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
TML_LANE_OP inline tml_emu_f32x4 __builtin_amdgcn_mfma_f32_16x16x32_f16(tml_emu_f16x8 a, tml_emu_f16x8 b, tml_emu_f32x4 c, int, int, int) {
    const tml_lane_pair<tml_emu_f16x8> ab{a, b};
    return tml_lane_product<_Float16, tml_emu_f32x4, 8>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
TML_LANE_OP inline tml_emu_i32x4 __builtin_amdgcn_mfma_i32_16x16x64_i8(tml_emu_i32x4 a, tml_emu_i32x4 b, tml_emu_i32x4 c, int, int, int) {
    const tml_lane_pair<tml_emu_i32x4> ab{a, b};
    return tml_lane_product<int8_t, tml_emu_i32x4, 16>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
// The 32 x 32 ones: A row l % 32, B column l % 32, the k of half l / 32; rows
// 8 j + 4 (l / 32) + i of column l % 32, in that order.
template <typename E, int N>
inline tml_emu_f32x16 tml_lane_product32(const tml_lane_meeting &m, tml_emu_f32x16 c) {
    tml_lane_whole_wave(m);
    const unsigned lane = tml_emu_lane();
    for (unsigned i = 0; i < 16; ++i)
        for (unsigned g = 0; g < 2; ++g) {
            E a[N], b[N];
            std::memcpy(a, m.data[32 * g + 8 * (i / 4) + 4 * (lane / 32) + i % 4], sizeof a);
            std::memcpy(b, m.data[32 * g + lane % 32] + sizeof a, sizeof b);
            for (int k = 0; k < N; ++k) c[i] += (float)a[k] * (float)b[k];
        }
    return c;
}
TML_LANE_OP inline tml_emu_f32x16 __builtin_amdgcn_mfma_f32_32x32x2f32(float a, float b, tml_emu_f32x16 c, int, int, int) {
    const tml_lane_pair<float> ab{a, b};
    return tml_lane_product32<float, 1>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
TML_LANE_OP inline tml_emu_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_bf16(tml_emu_bf16x8 a, tml_emu_bf16x8 b, tml_emu_f32x16 c, int, int, int) {
    const tml_lane_pair<tml_emu_bf16x8> ab{a, b};
    return tml_lane_product32<__bf16, 8>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
TML_LANE_OP inline tml_emu_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_f16(tml_emu_f16x8 a, tml_emu_f16x8 b, tml_emu_f32x16 c, int, int, int) {
    const tml_lane_pair<tml_emu_f16x8> ab{a, b};
    return tml_lane_product32<_Float16, 8>(tml_lane_meet(__builtin_return_address(0), &ab, sizeof ab), c);
}
// Lane i of 16 brings row i / 4, columns 4 (i % 4) and on, of a 4 x 16 block; gets column i.
typedef short tml_emu_s16x4 __attribute__((ext_vector_type(4)));
TML_LANE_OP inline tml_emu_s16x4 __builtin_amdgcn_ds_read_tr16_b64_v4i16(__attribute__((address_space(3))) tml_emu_s16x4 *p) {
    const tml_emu_s16x4 mine = *(const tml_emu_s16x4 *)p;
    const tml_lane_meeting &m = tml_lane_meet(__builtin_return_address(0), &mine, sizeof mine);
    tml_lane_whole_wave(m);
    const unsigned lane = tml_emu_lane();
    tml_emu_s16x4 out;
    for (unsigned j = 0; j < 4; ++j) {
        tml_emu_s16x4 four;
        std::memcpy(&four, m.data[(lane & ~15u) + 4 * j + lane % 16 / 4], sizeof four);
        out[j] = four[lane % 4];
    }
    return out;
}
// The upper half of the first and the lower half of the second change places.
TML_LANE_OP inline tml_emu_u32x2_swap __builtin_amdgcn_permlane32_swap(unsigned a, unsigned b, bool, bool) {
    const unsigned mine[2] = {a, b};
    const tml_lane_meeting &m = tml_lane_meet(__builtin_return_address(0), mine, sizeof mine);
    const unsigned lane = tml_emu_lane();
    unsigned other[2];
    std::memcpy(other, m.data[lane ^ 32], sizeof other);
    return lane < 32 ? tml_emu_u32x2_swap{a, other[0]} : tml_emu_u32x2_swap{other[1], b};
}
// The same for the odd 16s of the first and the even 16s of the second.
TML_LANE_OP inline tml_emu_u32x2_swap __builtin_amdgcn_permlane16_swap(unsigned a, unsigned b, bool, bool) {
    const unsigned mine[2] = {a, b};
    const tml_lane_meeting &m = tml_lane_meet(__builtin_return_address(0), mine, sizeof mine);
    const unsigned lane = tml_emu_lane();
    unsigned other[2];
    std::memcpy(other, m.data[lane ^ 16], sizeof other);
    return (lane & 16) == 0 ? tml_emu_u32x2_swap{a, other[0]} : tml_emu_u32x2_swap{other[1], b};
}
