// Driver of the lane emulation (lanes/hip/hip_runtime.h): runs the calls of a
// program file through the library's C ABI and writes the buffers back.
//
//   emu_lanes PROGRAM DATA
// PROGRAM holds, one a line,
//   buf BYTES        a device allocation of exactly that size, filled from DATA
//                    (where the buffers follow each other)
//   call NAME ARG..  a call of tml_hip_NAME_dev; an ARG is a number, `bI+OFF` (byte
//                    OFF of buffer I) or `null`
// Output: "ret CODE ALLOCATIONS MESSAGE" for each call, ALLOCATIONS being the device
// allocations alive after it; DATA is overwritten with the buffers' contents.
// ASan / UBSan end the process at the first bad access.
#include <fstream>
#include <iostream>
#include <sstream>
#include <string>
#include <tuple>
#include <utility>

#include <sanitizer/asan_interface.h>
#include <sanitizer/common_interface_defs.h>
#include <sys/mman.h>

#include "lanes/hip/hip_runtime.h"
#include "tomoul_hip.h"

// ------------------------------------------------------------------ lanes
extern "C" void tml_lane_switch(void **from, void *to);
asm(R"(
.text
.globl tml_lane_switch
.type tml_lane_switch,@function
tml_lane_switch:
    pushq %rbp
    pushq %rbx
    pushq %r12
    pushq %r13
    pushq %r14
    pushq %r15
    movq %rsp, (%rdi)
    movq %rsi, %rsp
    popq %r15
    popq %r14
    popq %r13
    popq %r12
    popq %rbx
    popq %rbp
    ret
.size tml_lane_switch,.-tml_lane_switch
)");

namespace {

constexpr size_t kStack = 256 << 10;
constexpr unsigned kMost = 1024;
enum State { kReady, kMeeting, kBarrier, kDone };

struct Lane {
    char *stack = nullptr;
    void *sp = nullptr;
    State state = kDone;
    const void *place = nullptr;
    unsigned char data[32];
    void *fake = nullptr;
};
Lane lanes[kMost];
unsigned current;
tml_lane_meeting meetings[kMost / 64];
void *scheduler_sp, *scheduler_fake;
const void *scheduler_stack;
size_t scheduler_size;
const std::function<void()> *body;

void to_scheduler(bool last) {
    Lane &l = lanes[current];
    __sanitizer_start_switch_fiber(last ? nullptr : &l.fake, scheduler_stack, scheduler_size);
    tml_lane_switch(&l.sp, scheduler_sp);
    __sanitizer_finish_switch_fiber(lanes[current].fake, &scheduler_stack, &scheduler_size);
}

__attribute__((no_sanitize("address", "undefined"), noinline)) void lane_entry() {
    __sanitizer_finish_switch_fiber(nullptr, &scheduler_stack, &scheduler_size);
    (*body)();
    lanes[current].state = kDone;
    to_scheduler(true);
    __builtin_trap();
}

void resume(unsigned t) {
    Lane &l = lanes[t];
    current = t;
    threadIdx.x = t;
    l.state = kReady;
    __sanitizer_start_switch_fiber(&scheduler_fake, l.stack, kStack);
    tml_lane_switch(&scheduler_sp, l.sp);
    __sanitizer_finish_switch_fiber(scheduler_fake, nullptr, nullptr);
}

// Runs a wave until all its lanes are at the block's barrier or done.
void run_wave(unsigned first, unsigned n) {
    for (unsigned l = 0; l < n; ++l)
        if (lanes[first + l].state == kReady) resume(first + l);
    for (;;) {
        // Of the places where lanes wait, the first in the program: lanes that are past
        // a loop wait for those still in it.
        const void *place = nullptr;
        for (unsigned l = 0; l < n; ++l)
            if (lanes[first + l].state == kMeeting && (place == nullptr || lanes[first + l].place < place)) place = lanes[first + l].place;
        if (place == nullptr) return;
        tml_lane_meeting &m = meetings[first / 64];
        m.here = 0;
        for (unsigned l = 0; l < n; ++l)
            if (lanes[first + l].state == kMeeting && lanes[first + l].place == place) {
                m.here |= 1ull << l;
                std::memcpy(m.data[l], lanes[first + l].data, sizeof m.data[l]);
            }
        const uint64_t here = m.here;
        for (unsigned l = 0; l < n; ++l)
            if (here >> l & 1) resume(first + l);
    }
}

void run_block(unsigned n, bool reverse) {
    for (unsigned t = 0; t < n; ++t) {
        Lane &l = lanes[t];
        if (l.stack == nullptr) {
            l.stack = (char *)mmap(nullptr, kStack, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
            if (l.stack == MAP_FAILED) std::abort();
        }
        // (what the last block's entry left marked)
        __asan_unpoison_memory_region(l.stack + kStack - 4096, 4096);
        void **sp = (void **)(l.stack + kStack - 64);
        *--sp = nullptr;
        *--sp = (void *)&lane_entry;
        for (int i = 0; i < 6; ++i) *--sp = nullptr;
        l.sp = sp;
        l.state = kReady;
    }
    const unsigned waves = (n + 63) / 64;
    for (;;) {
        for (unsigned i = 0; i < waves; ++i) {
            const unsigned first = 64 * (reverse ? waves - 1 - i : i);
            run_wave(first, std::min(64u, n - first));
        }
        bool any = false;
        for (unsigned t = 0; t < n; ++t)
            if (lanes[t].state == kBarrier) {
                lanes[t].state = kReady;
                any = true;
            }
        if (!any) return;
    }
}

}  // namespace

const tml_lane_meeting &tml_lane_meet(const void *place, const void *data, size_t bytes) {
    Lane &l = lanes[current];
    l.state = kMeeting;
    l.place = place;
    if (bytes) std::memcpy(l.data, data, bytes);
    to_scheduler(false);
    return meetings[current / 64];
}

void tml_lane_block_barrier() {
    lanes[current].state = kBarrier;
    to_scheduler(false);
}

bool tml_lane_run(dim3 g, dim3 b, size_t lds, const std::function<void()> &kernel) {
    const uint64_t limit = (uint64_t)1 << 32;
    if (b.y != 1 || b.z != 1 || b.x == 0 || b.x > kMost || g.x == 0 || g.y == 0 || g.z == 0 || (uint64_t)g.x * b.x >= limit ||
        lds > 160 << 10)
        return false;
    const char *r = std::getenv("EMU_REVERSE");
    const bool reverse = r != nullptr && *r == '1';
    body = &kernel;
    gridDim = g;
    blockDim = b;
    std::vector<char> dyn(lds, (char)0xFF);
    tml_emu_dyn_buf() = lds ? &dyn : nullptr;
    const uint64_t blocks = (uint64_t)g.x * g.y * g.z;
    for (uint64_t i = 0; i < blocks; ++i) {
        const uint64_t at = reverse ? blocks - 1 - i : i;
        blockIdx.x = (unsigned)(at % g.x);
        blockIdx.y = (unsigned)(at / g.x % g.y);
        blockIdx.z = (unsigned)(at / g.x / g.y);
        run_block(b.x, reverse);
    }
    tml_emu_dyn_buf() = nullptr;
    return true;
}

// ------------------------------------------------------------------ calls
namespace {

std::vector<std::pair<char *, size_t>> bufs;

template <typename T>
T arg(const std::string &s) {
    if constexpr (std::is_pointer_v<T>) {
        if (s == "null") return nullptr;
        if (s[0] != 'b') return (T)(uintptr_t)std::stoull(s);  // (an address that no call may touch)
        const size_t plus = s.find('+');
        return (T)(bufs.at(std::stoul(s.substr(1, plus - 1))).first + std::stoll(s.substr(plus + 1)));
    } else if constexpr (std::is_floating_point_v<T>) {
        return (T)std::stod(s);
    } else {
        return (T)std::stoll(s);
    }
}
template <typename... P, size_t... I>
int call_with(int (*f)(P...), const std::vector<std::string> &a, std::index_sequence<I...>) {
    return f(arg<P>(a.at(I))...);
}
template <typename... P>
int call(int (*f)(P...), const std::vector<std::string> &a) {
    if (a.size() != sizeof...(P)) {
        std::cerr << "EMU ERROR: " << a.size() << " arguments for " << sizeof...(P) << "\n";
        std::abort();
    }
    return call_with(f, a, std::index_sequence_for<P...>());
}

}  // namespace

int main(int argc, char **argv) {
    if (argc != 3) return 2;
    std::ifstream program(argv[1]), data(argv[2], std::ios::binary);
    std::string line;
    while (std::getline(program, line)) {
        std::istringstream in(line);
        std::string op, name;
        in >> op >> name;
        if (op == "buf") {
            const size_t n = std::stoull(name);
            void *p = nullptr;
            if (hipMalloc(&p, n) != hipSuccess) return 3;
            data.read((char *)p, (std::streamsize)n);
            bufs.push_back({(char *)p, n});
            continue;
        }
        std::vector<std::string> a;
        for (std::string s; in >> s;) a.push_back(s);
        int rc = -1;
        if (name == "kv_plan") rc = call(tml_hip_kv_plan_dev, a);
        else if (name == "kv_store") rc = call(tml_hip_kv_store_dev, a);
        else if (name == "paged_attention") rc = call(tml_hip_paged_attention_dev, a);
        else if (name == "rmsnorm") rc = call(tml_hip_rmsnorm_dev, a);
        else if (name == "matvec_q4g") rc = call(tml_hip_matvec_q4g_dev, a);
        else if (name == "quantize_groups") rc = call(tml_hip_quantize_groups_dev, a);
        else if (name == "gemm") rc = call(tml_hip_gemm_dev, a);
        else return 4;
        std::cout << "ret " << rc << " " << tml_emu_allocs().size() << " " << (rc ? tml_hip_last_error() : "") << std::endl;
    }
    data.close();
    std::ofstream out(argv[2], std::ios::binary);
    for (auto &b : bufs) out.write(b.first, (std::streamsize)b.second);
    return 0;
}
