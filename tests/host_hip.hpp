// The part of HIP that the attention, plan, keep, norm and rotation kernels use, on the CPU (test infrastructure): it
// stands in the place of tqt_hip_common.hpp where tests/host_kernels.py builds those sources for the host. A workgroup's
// threads are coroutines. One runs until it meets the others of its wave (a move between lanes, a vote, a matrix
// instruction, a wave barrier) or of its workgroup (a barrier); which wave and lane goes first is drawn anew each time, so that
// an order that the kernel does not enforce shows. Loads from memory to LDS arrive at the wait for them, not before. Lanes
// of a wave that meet at different operations end the process.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <functional>
#include <vector>

#include "tqt_gfx950_common.h"

#define __device__
#define __host__
#define __global__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __shared__ static

using std::max;
using std::min;
inline long long max(int a, long long b) { return std::max<long long>(a, b); }
inline long long min(int a, long long b) { return std::min<long long>(a, b); }

struct dim3
{
    unsigned x, y, z;
    dim3(unsigned x_ = 1, unsigned y_ = 1, unsigned z_ = 1) : x(x_), y(y_), z(z_) {}
};
typedef void *hipStream_t;

namespace host_hip {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kWave = 64, kMostThreads = 1024;
constexpr size_t kStack = 256 << 10, kSlot = 64;

[[noreturn]] inline void fail(const char *what)
{
    fprintf(stderr, "host_hip: %s\n", what);
    abort();
}

enum State { kRuns, kAtWave, kAtBlock, kDone };

struct Thread
{
    void *sp;
    dim3 idx;
    State state;
    int kind;                 // of the operation that it waits at
    std::vector<char> stack;
    std::vector<std::pair<const void *, void *>> loads;  // to LDS, on their way
};

struct Machine
{
    Thread threads[kMostThreads];
    int count = 0;
    Thread *self = nullptr;
    void *scheduler = nullptr;
    const std::function<void()> *kernel = nullptr;
    dim3 block, grid, block_dim;
    alignas(64) char slot[kMostThreads / kWave][kWave][kSlot];  // what lanes bring, and what they all see
    alignas(64) char seen[kMostThreads / kWave][kWave][kSlot];
    uint64_t active[kMostThreads / kWave];
    bool any = false, any_seen = false;
    uint64_t random = 88172645463325252ull;
    uint64_t draw()
    {
        random ^= random << 13;
        random ^= random >> 7;
        return random ^= random << 17;
    }
};

inline Machine &machine()
{
    static Machine *m = new Machine;
    return *m;
}

// Saves this coroutine's registers and stack in *save and goes on with the one of `load`.
extern "C" void host_hip_switch(void **save, void *load);
asm(R"(
.pushsection .text
.weak host_hip_switch
.type host_hip_switch, @function
host_hip_switch:
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
.popsection
)");

inline void thread_main()
{
    Machine &m = machine();
    (*m.kernel)();
    m.self->state = kDone;
    host_hip_switch(&m.self->sp, m.scheduler);
    fail("a finished thread went on");
}

inline int lane()
{
    return static_cast<int>(machine().self - machine().threads) % kWave;
}
inline int wave()
{
    return static_cast<int>(machine().self - machine().threads) / kWave;
}

inline void wait(State state, int kind)
{
    Machine &m = machine();
    m.self->state = state;
    m.self->kind = kind;
    host_hip_switch(&m.self->sp, m.scheduler);
}

// Meets the wave's lanes; what each of them brought.
template <typename V>
struct Brought
{
    const char (*from)[kSlot];
    uint64_t active;
    const V &operator[](int l) const
    {
        if (((active >> l) & 1) == 0) {
            fail("a value of a lane that has finished");
        }
        return *reinterpret_cast<const V *>(from[l]);
    }
};

template <typename V>
inline Brought<V> meet(const V &v, int kind)
{
    static_assert(sizeof(V) <= kSlot, "");
    Machine &m = machine();
    const int w = wave(), l = lane();
    memcpy(m.slot[w][l], &v, sizeof(V));
    wait(kAtWave, kind);
    return {m.seen[w], m.active[w]};
}

inline void run_block(const std::function<void()> &kernel)
{
    Machine &m = machine();
    m.kernel = &kernel;
    for (int t = 0; t < m.count; ++t) {
        Thread &x = m.threads[t];
        x.stack.resize(kStack);
        x.state = kRuns;
        x.idx = dim3(t, 0, 0);
        x.loads.clear();
        // six registers, then the address that the switch returns to, with the stack as after a call
        uintptr_t top = (reinterpret_cast<uintptr_t>(x.stack.data()) + kStack) & ~uintptr_t(63);
        void **sp = reinterpret_cast<void **>(top - 8);
        *--sp = reinterpret_cast<void *>(&thread_main);
        for (int i = 0; i < 6; ++i) {
            *--sp = nullptr;
        }
        x.sp = sp;
    }
    const int waves = (m.count + kWave - 1) / kWave;
    for (;;) {
        bool ran = false, done = true;
        const int w0 = static_cast<int>(m.draw() % waves);
        for (int i = 0; i < waves; ++i) {
            const int w = (w0 + i) % waves, first = w * kWave, lanes = std::min(kWave, m.count - first);
            const int l0 = static_cast<int>(m.draw() % lanes), step = (m.draw() & 1) ? 1 : lanes - 1;
            for (int j = 0, l = l0; j < lanes; ++j, l = (l + step) % lanes) {
                Thread &x = m.threads[first + l];
                if (x.state == kRuns) {
                    m.self = &x;
                    host_hip_switch(&m.scheduler, x.sp);
                    ran = true;
                }
            }
            int at_wave = 0, at_block = 0, kind = 0;
            uint64_t active = 0;
            for (int l = 0; l < lanes; ++l) {
                const Thread &x = m.threads[first + l];
                if (x.state == kAtWave) {
                    if (at_wave++ > 0 && x.kind != kind) {
                        fail("lanes of a wave at different operations");
                    }
                    kind = x.kind;
                    active |= 1ull << l;
                }
                at_block += x.state == kAtBlock;
            }
            if (at_wave > 0 && at_block > 0) {
                fail("lanes of a wave at a barrier and at an operation of the wave");
            }
            if (at_wave > 0) {
                memcpy(m.seen[w], m.slot[w], sizeof(m.seen[w]));
                m.active[w] = active;
                for (int l = 0; l < lanes; ++l) {
                    Thread &x = m.threads[first + l];
                    x.state = x.state == kAtWave ? kRuns : x.state;
                }
                ran = true;
            }
        }
        bool barrier = true;
        for (int t = 0; t < m.count; ++t) {
            done &= m.threads[t].state == kDone;
            barrier &= m.threads[t].state == kDone || m.threads[t].state == kAtBlock;
        }
        if (done) {
            return;
        }
        if (barrier) {
            m.any_seen = m.any;
            m.any = false;
            for (int t = 0; t < m.count; ++t) {
                m.threads[t].state = m.threads[t].state == kAtBlock ? kRuns : kDone;
            }
        } else if (!ran) {
            fail("a workgroup that waits for ever");
        }
    }
}

inline void launch(dim3 grid, dim3 block, const std::function<void()> &kernel)
{
    Machine &m = machine();
    m.count = static_cast<int>(block.x);
    m.grid = grid;
    m.block_dim = block;
    if (m.count > kMostThreads || block.y != 1 || block.z != 1 || grid.z != 1 || grid.x == 0 || grid.y == 0) {
        fail("a launch that this file does not know");
    }
    const uint64_t blocks = static_cast<uint64_t>(grid.x) * grid.y;
    // any workgroup may be the first
    const uint64_t at0 = m.draw() % blocks;
    for (uint64_t i = 0; i < blocks; ++i) {
        const uint64_t at = (at0 + i) % blocks;
        m.block = dim3(static_cast<unsigned>(at % grid.x), static_cast<unsigned>(at / grid.x));
        run_block(kernel);
    }
}

inline void wait_loads()
{
    for (auto &x : machine().self->loads) {
        memcpy(x.second, x.first, 16);
    }
    machine().self->loads.clear();
}

enum Kind { kLane = 1, kFirst, kBallot, kShfl, kShflUp, kShflXor, kDpp, kProduct16, kProduct32, kColumn, kBarrier, kHalves };

template <int kN, typename V, typename D>
inline D product(V a, V b, D c)
{
    struct Both
    {
        V a, b;
    };
    const auto x = meet(Both{a, b}, kN == 16 ? kProduct16 : kProduct32);
    const int l = lane(), col = l % kN, up = l / kN;
    for (int r = 0; r < static_cast<int>(sizeof(D) / 4); ++r) {
        const int row = kN == 16 ? 4 * up + r : 8 * (r / 4) + 4 * up + r % 4;
        float sum = c[r];
        for (int g = 0; g < 64 / kN; ++g) {
            for (int e = 0; e < 8; ++e) {
                sum += static_cast<float>(x[row + kN * g].a[e]) * static_cast<float>(x[col + kN * g].b[e]);
            }
        }
        c[r] = sum;
    }
    return c;
}

// The larger of this lane's value and that of lane ^ 32.
inline float max_across_halves(float x)
{
    const auto all = meet(x, kHalves);
    return fmaxf(x, all[lane() ^ 32]);
}

}  // namespace host_hip

#define threadIdx (host_hip::machine().self->idx)
#define blockIdx (host_hip::machine().block)
#define gridDim (host_hip::machine().grid)
#define hipLaunchKernelGGL(kernel, grid, block, bytes, stream, ...) \
    host_hip::launch(grid, block, [&] { (kernel)(__VA_ARGS__); })

inline int __builtin_amdgcn_readlane(int v, int l)
{
    return host_hip::meet(v, host_hip::kLane)[l];
}
inline int __builtin_amdgcn_readfirstlane(int v)
{
    const auto x = host_hip::meet(v, host_hip::kFirst);
    return x[__builtin_ctzll(x.active)];
}
inline unsigned long long __ballot(int p)
{
    const auto x = host_hip::meet(p, host_hip::kBallot);
    unsigned long long all = 0;
    for (int l = 0; l < host_hip::kWave; ++l) {
        all |= static_cast<unsigned long long>(((x.active >> l) & 1) != 0 && x[l] != 0) << l;
    }
    return all;
}
inline bool __any(int p) { return __ballot(p) != 0; }
inline bool __all(int p) { return __ballot(!p) == 0; }
template <typename T>
inline T __shfl(T v, int l)
{
    return host_hip::meet(v, host_hip::kShfl)[l & 63];
}
template <typename T>
inline T __shfl_up(T v, int n)
{
    const auto x = host_hip::meet(v, host_hip::kShflUp);
    const int l = host_hip::lane();
    return l >= n ? x[l - n] : v;
}
template <typename T>
inline T __shfl_xor(T v, int n)
{
    return host_hip::meet(v, host_hip::kShflXor)[host_hip::lane() ^ n];
}
// row_shr:n (0x110 + n) and the broadcasts of a row's and of the lower half's last lane
inline int __builtin_amdgcn_update_dpp(int old, int v, int ctrl, int rows, int, bool)
{
    const auto x = host_hip::meet(v, host_hip::kDpp);
    const int l = host_hip::lane();
    if (((rows >> (l / 16)) & 1) == 0) {
        return old;
    }
    if (ctrl > 0x110 && ctrl < 0x120) {
        const int n = ctrl - 0x110;
        return l % 16 >= n ? x[l - n] : old;
    }
    if (ctrl == 0x142) {
        return l >= 16 ? x[l / 16 * 16 - 1] : old;
    }
    if (ctrl == 0x143) {
        return l >= 32 ? x[31] : old;
    }
    host_hip::fail("a lane move that this file does not know");
}
inline uint32_t __builtin_amdgcn_perm(uint32_t a, uint32_t b, uint32_t select)
{
    const uint64_t both = static_cast<uint64_t>(a) << 32 | b;
    uint32_t y = 0;
    for (int i = 0; i < 4; ++i) {
        y |= static_cast<uint32_t>((both >> (8 * ((select >> (8 * i)) & 7))) & 0xff) << (8 * i);
    }
    return y;
}
inline float __builtin_amdgcn_exp2f(float x) { return exp2f(x); }
inline float __builtin_amdgcn_logf(float x) { return log2f(x); }
inline void __builtin_amdgcn_sched_barrier(int) {}
inline void __builtin_amdgcn_fence(int, const char *) {}
inline void __builtin_amdgcn_wave_barrier() { host_hip::meet(0, host_hip::kBarrier); }
inline void __syncthreads() { host_hip::wait(host_hip::kAtBlock, 0); }
inline int __syncthreads_or(int p)
{
    host_hip::machine().any |= p != 0;
    host_hip::wait(host_hip::kAtBlock, 0);
    return host_hip::machine().any_seen;
}
inline host_hip::f32x4 __builtin_amdgcn_mfma_f32_16x16x32_f16(host_hip::f16x8 a, host_hip::f16x8 b, host_hip::f32x4 c, int,
                                                              int, int)
{
    return host_hip::product<16>(a, b, c);
}
inline host_hip::f32x4 __builtin_amdgcn_mfma_f32_16x16x32_bf16(host_hip::bf16x8 a, host_hip::bf16x8 b, host_hip::f32x4 c,
                                                               int, int, int)
{
    return host_hip::product<16>(a, b, c);
}
inline host_hip::f32x16 __builtin_amdgcn_mfma_f32_32x32x16_f16(host_hip::f16x8 a, host_hip::f16x8 b, host_hip::f32x16 c,
                                                               int, int, int)
{
    return host_hip::product<32>(a, b, c);
}
inline host_hip::f32x16 __builtin_amdgcn_mfma_f32_32x32x16_bf16(host_hip::bf16x8 a, host_hip::bf16x8 b,
                                                                host_hip::f32x16 c, int, int, int)
{
    return host_hip::product<32>(a, b, c);
}
template <typename T>
inline T atomicAdd(T *p, T v)
{
    const T old = *p;
    *p = old + v;
    return old;
}
template <typename T>
inline T atomicMax(T *p, T v)
{
    const T old = *p;
    *p = std::max(old, v);
    return old;
}

#define TQT_FAIL(msg)                                       \
    do {                                                    \
        fprintf(stderr, "%s:%d %s\n", __FILE__, __LINE__, (msg)); \
        abort();                                            \
    } while (0)
#define TQT_REQUIRE(cond, msg) \
    do {                       \
        if (!(cond)) {         \
            TQT_FAIL(msg);     \
        }                      \
    } while (0)

namespace tqt {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Lane i of the wave writes lds + 16 i.
inline void dma_lds16(const int8_t *src, int8_t *lds)
{
    host_hip::machine().self->loads.emplace_back(src, lds + 16 * host_hip::lane());
}

// 4 rows x 16 columns of 16-bit elements: lane i of 16 gives the address of row i / 4, columns 4 (i % 4) .., and
// receives column i.
inline uint64_t host_read_column4(const void *p)
{
    const auto x = host_hip::meet(p, host_hip::kColumn);
    const int l = host_hip::lane(), i = l % 16;
    uint64_t y = 0;
    for (int e = 0; e < 4; ++e) {
        uint16_t v;
        memcpy(&v, static_cast<const char *>(x[l - i + 4 * e + i / 4]) + 2 * (i % 4), 2);
        y |= static_cast<uint64_t>(v) << (16 * e);
    }
    return y;
}

inline bool aligned16(const void *p)
{
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0;
}
inline hipStream_t as_stream(void *s)
{
    return s;
}
inline void check_launch(const char *) {}
inline void finish_sync(hipStream_t, const char *) {}

}  // namespace tqt
