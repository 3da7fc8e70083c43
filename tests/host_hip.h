// What csrc/*.hip name of HIP, as far as the kernels of the token operators need it, on the CPU: each thread
// of a launch runs on its own, one after the other.  Shuffles give back a lane's own value and matrix products
// their sum, so results mean nothing; which addresses are touched depends on sizes, strides, lengths and masks
// alone.  Buffers lie between pages that cannot be touched, so that an access outside is a fault that names
// the call.
#pragma once

#include <algorithm>
#include <csignal>
#include <cstdint>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <sys/mman.h>
#include <unistd.h>
#include <vector>

static char now[200];  // the call that runs
static void host_fault(int, siginfo_t *, void *) {
    ssize_t n = write(1, "out of range: ", 14);
    n += write(1, now, strlen(now));
    n += write(1, "\n", 1);
    _exit(1);
}

// bytes that end right before a page that cannot be touched, in a mapping kept for the next call
struct Guarded {
    char *base = nullptr;
    size_t room = 0;
    void *take(size_t bytes, size_t align = 16) {
        const size_t page = 4096, need = (bytes + page - 1) / page * page;
        if (need > room || !base) {
            if (base) munmap(base, room + 2 * page);
            room = need;
            base = static_cast<char *>(mmap(nullptr, room + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
            if (base == MAP_FAILED || (room && mprotect(base + page, room, PROT_READ | PROT_WRITE))) abort();
        }
        return base + page + (room - bytes) / align * align;
    }
};
static Guarded &lds_pages() {
    static Guarded g;
    return g;
}
static void name_faults() {
    struct sigaction s = {};
    s.sa_sigaction = host_fault;
    s.sa_flags = SA_SIGINFO;
    sigaction(SIGSEGV, &s, nullptr);
    sigaction(SIGBUS, &s, nullptr);
}

#define __device__
#define __global__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)
struct dim3 {
    uint32_t x, y, z;
    dim3(uint32_t a = 1, uint32_t b = 1, uint32_t c = 1) : x(a), y(b), z(c) {}
};
static dim3 threadIdx, blockIdx, blockDim, gridDim;
typedef void *hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
static hipError_t hipGetLastError() { return hipSuccess; }
using std::max;
using std::min;
template <class T> T __shfl_xor(T v, int) { return v; }
static void __syncthreads() {}
static float __fadd_rn(float a, float b) { return a + b; }
static float __fsub_rn(float a, float b) { return a - b; }
static float __fmul_rn(float a, float b) { return a * b; }
static float __uint_as_float(uint32_t u) { return __builtin_bit_cast(float, u); }
static uint32_t __float_as_uint(float f) { return __builtin_bit_cast(uint32_t, f); }
static float __int_as_float(int u) { return __builtin_bit_cast(float, u); }
static int __float_as_int(float f) { return __builtin_bit_cast(int, f); }
enum { hipFuncAttributeMaxDynamicSharedMemorySize };
static hipError_t hipFuncSetAttribute(const void *, int, int) { return hipSuccess; }
static uint64_t __ballot(bool x) { return x ? ~0ull : 0; }
static bool __any(bool x) { return x; }
template <class T> T __shfl(T v, int) { return v; }
static int __popcll(uint64_t x) { return __builtin_popcountll(x); }
static void atomicMin(int *p, int v) { *p = min(*p, v); }
static void atomicMax(int *p, int v) { *p = max(*p, v); }
static float __builtin_amdgcn_exp2f(float x) { return exp2f(x); }
static float __builtin_amdgcn_logf(float x) { return log2f(x); }
static void __builtin_amdgcn_s_waitcnt(int) {}
static float __builtin_amdgcn_fmed3f(float a, float, float) { return a; }
static int __builtin_amdgcn_update_dpp(int, int v, int, int, int, bool) { return v; }
static int __builtin_amdgcn_readlane(int v, int) { return v; }
static void __builtin_amdgcn_fence(int, const char *) {}
static void __builtin_amdgcn_wave_barrier() {}
static void __builtin_amdgcn_sched_group_barrier(int, int, int) {}
static uint32_t __builtin_amdgcn_perm(uint32_t a, uint32_t, uint32_t) { return a; }
template <class G, class L> void __builtin_amdgcn_global_load_lds(G *from, L *to, int bytes, int, int) {
    memcpy(reinterpret_cast<char *>((uintptr_t)to) + bytes * (threadIdx.x & 63), reinterpret_cast<const char *>((uintptr_t)from), bytes);
}
template <class A, class B, class C> C __builtin_amdgcn_mfma_f32_32x32x16_bf16(A, B, C c, int, int, int) { return c; }
typedef short host_s16x4 __attribute__((ext_vector_type(4)));
template <class P> host_s16x4 __builtin_amdgcn_ds_read_tr16_b64_v4i16(P *from) {
    host_s16x4 v;
    memcpy(&v, reinterpret_cast<const char *>((uintptr_t)from), 8);
    return v;
}

static uint16_t *host_lds;  // a launch's dynamic LDS, at its size
template <class F>
static void on_cpu(dim3 grid, dim3 block, F f) {
    gridDim = grid, blockDim = block;
    for (blockIdx.y = 0; blockIdx.y < grid.y; ++blockIdx.y)
        for (blockIdx.x = 0; blockIdx.x < grid.x; ++blockIdx.x)
            for (threadIdx.x = 0; threadIdx.x < block.x; ++threadIdx.x) f();
}
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) \
    host_lds = static_cast<uint16_t *>(lds_pages().take((size_t)(lds))), on_cpu(grid, block, [&] { (kernel)(__VA_ARGS__); })
