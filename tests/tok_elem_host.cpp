// The block boundary's kernels (csrc/tok_elem.hip) built for the CPU, each buffer between two pages
// that cannot be touched: a read or write one element past its end, or before its start, is a fault
// that names the call.  Every thread of a launch runs on its own, so sums over a row are not made and
// the values mean nothing; which addresses are touched depends on the sizes alone.
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
// (what the headers name beside; nothing below calls the matrix products)
static float __builtin_amdgcn_fmed3f(float a, float, float) { return a; }
static int __builtin_amdgcn_update_dpp(int, int v, int, int, int, bool) { return v; }
static int __builtin_amdgcn_readlane(int v, int) { return v; }
static void __builtin_amdgcn_fence(int, const char *) {}
static void __builtin_amdgcn_wave_barrier() {}
static void __builtin_amdgcn_sched_group_barrier(int, int, int) {}
static uint32_t __builtin_amdgcn_perm(uint32_t a, uint32_t, uint32_t) { return a; }
template <class... A> void __builtin_amdgcn_global_load_lds(A...) {}
template <class A, class B, class C> C __builtin_amdgcn_mfma_f32_32x32x16_bf16(A, B, C c, int, int, int) { return c; }
typedef short host_s16x4 __attribute__((ext_vector_type(4)));
template <class P> host_s16x4 __builtin_amdgcn_ds_read_tr16_b64_v4i16(P) { return host_s16x4{0, 0, 0, 0}; }

template <class F>
static void on_cpu(dim3 grid, dim3 block, F f) {
    gridDim = grid, blockDim = block;
    for (blockIdx.y = 0; blockIdx.y < grid.y; ++blockIdx.y)
        for (blockIdx.x = 0; blockIdx.x < grid.x; ++blockIdx.x)
            for (threadIdx.x = 0; threadIdx.x < block.x; ++threadIdx.x) f();
}
#define hipLaunchKernelGGL(kernel, grid, block, lds, stream, ...) on_cpu(grid, block, [&] { (kernel)(__VA_ARGS__); })

#include "../pcd_reg_hregnet_amd/csrc/tok_elem.hip"

static char now[200];  // the call that runs
static void fault(int, siginfo_t *, void *) {
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

int main() {
    struct sigaction s = {};
    s.sa_sigaction = fault;
    s.sa_flags = SA_SIGINFO;
    sigaction(SIGSEGV, &s, nullptr);
    sigaction(SIGBUS, &s, nullptr);
    static Guarded g[19];
    int calls = 0;
    // forms of the call: both norms and both gradients (the usual one), an RMS norm before alone, a norm
    // behind alone, the first norm of a stack; the gate for all, for some, for one of the rows, or none
    struct Form { int post, pre, f, bias; };
    const Form forms[] = {{2, 2, 1, 1}, {1, 1, 1, 0}, {0, 1, 1, 0}, {2, 0, 1, 1}, {0, 2, 0, 1}};
    std::vector<int> widths = {2048, 4096, 8191, 8192};  // (one more chunk than a whole row: 1032, 2056, ..)
    for (int C = 1; C <= 8192; C += C < 160 ? 1 : C < 1100 ? 8 : 44) widths.push_back(C);
    for (int C = 1024; C < 8192; C *= 2) widths.push_back(C + 8), widths.push_back(2 * C - 8);
    for (const int C : widths)
        for (int type = 0; type < 2; ++type) {
            const Form fm = forms[(C / 8 + type) % 5];
            for (int k = 0; k < 2; ++k) {
                const Form f = k ? fm : forms[0];
                const int R = C > 512 ? 2 : 6, kind = f.f ? (C / 8 + k) % 4 : 0, rows = kind == 1 ? R : kind == 2 ? R / 2 : 1;
                const int ptype = (C / 8 + type + k) % 2 ? HREG_TOK_F32 : type;
                const size_t e = type == HREG_TOK_F32 ? 4 : 2, pe = ptype == HREG_TOK_F32 ? 4 : 2, n = e * R * C;
                const size_t gn = e * C * (R / rows);
                snprintf(now, sizeof now, "type %d, parameters %d, %d rows of %d, norms %d and %d, gate rows %d, f %d", type, ptype, R,
                         C, f.post, f.pre, kind ? rows : 0, f.f);
                hreg_tok_block_t p = {};
                p.dtype = type, p.param_dtype = ptype, p.R = R, p.C = C, p.gate_rows = rows, p.post = f.post, p.pre = f.pre;
                p.scale = 1.f, p.eps = 1e-6f, p.step = C % 16 ? 0 : 6554, p.seed = 7;
                int at = 0;
                auto take = [&](size_t bytes, size_t align = 16) { return g[at++].take(bytes, align); };
                p.x = take(n);
                p.f = f.f ? take(n) : nullptr;
                p.gate = kind ? take(gn) : nullptr;
                p.post_w = f.post ? take(pe * C) : nullptr;
                p.post_b = f.post && f.bias ? take(pe * C) : nullptr;
                p.pre_w = f.pre ? take(pe * C) : nullptr;
                p.pre_b = f.pre && f.bias ? take(pe * C) : nullptr;
                p.y = f.f ? take(n) : nullptr;
                p.h = f.pre ? take(n) : nullptr;
                p.stats = static_cast<float *>(take(16 * R));
                if (hreg_tok_block_fwd(&p, nullptr) != HREG_OK) return 2;
                if (!f.f) p.y = const_cast<void *>(p.x), p.step = 0;
                p.dy = take(n);
                p.dh = f.pre ? take(n) : nullptr;
                p.dx = take(n);
                p.df = f.f ? take(n) : nullptr;
                p.dgate = kind ? take(gn) : nullptr;
                // (parameters' gradients are as long as the parameters, workspaces end at their size rounded up)
                static Guarded d[4], w;
                p.dpost_w = p.post_w ? d[0].take(pe * C, pe) : nullptr;
                p.dpost_b = p.post_b ? d[1].take(pe * C, pe) : nullptr;
                p.dpre_w = p.pre_w ? d[2].take(pe * C, pe) : nullptr;
                p.dpre_b = p.pre_b ? d[3].take(pe * C, pe) : nullptr;
                p.ws_bytes = hreg_tok_block_ws_bytes(&p);
                p.ws = w.take((p.ws_bytes + 255) / 256 * 256, 256);
                if (hreg_tok_block_bwd(&p, nullptr) != HREG_OK) return 3;
                ++calls;
            }
        }
    printf("%d calls inside their buffers\n", calls);
    return 0;
}
