"""Runs a generated operator kernel on the CPU, for its addresses only: each thread by itself, one after the other, every
operand between two pages that may not be touched.

Values mean nothing there (lanes exchange nothing, matrix instructions pass their accumulator on, LDS holds what earlier
threads left), so this shows reads and writes out of bounds of kernels whose addresses and loop counts depend on
positions and sizes alone -- without a GPU that such an access could fault.
"""
import os
import re
import subprocess
import tempfile

import pytest

from descent_amd import hip_backend

CLANG = "/opt/rocm/llvm/bin/clang++"

SHIM = r"""
#include <algorithm>
#include <cmath>
#include <csignal>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <sys/mman.h>
#include <type_traits>
#include <unistd.h>
#define __device__
#define __forceinline__ inline
#define __global__
#define __shared__ static
#define __restrict__
#define __launch_bounds__(...)
struct dim { unsigned x, y, z; };
static dim threadIdx, blockIdx;
struct float2 { float x, y; };
struct alignas(16) float4 { float x, y, z, w; };
static float4 make_float4(float a, float b, float c, float d) { return {a, b, c, d}; }
static float __uint_as_float(unsigned x) { float f; memcpy(&f, &x, 4); return f; }
static unsigned __float_as_uint(float x) { unsigned f; memcpy(&f, &x, 4); return f; }
static int __float_as_int(float x) { return (int)__float_as_uint(x); }
static float __int_as_float(int x) { return __uint_as_float((unsigned)x); }
template <class A, class B> auto min(A a, B b) { typedef std::common_type_t<A, B> C; return (C)a < (C)b ? (C)a : (C)b; }
template <class A, class B> auto max(A a, B b) { typedef std::common_type_t<A, B> C; return (C)a > (C)b ? (C)a : (C)b; }
template <class T> T __shfl_xor(T x, int) { return x; }
template <class T> T __shfl(T x, int) { return x; }
static bool __any(bool x) { return x; }
static void __syncthreads() {}
// (an operand that goes nowhere else counts as used, or the compiler would leave its loads out)
template <class A, class B, class C> C mfma(A a, B b, C c, int, int, int) { asm volatile("" ::"m"(a), "m"(b)); return c; }
struct swapped { unsigned v[2]; unsigned operator[](int i) const { return v[i]; } };
extern "C" __bf16 __truncsfbf2(float x) { const unsigned short h = (unsigned short)(__float_as_uint(x) >> 16); __bf16 y; memcpy(&y, &h, 2); return y; }
#define __builtin_amdgcn_readfirstlane(x) (x)
#define __builtin_amdgcn_sched_barrier(x)
#define __builtin_amdgcn_exp2f exp2f
#define __builtin_amdgcn_fmed3f(a, b, c) fminf(fmaxf(a, b), c)
#define __builtin_amdgcn_mov_dpp(v, ...) (v)
#define __builtin_amdgcn_permlane32_swap(a, b, ...) swapped{{a, b}}
#define __builtin_amdgcn_permlane16_swap(a, b, ...) swapped{{a, b}}
#define __builtin_amdgcn_mfma_f32_16x16x4f32 mfma
#define __builtin_amdgcn_mfma_f32_32x32x16_bf16 mfma
"""

MAIN = r"""
static void fault(int, siginfo_t* info, void*) {
    printf("block %u thread %u touches", blockIdx.x, threadIdx.x);
    for (int i = 0; i < BUFFERS; ++i) {
        const long at = (char*)info->si_addr - first[i];
        if (at >= -(long)GAP && at < (long)(sizes[i] + GAP)) printf(" byte %ld of operand %d, which has %ld", at, i, (long)sizes[i]);
    }
    printf("\n");
    fflush(stdout);
    _exit(1);
}
int main(int, char** argv) {
    const bool ends = argv[2][0] == '1';  // operands end at a page's end, or start at its start
    FILE* in = fopen(argv[1], "rb");
    for (int i = 0; i < BUFFERS; ++i) {
        const size_t room = (sizes[i] + 15) / 16 * 16, pages = (room + 4095) / 4096 * 4096;
        char* base = (char*)mmap(nullptr, pages + 2 * GAP, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS | MAP_NORESERVE, -1, 0);
        if (base == MAP_FAILED || mprotect(base + GAP, pages, PROT_READ | PROT_WRITE)) return 2;
        first[i] = base + GAP + (ends ? pages - room : 0);
        if (i < INPUTS && fread(first[i], 1, sizes[i], in) != sizes[i]) return 3;
    }
    struct sigaction act = {};
    act.sa_sigaction = fault;
    act.sa_flags = SA_SIGINFO;
    sigaction(SIGSEGV, &act, nullptr);
    sigaction(SIGBUS, &act, nullptr);
    for (blockIdx.x = 0; blockIdx.x < GRID; ++blockIdx.x)
        for (threadIdx.x = 0; threadIdx.x < BLOCK; ++threadIdx.x) CALL;
    printf("in bounds\n");
    return 0;
}
"""


def run(kernel, arrays, grid):
    """Fails if a thread of `grid` workgroups touches what lies outside the kernel's operands."""
    if not os.path.exists(CLANG):
        pytest.skip("no clang++")
    source = hip_backend.codegen_source(kernel)
    source = re.sub(r"asm( volatile)?\((.|\n)*?\);", "", source)  # (other kernels' helpers in the common prelude)
    entry, parameters = re.search(r'extern "C" __global__ __launch_bounds__\([^)]*\) void (\w+)\(([^)]*)\)', source).groups()
    block = int(re.search(r'extern "C" __global__ __launch_bounds__\((\d+)', source).group(1))
    sizes = [a.nbytes for a in arrays] + [kernel.result_shapes()[i].buffer_size() for i in kernel.results]
    assert parameters.count("float* b") == len(sizes)
    call = entry + "(" + ", ".join(f"(float*)first[{i}]" for i in range(len(sizes))) + ", nullptr, 0u)"
    text = SHIM + source.replace('extern "C"', "static") + (
        f"\nenum {{ BUFFERS = {len(sizes)}, INPUTS = {len(arrays)}, BLOCK = {block}, GRID = {grid}, GAP = 1 << 20 }};\n"
        f"static const size_t sizes[] = {{{', '.join(map(str, sizes))}}};\nstatic char* first[BUFFERS];\n" + MAIN.replace("CALL", call)
    )
    with tempfile.TemporaryDirectory() as tmp:
        path = os.path.join(tmp, "kernel")
        with open(path + ".cpp", "w") as f:
            f.write(text)
        with open(path + ".in", "wb") as f:
            for a in arrays:
                f.write(a.tobytes())
        subprocess.run([CLANG, "-O1", "-w", "-std=c++17", "-ffp-contract=off", path + ".cpp", "-o", path], check=True)
        for ends in "10":
            out = subprocess.run([path, path + ".in", ends], capture_output=True, text=True, timeout=300)
            assert out.returncode == 0, out.stdout + out.stderr
