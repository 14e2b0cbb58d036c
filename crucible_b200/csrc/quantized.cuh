// What the products over quantised weights share: how a code becomes a bf16 weight, and how a fp32
// row becomes three bf16 ones.
//
// (code - 8) * scale has at most 3 + 4 significant bits for an e4m3 scale, so it is a bf16 number and
// the tensor cores multiply the weights themselves.  Code bits put into the mantissa of 16 are
// 16 + code, and one fused multiply-add, (16 + code) scale - 24 scale, is exact (24 scale has 2 + 4
// significant bits).
//
// A fp32 row is the sum of three bf16 rows exactly: the 24 bits of the mantissa, 8 by 8 (of numbers below 2^-110
// what lies below 2^-133, the last bit that bf16 has, is lost).  Their
// products with the weights are exact too, and only fp32 sums are rounded.  The first part has a sum of
// its own: the numbers of the others are 2^-8 of it and less, and a sum that held the first would
// cut off their last bits at every addition (rows of 8,192: 2.4e-6 off with one sum).
#pragma once
#include "common.cuh"

// K of a product at the most: indices along K, and the products that stand for divisions of them, are 32-bit
constexpr int MOST_K = 1 << 20;
constexpr int MOST_PITCH = 1 << 24;     // bytes from one feature's weights to the next: a block's offsets are 32-bit

enum QuantizedKind { FOUR_BF16 = 0, FOUR_F32 = 1, EIGHT = 2 };

struct QuantizedArgs {
    const void* rows;                   // bf16, fp32 or e4m3 [M, ldr elements]
    long long ldr;
    const float* row_scale;             // EIGHT: [M]
    const void* w;                      // codes int32 [N, K / 8], or e4m3 [N, ldw]
    long long ldw;                      // bytes
    const uint8_t* group_scale;         // e4m3 [N, K / group]
    const float* feature_scale;         // [N]
    const float* add;                   // fp32 [M, lda] or null
    long long lda;
    void* out;                          // [M, ldo]
    long long ldo;
    int M, N, K, group, out_bf16, groups;           // groups: K / group
};

// An e4m3 scale as a pair of equal bf16 numbers, and -24 and -136 times that: all exact.
struct ScalePair {
    uint32_t s, c24, c136;
};

// Two e4m3 scales (the lower two bytes).
__device__ __forceinline__ void scale_pairs(uint32_t e4m3x2, ScalePair (&scale)[2]) {
    uint32_t h2;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h2) : "h"((uint16_t)e4m3x2));
    float s[2];
    asm("{\n\t.reg .f16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\tcvt.f32.f16 %0, lo;\n\tcvt.f32.f16 %1, hi;\n\t}"
        : "=f"(s[0]), "=f"(s[1]) : "r"(h2));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        asm("cvt.rn.bf16x2.f32 %0, %1, %1;" : "=r"(scale[i].s) : "f"(s[i]));
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(scale[i].c24) : "r"(scale[i].s), "r"(0xC1C0C1C0u));       // -24
        asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(scale[i].c136) : "r"(scale[i].s), "r"(0xC308C308u));      // -136
    }
}

// Pair i (k = 2i, 2i + 1) of a word of eight codes as two bf16 weights.  (The mask and the 16s come as registers: with
// both as constants the compiler takes two instructions for them, and the unit that runs them is what a product of a few rows
// waits for.)
__device__ __forceinline__ uint32_t weight_pair(uint32_t word, int i, const ScalePair& scale) {
    uint32_t magic, r;
    if (i == 0) asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(magic) : "r"(word), "r"(0x000F000Fu), "r"(0x43004300u));      // 128 + code, twice
    else asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(magic) : "r"(word >> (4 * i - 3)), "r"(0x00780078u), "r"(0x41804180u));   // 16 + code
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(magic), "r"(scale.s), "r"(i == 0 ? scale.c136 : scale.c24));
    return r;
}

// Two fp32 numbers as three pairs of bf16 whose sum they are.  (Cut, not rounded: what is left is
// exact.  An infinity or a NaN stands in the first pair alone.)
__device__ __forceinline__ void three_parts(float x, float y, uint32_t (&p)[3]) {
    const float v[2] = {x, y};
    uint32_t part[2][3];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t bits = __float_as_uint(v[i]);
        const bool finite = (bits & 0x7F800000u) != 0x7F800000u;
        const float rest = finite ? v[i] - __uint_as_float(bits & 0xFFFF0000u) : 0.f;
        const float second = __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
        part[i][0] = finite || (bits & 0x007FFFFFu) == 0 ? bits >> 16 : 0x7FC0u;
        part[i][1] = __float_as_uint(second) >> 16;
        part[i][2] = __float_as_uint(rest - second) >> 16;
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) p[j] = part[0][j] | (part[1][j] << 16);
}

// fp32 rows as three bf16 ones: parts [3, M, K].  Four numbers a thread.  (A template, so that only the sources that launch it
// carry it.)
template <int THREADS> __global__ void __launch_bounds__(THREADS) split_rows_kernel(const float* __restrict__ rows, long long ldr,
                                                         __nv_bfloat16* __restrict__ parts, int M, int K) {
    cb_pdl_wait();
    cb_pdl_trigger();
    const long long total = (long long)M * (K / 4);
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
        const long long m = i / (K / 4), k = i % (K / 4) * 4;
        const float4 v = __ldg(reinterpret_cast<const float4*>(rows + m * ldr + k));
        uint32_t a[3], b[3];
        three_parts(v.x, v.y, a);
        three_parts(v.z, v.w, b);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            *reinterpret_cast<uint2*>(parts + ((long long)j * M + m) * K + k) = make_uint2(a[j], b[j]);
    }
}

template <int THREADS = 256> void split_rows(const float* rows, long long ldr, __nv_bfloat16* parts, int M, int K, cudaStream_t stream) {
    const long long quads = (long long)M * (K / 4);
    const int blocks = (int)(quads / THREADS + 1 < 148 * 8 ? quads / THREADS + 1 : 148 * 8);
    cb_launch(split_rows_kernel<THREADS>, dim3(blocks), dim3(THREADS), 0, stream, rows, ldr, parts, M, K);
}

// K of one sum over 4-bit weights by mma.sync, fp32 results.  The tensor cores cut off, towards zero, what an addition leaves
// below the sum's last bit, and over a long K that adds up (a warp's share of 8,192 in one sum: 1.5e-6 of the result's norm; 2.7e-7
// in sums of 2,048).
constexpr int MMA_CHUNK = 2048;

// Room for the sums of a warp's chunks before the present one, zeroed, by an address that the compiler does not see through:
// they stay in memory, and a loop whose registers are all taken keeps them (8 rows of 14,336 by 28,672 through the ring
// 58.4 us in one sum, 59.5 like this, 62.6 with the sums in registers).
template <int N> __device__ __forceinline__ float* set_aside(float (&room)[N]) {
    float* at = room;
    asm volatile("" : "+l"(at));
#pragma unroll
    for (int i = 0; i < N; ++i) at[i] = 0.f;
    return at;
}

// A sum's way out: its scales, the addition, the rounding.
__device__ __forceinline__ void finish(const QuantizedArgs& p, float v, float row_scale, float feature_scale, int m, int n) {
    v *= feature_scale;
    v *= row_scale;
    if (p.add != nullptr) v += p.add[(long long)m * p.lda + n];
    const long long at = (long long)m * p.ldo + n;
    if (p.out_bf16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    else static_cast<float*>(p.out)[at] = v;
}

// Shared memory beyond the default, asked for once a kernel and device.
template <typename Kernel>
static inline int allow_shared(Kernel kernel, int bytes, bool (&configured)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64 && configured[dev]) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) configured[dev] = true;
    return (int)e;
}
