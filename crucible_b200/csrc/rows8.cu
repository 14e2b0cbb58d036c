// Rows of activations in 8 bits: e4m3 numbers with one fp32 scale a row.
//
//   norm8:  sum = x + delta,  y = sum / sqrt(mean(sum^2) + eps) * gain
//   glu8:   y = silu(g) * u of a row [g : u], or the capped pair
//   both:   scale = max(max |y|, 1e-30) / 448,  q = e4m3(y * (448 / max(max |y|, 1e-30)))
//
// e4m3 reaches 448, so a row's largest number lands there; 1e-30 keeps 448 / max finite and gives
// rows of zeros a scale.  Everything up to the one rounding to e4m3 (to nearest, ties to even, half
// a step 2^-4) is fp32.  A NaN anywhere in a row makes the scale NaN and with it the row.
//
// Memory bounds both: one pass over the data, a row's numbers stay in the registers of the threads
// that fetched them (16 bytes a chunk) while the row's sum of squares and largest magnitude are taken.
// (In a chain over inputs that are not in L2: 2,048 rows of 4,096 with a bf16 delta 17.0 us, 5.4 TB/s; 2,048 of 14,336 bf16
// pairs 27.2, 5.4 TB/s.)
#define CB_PDL_BIT 6      // this file's bit in CRUCIBLE_PDL
#include "quantized.cuh"
#include "tc_common.cuh"

namespace {

constexpr float E4M3_TOP = 448.f;
constexpr float LEAST = 1e-30f;
constexpr float BIG_R = 262144.f;       // a factor r up to here: neither r * (448 / LEAST) nor 448 / max |v| of a max |v| r from LEAST on overflows

// two fp32 to two e4m3 (the lower byte is `lo`): to nearest even, beyond 448 to 448, NaN stays NaN
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// E consecutive elements from `at` of a row of `width`; zeros beyond it.
template <typename T, int E, bool VEC>
__device__ __forceinline__ void load_chunk(const T* __restrict__ row, int at, int width, float (&v)[E]) {
    if constexpr (VEC && sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < E; i += 4) {
            const float4 x = *reinterpret_cast<const float4*>(row + at + i);
            v[i] = x.x, v[i + 1] = x.y, v[i + 2] = x.z, v[i + 3] = x.w;
        }
    } else if constexpr (VEC) {
        uint32_t w[E / 2];
        if constexpr (E == 8) {
            const uint4 x = *reinterpret_cast<const uint4*>(row + at);
            w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(row + at);
            w[0] = x.x, w[1] = x.y;
        }
#pragma unroll
        for (int i = 0; i < E / 2; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i) v[i] = at + i < width ? cb_to_float(row[at + i]) : 0.f;
    }
}

template <int E, bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* __restrict__ row, int at, int width, const float (&v)[E], float inv) {
    uint32_t word[E / 4];
#pragma unroll
    for (int i = 0; i < E / 4; ++i)
        word[i] = e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) | (e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
    if constexpr (VEC && E == 8) {
        *reinterpret_cast<uint2*>(row + at) = make_uint2(word[0], word[1]);
    } else if constexpr (VEC) {
        *reinterpret_cast<uint32_t*>(row + at) = word[0];
    } else {
#pragma unroll
        for (int i = 0; i < E; ++i)
            if (at + i < width) row[at + i] = (uint8_t)(word[i >> 2] >> (8 * (i & 3)));
    }
}

// Over the threads of one row (a warp, or the whole block): the sum in a fixed order, or the largest of
// non-negative floats by their bits, by which a (positive) NaN is larger than every number.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    if (WARP) return cb_warp_sum(v);
    return cb_block_sum(v, scratch);
}

template <bool WARP>
__device__ __forceinline__ float row_max(float m, uint32_t* scratch) {
    uint32_t v = __reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7FFFFFFFu);
    if (!WARP) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        for (unsigned w = 0; w < blockDim.x / 32; ++w) v = max(v, scratch[w]);
    }
    return __uint_as_float(v);
}

// The larger of m and every |v|; a NaN is larger than all.
template <int E> __device__ __forceinline__ float magnitude(float m, const float (&v)[E]) {
#pragma unroll
    for (int i = 0; i < E; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(fabsf(v[i])));
    return m;
}

// max(v, LEAST) that keeps a NaN
__device__ __forceinline__ float at_least(float v) { return v < LEAST ? LEAST : v; }

// CH: chunks a thread.  WARP: a warp a row (blockDim.y rows a block), else a block a row.
template <typename D, int CH, bool WARP, bool VEC>
__global__ void __launch_bounds__(WARP ? 128 : (CH < 8 ? 512 : 1024))
norm8_kernel(const float* x, long long ldx, const D* delta, long long ldd, const float* __restrict__ gain,
             float eps, float* sum_out, long long lds, uint8_t* __restrict__ q, long long ldq,
             float* __restrict__ scales, int rows, int width) {
    constexpr int E = 4;
    __shared__ float scratch[32];
    cb_pdl_wait();
    cb_pdl_trigger();
    const long long row = (long long)blockIdx.x * (WARP ? blockDim.y : 1) + (WARP ? threadIdx.y : 0);
    if (row >= rows) return;                           // (a whole warp at a time: only with WARP)
    const int step = E * (WARP ? 32 : blockDim.x), at0 = E * threadIdx.x;
    const float* xr = x + row * ldx;
    float v[CH][E];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
#pragma unroll
        for (int i = 0; i < E; ++i) v[c][i] = 0.f;
        if (at < width) load_chunk<float, E, VEC>(xr, at, width, v[c]);
    }
    if (delta != nullptr) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = at0 + c * step;
            if (at < width) {
                float d[E];
                load_chunk<D, E, VEC>(delta + row * ldd, at, width, d);
#pragma unroll
                for (int i = 0; i < E; ++i) v[c][i] += d[i];
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c) ss += (v[c][0] * v[c][0] + v[c][1] * v[c][1]) + (v[c][2] * v[c][2] + v[c][3] * v[c][3]);
    if (sum_out != nullptr) {
        float* sr = sum_out + row * lds;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = at0 + c * step;
            if (VEC) {
                if (at < width) *reinterpret_cast<float4*>(sr + at) = make_float4(v[c][0], v[c][1], v[c][2], v[c][3]);
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (at + i < width) sr[at + i] = v[c][i];
            }
        }
    }
    ss = row_sum<WARP>(ss, scratch);
    float r = 1.0f / sqrtf(ss / (float)width + eps);
    // y = v r with v = sum * gain: the row's factor r is in its largest number as well, so 448 / max |v| takes v to e4m3 with
    // three roundings, whatever r was rounded to
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) {
            float w[E];
            load_chunk<float, E, VEC>(gain, at, width, w);
#pragma unroll
            for (int i = 0; i < E; ++i) v[c][i] *= w[i];
            top = magnitude(top, v[c]);
        }
    }
    float top_v = row_max<WARP>(top, reinterpret_cast<uint32_t*>(scratch));
    const float top_y = top_v * r;
    if (r > BIG_R) {                                   // (eps below 1.5e-11 and a row of next to nothing)
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
            for (int i = 0; i < E; ++i) v[c][i] *= r;
        top_v = top_y, r = 1.f;
    }
    const float most = at_least(top_y);
    const float factor = top_y >= LEAST ? E4M3_TOP / top_v : (top_y < LEAST ? r * (E4M3_TOP / LEAST) : top_y);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) store_e4m3<E, VEC>(q + row * ldq, at, width, v[c], factor);
    }
    if (threadIdx.x == 0) scales[row] = most / E4M3_TOP;
}

// Two fp32 numbers in one register pair: one instruction for both.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float x, float y) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void apart(F2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// z / (1 + e^-a z) by the hardware's unit, 2^-22 and 2^-23 for the power of two and the reciprocal, of two numbers at a
// time.  t = x log2 e (x = -a z) is rounded, up to 2^-18 of the power, so e^x = 2^t (1 + d) with d = x - t ln 2, which two
// fused multiply-adds give.  (With expf and the exact division 2,048 rows of 14,336 bf16 pairs took 77 us, which is what
// those instructions take.)
__device__ __forceinline__ F2 gated(F2 z, float alpha) {
    float x0, x1, n0, n1, e0, e1;
    apart(mul2(z, f2(-alpha, -alpha)), x0, x1);
    // (beyond e^88 there is nothing of z left, below e^-88 all of it; a NaN is in z as well)
    const F2 x = f2(fmaxf(fminf(x0, 88.f), -88.f), fmaxf(fminf(x1, 88.f), -88.f));
    const F2 minus_t = mul2(x, f2(-1.44269504f, -1.44269504f));
    const F2 d = fma2(minus_t, f2(-1.90465430e-9f, -1.90465430e-9f), fma2(minus_t, f2(0.693147182f, 0.693147182f), x));
    apart(minus_t, n0, n1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(-n0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(-n1));
    const F2 e = f2(e0, e1);
    apart(add2(fma2(e, d, e), f2(1.f, 1.f)), e0, e1);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(e0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(e1));
    return mul2(z, f2(e0, e1));
}

// the smaller one; NaN stays NaN
__device__ __forceinline__ float less(float v, float limit) {
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(v) : "f"(limit));
    return v;
}

template <bool CAPPED>
__device__ __forceinline__ void pair8(float g0, float g1, float u0, float u1, float limit, float alpha, float offset, float& y0, float& y1) {
    if (CAPPED) {
        g0 = less(g0, limit), g1 = less(g1, limit);
        u0 = -less(-less(u0, limit), limit), u1 = -less(-less(u1, limit), limit);
        apart(mul2(gated(f2(g0, g1), alpha), add2(f2(u0, u1), f2(offset, offset))), y0, y1);
    } else {
        apart(mul2(gated(f2(g0, g1), 1.0f), f2(u0, u1)), y0, y1);
    }
}

template <typename T, int CH, bool WARP, bool VEC, bool CAPPED>
__global__ void __launch_bounds__(WARP ? 128 : 1024)
glu8_kernel(const T* __restrict__ both, long long ldb, uint8_t* __restrict__ q, long long ldq,
            float* __restrict__ scales, int rows, int width, float limit, float alpha, float offset) {
    constexpr int E = 16 / sizeof(T);
    __shared__ uint32_t scratch[32];
    cb_pdl_wait();
    cb_pdl_trigger();
    const long long row = (long long)blockIdx.x * (WARP ? blockDim.y : 1) + (WARP ? threadIdx.y : 0);
    if (row >= rows) return;
    const int step = E * (WARP ? 32 : blockDim.x), at0 = E * threadIdx.x;
    const T* gr = both + row * ldb;
    const T* ur = gr + width;
    float v[CH][E];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) {
            float g[E], u[E];
            load_chunk<T, E, VEC>(gr, at, width, g);
            load_chunk<T, E, VEC>(ur, at, width, u);
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                pair8<CAPPED>(g[i], g[i + 1], u[i], u[i + 1], limit, alpha, offset, v[c][i], v[c][i + 1]);
                if (!VEC && at + i >= width) v[c][i] = 0.f;        // (an offset makes something of the zeros beyond the row)
                if (!VEC && at + i + 1 >= width) v[c][i + 1] = 0.f;
            }
            top = magnitude(top, v[c]);
        }
    }
    const float most = at_least(row_max<WARP>(top, scratch));
    const float inv = E4M3_TOP / most;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) store_e4m3<E, VEC>(q + row * ldq, at, width, v[c], inv);
    }
    if (threadIdx.x == 0) scales[row] = most / E4M3_TOP;
}

// The same for many long rows: a block stays on its SM and walks rows, which one thread brings into shared memory, as
// many ahead as fit.  (A block a row has nothing on its way while it computes and takes the row's maximum.  us, 2,048 rows,
// this / a block a row: 14,336 bf16 pairs 27.2 / 31.9, 11,008 22.0 / 27.5, 10,240 20.7 / 21.8, 8,192 17.8 / 17.4; 7,168 fp32
// pairs 24.5 / 27.8, 4,096 15.6 / 15.5.)
constexpr int RING_ROWS = 8;            // stages at most
constexpr int RING_BYTES = 32768;       // rows of more than this
constexpr int RING_MANY = 1024;         // and so many of them (512 of 14,336 bf16 pairs: 8.8 either way), where two blocks fit on an SM

template <typename T, int THREADS, bool CAPPED>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS)
glu8_ring_kernel(const T* __restrict__ both, long long ldb, uint8_t* __restrict__ q, long long ldq, float* __restrict__ scales,
                 int rows, int width, float limit, float alpha, float offset, int stages, int* __restrict__ status) {
    constexpr int E = 16 / sizeof(T), CH = 4, WARPS = THREADS / 32;
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ __align__(8) uint64_t full[RING_ROWS];
    __shared__ uint32_t tops[2][WARPS];
    __shared__ int abort_word;
    volatile int* abort_flag = &abort_word;
    const int bytes = 2 * width * (int)sizeof(T);
    if (threadIdx.x == 0) {
        for (int i = 0; i < stages; ++i) tc::mbar_init(&full[i], 1);
        abort_word = 0;
        tc::fence_barrier_init();
    }
    __syncthreads();
    cb_pdl_wait();
    cb_pdl_trigger();
    int brought = 0;
    auto bring = [&](int row, int st) {
        if (row >= rows) return;
        ++brought;
        tc::mbar_expect_tx(&full[st], bytes);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     ::"r"(tc::smem_u32(ring + (size_t)st * bytes)), "l"(both + row * ldb), "r"(bytes), "r"(tc::smem_u32(&full[st])) : "memory");
    };
    const int step = gridDim.x;
    if (threadIdx.x == 0)
        for (int i = 0; i < stages; ++i) bring(blockIdx.x + i * step, i);
    bool ok = true;
    int st = 0, turn = 0;
    uint32_t parity = 0;
    for (int row = blockIdx.x; row < rows; row += step, turn ^= 1) {
        // (where a wait runs out the rest is gone through without waiting, and not stored)
        if (ok && !tc::mbar_wait(&full[st], parity, abort_flag)) {
            ok = false;
            tc::give_up(abort_flag, status, tc::ST_PRODUCER_TIMEOUT);
        }
        const T* gr = reinterpret_cast<const T*>(ring + (size_t)st * bytes);
        float v[CH][E];
        float top = 0.f;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = E * (threadIdx.x + c * THREADS);
            if (at < width) {
                float g[E], u[E];
                load_chunk<T, E, true>(gr, at, width, g);
                load_chunk<T, E, true>(gr + width, at, width, u);
#pragma unroll
                for (int i = 0; i < E; i += 2)
                    pair8<CAPPED>(g[i], g[i + 1], u[i], u[i + 1], limit, alpha, offset, v[c][i], v[c][i + 1]);
                top = magnitude(top, v[c]);
            }
        }
        const uint32_t mine = __reduce_max_sync(0xffffffffu, __float_as_uint(top) & 0x7FFFFFFFu);
        if ((threadIdx.x & 31) == 0) tops[turn][threadIdx.x >> 5] = mine;
        __syncthreads();                // the row has been read, and every warp's part is there
        if (threadIdx.x == 0 && *abort_flag == 0) bring(row + stages * step, st);
        const float most = at_least(__uint_as_float(__reduce_max_sync(0xffffffffu, tops[turn][threadIdx.x % WARPS])));
        const float inv = E4M3_TOP / most;
        if (*abort_flag == 0) {
#pragma unroll
            for (int c = 0; c < CH; ++c) {
                const int at = E * (threadIdx.x + c * THREADS);
                if (at < width) store_e4m3<E, true>(q + row * ldq, at, width, v[c], inv);
            }
            if (threadIdx.x == 0) scales[row] = most / E4M3_TOP;
        }
        if (++st == stages) st = 0, parity ^= 1;
    }
    if (*abort_flag)                    // (thread 0's copies land before the block's shared memory goes away)
        for (int i = max(0, brought - stages); i < brought; ++i)
            for (uint32_t j = 0; j < tc::WAIT_LIMIT; ++j)
                if (tc::mbar_try_wait(&full[i % stages], (i / stages) & 1)) break;
}

constexpr int WARP_ROW = 512;           // widths up to here: a warp a row, 4 rows a block
constexpr int WIDEST = 32768;
constexpr int MANY_ROWS = 296;          // two for every SM
constexpr int N_SMS = 148;

struct Shape {
    int chunks;                         // a thread: 1, 2, 4 or 8
    bool warp;
    dim3 grid, block;
};

// A block a row, of at most `most` threads (twice that where a row needs it).  Many rows: as many chunks of `e` a thread
// as leave a block `least` threads (`least_two`, for two chunks), so that several blocks are on an SM and one's loads run
// beside another's sums; few rows: as few chunks as there are threads for, since then the chain of one row is all there
// is.  us, 2,048 rows: norms of 4,096 with 256 and 512 threads 17.2 and 18.6, of 2,048 with 128 and 256 7.3 and 8.3; bf16 pairs by one, two
// and four chunks, of 4,096 8.7, 8.0 and 8.8, of 5,632 17.2, 13.3 and 15.3, of 2,816 6.8, 6.3 and -, of 8,192 -, 17.4 and
// 20.5; fp32 pairs of 2,816 15.1, 10.9 and 12.9.
inline Shape shape_of(int rows, int width, int e, int least, int least_two, int most) {
    Shape s;
    const int all = (width + e - 1) / e;
    s.warp = width <= WARP_ROW;
    if (s.warp) {
        s.chunks = all <= 32 ? 1 : (all <= 64 ? 2 : 4);
        s.block = dim3(32, 4);
        s.grid = dim3((rows + 3) / 4);
        return s;
    }
    s.chunks = 32 / e;
    if (s.chunks == 8 && all <= 4 * most) s.chunks = 4;
    if (rows < MANY_ROWS) least = least_two = most;
    while (s.chunks > 1 && (all + s.chunks - 1) / s.chunks < (s.chunks > 2 ? least : least_two) && (all + s.chunks / 2 - 1) / (s.chunks / 2) <= most) s.chunks /= 2;
    s.block = dim3(((all + s.chunks - 1) / s.chunks + 31) / 32 * 32);
    s.grid = dim3(rows);
    return s;
}

inline bool aligned(const void* p, int bytes) { return ((uintptr_t)p & (uintptr_t)(bytes - 1)) == 0; }

template <typename D, bool VEC>
void launch_norm8(const Shape& s, const float* x, long long ldx, const D* delta, long long ldd, const float* gain,
                  float eps, float* sum_out, long long lds, uint8_t* q, long long ldq, float* scales, int rows,
                  int width, cudaStream_t stream) {
#define CB_NORM8(CH, WARP)                                                                                        \
    cb_launch(norm8_kernel<D, CH, WARP, VEC>, s.grid, s.block, 0, stream, x, ldx, delta, ldd, gain, eps, sum_out, \
              lds, q, ldq, scales, rows, width)
    if (s.warp)
        s.chunks == 1 ? CB_NORM8(1, true) : (s.chunks == 2 ? CB_NORM8(2, true) : CB_NORM8(4, true));
    else
        s.chunks == 1 ? CB_NORM8(1, false) : (s.chunks == 2 ? CB_NORM8(2, false) : (s.chunks == 4 ? CB_NORM8(4, false) : CB_NORM8(8, false)));
#undef CB_NORM8
}

template <typename T, bool VEC, bool CAPPED>
void launch_glu8_as(const Shape& s, const T* both, long long ldb, uint8_t* q, long long ldq, float* scales, int rows,
                 int width, float limit, float alpha, float offset, cudaStream_t stream) {
#define CB_GLU8(CH, WARP)                                                                                        \
    cb_launch(glu8_kernel<T, CH, WARP, VEC, CAPPED>, s.grid, s.block, 0, stream, both, ldb, q, ldq, scales, rows, width, \
              limit, alpha, offset)
    constexpr bool F32 = sizeof(T) == 4;               // (bf16 chunks are 8 long: no row has more than 4 a thread)
    if (s.warp)
        s.chunks == 1 ? CB_GLU8(1, true) : (s.chunks == 2 ? CB_GLU8(2, true) : CB_GLU8(4, true));
    else
        s.chunks == 1 ? CB_GLU8(1, false) : (s.chunks == 2 ? CB_GLU8(2, false) : (s.chunks == 4 ? CB_GLU8(4, false) : CB_GLU8((F32 ? 8 : 4), false)));
#undef CB_GLU8
}

// Shared memory of a block of the ring, and its rows: two blocks of 512 threads an SM, or one of 1,024.
constexpr int ring_room(int threads) { return (threads == 512 ? 112 : 225) * 1024; }

// Threads of a block of the ring, or 0: a block a row.  (The ring waits for its copies, and a wait that runs out has to be told:
// without a place for that, null, a block a row, which waits for nothing.)
inline int ring_threads(int rows, int width, int size, const int* status) {
    if (status == nullptr) return 0;
    const int bytes = 2 * width * size;
    if (bytes <= RING_BYTES || 2 * bytes > ring_room(1024)) return 0;
    const int threads = 2 * bytes <= ring_room(512) ? 512 : 1024;
    return rows >= (threads == 512 ? RING_MANY : MANY_ROWS) ? threads : 0;
}

template <typename T, int THREADS, bool CAPPED>
int launch_glu8_ring(const T* both, long long ldb, uint8_t* q, long long ldq, float* scales, int rows, int width, float limit,
                     float alpha, float offset, int* status, cudaStream_t stream) {
    constexpr int ROOM = ring_room(THREADS), BLOCKS = 1024 / THREADS;
    static_assert(ROOM / 2 / 2 / 16 <= 4 * THREADS, "a thread has four chunks of either half of a row");
    const int bytes = 2 * width * (int)sizeof(T), stages = ROOM / bytes < RING_ROWS ? ROOM / bytes : RING_ROWS;
    static bool configured[64] = {};
    auto kernel = glu8_ring_kernel<T, THREADS, CAPPED>;
    const int rc = allow_shared(kernel, ROOM, configured);
    if (rc != 0) return rc;
    cb_launch(kernel, dim3(rows < N_SMS * BLOCKS ? rows : N_SMS * BLOCKS), dim3(THREADS), stages * bytes, stream, both, ldb, q, ldq,
              scales, rows, width, limit, alpha, offset, stages, status);
    return cb_last_error();
}

template <typename T>
int launch_glu8_ring(int threads, const T* both, long long ldb, uint8_t* q, long long ldq, float* scales, int rows, int width,
                     float limit, float alpha, float offset, int* status, cudaStream_t st) {
    if (threads == 512)
        return limit > 0.f ? launch_glu8_ring<T, 512, true>(both, ldb, q, ldq, scales, rows, width, limit, alpha, offset, status, st)
                           : launch_glu8_ring<T, 512, false>(both, ldb, q, ldq, scales, rows, width, limit, alpha, offset, status, st);
    return limit > 0.f ? launch_glu8_ring<T, 1024, true>(both, ldb, q, ldq, scales, rows, width, limit, alpha, offset, status, st)
                       : launch_glu8_ring<T, 1024, false>(both, ldb, q, ldq, scales, rows, width, limit, alpha, offset, status, st);
}

template <typename T, bool VEC>
void launch_glu8(const Shape& s, const T* both, long long ldb, uint8_t* q, long long ldq, float* scales, int rows,
                 int width, float limit, float alpha, float offset, cudaStream_t stream) {
    if (limit > 0.f) launch_glu8_as<T, VEC, true>(s, both, ldb, q, ldq, scales, rows, width, limit, alpha, offset, stream);
    else launch_glu8_as<T, VEC, false>(s, both, ldb, q, ldq, scales, rows, width, limit, alpha, offset, stream);
}

}  // namespace

CB_EXPORT int cb_rows8_widest() { return WIDEST; }

// Strides in elements.  `delta` and `sum_out` may be null; `sum_out` may be `x` or `delta`.
CB_EXPORT int cb_norm8(const float* x, long long ldx, const void* delta, int delta_dtype, long long ldd,
                       const float* gain, float eps, float* sum_out, long long lds, void* q, long long ldq,
                       float* scales, int rows, int width, void* stream) {
    if (rows <= 0) return 0;
    if (width <= 0 || width > WIDEST) return CB_ERR_UNSUPPORTED;
    const Shape s = shape_of(rows, width, 4, 128, 128, 512);
    const int dsize = delta_dtype == CB_BF16 ? 2 : 4;
    const bool vec = width % 4 == 0 && ldx % 4 == 0 && ldq % 4 == 0 && aligned(x, 16) && aligned(gain, 16) &&
                     aligned(q, 4) && (!sum_out || (lds % 4 == 0 && aligned(sum_out, 16))) &&
                     (!delta || (ldd % 4 == 0 && aligned(delta, 4 * dsize)));
    cudaStream_t st = (cudaStream_t)stream;
    if (delta_dtype == CB_BF16) {
        const __nv_bfloat16* d = (const __nv_bfloat16*)delta;
        vec ? launch_norm8<__nv_bfloat16, true>(s, x, ldx, d, ldd, gain, eps, sum_out, lds, (uint8_t*)q, ldq, scales, rows, width, st)
            : launch_norm8<__nv_bfloat16, false>(s, x, ldx, d, ldd, gain, eps, sum_out, lds, (uint8_t*)q, ldq, scales, rows, width, st);
    } else {
        const float* d = (const float*)delta;
        vec ? launch_norm8<float, true>(s, x, ldx, d, ldd, gain, eps, sum_out, lds, (uint8_t*)q, ldq, scales, rows, width, st)
            : launch_norm8<float, false>(s, x, ldx, d, ldd, gain, eps, sum_out, lds, (uint8_t*)q, ldq, scales, rows, width, st);
    }
    return cb_last_error();
}

// The fewest rows that are brought by copies which a kernel waits for, whatever their width.
CB_EXPORT int cb_glu8_waits_from() { return MANY_ROWS < RING_MANY ? MANY_ROWS : RING_MANY; }

// Whether so many pairs of rows that begin on 16 bytes are brought by such copies, with a place to tell of waits that run out
// (`status`) or without.
CB_EXPORT int cb_glu8_waits(int dtype, int rows, int width, const int* status) {
    return ring_threads(rows, width, dtype == CB_BF16 ? 2 : 4, status) != 0;
}

// limit <= 0: silu(g) * u; else the capped pair.  `status` (may be null): where a wait for memory that runs out is told.
CB_EXPORT int cb_glu8(const void* both, int dtype, long long ldb, void* q, long long ldq, float* scales, int rows,
                      int width, float limit, float alpha, float offset, int* status, void* stream) {
    if (rows <= 0) return 0;
    if (width <= 0 || width > WIDEST) return CB_ERR_UNSUPPORTED;
    const int e = dtype == CB_BF16 ? 8 : 4;            // 16 bytes
    const Shape s = shape_of(rows, width, e, 1024, 160, 1024);
    const bool vec = width % e == 0 && ldb % e == 0 && ldq % e == 0 && aligned(both, 16) && aligned(q, e);
    cudaStream_t st = (cudaStream_t)stream;
    const int ring = vec ? ring_threads(rows, width, 16 / e, status) : 0;
    if (ring != 0)
        return dtype == CB_BF16 ? launch_glu8_ring(ring, (const __nv_bfloat16*)both, ldb, (uint8_t*)q, ldq, scales, rows, width, limit, alpha, offset, status, st)
                                : launch_glu8_ring(ring, (const float*)both, ldb, (uint8_t*)q, ldq, scales, rows, width, limit, alpha, offset, status, st);
    if (dtype == CB_BF16) {
        const __nv_bfloat16* b = (const __nv_bfloat16*)both;
        vec ? launch_glu8<__nv_bfloat16, true>(s, b, ldb, (uint8_t*)q, ldq, scales, rows, width, limit, alpha, offset, st)
            : launch_glu8<__nv_bfloat16, false>(s, b, ldb, (uint8_t*)q, ldq, scales, rows, width, limit, alpha, offset, st);
    } else {
        const float* b = (const float*)both;
        vec ? launch_glu8<float, true>(s, b, ldb, (uint8_t*)q, ldq, scales, rows, width, limit, alpha, offset, st)
            : launch_glu8<float, false>(s, b, ldb, (uint8_t*)q, ldq, scales, rows, width, limit, alpha, offset, st);
    }
    return cb_last_error();
}
