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
// that fetched them (4 consecutive ones a chunk) while the row's sum of squares and largest
// magnitude are taken.
#define CB_PDL_BIT 6      // this file's bit in CRUCIBLE_PDL
#include "common.cuh"

namespace {

constexpr float E4M3_TOP = 448.f;
constexpr float LEAST = 1e-30f;

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
    const float r = 1.0f / sqrtf(ss / (float)width + eps);
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
    const float top_v = row_max<WARP>(top, reinterpret_cast<uint32_t*>(scratch)), top_y = top_v * r;
    const float most = at_least(top_y);
    const float factor = top_y >= LEAST ? E4M3_TOP / top_v : (top_y < LEAST ? r * (E4M3_TOP / LEAST) : top_y);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) store_e4m3<E, VEC>(q + row * ldq, at, width, v[c], factor);
    }
    if (threadIdx.x == 0) scales[row] = most / E4M3_TOP;
}

// z / (1 + e^-a z) by the hardware's unit, 2^-22 and 2^-23 for the power of two and the reciprocal.  t = -a z log2 e loses
// 2^-24 of itself, up to 2^-18 of the power, unless its rest, which one fused multiply-add gives, goes back into it.
// (With expf and the exact division 2,048 rows of 14,336 bf16 pairs took 77 us, which is what those instructions take.)
__device__ __forceinline__ float gated(float z, float alpha) {
    // (beyond e^88 there is nothing of z left, below e^-88 all of it; a NaN is in z as well)
    const float x = fmaxf(fminf(-alpha * z, 88.f), -88.f), log2e = 1.44269504f;
    const float t = x * log2e;
    const float rest = fmaf(x, log2e, -t) + x * 1.92596299e-8f;       // log2 e has more digits, too
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    e = fmaf(e, rest * 0.693147182f, e);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
    return z * r;
}

template <bool CAPPED>
__device__ __forceinline__ float pair8(float g, float u, float limit, float alpha, float offset) {
    if (CAPPED) {
        // (written so that a NaN stays one)
        g = g > limit ? limit : g;
        u = (u > limit ? limit : (u < -limit ? -limit : u)) + offset;
        return gated(g, alpha) * u;
    }
    return gated(g, 1.0f) * u;
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
            for (int i = 0; i < E; ++i) {
                v[c][i] = pair8<CAPPED>(g[i], u[i], limit, alpha, offset);
                if (!VEC && at + i >= width) v[c][i] = 0.f;        // (an offset makes something of the zeros beyond the row)
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

constexpr int WARP_ROW = 512;           // widths up to here: a warp a row, 4 rows a block
constexpr int WIDEST = 32768;
constexpr int MANY_ROWS = 296;          // two for every SM

struct Shape {
    int chunks;                         // a thread: 1, 2, 4 or 8
    bool warp;
    dim3 grid, block;
};

// A block a row, of at most `most` threads (twice that where a row needs it).  Many rows: as many chunks of `e` a thread
// as leave a block `least` threads, so that several blocks are on an SM and one's loads run beside another's sums; few
// rows: as few chunks as there are threads for, since then the chain of one row is all there is.  us, 2,048 rows: norms
// of 4,096 with 256 and 512 threads 17.9 and 18.1, of 2,048 8.0 and 11.3; pairs of 14,336 bf16 with 448 and 896 39.8
// and 32.3, of 8,192 with 256 and 512 22.5 and 17.7.
inline Shape shape_of(int rows, int width, int e, int least, int most) {
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
    if (rows < MANY_ROWS) least = most;
    while (s.chunks > 1 && (all + s.chunks - 1) / s.chunks < least && (all + s.chunks / 2 - 1) / (s.chunks / 2) <= most) s.chunks /= 2;
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
    const Shape s = shape_of(rows, width, 4, 256, 512);
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

// limit <= 0: silu(g) * u; else the capped pair.
CB_EXPORT int cb_glu8(const void* both, int dtype, long long ldb, void* q, long long ldq, float* scales, int rows,
                      int width, float limit, float alpha, float offset, void* stream) {
    if (rows <= 0) return 0;
    if (width <= 0 || width > WIDEST) return CB_ERR_UNSUPPORTED;
    const int e = dtype == CB_BF16 ? 8 : 4;            // 16 bytes
    const Shape s = shape_of(rows, width, e, 512, 1024);
    const bool vec = width % e == 0 && ldb % e == 0 && ldq % e == 0 && aligned(both, 16) && aligned(q, e);
    cudaStream_t st = (cudaStream_t)stream;
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
