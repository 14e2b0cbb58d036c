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

// 4 consecutive elements from `at` of a row of `width`; zeros beyond it.
template <typename T, bool VEC>
__device__ __forceinline__ float4 load4(const T* __restrict__ row, int at, int width) {
    float v[4];
    if (VEC) {
        if constexpr (sizeof(T) == 4) {
            return *reinterpret_cast<const float4*>(row + at);
        } else {
            const uint2 raw = *reinterpret_cast<const uint2*>(row + at);
            return make_float4(__uint_as_float(raw.x << 16), __uint_as_float(raw.x & 0xFFFF0000u),
                               __uint_as_float(raw.y << 16), __uint_as_float(raw.y & 0xFFFF0000u));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = at + i < width ? cb_to_float(row[at + i]) : 0.f;
    return make_float4(v[0], v[1], v[2], v[3]);
}

template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* __restrict__ row, int at, int width, float4 v, float inv) {
    const uint32_t lo = e4m3x2(v.x * inv, v.y * inv), hi = e4m3x2(v.z * inv, v.w * inv);
    const uint32_t word = lo | (hi << 16);
    if (VEC) {
        *reinterpret_cast<uint32_t*>(row + at) = word;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i < width) row[at + i] = (uint8_t)(word >> (8 * i));
    }
}

// Over the threads of one row (a warp, or the whole block): the sum in a fixed order, or the largest of
// non-negative floats by their bits, by which a NaN is larger than every number.
template <bool WARP>
__device__ __forceinline__ float row_sum(float v, float* scratch) {
    if (WARP) return cb_warp_sum(v);
    return cb_block_sum(v, scratch);
}

template <bool WARP>
__device__ __forceinline__ float row_max(uint32_t v, uint32_t* scratch) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (!WARP) {
        __syncthreads();
        if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
        __syncthreads();
        for (unsigned w = 0; w < blockDim.x / 32; ++w) v = max(v, scratch[w]);
    }
    return __uint_as_float(v);
}

__device__ __forceinline__ uint32_t magnitude(float4 v) {
    const uint32_t m = 0x7FFFFFFFu;
    return max(max(__float_as_uint(v.x) & m, __float_as_uint(v.y) & m),
               max(__float_as_uint(v.z) & m, __float_as_uint(v.w) & m));
}

// max(v, LEAST) that keeps a NaN
__device__ __forceinline__ float at_least(float v) { return v < LEAST ? LEAST : v; }

// CH: chunks of 4 a thread.  WARP: a warp a row (blockDim.y rows a block), else a block a row.
template <typename D, int CH, bool WARP, bool VEC>
__global__ void __launch_bounds__(WARP ? 128 : 1024) norm8_kernel(const float* x, long long ldx, const D* __restrict__ delta, long long ldd,
                             const float* __restrict__ gain, float eps, float* sum_out, long long lds,
                             uint8_t* __restrict__ q, long long ldq, float* __restrict__ scales, int rows, int width) {
    __shared__ float scratch[32];
    cb_pdl_wait();
    const long long row = (long long)blockIdx.x * (WARP ? blockDim.y : 1) + (WARP ? threadIdx.y : 0);
    if (row >= rows) return;                           // (a whole warp at a time: only with WARP)
    const int step = 4 * (WARP ? 32 : blockDim.x), at0 = 4 * threadIdx.x;
    const float* xr = x + row * ldx;
    float4 v[CH];
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at < width) v[c] = load4<float, VEC>(xr, at, width);
    }
    if (delta != nullptr) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = at0 + c * step;
            if (at < width) {
                const float4 d = load4<D, VEC>(delta + row * ldd, at, width);
                v[c].x += d.x, v[c].y += d.y, v[c].z += d.z, v[c].w += d.w;
            }
        }
    }
#pragma unroll
    for (int c = 0; c < CH; ++c)
        ss += (v[c].x * v[c].x + v[c].y * v[c].y) + (v[c].z * v[c].z + v[c].w * v[c].w);
    if (sum_out != nullptr) {
        float* sr = sum_out + row * lds;
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int at = at0 + c * step;
            if (VEC) {
                if (at < width) *reinterpret_cast<float4*>(sr + at) = v[c];
            } else {
                const float e[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (at + i < width) sr[at + i] = e[i];
            }
        }
    }
    ss = row_sum<WARP>(ss, scratch);
    const float r = 1.0f / sqrtf(ss / (float)width + eps);
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) {
            const float4 w = load4<float, VEC>(gain, at, width);
            v[c].x = v[c].x * r * w.x, v[c].y = v[c].y * r * w.y;
            v[c].z = v[c].z * r * w.z, v[c].w = v[c].w * r * w.w;
            top = max(top, magnitude(v[c]));
        }
    }
    const float most = at_least(row_max<WARP>(top, reinterpret_cast<uint32_t*>(scratch)));
    const float inv = E4M3_TOP / most;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) store_e4m3<VEC>(q + row * ldq, at, width, v[c], inv);
    }
    if (threadIdx.x == 0) scales[row] = most / E4M3_TOP;
}

__device__ __forceinline__ float pair8(float g, float u, float limit, float alpha, float offset) {
    if (limit > 0.f) {
        // (written so that a NaN stays one)
        g = g > limit ? limit : g;
        u = (u > limit ? limit : (u < -limit ? -limit : u)) + offset;
        return g / (1.0f + expf(-alpha * g)) * u;
    }
    return g / (1.0f + expf(-g)) * u;
}

template <typename T, int CH, bool WARP, bool VEC>
__global__ void __launch_bounds__(WARP ? 128 : 1024) glu8_kernel(const T* __restrict__ both, long long ldb, uint8_t* __restrict__ q, long long ldq,
                            float* __restrict__ scales, int rows, int width, float limit, float alpha, float offset) {
    __shared__ uint32_t scratch[32];
    cb_pdl_wait();
    const long long row = (long long)blockIdx.x * (WARP ? blockDim.y : 1) + (WARP ? threadIdx.y : 0);
    if (row >= rows) return;
    const int step = 4 * (WARP ? 32 : blockDim.x), at0 = 4 * threadIdx.x;
    const T* gr = both + row * ldb;
    const T* ur = gr + width;
    float4 v[CH];
    uint32_t top = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (at < width) {
            const float4 g = load4<T, VEC>(gr, at, width), u = load4<T, VEC>(ur, at, width);
            v[c].x = pair8(g.x, u.x, limit, alpha, offset), v[c].y = pair8(g.y, u.y, limit, alpha, offset);
            v[c].z = pair8(g.z, u.z, limit, alpha, offset), v[c].w = pair8(g.w, u.w, limit, alpha, offset);
            if (!VEC) {                                // (an offset makes something of the zeros beyond the row)
                if (at + 1 >= width) v[c].y = 0.f;
                if (at + 2 >= width) v[c].z = 0.f;
                if (at + 3 >= width) v[c].w = 0.f;
            }
            top = max(top, magnitude(v[c]));
        }
    }
    const float most = at_least(row_max<WARP>(top, scratch));
    const float inv = E4M3_TOP / most;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int at = at0 + c * step;
        if (at < width) store_e4m3<VEC>(q + row * ldq, at, width, v[c], inv);
    }
    if (threadIdx.x == 0) scales[row] = most / E4M3_TOP;
}

constexpr int WARP_ROW = 512;           // widths up to here: a warp a row, 4 rows a block
constexpr int WIDEST = 32768;

struct Shape {
    int chunks;                         // of 4 a thread: 1, 2, 4 or 8
    bool warp;
    dim3 grid, block;
};

// A block a row: as few threads as hold it with 4 chunks each (8 beyond 16,384 numbers).
inline Shape shape_of(int rows, int width) {
    Shape s;
    const int quads = (width + 3) / 4;
    s.warp = width <= WARP_ROW;
    if (s.warp) {
        s.chunks = quads <= 32 ? 1 : (quads <= 64 ? 2 : 4);
        s.block = dim3(32, 4);
        s.grid = dim3((rows + 3) / 4);
        return s;
    }
    s.chunks = quads <= 4096 ? 4 : 8;
    s.block = dim3(((quads + s.chunks - 1) / s.chunks + 31) / 32 * 32);
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
        s.chunks == 4 ? CB_NORM8(4, false) : CB_NORM8(8, false);
#undef CB_NORM8
}

template <typename T, bool VEC>
void launch_glu8(const Shape& s, const T* both, long long ldb, uint8_t* q, long long ldq, float* scales, int rows,
                 int width, float limit, float alpha, float offset, cudaStream_t stream) {
#define CB_GLU8(CH, WARP)                                                                                        \
    cb_launch(glu8_kernel<T, CH, WARP, VEC>, s.grid, s.block, 0, stream, both, ldb, q, ldq, scales, rows, width, \
              limit, alpha, offset)
    if (s.warp)
        s.chunks == 1 ? CB_GLU8(1, true) : (s.chunks == 2 ? CB_GLU8(2, true) : CB_GLU8(4, true));
    else
        s.chunks == 4 ? CB_GLU8(4, false) : CB_GLU8(8, false);
#undef CB_GLU8
}

}  // namespace

CB_EXPORT int cb_rows8_widest() { return WIDEST; }

// Strides in elements.  `delta` and `sum_out` may be null; `sum_out` may be `x`.
CB_EXPORT int cb_norm8(const float* x, long long ldx, const void* delta, int delta_dtype, long long ldd,
                       const float* gain, float eps, float* sum_out, long long lds, void* q, long long ldq,
                       float* scales, int rows, int width, void* stream) {
    if (rows <= 0) return 0;
    if (width <= 0 || width > WIDEST) return CB_ERR_UNSUPPORTED;
    const Shape s = shape_of(rows, width);
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
    const Shape s = shape_of(rows, width);
    const int size = dtype == CB_BF16 ? 2 : 4;
    const bool vec = width % 4 == 0 && ldb % 4 == 0 && ldq % 4 == 0 && aligned(both, 4 * size) && aligned(q, 4);
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
