// Writing the cache in 4 bits, and reading it back as it stands.
//
//   append4   a row's q and k are rotated by its position, k and v go to the row's place in the pages.
//             One warp a (row, head): lane L holds the features L + 32 i, so that a group's least and
//             largest number are warp reductions, and a word of codes is put together from four lanes.
//   bounds4   of every page that the step wrote: each feature's largest and least key over the tokens that
//             the page now holds, in 8 bits with one scale.  A block a (row, kv head); only the last row of
//             each page's run does anything.
//   values4   the whole pool as float32 or bfloat16 rows.
//   expand4   the pages of some requests as rows of float32 or bfloat16 in pages of 64 tokens, for attention
//             over many rows.
//
// All are bound by memory in large calls and by their launch in small ones.
#define CB_PDL_BIT 6      // with the other quantised operators
#include "cache4.cuh"

namespace {

__device__ __forceinline__ float warp_least(float v) {
    float r;
    asm("redux.sync.min.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_largest(float v) {
    float r;
    asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

struct AppendParams {
    const void* qkv;
    long long qkv_stride;
    void* q;
    long long q_stride;
    const float* cos_t;
    const float* sin_t;
    int rotary, n_positions, neighbours, write;
    const int* positions;
    const int* row_request;
    const int* table;
    int table_stride, n_requests;
    uint32_t* codes;
    uint32_t* scales;
    int n_pages, page_tokens, n_heads, kv_heads;
    int rows;
    int8_t* bounds;
    float* bound_scales;
};

// One group: what its numbers are coded with.
struct Coding {
    float low, inverse;
    uint32_t pair;
};

__device__ __forceinline__ Coding coding_of(float least, float largest) {
    Coding c;
    const __nv_bfloat16 low = __float2bfloat16_rd(least);
    c.low = __bfloat162float(low);
    const float range = __fsub_rn(largest, c.low);
    __nv_bfloat16 step = __float2bfloat16_rn(__fmul_rn(range, 1.0f / 15.0f));
    c.inverse = 0.f;
    if (!(range <= 3.4e38f) || !(c.low >= -3.4e38f)) {       // a number that is not finite, or a range that is none
        c.pair = 0x7fff7fffu;
        c.low = 0.f;
        return c;
    }
    if (__bfloat162float(step) < C4_LEAST_STEP) step = __float2bfloat16_rn(0.f);
    else c.inverse = __frcp_rn(__bfloat162float(step));
    c.pair = (uint32_t)__bfloat16_as_ushort(step) | ((uint32_t)__bfloat16_as_ushort(low) << 16);
    return c;
}

__device__ __forceinline__ uint32_t code_of(float x, const Coding& c) {
    const float v = rintf(__fmul_rn(__fsub_rn(x, c.low), c.inverse));
    return (uint32_t)fminf(fmaxf(v, 0.f), 15.f);
}

template <int D, int GROUP, typename T>
__global__ void __launch_bounds__(256) append4_kernel(const AppendParams p) {
    cb_pdl_trigger();
    cb_pdl_wait();
    constexpr int NI = D / 32, W = D / 64, NG = D / GROUP;
    const int lane = threadIdx.x & 31;
    const int heads = p.n_heads + (p.write ? 2 * p.kv_heads : 0);
    const long long items = (long long)p.rows * heads;
    for (long long item = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); item < items; item += (long long)gridDim.x * 8) {
        const int row = (int)(item / heads), head = (int)(item - (long long)row * heads);
        const int request = p.row_request[row], pos = p.positions[row];
        if (request < 0 || request >= p.n_requests || pos < 0 || (p.rotary > 0 && pos >= p.n_positions)) continue;
        const T* src = reinterpret_cast<const T*>(p.qkv) + (size_t)row * p.qkv_stride + (size_t)head * D;
        float x[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) x[i] = cb_to_float(src[lane + 32 * i]);
        if (head < p.n_heads + p.kv_heads && p.rotary > 0) {
            const int half = p.rotary >> 1;
            const float* cs = p.cos_t + (size_t)pos * half;
            const float* sn = p.sin_t + (size_t)pos * half;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int f = lane + 32 * i;
                if (f < p.rotary) {
                    const bool first = p.neighbours ? (f & 1) == 0 : f < half;
                    const int at = p.neighbours ? f >> 1 : first ? f : f - half;
                    const int other = p.neighbours ? f ^ 1 : first ? f + half : f - half;
                    const float y = cb_to_float(src[other]);
                    const float own = __fmul_rn(x[i], cs[at]), cross = __fmul_rn(y, sn[at]);
                    x[i] = first ? __fsub_rn(own, cross) : __fadd_rn(cross, own);
                }
            }
        }
        if (head < p.n_heads) {
            __syncwarp();                     // q may take its own place: every lane has read what it turns
            T* dst = reinterpret_cast<T*>(p.q) + (size_t)row * p.q_stride + (size_t)head * D;
#pragma unroll
            for (int i = 0; i < NI; ++i) dst[lane + 32 * i] = cb_from_float<T>(x[i]);
            continue;
        }
        const int side = head >= p.n_heads + p.kv_heads;
        const int kv = head - p.n_heads - side * p.kv_heads;
        long long at = c4_row(p.table + (size_t)request * p.table_stride, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
        if (at < 0) continue;
        at += (long long)kv * p.page_tokens + (long long)side * p.n_pages * p.kv_heads * p.page_tokens;
        constexpr int PER = GROUP / 32;
        uint32_t code[NI], pair = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float least = x[g * PER], largest = x[g * PER];
#pragma unroll
            for (int i = 1; i < PER; ++i) {
                // (a NaN has to stay one)
                const float v = x[g * PER + i];
                least = least <= v ? least : v != v ? v : least != least ? least : v;
                largest = largest >= v ? largest : v != v ? v : largest != largest ? largest : v;
            }
            const Coding c = coding_of(warp_least(least), warp_largest(largest));
#pragma unroll
            for (int i = 0; i < PER; ++i) code[g * PER + i] = code_of(x[g * PER + i], c);
            if (lane == g) pair = c.pair;
        }
        if (lane < NG) p.scales[at * NG + lane] = pair;
        const int shift = c4_shift(lane >> 3);             // of feature k = lane / 8; k + 4 lies 8 bits higher
        uint32_t word[W];
#pragma unroll
        for (int w = 0; w < W; ++w) {
            word[w] = (code[2 * w] << shift) | (code[2 * w + 1] << (shift + 8));
            word[w] |= __shfl_xor_sync(0xffffffffu, word[w], 8);
            word[w] |= __shfl_xor_sync(0xffffffffu, word[w], 16);
        }
        if (lane < 8) {
            uint32_t* dst = p.codes + at * (D / 8) + lane * W;
            if constexpr (W == 1) dst[0] = word[0];
            else if constexpr (W == 2) *reinterpret_cast<uint2*>(dst) = make_uint2(word[0], word[1]);
            else if constexpr (W == 4) *reinterpret_cast<uint4*>(dst) = make_uint4(word[0], word[1], word[2], word[3]);
            else {
#pragma unroll
                for (int w = 0; w < W; ++w) dst[w] = word[w];
            }
        }
    }
}

// The value of feature f of the row `at`.
template <int D>
__device__ __forceinline__ float value_of(const uint32_t* codes, const uint32_t* scales, long long at, int group, int f) {
    const uint32_t word = codes[at * (D / 8) + (f & 7) * (D / 64) + (f >> 6)];
    const uint32_t pair = scales[at * (D / group) + f / group];
    return fmaf((float)((word >> c4_shift((f >> 3) & 7)) & 15u), c4_step(pair), c4_low(pair));
}

// A block of D threads a feature each, four threads a feature over the tokens.
template <int D>
__global__ void __launch_bounds__(4 * D) bounds4_kernel(const AppendParams p, int group) {
    cb_pdl_trigger();
    cb_pdl_wait();
    __shared__ float part[2][4][D];
    __shared__ float largest[8];
    const int row = blockIdx.x / p.kv_heads, kv = blockIdx.x - row * p.kv_heads;
    const int request = p.row_request[row], pos = p.positions[row];
    if (request < 0 || request >= p.n_requests || pos < 0 || (p.rotary > 0 && pos >= p.n_positions)) return;
    const int index = pos / p.page_tokens;
    if (row + 1 < p.rows && p.row_request[row + 1] == request && p.positions[row + 1] / p.page_tokens == index) return;
    long long at = c4_row(p.table + (size_t)request * p.table_stride, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
    if (at < 0) return;
    const int held = pos - index * p.page_tokens + 1;
    const long long page = (at - (held - 1)) / ((long long)p.kv_heads * p.page_tokens);
    at += (long long)kv * p.page_tokens - (held - 1);
    const int f = threadIdx.x % D, q = threadIdx.x / D;
    float hi = -INFINITY, lo = INFINITY;
    for (int i = q; i < held; i += 4) {
        const float v = value_of<D>(p.codes, p.scales, at + i, group, f);
        hi = fmaxf(hi, v);
        lo = fminf(lo, v);
    }
    part[0][q][f] = hi;
    part[1][q][f] = lo;
    __syncthreads();
    if (q == 0) {
#pragma unroll
        for (int i = 1; i < 4; ++i) {
            hi = fmaxf(hi, part[0][i][f]);
            lo = fminf(lo, part[1][i][f]);
        }
        if (!(lo <= hi)) hi = lo = 0.f;          // (a feature of which no token's key is a number)
        const float most = cb_warp_max(fmaxf(fabsf(hi), fabsf(lo)));
        if ((f & 31) == 0) largest[f >> 5] = most;
    }
    __syncthreads();
    if (q != 0) return;
    float most = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i) most = fmaxf(most, largest[i]);
    const float scale = __fmul_rn(most, 1.0f / 127.0f);
    const float inverse = scale > 0.f ? __frcp_rn(scale) : 0.f;
    const long long to = page * p.kv_heads + kv;
    p.bounds[(to * 2) * D + f] = (int8_t)(int)fminf(fmaxf(rintf(__fmul_rn(hi, inverse)), -127.f), 127.f);
    p.bounds[(to * 2 + 1) * D + f] = (int8_t)(int)fminf(fmaxf(rintf(__fmul_rn(lo, inverse)), -127.f), 127.f);
    if (f == 0) p.bound_scales[to] = scale;
}

// Eight neighbouring features of a row.
template <int D>
__device__ __forceinline__ void eight_values(const uint32_t* codes, const uint32_t* scales, long long at, int group, int f,
                                             float (&v)[8]) {
    const uint32_t* words = codes + at * (D / 8) + (f >> 6);
    const uint32_t pair = scales[at * (D / group) + f / group];
    const float step = c4_step(pair), low = c4_low(pair);
    const int shift = c4_shift((f >> 3) & 7);
#pragma unroll
    for (int g = 0; g < 8; ++g) v[g] = fmaf((float)((words[g * (D / 64)] >> shift) & 15u), step, low);
}

template <typename T>
__device__ __forceinline__ void store_eight(T* dst, const float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        __nv_bfloat162 b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(b);
    }
}

template <int D, typename T>
__global__ void __launch_bounds__(256) values4_kernel(const uint32_t* codes, const uint32_t* scales, int group, long long rows,
                                                      T* out) {
    cb_pdl_trigger();
    cb_pdl_wait();
    const long long items = rows * (D / 8);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < items; i += (long long)gridDim.x * 256) {
        const long long at = i / (D / 8);
        const int f = (int)(i - at * (D / 8)) * 8;
        float v[8];
        eight_values<D>(codes, scales, at, group, f, v);
        store_eight(out + at * D + f, v);
    }
}

struct ExpandParams {
    const uint32_t* codes;
    const uint32_t* scales;
    int n_pages, page_tokens, kv_heads, group;
    const int* row_start;
    const int* first_pos;
    const int* table;
    int table_stride, n_requests;
    int window;
    void* keys;              // [blocks of 64 tokens][kv heads][64][D]
    void* values;
    int* blocks;             // [requests][block_stride]: where each request's blocks of 64 tokens lie
    int block_stride, n_blocks;
};

// A block of threads a block of 64 tokens and kv head.  Which request the block of tokens is of follows from how many
// blocks the requests before it have; tokens that no row of the step sees are left out, as zeros.
template <int D, typename T>
__global__ void __launch_bounds__(256) expand4_kernel(const ExpandParams p) {
    cb_pdl_trigger();
    cb_pdl_wait();
    int request = 0, before = 0, count = 0, held = 0, first = 0;
    const int block = blockIdx.x;
    for (; request < p.n_requests; ++request) {
        first = p.first_pos[request];
        held = first + p.row_start[request + 1] - p.row_start[request];
        count = (held + 63) >> 6;
        if (block < before + count) break;
        before += count;
    }
    if (request == p.n_requests) return;
    const int index = block - before;
    if (index >= p.block_stride) return;
    if (blockIdx.y == 0 && threadIdx.x == 0) p.blocks[(size_t)request * p.block_stride + index] = block;
    const int lo = p.window > 0 ? max(0, first - p.window + 1) : 0;
    const int* table = p.table + (size_t)request * p.table_stride;
    for (int i = threadIdx.x; i < 64 * (D / 8); i += 256) {
        const int t = i / (D / 8), f = (i - t * (D / 8)) * 8, pos = index * 64 + t;
        const long long to = (((long long)block * p.kv_heads + blockIdx.y) * 64 + t) * D + f;
        float k[8] = {0.f}, v[8] = {0.f};
        if (pos < held && pos >= lo) {
            long long at = c4_row(table, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
            if (at >= 0) {
                at += (long long)blockIdx.y * p.page_tokens;
                eight_values<D>(p.codes, p.scales, at, p.group, f, k);
                eight_values<D>(p.codes, p.scales, at + (long long)p.n_pages * p.kv_heads * p.page_tokens, p.group, f, v);
            }
        }
        store_eight(reinterpret_cast<T*>(p.keys) + to, k);
        store_eight(reinterpret_cast<T*>(p.values) + to, v);
    }
}

template <int D, int GROUP>
int append_of(const AppendParams& p, int dtype, cudaStream_t stream) {
    const long long items = (long long)p.rows * (p.n_heads + 2 * p.kv_heads);
    const dim3 grid((unsigned)min((items + 7) / 8, 148LL * 8));
    int rc;
    if (dtype == CB_F32) rc = cb_launch(append4_kernel<D, GROUP, float>, grid, dim3(256), 0, stream, p);
    else rc = cb_launch(append4_kernel<D, GROUP, __nv_bfloat16>, grid, dim3(256), 0, stream, p);
    if (rc == 0 && p.write && p.bounds != nullptr)
        rc = cb_launch(bounds4_kernel<D>, dim3((unsigned)p.rows * p.kv_heads), dim3(4 * D), 0, stream, p, GROUP);
    return rc;
}

template <int D>
int append_dim(const AppendParams& p, int group, int dtype, cudaStream_t stream) {
    if (group == 32) return append_of<D, 32>(p, dtype, stream);
    if (group == 64) return append_of<D, 64>(p, dtype, stream);
    if constexpr (D % 128 == 0)
        if (group == 128) return append_of<D, 128>(p, dtype, stream);
    return CB_ERR_UNSUPPORTED;
}

}  // namespace

CB_EXPORT int cb_append4(const void* qkv, int dtype, long long qkv_stride, void* q, long long q_stride, const float* cos_t,
                         const float* sin_t, int rotary, int n_positions, int neighbours, int write, const int* positions,
                         const int* row_request, const int* table, int table_stride, int n_requests, void* codes,
                         void* scales, int n_pages, int page_tokens, int n_heads, int kv_heads, int head_dim, int group,
                         int rows, void* bounds, float* bound_scales, void* stream) {
    if (rows <= 0) return 0;
    AppendParams p = {qkv, qkv_stride, q, q_stride, cos_t, sin_t, rotary, n_positions, neighbours, write, positions, row_request,
                      table, table_stride, n_requests, reinterpret_cast<uint32_t*>(codes), reinterpret_cast<uint32_t*>(scales),
                      n_pages, page_tokens, n_heads, kv_heads, rows, reinterpret_cast<int8_t*>(bounds), bound_scales};
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int rc = CB_ERR_UNSUPPORTED;
    if (head_dim == 64) rc = append_dim<64>(p, group, dtype, s);
    else if (head_dim == 128) rc = append_dim<128>(p, group, dtype, s);
    else if (head_dim == 192) rc = append_dim<192>(p, group, dtype, s);
    else if (head_dim == 256) rc = append_dim<256>(p, group, dtype, s);
    if (rc == CB_ERR_UNSUPPORTED) return rc;
    return cb_last_error();
}

CB_EXPORT int cb_values4(const void* codes, const void* scales, int group, long long rows, int head_dim, void* out, int dtype,
                         void* stream) {
    if (rows <= 0) return 0;
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes);
    const uint32_t* sc = reinterpret_cast<const uint32_t*>(scales);
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)min((rows * (head_dim / 8) + 255) / 256, 148LL * 32));
#define VALUES(D)                                                                                                        \
    if (head_dim == D) {                                                                                                 \
        if (dtype == CB_F32) cb_launch(values4_kernel<D, float>, grid, dim3(256), 0, s, c, sc, group, rows, (float*)out); \
        else cb_launch(values4_kernel<D, __nv_bfloat16>, grid, dim3(256), 0, s, c, sc, group, rows, (__nv_bfloat16*)out); \
        return cb_last_error();                                                                                          \
    }
    VALUES(64) VALUES(128) VALUES(192) VALUES(256)
#undef VALUES
    return CB_ERR_UNSUPPORTED;
}

CB_EXPORT int cb_expand4(const void* codes, const void* scales, int n_pages, int page_tokens, int kv_heads, int head_dim,
                         int group, const int* row_start, const int* first_pos, const int* table, int table_stride,
                         int n_requests, int window, void* keys, void* values, int dtype, int* blocks, int block_stride,
                         int n_blocks, void* stream) {
    if (n_blocks <= 0) return 0;
    const ExpandParams p = {reinterpret_cast<const uint32_t*>(codes), reinterpret_cast<const uint32_t*>(scales), n_pages,
                            page_tokens, kv_heads, group, row_start, first_pos, table, table_stride, n_requests, window,
                            keys, values, blocks, block_stride, n_blocks};
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 grid((unsigned)n_blocks, (unsigned)kv_heads);
#define EXPAND(D)                                                                              \
    if (head_dim == D) {                                                                       \
        if (dtype == CB_F32) cb_launch(expand4_kernel<D, float>, grid, dim3(256), 0, s, p);    \
        else cb_launch(expand4_kernel<D, __nv_bfloat16>, grid, dim3(256), 0, s, p);            \
        return cb_last_error();                                                                \
    }
    EXPAND(64) EXPAND(128) EXPAND(192) EXPAND(256)
#undef EXPAND
    return CB_ERR_UNSUPPORTED;
}
