// Writing the cache in 4 bits, and reading it back as it stands.
//
//   append4   a row's q and k are rotated by its position, k and v go to the row's place in the pages.
//             A block a row and a run of its heads, so that its position, place and angles are fetched once; D/8
//             lanes a head, eight neighbouring features a lane: 16 bytes a load where rows are aligned, the next
//             head's before this one's are worked on.  Lane l of eight takes the features whose codes lie at bits
//             4l.. 4l + 3 of their words, so that eight lanes' codes are turned into eight words by a transposition
//             of 8 x 8 nibbles, three shuffles; a group's least and largest number take two to four shuffles each.
//             2,048 rows of 32 + 16 heads of 128 in bfloat16: 13.8 us, 3.1 TB/s of rows and words (a block's chain of
//             position, place, angles, numbers, shuffles, with three blocks an SM to hide it); 64 rows 2.5 us, one 2.
//   bounds4   of every page that the step wrote: each feature's largest and least key over the tokens that
//             the page now holds, in 8 bits with one scale.  A block a (row, kv head), a thread a word of codes and
//             every 16th token; only the last row of each page's run does anything.  64 rows of 8 heads of 128,
//             pages of 64: 5.5 us, a thread's chain through place, codes and pairs, then a block's largest.
//   values4   the whole pool as float32 or bfloat16 rows.
//   span4     before expand4: how large the numbers of every 64 tokens can be.
//   expand4   the pages of some requests as float16 rows in pages of 64 tokens, for attention over many rows: 2,048 tokens
//             of 8 heads of 128, 11 MB, both 9 us, two chains of place, words and pairs one behind the other.
#define CB_PDL_BIT 6      // with the other quantised operators
#include "cache4.cuh"

namespace {

// (fminf and fmaxf would lose a NaN)
__device__ __forceinline__ float least_of(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float largest_of(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
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

// Eight codes of a group, the e-th in bits 4e.. 4e + 3.  (x - low) * inverse lies in 0 .. 15.06 (low is not above x, and the
// step is off by 2^-8 of it at most), so that adding 1.5 2^23 rounds it to the nearest, ties to even, and leaves the code in
// the lowest bits; what else these numbers' bits hold is the same for all eight and goes with one subtraction.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], const Coding& c) {
    uint32_t m = 0u - 0x4b400000u * 0x11111111u;
#pragma unroll
    for (int e = 0; e < 8; ++e)
        m += __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x[e], c.low), c.inverse), 12582912.f)) << (4 * e);
    return m;
}

// Eight neighbouring numbers (VEC: aligned to 16 bytes).
template <typename T, bool VEC>
__device__ __forceinline__ void load_eight(const T* src, float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = cb_to_float(src[e]);
    } else if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 a = *reinterpret_cast<const uint4*>(src);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __uint_as_float(w[e] << 16);
            v[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store_eight(T* dst, const float (&v)[8]) {
    if constexpr (!VEC) {
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[e] = cb_from_float<T>(v[e]);
    } else if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4*>(dst)[0] = make_float4(v[0], v[1], v[2], v[3]);
        reinterpret_cast<float4*>(dst)[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
        __nv_bfloat162 b[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(b);
    }
}

// A word's eight codes, the lowest bits' first.  (A code under the exponent of 2^23 is 2^23 + code; one that lies 4 e bits
// higher, up to bit 19, is taken down by 16^-e: no shift, no conversion.)
__device__ __forceinline__ void codes_as_floats(uint32_t m, float (&v)[8]) {
    const uint32_t upper = m >> 20;
    constexpr float DOWN[5] = {1.f, 0.0625f, 0.00390625f, 0.000244140625f, 0.0000152587890625f};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int at = e < 5 ? e : e - 5;
        const uint32_t bits = ((e < 5 ? m : upper) & (15u << (4 * at))) | 0x4b000000u;
        v[e] = (__uint_as_float(bits) - 8388608.f) * DOWN[at];
    }
}

// Eight numbers as they come from memory.
template <typename T>
struct Eight {
    uint32_t raw[2 * sizeof(T)] = {};
    template <bool VEC>
    __device__ __forceinline__ void load(const T* src) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(raw)[i] = reinterpret_cast<const uint4*>(src)[i];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) reinterpret_cast<T*>(raw)[e] = src[e];
        }
    }
    __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            v[e] = sizeof(T) == 4 ? __uint_as_float(raw[e % (2 * sizeof(T))])
                                  : __uint_as_float(e & 1 ? raw[e / 2] & 0xffff0000u : raw[e / 2] << 16);
    }
};

// Nibbles of eight lanes' words, transposed: nibble n of lane l becomes nibble l of lane n (lanes in runs of eight).
__device__ __forceinline__ uint32_t transposed(uint32_t m, int l) {
    uint32_t other = __shfl_xor_sync(0xffffffffu, m, 4);
    m = (l & 4) ? __byte_perm(other, m, 0x7632) : __byte_perm(m, other, 0x5410);
    other = __shfl_xor_sync(0xffffffffu, m, 2);
    m = (l & 2) ? __byte_perm(other, m, 0x7351) : __byte_perm(m, other, 0x6240);
    other = __shfl_xor_sync(0xffffffffu, m, 1);
    return (l & 1) ? ((other >> 4) & 0x0f0f0f0fu) | (m & 0xf0f0f0f0u) : (m & 0x0f0f0f0fu) | ((other << 4) & 0xf0f0f0f0u);
}

// The eights of a row, D/8 lanes: lane 8 w + l has the word of g = l, and of the transposed words the codes of the
// features from f on.
template <int D>
__device__ __forceinline__ int eight_of(int within) {
    const int l = within & 7;
    return 64 * (within >> 3) + 8 * ((l & 1) | ((l & 2) << 1) | ((l & 4) >> 1));         // (0, 1, 4, 5, 2, 3, 6, 7)[l]
}

// VEC: rows are aligned to 16 bytes, and half of the rotated features is a multiple of eight.
template <int D, int GROUP, typename T, bool VEC>
__global__ void __launch_bounds__(256, 3) append4_kernel(const AppendParams p, int heads_each) {
    cb_pdl_wait();
    cb_pdl_trigger();              // (after the wait: the kernel of the bounds reads the step's numbers before its own)
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES, W = D / 64, NG = D / GROUP, STEP = 8 * PER_WARP;
    const int lane = threadIdx.x & 31, within = lane % LANES;
    const int w = within >> 3, l = within & 7, f = eight_of<D>(within);
    const int row = blockIdx.x, heads = p.n_heads + (p.write ? 2 * p.kv_heads : 0);
    const int end = min(heads, ((int)blockIdx.y + 1) * heads_each);
    int head = blockIdx.y * heads_each + (threadIdx.x >> 5) * PER_WARP + lane / LANES;
    if (lane >= LANES * PER_WARP) head = end;                 // (lanes that have no head go along: shuffles)
    const T* row_src = reinterpret_cast<const T*>(p.qkv) + (size_t)row * p.qkv_stride;
    const int half = p.rotary >> 1;
    const bool first = f < half, halves = VEC && !p.neighbours && f < p.rotary;
    const int other_f = first ? f + half : f - half;
    Eight<T> ahead_x[2], ahead_y[2];                           // the next two heads' numbers, and those they turn with
    auto load = [&](int h, Eight<T>& x, Eight<T>& y) {
        if (h >= end) return;
        x.template load<VEC>(row_src + (size_t)h * D + f);
        if (halves && h < p.n_heads + p.kv_heads) y.template load<VEC>(row_src + (size_t)h * D + other_f);
    };
    load(head, ahead_x[0], ahead_y[0]);
    load(head + STEP, ahead_x[1], ahead_y[1]);
    const int request = p.row_request[row], pos = p.positions[row];
    if (request < 0 || request >= p.n_requests || pos < 0 || (p.rotary > 0 && pos >= p.n_positions)) return;
    const float* cs = p.cos_t + (size_t)pos * half;
    const float* sn = p.sin_t + (size_t)pos * half;
    float c[8], s[8];
    if (halves) {
        load_eight<float, VEC>(cs + (first ? f : other_f), c);
        load_eight<float, VEC>(sn + (first ? f : other_f), s);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] = first ? -s[e] : s[e];           // a cos - b sin is a cos + b (-sin) to the bit
    }
    const long long place = c4_row(p.table + (size_t)request * p.table_stride, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
    auto one = [&](int turn, Eight<T>& next_x, Eight<T>& next_y) {
        const bool live = head < end;
        float x[8];
        next_x.get(x);
        if (live && f < p.rotary && head < p.n_heads + p.kv_heads) {
            if (halves) {
                float y[8];
                next_y.get(y);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = __fadd_rn(__fmul_rn(x[e], c[e]), __fmul_rn(y[e], s[e]));
            } else if (p.neighbours) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (f + 2 * e >= p.rotary) break;
                    const float a = x[2 * e], b = x[2 * e + 1], co = cs[(f >> 1) + e], si = sn[(f >> 1) + e];
                    x[2 * e] = __fsub_rn(__fmul_rn(a, co), __fmul_rn(b, si));
                    x[2 * e + 1] = __fadd_rn(__fmul_rn(a, si), __fmul_rn(b, co));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if (f + e >= p.rotary) break;
                    const bool lower = f + e < half;
                    const int j = lower ? f + e : f + e - half;
                    const float v = cb_to_float(row_src[(size_t)head * D + (lower ? j + half : j)]);
                    const float own = __fmul_rn(x[e], cs[j]), cross = __fmul_rn(v, sn[j]);
                    x[e] = lower ? __fsub_rn(own, cross) : __fadd_rn(cross, own);
                }
            }
        }
        __syncwarp();                     // q may take its own place: every lane has read what it turns
        load(head + 2 * STEP, next_x, next_y);
        if (live && head < p.n_heads)
            store_eight<T, VEC>(reinterpret_cast<T*>(p.q) + (size_t)row * p.q_stride + (size_t)head * D + f, x);
        if (turn + PER_WARP <= p.n_heads) return;                // queries alone
        // groups of 32 are the lanes of equal l & 2, of 64 all eight, of 128 two eights
        float least = x[0], largest = x[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) {
            least = least_of(least, x[e]);
            largest = largest_of(largest, x[e]);
        }
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            if (o == 2 && GROUP < 64) continue;
            if (o == 8 && GROUP < 128) continue;
            least = least_of(least, __shfl_xor_sync(0xffffffffu, least, o));
            largest = largest_of(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        }
        const Coding coding = coding_of(least, largest);
        const uint32_t m = transposed(codes_of(x, coding), l);
        if (live && head >= p.n_heads && place >= 0) {
            const int side = head >= p.n_heads + p.kv_heads;
            const long long at = place + (long long)(head - p.n_heads - side * p.kv_heads) * p.page_tokens
                + (long long)side * p.n_pages * p.kv_heads * p.page_tokens;
            p.codes[at * (D / 8) + l * W + w] = m;
            // (the first lane of a group)
            const bool leads = GROUP == 32 ? (l & ~2) == 0 : GROUP == 64 ? l == 0 : (within & 15) == 0;
            if (leads) p.scales[at * NG + f / GROUP] = coding.pair;
        }
    };
    // (as many turns for every lane of a warp)
    for (int turn = blockIdx.y * heads_each + (threadIdx.x >> 5) * PER_WARP; turn < end; turn += 2 * STEP) {
        one(turn, ahead_x[0], ahead_y[0]);
        head += STEP;
        if (turn + STEP >= end) break;
        one(turn + STEP, ahead_x[1], ahead_y[1]);
        head += STEP;
    }
}

template <int D>
__global__ void __launch_bounds__(2 * D) bounds4_kernel(const AppendParams p, int group) {
    constexpr int WORDS = D / 8, W = D / 64;                 // 16 threads a word, neighbours take neighbouring words
    __shared__ float ends[2][8][16][WORDS];
    __shared__ float largest[2 * D / 32];
    __shared__ __align__(16) int8_t rounded[2 * D];
    const int row = blockIdx.x / p.kv_heads, kv = blockIdx.x - row * p.kv_heads;
    const int request = p.row_request[row], pos = p.positions[row], index = pos / p.page_tokens;
    long long at = -1;
    if (request >= 0 && request < p.n_requests && pos >= 0 && !(p.rotary > 0 && pos >= p.n_positions)
        && !(row + 1 < p.rows && p.row_request[row + 1] == request && p.positions[row + 1] / p.page_tokens == index
             && !(p.rotary > 0 && p.positions[row + 1] >= p.n_positions)))           // (a row that is left out is nobody's last)
        at = c4_row(p.table + (size_t)request * p.table_stride, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
    if (at < 0) {
        cb_pdl_wait();             // (every block waits: what is launched behind this kernel waits for it alone)
        return;
    }
    const int held = pos - index * p.page_tokens + 1;
    const long long page = (at - (held - 1)) / ((long long)p.kv_heads * p.page_tokens);
    at += (long long)kv * p.page_tokens - (held - 1);
    const int tid = threadIdx.x, lane = tid & 31, word = tid % WORDS, t = tid / WORDS;
    const int g = word / W, f = 64 * (word - g * W) + g;              // features f + 8 k
    const uint32_t* codes = p.codes + at * WORDS + word;
    const uint32_t* scales = p.scales + at * (D / group);
    const int g0 = f / group, g1 = (f + 32) / group;                  // k < 4, k >= 4
    float hi[8], lo[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) hi[k] = -INFINITY, lo[k] = INFINITY;
    cb_pdl_wait();                 // (what is above is the step's numbers, which were there before the rows were written)
    cb_pdl_trigger();
#pragma unroll 4
    for (int i = t; i < held; i += 16) {
        const uint32_t c = codes[(size_t)i * WORDS];
        const uint32_t a = scales[(size_t)i * (D / group) + g0], b = scales[(size_t)i * (D / group) + g1];
        float code[8];
        codes_as_floats(c, code);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t pair = k < 4 ? a : b;
            const float v = fmaf(code[c4_shift(k) / 4], c4_step(pair), c4_low(pair));
            hi[k] = fmaxf(hi[k], v);
            lo[k] = fminf(lo[k], v);
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        ends[0][k][t][word] = hi[k];
        ends[1][k][t][word] = lo[k];
    }
    __syncthreads();
    // a thread a feature's end: the first D threads the largest, the others the least
    const int side = tid / D, mine = tid - side * D, my_word = mine % WORDS, my_k = mine / WORDS;
    float end = ends[side][my_k][0][my_word];
#pragma unroll
    for (int i = 1; i < 16; ++i) {
        const float v = ends[side][my_k][i][my_word];
        end = side ? fminf(end, v) : fmaxf(end, v);
    }
    if (fabsf(end) == INFINITY) end = 0.f;                   // (a feature of which no token's key is a number)
    float most = cb_warp_max(fabsf(end));
    if (lane == 0) largest[tid >> 5] = most;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2 * D / 32; ++i) most = fmaxf(most, largest[i]);
    const float scale = __fmul_rn(most, 1.0f / 127.0f);
    const float inverse = scale > 0.f ? __frcp_rn(scale) : 0.f;
    const int my_g = my_word / W;
    rounded[side * D + 64 * (my_word - my_g * W) + my_g + 8 * my_k] =
        (int8_t)(int)fminf(fmaxf(rintf(__fmul_rn(end, inverse)), -127.f), 127.f);
    __syncthreads();
    const long long to = page * p.kv_heads + kv;
    if (tid < 2 * D / 16)
        reinterpret_cast<int4*>(p.bounds + to * 2 * D)[tid] = reinterpret_cast<const int4*>(rounded)[tid];
    if (tid == 0) p.bound_scales[to] = scale;
}

// Eight neighbouring features of a row: its word and pair, then their values (every lane of the warp takes part).
template <int D>
__device__ __forceinline__ uint2 eight_fetched(const uint32_t* codes, const uint32_t* scales, long long at, bool there, int group,
                                               int within) {
    return there ? make_uint2(codes[at * (D / 8) + (within & 7) * (D / 64) + (within >> 3)], scales[at * (D / group) + eight_of<D>(within) / group])
                 : make_uint2(0u, 0u);
}

__device__ __forceinline__ void eight_values(uint2 from, int within, float (&v)[8]) {
    const uint32_t m = transposed(from.x, within & 7);
    const float step = c4_step(from.y), low = c4_low(from.y);
    codes_as_floats(m, v);
#pragma unroll
    for (int g = 0; g < 8; ++g) v[g] = fmaf(v[g], step, low);
}

template <int D, typename T>
__global__ void __launch_bounds__(256) values4_kernel(const uint32_t* codes, const uint32_t* scales, int group, long long rows,
                                                      T* out) {
    cb_pdl_trigger();
    cb_pdl_wait();
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
    const int lane = threadIdx.x & 31, within = lane % LANES;
    const long long stride = (long long)gridDim.x * 8 * PER_WARP;
    for (long long row = ((long long)blockIdx.x * 8 + (threadIdx.x >> 5)) * PER_WARP; row < rows; row += 2 * stride) {
        float v[2][8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long long at = row + j * stride + lane / LANES;
            eight_values(eight_fetched<D>(codes, scales, at, at < rows && lane < LANES * PER_WARP, group, within), within, v[j]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const long long at = row + j * stride + lane / LANES;
            if (at < rows && lane < LANES * PER_WARP) store_eight<T, true>(out + at * D + eight_of<D>(within), v[j]);
        }
    }
}

__global__ void __launch_bounds__(256) bound_values4_kernel(const uint32_t* bounds, const float* scales, int words_each,
                                                            long long words, float* out) {
    cb_pdl_trigger();
    cb_pdl_wait();
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < words; i += (long long)gridDim.x * 256) {
        const uint32_t w = bounds[i];
        const float a = scales[i / words_each];
        reinterpret_cast<float4*>(out)[i] = make_float4((float)(int8_t)w * a, (float)(int8_t)(w >> 8) * a,
                                                        (float)(int8_t)(w >> 16) * a, (float)(int8_t)(w >> 24) * a);
    }
}

constexpr int C4_LEAST_SPAN = -100;      // the smallest exponent of a request's numbers that counts

struct ExpandParams {
    const uint32_t* codes;
    const uint32_t* scales;
    int n_pages, page_tokens, kv_heads, group;
    const int* row_start;
    const int* first_pos;
    const int* table;
    int table_stride, n_requests;
    int window;
    __half* keys;            // [blocks of 64 tokens][kv heads][64][D]
    __half* values;
    int* spans;              // [blocks of 64 tokens][kv heads][keys, values]
    float2* factors;         // [requests][kv heads]: what keys and values were divided by
    uint32_t* seen;          // [requests][block_stride][2]: a bit a token that is there
    int* blocks;             // [requests][block_stride]: which blocks of 64 tokens are a request's
    int block_stride, n_blocks;
    int rows;                // of the step's tensors: what requests have beyond them is not there
};

// Which request a block of 64 tokens is of, from how many blocks the requests before it have: from the one that holds the
// first token that a row sees to the one that holds the last.
struct Laid {
    int request, before, count, first, held, lo;
    __device__ __forceinline__ int index_of(int block) const { return block - before + (lo >> 6); }
};

__device__ __forceinline__ Laid laid_at(const ExpandParams& p, int request, int before) {
    Laid at = {request, before, 0, 0, 0, 0};
    at.first = p.first_pos[request];
    const int row = p.row_start[request];
    at.held = row < 0 ? 0 : at.first + max(0, min(p.row_start[request + 1], p.rows) - row);
    at.lo = p.window > 0 ? max(0, at.first - p.window + 1) : 0;
    at.count = max(0, min((at.held + 63) >> 6, p.block_stride) - (at.lo >> 6));
    return at;
}

__device__ __forceinline__ Laid laid_of(const ExpandParams& p, int block) {
    Laid at = {0, 0, 0, 0, 0, 0};
    for (int r = 0; r < p.n_requests; ++r) {
        at = laid_at(p, r, at.before + at.count);
        if (block < at.before + at.count) return at;
    }
    at.request = p.n_requests;
    return at;
}

__device__ __forceinline__ float two_to(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

__device__ __forceinline__ void store_halves(__half* dst, const float (&v)[8]) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(h);
}

// A block of threads a block of 64 tokens and kv head: the exponents of the largest finite numbers that its keys and values
// can hold, from their groups' pairs.
template <int D>
__global__ void __launch_bounds__(128) span4_kernel(const ExpandParams p) {
    cb_pdl_wait();
    cb_pdl_trigger();              // (after the wait: the tiles' kernel reads where rows begin, and queries, before its own)
    const Laid in = laid_of(p, blockIdx.x);
    const int side = threadIdx.x >> 6, pos = in.index_of(blockIdx.x) * 64 + (threadIdx.x & 63);
    int e = C4_LEAST_SPAN;
    if (in.request < p.n_requests && pos < in.held && pos >= in.lo) {
        const long long at = c4_row(p.table + (size_t)in.request * p.table_stride, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
        if (at >= 0) {
            const long long row = at + ((long long)side * p.n_pages * p.kv_heads + blockIdx.y) * p.page_tokens;
            for (int g = 0; g < D / p.group; ++g) {
                const uint32_t pair = p.scales[row * (D / p.group) + g];
                const float most = fmaxf(fabsf(c4_low(pair)), fabsf(fmaf(15.f, c4_step(pair), c4_low(pair))));
                if (most == most) e = max(e, min((int)(__float_as_uint(most) >> 23) - 127, 127));
            }
        }
    }
    e = __reduce_max_sync(0xffffffffu, e);
    __shared__ int of_warps[4];
    if ((threadIdx.x & 31) == 0) of_warps[threadIdx.x >> 5] = e;
    __syncthreads();
    if (threadIdx.x < 2)
        p.spans[((size_t)blockIdx.x * p.kv_heads + blockIdx.y) * 2 + threadIdx.x] = max(of_warps[2 * threadIdx.x], of_warps[2 * threadIdx.x + 1]);
}

// Keys (x) and values (y) of a request and kv head go into float16 times 2^(14 - e), e the largest of its blocks' exponents:
// the largest lies below 2^15, and what is up to 2^28 times smaller keeps float16's eleven bits.  Whole warps.
__device__ __forceinline__ int2 exponents_of(const ExpandParams& p, const Laid& in, int kv) {
    int2 e = make_int2(C4_LEAST_SPAN, C4_LEAST_SPAN);
    for (int i = threadIdx.x & 31; i < in.count && in.before + i < p.n_blocks; i += 32) {
        const int2 of = reinterpret_cast<const int2*>(p.spans)[(size_t)(in.before + i) * p.kv_heads + kv];
        e = make_int2(max(e.x, of.x), max(e.y, of.y));
    }
    return make_int2(__reduce_max_sync(0xffffffffu, e.x) - 14, __reduce_max_sync(0xffffffffu, e.y) - 14);
}

// A block of threads a block of 64 tokens and kv head; block n_blocks is of zeros, for what the table has behind a request's
// last token.  Tokens that no row of the step sees are left out, as zeros; of those whose table entry names no page `seen`
// has no bit.  A value that is no number becomes its key's: attention by tiles multiplies the values of masked keys by
// zero, but does not take their scores.
template <int D>
__global__ void __launch_bounds__(256) expand4_kernel(const ExpandParams p) {
    cb_pdl_wait();
    cb_pdl_trigger();              // (after the wait: the tiles' kernel reads where rows begin, and queries, before its own)
    __shared__ uint32_t bad[64];
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES, ROUNDS = 64 / (8 * PER_WARP);
    const int block = blockIdx.x, lane = threadIdx.x & 31, within = lane % LANES;
    if (block == 0 && blockIdx.y == 0) {
        Laid at = {0, 0, 0, 0, 0, 0};
        for (int r = 0; r < p.n_requests; ++r) {
            at = laid_at(p, r, at.before + at.count);
            for (int i = threadIdx.x; i < p.block_stride; i += 256) {
                const int one = at.before + i - (at.lo >> 6);
                const bool some = one >= at.before && one < min(at.before + at.count, p.n_blocks);
                p.blocks[(size_t)r * p.block_stride + i] = some ? one : p.n_blocks;
                if (!some) reinterpret_cast<uint2*>(p.seen)[(size_t)r * p.block_stride + i] = make_uint2(0u, 0u);
            }
        }
    }
    const Laid in = laid_of(p, block);
    const int request = in.request, held = in.held, lo = in.lo, index = in.index_of(block);
    const bool some = block < p.n_blocks && request < p.n_requests;
    const int* table = p.table + (size_t)request * p.table_stride;
    __shared__ int there[64];
    if (threadIdx.x < 64) bad[threadIdx.x] = 0;
    const int f = eight_of<D>(within);
    const long long side_rows = (long long)p.n_pages * p.kv_heads * p.page_tokens;
    uint2 key[ROUNDS], value[ROUNDS];
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
        const int pos = index * 64 + (j * 8 + (threadIdx.x >> 5)) * PER_WARP + lane / LANES;
        long long at = -1;
        if (some && lane < LANES * PER_WARP && pos < held && pos >= lo)
            at = c4_row(table, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, pos);
        if (within == 0 && lane < LANES * PER_WARP) there[pos - index * 64] = at >= 0;
        if (at >= 0) at += (long long)blockIdx.y * p.page_tokens;
        key[j] = eight_fetched<D>(p.codes, p.scales, at, at >= 0, p.group, within);
        value[j] = eight_fetched<D>(p.codes, p.scales, at + side_rows, at >= 0, p.group, within);
    }
    const int2 e = some ? exponents_of(p, in, blockIdx.y) : make_int2(0, 0);
    const float down_k = two_to(-e.x), down_v = two_to(-e.y);
    if (some && block == in.before && threadIdx.x == 0)
        p.factors[(size_t)request * p.kv_heads + blockIdx.y] = make_float2(two_to(e.x), two_to(e.y));
    __syncthreads();
    if (some && index < p.block_stride && blockIdx.y == 0 && threadIdx.x < 64) {
        const uint32_t bits = __ballot_sync(0xffffffffu, there[threadIdx.x] != 0);
        if (lane == 0) p.seen[((size_t)request * p.block_stride + index) * 2 + (threadIdx.x >> 5)] = bits;
    }
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j)
        if (c4_low(value[j].y) != c4_low(value[j].y)) {
            bad[(j * 8 + (threadIdx.x >> 5)) * PER_WARP + lane / LANES] = 1;
            value[j] = make_uint2(0u, 0u);
        }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ROUNDS; ++j) {
        const int t = (j * 8 + (threadIdx.x >> 5)) * PER_WARP + lane / LANES;
        const long long to = (((long long)block * p.kv_heads + blockIdx.y) * 64 + t) * D + f;
        float k[8], v[8];
        eight_values(key[j], within, k);
        eight_values(value[j], within, v);
        if (lane >= LANES * PER_WARP) continue;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (bad[t]) k[e] = __int_as_float(0x7fffffff);
            else if (k[e] == k[e]) k[e] = fminf(fmaxf(k[e] * down_k, -65504.f), 65504.f);
            v[e] = fminf(fmaxf(v[e] * down_v, -65504.f), 65504.f);
        }
        store_halves(p.keys + to, k);
        store_halves(p.values + to, v);
    }
}

template <int D, int GROUP>
int append_of(const AppendParams& p, int dtype, cudaStream_t stream) {
    const int size = dtype == CB_F32 ? 4 : 2;
    // heads a block: all of a row's where there are rows for every SM, else as few turns of a block's warps as fill them
    const int step = 8 * (32 / (D / 8)), heads = p.n_heads + (p.write ? 2 * p.kv_heads : 0), turns = (heads + step - 1) / step;
    const int runs = max(1, min(turns, 148 * 4 / p.rows)), heads_each = (turns + runs - 1) / runs * step;
    const dim3 grid((unsigned)p.rows, (unsigned)((heads + heads_each - 1) / heads_each));
    const bool vec = ((uintptr_t)p.qkv | (uintptr_t)p.q | (uintptr_t)p.cos_t | (uintptr_t)p.sin_t) % 16 == 0
        && p.qkv_stride * size % 16 == 0 && p.q_stride * size % 16 == 0 && (p.rotary / 2) % 8 == 0;
    int rc;
    if (dtype == CB_F32) rc = cb_launch(vec ? append4_kernel<D, GROUP, float, true> : append4_kernel<D, GROUP, float, false>,
                                        grid, dim3(256), 0, stream, p, heads_each);
    else rc = cb_launch(vec ? append4_kernel<D, GROUP, __nv_bfloat16, true> : append4_kernel<D, GROUP, __nv_bfloat16, false>,
                        grid, dim3(256), 0, stream, p, heads_each);
    if (rc == 0 && p.write && p.bounds != nullptr)
        rc = cb_launch(bounds4_kernel<D>, dim3((unsigned)p.rows * p.kv_heads), dim3(2 * D), 0, stream, p, GROUP);
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
    const dim3 grid((unsigned)min((rows * (head_dim / 8) + 511) / 512, 148LL * 64));
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

CB_EXPORT int cb_bound_values4(const void* bounds, const float* scales, int heads, int head_dim, float* out, void* stream) {
    const long long words = (long long)heads * head_dim / 2;
    cb_launch(bound_values4_kernel, dim3((unsigned)min((words + 255) / 256, 148LL * 32)), dim3(256), 0,
              reinterpret_cast<cudaStream_t>(stream), reinterpret_cast<const uint32_t*>(bounds), scales, head_dim / 2, words, out);
    return cb_last_error();
}

CB_EXPORT int cb_expand4(const void* codes, const void* scales, int n_pages, int page_tokens, int kv_heads, int head_dim,
                         int group, const int* row_start, const int* first_pos, const int* table, int table_stride,
                         int n_requests, int window, void* keys, void* values, int* spans, float* factors, uint32_t* seen,
                         int* blocks, int block_stride, int n_blocks, int rows, void* stream) {
    if (n_blocks <= 0) return 0;
    const ExpandParams p = {reinterpret_cast<const uint32_t*>(codes), reinterpret_cast<const uint32_t*>(scales), n_pages,
                            page_tokens, kv_heads, group, row_start, first_pos, table, table_stride, n_requests, window,
                            reinterpret_cast<__half*>(keys), reinterpret_cast<__half*>(values), spans,
                            reinterpret_cast<float2*>(factors), seen, blocks, block_stride, n_blocks, rows};
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const dim3 spans_grid((unsigned)n_blocks, (unsigned)kv_heads);
    const dim3 grid((unsigned)n_blocks + 1, (unsigned)kv_heads);
    if (head_dim == 64) {
        cb_launch(span4_kernel<64>, spans_grid, dim3(128), 0, s, p);
        cb_launch(expand4_kernel<64>, grid, dim3(256), 0, s, p);
    } else if (head_dim == 128) {
        cb_launch(span4_kernel<128>, spans_grid, dim3(128), 0, s, p);
        cb_launch(expand4_kernel<128>, grid, dim3(256), 0, s, p);
    } else return CB_ERR_UNSUPPORTED;
    return cb_last_error();
}
