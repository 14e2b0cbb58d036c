// out[M,N] = rows[M,K] . W[N,K]^T over quantised weights, for few rows (decoded tokens).
//
//   FOUR_BF16  W = (codes - 8) * group scale, rows bf16
//   FOUR_F32   the same, rows fp32
//   EIGHT      W = e4m3 values, rows e4m3 with a scale each
//   all        times a scale per output feature, plus `add` if given; fp32 or bf16 out
//
// Such a product reads its weights once and does little else, so they go from memory straight into the
// registers that hold the operands of mma.sync (weights: 16 features by 16 or 32 k; rows: 8 at a time;
// fp32 sums): no descriptor, barrier or tensor memory stands between a load and its use.  A dot
// product does not see the order of k, so a thread takes 16 neighbouring bytes of a feature's
// weights and the same k of its row of the step, whatever k the instruction calls them.
//
// A block owns 32 features and 8 or 16 rows; its warps take segments of K in turn and their sums are added
// in the warps' order, so the order of a dot product's sum depends on K alone.  A warp asks for its next
// segments' weights before it multiplies the present ones.
//
// LONG: fp32 results over 4-bit weights where a warp's share of K is above MMA_CHUNK: so many k a sum, and the sums are added
// with rounding.
#define CB_PDL_BIT 6      // this file's bit in CRUCIBLE_PDL
#include "quantized.cuh"

namespace {

constexpr int PAIRS = 2;                // 16 features each: a block's
constexpr int FEATURES = 16 * PAIRS;
constexpr int BATCH = 2;                // segments of weights that a warp asks for together

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_e4m3(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// What a thread holds of a segment's weights: 16 bytes of each of its features, and their scales.  (Those of features g and
// g + 8 are put together when they are needed: where they are asked for, that would wait for them, 8 rows of 768 by
// 1,280 3.0 us, not 2.8.)
struct Held {
    uint4 w[PAIRS][2];
    uint32_t scale[PAIRS][2];
};

// NT: groups of 8 rows.  WARPS share K.
template <int KIND, int NT, int WARPS, bool LONG>
__global__ void __launch_bounds__(WARPS * 32, (KIND == FOUR_F32 ? 8 : 16) / WARPS)
linear_few_kernel(const QuantizedArgs p, uint32_t run_magic) {
    constexpr int SEG = KIND == EIGHT ? 64 : 128;       // k of a segment: 64 bytes of a feature's weights
    constexpr int MINE = SEG / 4;                       // k of a thread: 16 bytes
    constexpr int SIZE = KIND == EIGHT ? 1 : (KIND == FOUR_F32 ? 4 : 2);
    constexpr int ROWS = 8 * NT;
    __shared__ float sums[WARPS][FEATURES][ROWS + 1];
    cb_pdl_wait();
    cb_pdl_trigger();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * FEATURES, m0 = blockIdx.y * ROWS;
    const int K = p.K, whole = K / SEG;                 // (segments that do not end in K's tail)
    // the thread's features (beyond the last: the last, whose sums nobody stores) and rows
    const uint8_t* w[PAIRS][2];
    uint32_t scales[PAIRS][2];                          // offsets, in a matrix of group scales
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int f = min(n0 + 16 * i + 8 * h + g, p.N - 1);
            w[i][h] = static_cast<const uint8_t*>(p.w) + f * p.ldw + 16 * t;
            scales[i][h] = KIND == EIGHT ? 0 : (uint32_t)(f - n0) * (uint32_t)p.groups;
        }
    const uint8_t* const block_scales = KIND == EIGHT ? nullptr : p.group_scale + (long long)n0 * p.groups;
    const uint8_t* rows[NT];
    bool has_row[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        has_row[i] = m0 + 8 * i + g < p.M;
        rows[i] = static_cast<const uint8_t*>(p.rows) + (has_row[i] ? m0 + 8 * i + g : 0) * p.ldr * SIZE + t * MINE * SIZE;
    }
    float acc[PAIRS][NT][4], rest[KIND == FOUR_F32 ? PAIRS : 1][NT][4];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = rest[KIND == FOUR_F32 ? i : 0][j][e] = 0.f;

    // 16 e4m3 numbers from `at`; zeros beyond K, where a row may end inside them
    auto load16 = [&](const uint8_t* at, int left) -> uint4 {
        if (left >= 16) return __ldg(reinterpret_cast<const uint4*>(at));
        uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < left) word[i >> 2] |= (uint32_t)at[i] << (8 * (i & 3));
        return make_uint4(word[0], word[1], word[2], word[3]);
    };
    // TAIL: the segment in which K ends; a thread whose k lie beyond it has zeros
    auto fetch = [&](Held& h, int seg, bool tail) {
        const int k = seg * SEG + t * MINE;
        if (tail && k >= K) {
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) h.w[i][0] = h.w[i][1] = make_uint4(0, 0, 0, 0), h.scale[i][0] = h.scale[i][1] = 0;
            return;
        }
        // the scale of a run of 32 k: 2 (k / 32) over the runs that share one, by half their reciprocal
        const uint32_t at = KIND == EIGHT ? 0 : __umulhi((uint32_t)k >> 4, run_magic);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint8_t* from = w[i][j] + seg * 64;
                h.w[i][j] = KIND == EIGHT && tail ? load16(from, K - k) : __ldg(reinterpret_cast<const uint4*>(from));
            }
            if (KIND != EIGHT)
                h.scale[i][0] = __ldg(block_scales + (scales[i][0] + at)), h.scale[i][1] = __ldg(block_scales + (scales[i][1] + at));
        }
    };
    auto multiply = [&](const Held& h, int seg, bool tail) {
        const int k = seg * SEG + t * MINE;
        if constexpr (KIND == EIGHT) {
            uint4 r[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                r[j] = make_uint4(0, 0, 0, 0);
                if (has_row[j] && (!tail || k < K)) r[j] = load16(rows[j] + seg * SEG, tail ? K - k : 16);
            }
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) {
                const uint4 x = h.w[i][0], y = h.w[i][1];
                const uint32_t lo[4] = {x.x, y.x, x.y, y.y}, hi[4] = {x.z, y.z, x.w, y.w};
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    mma_e4m3(acc[i][j], lo, r[j].x, r[j].y);
                    mma_e4m3(acc[i][j], hi, r[j].z, r[j].w);
                }
            }
        } else {
            uint4 b16[KIND == FOUR_BF16 ? NT : 1][4];
            if constexpr (KIND == FOUR_BF16) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        b16[j][c] = make_uint4(0, 0, 0, 0);
                        if (has_row[j] && (!tail || k < K))
                            b16[j][c] = __ldg(reinterpret_cast<const uint4*>(rows[j] + seg * SEG * SIZE) + c);
                    }
            }
            ScalePair s[PAIRS][2];
#pragma unroll
            for (int i = 0; i < PAIRS; ++i) scale_pairs(__byte_perm(h.scale[i][0], h.scale[i][1], 0x0040), s[i]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {               // eight k at a time
                uint32_t b[NT][3][4];                   // [rows][part][pairs of k]
                if constexpr (KIND == FOUR_F32) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (has_row[j] && (!tail || k < K))
                                r = __ldg(reinterpret_cast<const float4*>(rows[j] + seg * SEG * SIZE) + 2 * c + q);
                            uint32_t one[3], two[3];
                            three_parts(r.x, r.y, one);
                            three_parts(r.z, r.w, two);
#pragma unroll
                            for (int i = 0; i < 3; ++i) b[j][i][2 * q] = one[i], b[j][i][2 * q + 1] = two[i];
                        }
                } else {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        b[j][0][0] = b16[j][c].x, b[j][0][1] = b16[j][c].y, b[j][0][2] = b16[j][c].z, b[j][0][3] = b16[j][c].w;
                }
#pragma unroll
                for (int i = 0; i < PAIRS; ++i) {
                    const uint4 &x = h.w[i][0], &y = h.w[i][1];
                    const uint32_t xw = c == 0 ? x.x : (c == 1 ? x.y : (c == 2 ? x.z : x.w));
                    const uint32_t yw = c == 0 ? y.x : (c == 1 ? y.y : (c == 2 ? y.z : y.w));
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t a[4] = {weight_pair(xw, 2 * q, s[i][0]), weight_pair(yw, 2 * q, s[i][1]),
                                               weight_pair(xw, 2 * q + 1, s[i][0]), weight_pair(yw, 2 * q + 1, s[i][1])};
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            mma_bf16(acc[i][j], a, b[j][0][2 * q], b[j][0][2 * q + 1]);
                            if constexpr (KIND == FOUR_F32) {
                                mma_bf16(rest[i][j], a, b[j][1][2 * q], b[j][1][2 * q + 1]);
                                mma_bf16(rest[i][j], a, b[j][2][2 * q], b[j][2][2 * q + 1]);
                            }
                        }
                    }
                }
            }
        }
    };

    // Two batches take turns: one is on its way while the other is multiplied.
    Held x[BATCH], y[BATCH];
    int seg = warp;
    auto more = [&]() { return seg + (BATCH - 1) * WARPS < whole; };
    auto ask = [&](Held (&h)[BATCH]) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) fetch(h[b], seg + b * WARPS, false);
    };
    auto take = [&](const Held (&h)[BATCH], int from) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) multiply(h[b], from + b * WARPS, false);
    };
    constexpr int SUMS = PAIRS * NT * 4;
    float room[LONG ? SUMS : 1];
    float* const aside = LONG ? set_aside(room) : nullptr;
    auto end_of_chunk = [&]() {
#pragma unroll
        for (int q = 0; q < SUMS; ++q) {
            float &v = acc[q / (NT * 4)][q / 4 % NT][q % 4], &r = rest[KIND == FOUR_F32 ? q / (NT * 4) : 0][q / 4 % NT][q % 4];
            aside[q] += KIND == FOUR_F32 ? v + r : v;
            v = r = 0.f;
        }
    };
    bool have = more();
    if (have) ask(x);
    int left = MMA_CHUNK / (2 * BATCH * SEG);
#pragma unroll 1
    while (have) {
        int from = seg;
        seg += WARPS * BATCH;
        have = more();
        if (have) ask(y);
        take(x, from);
        if (!have) break;
        from = seg;
        seg += WARPS * BATCH;
        have = more();
        if (have) ask(x);
        take(y, from);
        if (LONG && --left == 0) {
            left = MMA_CHUNK / (2 * BATCH * SEG);
            end_of_chunk();
        }
    }
    if (LONG) end_of_chunk();
#pragma unroll 1
    for (; seg * SEG < K; seg += WARPS) {
        fetch(x[0], seg, true);
        multiply(x[0], seg, true);
    }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = acc[i][j][e];
                if constexpr (KIND == FOUR_F32) v += rest[i][j][e];
                if (LONG) v += aside[(i * NT + j) * 4 + e];
                sums[warp][16 * i + 8 * (e >> 1) + g][8 * j + 2 * t + (e & 1)] = v;
            }
    __syncthreads();
#pragma unroll 1
    for (int at = threadIdx.x; at < FEATURES * ROWS; at += WARPS * 32) {
        const int f = at % FEATURES, m = at / FEATURES;
        if (n0 + f >= p.N || m0 + m >= p.M) continue;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) v += sums[i][f][m];
        finish(p, v, KIND == EIGHT ? __ldg(p.row_scale + m0 + m) : 1.f, __ldg(p.feature_scale + n0 + f), m0 + m, n0 + f);
    }
}

template <int KIND, int NT>
void launch(const QuantizedArgs& p, uint32_t run_magic, cudaStream_t s) {
    const dim3 grid((p.N + FEATURES - 1) / FEATURES, (p.M + 8 * NT - 1) / (8 * NT));
    constexpr int SHORT_K = 6144;
    static_assert(SHORT_K / 4 <= MMA_CHUNK, "four warps' sums are never long");
    if (p.K <= SHORT_K) {
        cb_launch(linear_few_kernel<KIND, NT, 4, false>, grid, dim3(128), 0, s, p, run_magic);
        return;
    }
    // (e4m3 products have 8 bits, and their sums lose nothing to speak of: 2.9e-7 of the norm for a K of 262,144)
    if constexpr (KIND != EIGHT) {
        if (!p.out_bf16 && p.K > 8 * MMA_CHUNK) {
            cb_launch(linear_few_kernel<KIND, NT, 8, true>, grid, dim3(256), 0, s, p, run_magic);
            return;
        }
    }
    cb_launch(linear_few_kernel<KIND, NT, 8, false>, grid, dim3(256), 0, s, p, run_magic);
}

template <int KIND>
void launch_rows(const QuantizedArgs& p, uint32_t run_magic, cudaStream_t s) {
    if (p.M <= 8) launch<KIND, 1>(p, run_magic, s);
    else launch<KIND, 2>(p, run_magic, s);
}

}  // namespace

// Strides of rows, add and out in elements, of w in bytes.  Whole segments are fetched 16 bytes at a
// time: `rows` and `w` 16-byte aligned, their strides multiples of 16 bytes.
CB_EXPORT int cb_linear_quantized_few(int kind, const void* rows, long long ldr, const float* row_scale, const void* w,
                                      long long ldw, const void* group_scale, const float* feature_scale,
                                      const float* add, long long lda, void* out, int out_dtype, long long ldo, int M,
                                      int N, int K, int group, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    const int size = kind == EIGHT ? 1 : (kind == FOUR_F32 ? 4 : 2);
    if (K <= 0 || K > MOST_K || ldw > MOST_PITCH || (((uintptr_t)rows | (uintptr_t)w | (uintptr_t)(ldr * size) | (uintptr_t)ldw) & 15) ||
        (M + 15) / 16 > 65535 || (kind != EIGHT && (group <= 0 || group % 32 || K % group)))
        return CB_ERR_UNSUPPORTED;
    const QuantizedArgs p = {rows, ldr, row_scale, w, ldw, (const uint8_t*)group_scale, feature_scale, add, lda, out, ldo,
                             M, N, K, group, out_dtype == CB_BF16, group > 0 ? K / group : 0};
    // half the reciprocal of the runs that share a scale, ceil(2^31 / runs): its products with 2 (k / 32) are exact
    // while K / 32 * runs < 2^31
    const uint32_t runs = (uint32_t)group / 32;
    const uint32_t run_magic = runs > 0 ? (uint32_t)(((1ull << 31) + runs - 1) / runs) : 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (kind == FOUR_BF16) launch_rows<FOUR_BF16>(p, run_magic, s);
    else if (kind == FOUR_F32) launch_rows<FOUR_F32>(p, run_magic, s);
    else if (kind == EIGHT) launch_rows<EIGHT>(p, run_magic, s);
    else return CB_ERR_UNSUPPORTED;
    return cb_last_error();
}
