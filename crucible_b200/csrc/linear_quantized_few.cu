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
#include "quantized.cuh"

namespace {

constexpr int WARPS = 8;
constexpr int PAIRS = 2;                // 16 features each: a block's
constexpr int FEATURES = 16 * PAIRS;

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

// What a thread holds of a segment's weights: 16 bytes of each of its features, and their scales.
template <int KIND> struct Held {
    uint4 w[PAIRS][2];
    uint8_t scale[PAIRS][2];
};

// NT: groups of 8 rows.  BATCH: segments of weights a warp has in flight.
template <int KIND, int NT, int BATCH>
__global__ void __launch_bounds__(WARPS * 32, KIND == FOUR_F32 ? 1 : 2) linear_few_kernel(const QuantizedArgs p, uint32_t run_magic) {
    constexpr int SEG = KIND == EIGHT ? 64 : 128;       // k of a segment: 64 bytes of a feature's weights
    constexpr int MINE = SEG / 4;                       // k of a thread: 16 bytes
    constexpr int ROWS = 8 * NT;
    __shared__ float sums[WARPS][FEATURES][ROWS + 1];
    cb_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * FEATURES, m0 = blockIdx.y * ROWS;
    const int K = p.K, segments = (K + SEG - 1) / SEG;
    const int groups = KIND == EIGHT ? 0 : K / p.group;
    // the thread's features (beyond the last: the last, whose sums nobody stores) and rows
    const uint8_t *w[PAIRS][2], *scales[PAIRS][2];
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const long long f = min(n0 + 16 * i + 8 * h + g, p.N - 1);
            w[i][h] = static_cast<const uint8_t*>(p.w) + f * p.ldw;
            scales[i][h] = p.group_scale + f * groups;
        }
    constexpr int SIZE = KIND == EIGHT ? 1 : (KIND == FOUR_F32 ? 4 : 2);
    const uint8_t* rows[NT];
    bool has_row[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
        has_row[i] = m0 + 8 * i + g < p.M;
        rows[i] = static_cast<const uint8_t*>(p.rows) + (has_row[i] ? m0 + 8 * i + g : 0) * p.ldr * SIZE;
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
    auto fetch = [&](Held<KIND>& h, int seg) {
        const int k = seg * SEG + t * MINE;
        // the run of 32 k's scale: k / 32 over the runs that share one, by its reciprocal (0: one run)
        const uint32_t at = KIND == EIGHT ? 0 : (run_magic ? __umulhi((uint32_t)k >> 5, run_magic) : (uint32_t)k >> 5);
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                h.w[i][j] = make_uint4(0, 0, 0, 0);
                h.scale[i][j] = 0;
                if (k < K) {
                    if constexpr (KIND == EIGHT) {
                        h.w[i][j] = load16(w[i][j] + k, K - k);
                    } else {
                        h.w[i][j] = __ldg(reinterpret_cast<const uint4*>(w[i][j] + (k >> 1)));
                        h.scale[i][j] = __ldg(scales[i][j] + at);
                    }
                }
            }
    };
    auto multiply = [&](const Held<KIND>& h, int seg) {
        const int k = seg * SEG + t * MINE;
        if constexpr (KIND == EIGHT) {
            uint4 r[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                r[j] = make_uint4(0, 0, 0, 0);
                if (has_row[j] && k < K) r[j] = load16(rows[j] + k, K - k);
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
            uint32_t s2[PAIRS][2], c2[PAIRS][2];
#pragma unroll
            for (int i = 0; i < PAIRS; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) scale_pairs(h.scale[i][j], s2[i][j], c2[i][j]);
            uint4 b16[KIND == FOUR_BF16 ? NT : 1][4];
            if constexpr (KIND == FOUR_BF16) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        b16[j][c] = make_uint4(0, 0, 0, 0);
                        if (has_row[j] && k < K) b16[j][c] = __ldg(reinterpret_cast<const uint4*>(rows[j] + 2 * k) + c);
                    }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {               // eight k at a time
                uint32_t b[NT][3][4];                   // [rows][part][pairs of k]
                if constexpr (KIND == FOUR_F32) {
#pragma unroll
                    for (int j = 0; j < NT; ++j)
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (has_row[j] && k < K) r = __ldg(reinterpret_cast<const float4*>(rows[j] + 4 * k) + 2 * c + q);
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
                        const uint32_t a[4] = {weight_pair(xw, 2 * q, s2[i][0], c2[i][0]), weight_pair(yw, 2 * q, s2[i][1], c2[i][1]),
                                               weight_pair(xw, 2 * q + 1, s2[i][0], c2[i][0]), weight_pair(yw, 2 * q + 1, s2[i][1], c2[i][1])};
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

    Held<KIND> now[BATCH], then[BATCH];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) fetch(now[b], warp + b * WARPS);
    for (int seg = warp; seg < segments; seg += WARPS * BATCH) {
#pragma unroll
        for (int b = 0; b < BATCH; ++b) fetch(then[b], seg + (BATCH + b) * WARPS);
#pragma unroll
        for (int b = 0; b < BATCH; ++b) multiply(now[b], seg + b * WARPS);
#pragma unroll
        for (int b = 0; b < BATCH; ++b) now[b] = then[b];
    }
#pragma unroll
    for (int i = 0; i < PAIRS; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = acc[i][j][e];
                if constexpr (KIND == FOUR_F32) v += rest[i][j][e];
                sums[warp][16 * i + 8 * (e >> 1) + g][8 * j + 2 * t + (e & 1)] = v;
            }
    __syncthreads();
#pragma unroll
    for (int at = threadIdx.x; at < FEATURES * ROWS; at += WARPS * 32) {
        const int f = at % FEATURES, m = at / FEATURES;
        if (n0 + f >= p.N || m0 + m >= p.M) continue;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) v += sums[i][f][m];
        finish(p, v, KIND == EIGHT ? __ldg(p.row_scale + m0 + m) : 1.f, __ldg(p.feature_scale + n0 + f), m0 + m, n0 + f);
    }
}

template <int KIND>
void launch(const QuantizedArgs& p, uint32_t run_magic, cudaStream_t s) {
    const unsigned tiles = (p.N + FEATURES - 1) / FEATURES;
    if (p.M <= 8) cb_launch(linear_few_kernel<KIND, 1, 2>, dim3(tiles), dim3(WARPS * 32), 0, s, p, run_magic);
    else cb_launch(linear_few_kernel<KIND, 2, 1>, dim3(tiles, (p.M + 15) / 16), dim3(WARPS * 32), 0, s, p, run_magic);
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
    if (K <= 0 || K > MOST_K || (((uintptr_t)rows | (uintptr_t)w | (uintptr_t)(ldr * size) | (uintptr_t)ldw) & 15) ||
        (M + 15) / 16 > 65535 || (kind != EIGHT && (group <= 0 || group % 32 || K % group)))
        return CB_ERR_UNSUPPORTED;
    const QuantizedArgs p = {rows, ldr, row_scale, w, ldw, (const uint8_t*)group_scale, feature_scale, add, lda, out, ldo,
                             M, N, K, group, out_dtype == CB_BF16};
    const uint32_t sub = (uint32_t)group / 32;          // ceil(2^32 / sub): exact while K / 32 * sub < 2^32
    const uint32_t run_magic = sub > 1 ? (uint32_t)(((1ull << 32) + sub - 1) / sub) : 0;
    cudaStream_t s = (cudaStream_t)stream;
    if (kind == FOUR_BF16) launch<FOUR_BF16>(p, run_magic, s);
    else if (kind == FOUR_F32) launch<FOUR_F32>(p, run_magic, s);
    else if (kind == EIGHT) launch<EIGHT>(p, run_magic, s);
    else return CB_ERR_UNSUPPORTED;
    return cb_last_error();
}
