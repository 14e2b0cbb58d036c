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
// A block owns 16 features and 8 rows; its warps take segments of K in turn and their sums are added
// in the warps' order, so the order of a dot product's sum depends on K alone.
#include "quantized.cuh"

namespace {

constexpr int WARPS = 8;
constexpr int FEATURES = 16;            // a block
constexpr int ROWS = 8;
constexpr int BATCH = 2;                // segments of weights a warp has in flight

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

template <int KIND>
__global__ void __launch_bounds__(WARPS * 32) linear_few_kernel(const QuantizedArgs p) {
    constexpr int SEG = KIND == EIGHT ? 64 : 128;       // k of a segment: 64 bytes of a feature's weights
    constexpr int MINE = SEG / 4;                       // k of a thread: 16 bytes
    __shared__ float sums[WARPS][FEATURES][ROWS + 1];
    cb_pdl_wait();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const int n0 = blockIdx.x * FEATURES, m0 = blockIdx.y * ROWS;
    const int K = p.K;
    // the thread's two features (beyond the last: the last, whose sums nobody stores) and its row
    const int f0 = min(n0 + g, p.N - 1), f1 = min(n0 + g + 8, p.N - 1);
    const bool has_row = m0 + g < p.M;
    const long long row = has_row ? m0 + g : 0;
    const int wb = KIND == EIGHT ? 1 : 2;               // weights a byte
    const uint8_t* w0 = static_cast<const uint8_t*>(p.w) + (long long)f0 * p.ldw;
    const uint8_t* w1 = static_cast<const uint8_t*>(p.w) + (long long)f1 * p.ldw;
    const int groups = KIND == EIGHT ? 0 : K / p.group;
    const uint8_t* s0 = p.group_scale + (long long)f0 * groups;
    const uint8_t* s1 = p.group_scale + (long long)f1 * groups;
    float acc[4] = {0.f, 0.f, 0.f, 0.f}, rest[4] = {0.f, 0.f, 0.f, 0.f};
    const int segments = (K + SEG - 1) / SEG;

    // 16 e4m3 numbers from `at`; zeros beyond K, where a row may end inside them
    auto load16 = [&](const uint8_t* at, int left) -> uint4 {
        if (left >= 16) return __ldg(reinterpret_cast<const uint4*>(at));
        uint32_t word[4] = {0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < left) word[i >> 2] |= (uint32_t)at[i] << (8 * (i & 3));
        return make_uint4(word[0], word[1], word[2], word[3]);
    };

    for (int seg0 = warp; seg0 < segments; seg0 += WARPS * BATCH) {
        uint4 wv[BATCH][2];
        uint8_t sc[BATCH][2];
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int k0 = (seg0 + b * WARPS) * SEG + t * MINE;
            wv[b][0] = wv[b][1] = make_uint4(0, 0, 0, 0);
            sc[b][0] = sc[b][1] = 0;
            if (k0 < K) {
                if (KIND == EIGHT) {
                    wv[b][0] = load16(w0 + k0, K - k0);
                    wv[b][1] = load16(w1 + k0, K - k0);
                } else {
                    wv[b][0] = __ldg(reinterpret_cast<const uint4*>(w0 + k0 / wb));
                    wv[b][1] = __ldg(reinterpret_cast<const uint4*>(w1 + k0 / wb));
                    sc[b][0] = __ldg(s0 + k0 / p.group);
                    sc[b][1] = __ldg(s1 + k0 / p.group);
                }
            }
        }
#pragma unroll
        for (int b = 0; b < BATCH; ++b) {
            const int k0 = (seg0 + b * WARPS) * SEG + t * MINE;
            const bool here = has_row && k0 < K;
            const uint32_t x[2][4] = {{wv[b][0].x, wv[b][0].y, wv[b][0].z, wv[b][0].w},
                                      {wv[b][1].x, wv[b][1].y, wv[b][1].z, wv[b][1].w}};
            if constexpr (KIND == EIGHT) {
                uint4 r = make_uint4(0, 0, 0, 0);
                if (here) r = load16(static_cast<const uint8_t*>(p.rows) + row * p.ldr + k0, K - k0);
                const uint32_t lo[4] = {x[0][0], x[1][0], x[0][1], x[1][1]}, hi[4] = {x[0][2], x[1][2], x[0][3], x[1][3]};
                mma_e4m3(acc, lo, r.x, r.y);
                mma_e4m3(acc, hi, r.z, r.w);
            } else {
                uint32_t s2[2], c2[2];
                scale_pairs(sc[b][0], s2[0], c2[0]);
                scale_pairs(sc[b][1], s2[1], c2[1]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {           // eight k at a time
                    uint32_t a[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        a[h][0] = weight_pair(x[0][j], 2 * h, s2[0], c2[0]);
                        a[h][1] = weight_pair(x[1][j], 2 * h, s2[1], c2[1]);
                        a[h][2] = weight_pair(x[0][j], 2 * h + 1, s2[0], c2[0]);
                        a[h][3] = weight_pair(x[1][j], 2 * h + 1, s2[1], c2[1]);
                    }
                    if constexpr (KIND == FOUR_BF16) {
                        uint4 r = make_uint4(0, 0, 0, 0);
                        if (here)
                            r = __ldg(reinterpret_cast<const uint4*>(
                                static_cast<const __nv_bfloat16*>(p.rows) + row * p.ldr + k0 + 8 * j));
                        mma_bf16(acc, a[0], r.x, r.y);
                        mma_bf16(acc, a[1], r.z, r.w);
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
                            if (here)
                                r = __ldg(reinterpret_cast<const float4*>(
                                    static_cast<const float*>(p.rows) + row * p.ldr + k0 + 8 * j + 4 * h));
                            uint32_t b0[3], b1[3];
                            three_parts(r.x, r.y, b0);
                            three_parts(r.z, r.w, b1);
#pragma unroll
                            for (int i = 0; i < 3; ++i) mma_bf16(i == 0 ? acc : rest, a[h], b0[i], b1[i]);
                        }
                    }
                }
            }
        }
    }
    if constexpr (KIND == FOUR_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] += rest[i];
    }
    sums[warp][g][2 * t] = acc[0], sums[warp][g][2 * t + 1] = acc[1];
    sums[warp][g + 8][2 * t] = acc[2], sums[warp][g + 8][2 * t + 1] = acc[3];
    __syncthreads();
    const int f = threadIdx.x & 15, m = threadIdx.x >> 4;
    if (m >= ROWS || n0 + f >= p.N || m0 + m >= p.M) return;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) v += sums[w][f][m];
    finish(p, v, KIND == EIGHT ? __ldg(p.row_scale + m0 + m) : 1.f, __ldg(p.feature_scale + n0 + f), m0 + m, n0 + f);
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
    if (K <= 0 || (((uintptr_t)rows | (uintptr_t)w | (uintptr_t)(ldr * size) | (uintptr_t)ldw) & 15) ||
        (M + ROWS - 1) / ROWS > 65535 || (kind != EIGHT && (group <= 0 || group % 32 || K % group)))
        return CB_ERR_UNSUPPORTED;
    const QuantizedArgs p = {rows, ldr, row_scale, w, ldw, (const uint8_t*)group_scale, feature_scale, add, lda, out, ldo,
                    M, N, K, group, out_dtype == CB_BF16};
    const dim3 grid((N + FEATURES - 1) / FEATURES, (M + ROWS - 1) / ROWS), block(WARPS * 32);
    cudaStream_t s = (cudaStream_t)stream;
    if (kind == FOUR_BF16) cb_launch(linear_few_kernel<FOUR_BF16>, grid, block, 0, s, p);
    else if (kind == FOUR_F32) cb_launch(linear_few_kernel<FOUR_F32>, grid, block, 0, s, p);
    else if (kind == EIGHT) cb_launch(linear_few_kernel<EIGHT>, grid, block, 0, s, p);
    else return CB_ERR_UNSUPPORTED;
    return cb_last_error();
}
