// out[M,N] = rows[M,K] . W[N,K]^T for few rows (decoded tokens) and 4-bit weights whose K is a multiple of 256.  Rows are
// bf16; up to five fp32 ones are made three bf16 ones each by a kernel before this one, whose sums meet at the way out.
//
// The arithmetic of linear_quantized_few: codes become bf16 weights, exactly (see quantized.cuh), in the registers
// that hold mma.sync's operands.  Here codes and rows come through a ring of stages in shared memory that one
// thread keeps full by TMA: loads into registers and the instructions that take codes apart (2 to 3 a
// weight, of which a unit at half rate runs one) took turns in a warp, one's 12 us behind the other's 17 (a row
// of 4,096 by 28,672).
//
// A block's warps form groups: each owns 32 features, and the warps of a group take segments of 128 k in
// turn, one of every stage.  Few features: the blocks (x, y, 0..S-1) form a cluster that splits K.  The warps' and the
// blocks' sums are added in their order, so the order of a dot product's sum depends on the sizes alone.  A thread takes
// 16 neighbouring bytes of a feature's codes, 32 k, and the same k of its row.
//
// LONG: fp32 results where a warp's share of K is above MMA_CHUNK: so many k a sum, and the sums are added with rounding.
//
// What it takes is instructions (8 rows of 4,096 by 128,256, 69 us: issue slots 58%, the unit of shifts and masks 53%,
// memory 45%): more warps an SM, fewer waits, group scales through shared memory and blocks that stay and share the
// features evenly changed nothing.
#define CB_PDL_BIT 6      // this file's bit in CRUCIBLE_PDL
#include "quantized.cuh"
#include "tc_common.cuh"

namespace {

constexpr int SEG = 128;                // k: 64 bytes of a feature's codes, 256 of a row
constexpr int PAIRS = 2;                // 16 features each: a group's

template <int NT, int GROUPS, int SHARE> struct Sizes {
    static constexpr int WARPS = GROUPS * SHARE, FEATURES = GROUPS * 16 * PAIRS, ROWS = 8 * NT;
    static constexpr int CODES_BYTES = FEATURES * 64 * SHARE, ROWS_BYTES = ROWS * 256 * SHARE;
    static constexpr int BLOCKS = 16 / WARPS;
    static constexpr int FIT = 216 * 1024 / BLOCKS / (CODES_BYTES + ROWS_BYTES);
    static constexpr int STAGES = FIT > 6 ? 6 : FIT;
    static_assert(STAGES >= 2, "a ring");
};

template <int NT, int GROUPS, int SHARE> struct Storage {
    using S = Sizes<NT, GROUPS, SHARE>;
    alignas(1024) uint8_t codes[S::STAGES][S::CODES_BYTES];           // [256 k][feature][128 bytes], 128-byte swizzle
    alignas(1024) uint8_t rows[S::STAGES][S::ROWS_BYTES];             // [64 k][row][128 bytes], the same
    alignas(8) uint64_t full[S::STAGES], empty[S::STAGES];
    int abort_flag;
};

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int c) { return c == 0 ? v.x : (c == 1 ? v.y : (c == 2 ? v.z : v.w)); }

template <int NT, int GROUPS, int SHARE, bool LONG>
__global__ void __launch_bounds__(GROUPS * SHARE * 32 + 32, Sizes<NT, GROUPS, SHARE>::BLOCKS)
linear_ring_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_w,
                   const QuantizedArgs p, uint32_t run_magic, int parts, int splits, int* __restrict__ status) {
    using S = Sizes<NT, GROUPS, SHARE>;
    extern __shared__ uint8_t smem_raw[];
    Storage<NT, GROUPS, SHARE>& s = *reinterpret_cast<Storage<NT, GROUPS, SHARE>*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * S::FEATURES, m0 = blockIdx.y * S::ROWS;
    const int segments = (p.K + SEG - 1) / SEG, stages = (segments + SHARE - 1) / SHARE;
    // this block's share of K; the launcher keeps it from being empty
    const int per = (stages + splits - 1) / splits, begin = (int)blockIdx.z * per, end = min(stages, begin + per);
    volatile int* abort_flag = &s.abort_flag;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            tc::mbar_init(&s.full[i], 1);
            tc::mbar_init(&s.empty[i], S::WARPS);
        }
        s.abort_flag = 0;
        tc::fence_barrier_init();
    }
    __syncthreads();
    cb_pdl_wait();                      // (the barriers are ready; what earlier kernels wrote is read from here on)
    cb_pdl_trigger();
    float acc[PAIRS][NT][4];
    const int group = warp / SHARE, turn = warp % SHARE;
    const int g = lane >> 2, t = lane & 3;
    // Which of 8 features a lane's rows of the operand stand for: a 16-byte load of 8 lanes then takes one row from
    // either half of the swizzle's 8, and no two of them the same banks.
    const int mine = (g >> 1) | (g & 1) << 2;
    bool ok = true;
    if (warp == S::WARPS) {
        if (tc::elect_one()) {
            int st = 0, sent = 0;
            uint32_t parity = 1;
            for (int i = 0; i < end - begin; ++i) {
                if (i >= S::STAGES && !tc::mbar_wait(&s.empty[st], parity, abort_flag)) {
                    tc::give_up(abort_flag, status, tc::ST_PRODUCER_TIMEOUT);
                    break;
                }
                tc::mbar_expect_tx(&s.full[st], S::CODES_BYTES + S::ROWS_BYTES);
                tc::tma_load_3d(s.codes[st], &map_w, &s.full[st], 0, n0, (begin + i) * (SHARE / 2));
                tc::tma_load_3d(s.rows[st], &map_rows, &s.full[st], 0, m0, (begin + i) * (SHARE * 2));
                sent = i + 1;
                if (++st == S::STAGES) st = 0, parity ^= 1;
            }
            if (*abort_flag)        // our own copies land before the block's shared memory goes away
                for (int i = max(0, sent - S::STAGES); i < sent; ++i)
                    for (uint32_t j = 0; j < tc::WAIT_LIMIT; ++j)
                        if (tc::mbar_try_wait(&s.full[i % S::STAGES], (i / S::STAGES) & 1)) break;
        }
    } else {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = 0.f;
        const uint8_t* const scales = p.group_scale + (long long)n0 * p.groups;
        uint32_t s_off[PAIRS][2];
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                s_off[i][h] = (uint32_t)(min(n0 + 32 * group + 16 * i + 8 * h + mine, p.N - 1) - n0) * (uint32_t)p.groups;
        // The scales of a segment's codes, asked for a stage ahead.  (The bytes stay apart until they are needed: put together
        // here they would be waited for here, which took 2 to 8% of the time.)
        auto ask = [&](uint32_t (&scale)[PAIRS][2], int seg) {
            if (seg >= segments) return;
            // the scale of a run of 32 k: 2 (k / 32) over the runs that share one, by half their reciprocal
            const uint32_t at = __umulhi((uint32_t)(8 * seg + 2 * t), run_magic);
#pragma unroll
            for (int i = 0; i < PAIRS; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) scale[i][h] = __ldg(scales + (s_off[i][h] + at));
        };
        // where the thread's codes and rows lie in a stage
        const int codes_at = (turn >> 1) * (S::FEATURES * 128) + (32 * group + mine) * 128 + ((((turn & 1) * 4 + t) ^ mine) << 4);
        const int rows_at = (turn * 2 + (t >> 1)) * (S::ROWS * 128) + g * 128;
        const int piece0 = (t & 1) * 4;
        uint32_t scale[PAIRS][2], next[PAIRS][2];
        ask(next, begin * SHARE + turn);
        constexpr int SUMS = PAIRS * NT * 4;
        float room[LONG ? SUMS : 1];
        float* const aside = LONG ? set_aside(room) : nullptr;
        int st = 0, left = MMA_CHUNK / SEG;
        uint32_t parity = 0;
#pragma unroll 1
        for (int i = begin; i < end; ++i) {
#pragma unroll
            for (int q = 0; q < PAIRS; ++q) scale[q][0] = next[q][0], scale[q][1] = next[q][1];
            const int seg = i * SHARE + turn;
            ask(next, seg + SHARE);
            ok = tc::mbar_wait(&s.full[st], parity, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                tc::give_up(abort_flag, status, tc::ST_MMA_TIMEOUT);
                break;
            }
            if (seg < segments) {
                const uint8_t* codes = s.codes[st] + codes_at;
                const uint8_t* rows = s.rows[st] + rows_at;
                uint4 x[PAIRS], y[PAIRS];
                ScalePair both[PAIRS][2];
#pragma unroll
                for (int q = 0; q < PAIRS; ++q) {
                    x[q] = *reinterpret_cast<const uint4*>(codes + q * 2048);
                    y[q] = *reinterpret_cast<const uint4*>(codes + q * 2048 + 1024);
                    scale_pairs(__byte_perm(scale[q][0], scale[q][1], 0x0040), both[q]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {               // eight k at a time
                    uint4 b[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) b[j] = *reinterpret_cast<const uint4*>(rows + j * 1024 + (((piece0 + c) ^ g) << 4));
#pragma unroll
                    for (int q = 0; q < PAIRS; ++q) {
                        const uint32_t xw = word_of(x[q], c), yw = word_of(y[q], c);
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t a[4] = {weight_pair(xw, 2 * e, both[q][0]), weight_pair(yw, 2 * e, both[q][1]),
                                                   weight_pair(xw, 2 * e + 1, both[q][0]), weight_pair(yw, 2 * e + 1, both[q][1])};
#pragma unroll
                            for (int j = 0; j < NT; ++j) mma_bf16(acc[q][j], a, e ? b[j].z : b[j].x, e ? b[j].w : b[j].y);
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s.empty[st]);
            if (++st == S::STAGES) st = 0, parity ^= 1;
            if (LONG && --left == 0) {
                left = MMA_CHUNK / SEG;
#pragma unroll
                for (int q = 0; q < SUMS; ++q) {
                    float& v = acc[q / (NT * 4)][q / 4 % NT][q % 4];
                    aside[q] += v, v = 0.f;
                }
            }
        }
        if (LONG) {
#pragma unroll
            for (int q = 0; q < SUMS; ++q) acc[q / (NT * 4)][q / 4 % NT][q % 4] += aside[q];
        }
    }
    __syncthreads();
    // every stage has landed and been read: the ring is free
    float* const sums = reinterpret_cast<float*>(s.codes[0]);         // [SHARE][FEATURES][ROWS + 1]
    static_assert(SHARE * S::FEATURES * (S::ROWS + 1) * 4 <= (int)(sizeof(s.codes) + sizeof(s.rows)), "the sums fit in the ring");
    const bool whole = *abort_flag == 0;
    if (warp < S::WARPS && whole) {
#pragma unroll
        for (int i = 0; i < PAIRS; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    sums[(turn * S::FEATURES + 32 * group + 16 * i + 8 * (e >> 1) + mine) * (S::ROWS + 1) + 8 * j + 2 * t + (e & 1)] = acc[i][j][e];
    }
    __syncthreads();
    auto each = [&](int first, int step, auto sum_of) {
#pragma unroll 1
        for (int at = first; at < S::FEATURES * S::ROWS; at += step) {
            const int f = at % S::FEATURES, m = at / S::FEATURES;
            if (m0 + m >= p.M) break;
            if (n0 + f >= p.N) continue;
            float v = sum_of(f, m);
            if (parts == 3) v += sum_of(f, p.M + m) + sum_of(f, 2 * p.M + m);
            finish(p, v, 1.f, __ldg(p.feature_scale + n0 + f), m0 + m, n0 + f);
        }
    };
    auto warps_sum = [&](int f, int m) {
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < SHARE; ++i) v += sums[(i * S::FEATURES + f) * (S::ROWS + 1) + m];
        return v;
    };
    constexpr int THREADS = S::WARPS * 32 + 32;
    if (splits == 1) {
        if (whole) each(threadIdx.x, THREADS, warps_sum);
        return;
    }
    // The blocks of a cluster split K: each leaves its sums in its shared memory, and each adds up a share of the numbers from all
    // of them, in their order.
    float* const mine_of_k = sums + SHARE * S::FEATURES * (S::ROWS + 1);            // [ROWS][FEATURES]
    static_assert((SHARE * (S::ROWS + 1) + S::ROWS) * S::FEATURES * 4 <= (int)(sizeof(s.codes) + sizeof(s.rows)), "the sums fit in the ring");
    for (int at = threadIdx.x; at < S::FEATURES * S::ROWS; at += THREADS) mine_of_k[at] = warps_sum(at % S::FEATURES, at / S::FEATURES);
    __syncwarp();
    tc::cluster_sync_all();
    const uint32_t theirs = tc::smem_u32(mine_of_k);
    if (whole)
        each((int)blockIdx.z * THREADS + threadIdx.x, splits * THREADS, [&](int f, int m) {
            float v = 0.f;
#pragma unroll 4
            for (int q = 0; q < splits; ++q) {
                float x;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(tc::cluster_map(theirs + 4 * (m * S::FEATURES + f), (uint32_t)q)) : "memory");
                v += x;
            }
            return v;
        });
    __syncwarp();
    tc::cluster_sync_all();             // nobody goes while his shared memory is read
}

// A matrix of rows of `row_bytes` bytes (a multiple of 128) as [128 bytes of a row][row][128 bytes], read in boxes of `depth`
// of `box_rows` rows with the 128-byte swizzle; beyond it zeros.
bool ring_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t row_bytes, uint64_t pitch, uint32_t box_rows, uint32_t depth) {
    tc::EncodeTiledFn fn = tc::encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {128, rows, row_bytes / 128};
    cuuint64_t strides[2] = {pitch, 128};
    cuuint32_t box[3] = {128, box_rows, depth};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT, int GROUPS, int SHARE, bool LONG>
int launch_as(const QuantizedArgs& p, uint32_t run_magic, int parts, int splits, int* status, cudaStream_t stream) {
    using S = Sizes<NT, GROUPS, SHARE>;
    constexpr int SMEM = (int)sizeof(Storage<NT, GROUPS, SHARE>) + 1024;
    CUtensorMap mr, mw;
    if (!ring_map(&mw, p.w, (uint64_t)p.N, (uint64_t)p.K / 2, (uint64_t)p.ldw, S::FEATURES, SHARE / 2) ||
        !ring_map(&mr, p.rows, (uint64_t)p.M * parts, (uint64_t)p.K * 2, (uint64_t)p.ldr * 2, S::ROWS, SHARE * 2))
        return CB_ERR_UNSUPPORTED;
    static bool configured[64] = {};
    auto kernel = linear_ring_kernel<NT, GROUPS, SHARE, LONG>;
    const int rc = allow_shared(kernel, SMEM, configured);
    if (rc != 0) return rc;
    cb_launch_cluster(kernel, dim3((p.N + S::FEATURES - 1) / S::FEATURES, (p.M + S::ROWS - 1) / S::ROWS, splits),
                      dim3(S::WARPS * 32 + 32), SMEM, stream, splits, mr, mw, p, run_magic, parts, splits, status);
    return cb_last_error();
}

template <int NT, int GROUPS, int SHARE>
int launch(const QuantizedArgs& p, uint32_t run_magic, int parts, int splits, int* status, cudaStream_t stream) {
    const int stages = (p.K + SHARE * SEG - 1) / (SHARE * SEG);
    if (splits > stages) splits = stages;
    while (splits > 1 && (splits - 1) * ((stages + splits - 1) / splits) >= stages) --splits;
    const bool one_sum = p.out_bf16 || (stages + splits - 1) / splits * SEG <= MMA_CHUNK;
    return one_sum ? launch_as<NT, GROUPS, SHARE, false>(p, run_magic, parts, splits, status, stream)
                   : launch_as<NT, GROUPS, SHARE, true>(p, run_magic, parts, splits, status, stream);
}

template <int NT>
int launch_block(const QuantizedArgs& p, int groups, int share, int splits, uint32_t run_magic, int parts, int* status, cudaStream_t stream) {
    if (groups == 1 && share == 8) return launch<NT, 1, 8>(p, run_magic, parts, splits, status, stream);
    if (groups == 1 && share == 4) return launch<NT, 1, 4>(p, run_magic, parts, splits, status, stream);
    if (groups == 2 && share == 4) return launch<NT, 2, 4>(p, run_magic, parts, splits, status, stream);
    if (groups == 2 && share == 2) return launch<NT, 2, 2>(p, run_magic, parts, splits, status, stream);
    return CB_ERR_UNSUPPORTED;
}

}  // namespace

// `groups` of `share` warps a block, of 32 features a group: 1 x 8, 2 x 4, 1 x 4 or 2 x 2; `splits`:
// shares of K, 1 to 8 (as many as leave none empty).  K a multiple of 256;
// rows bf16, or up to five of fp32 and `parts`, bf16 [3, M, K], where they are split to.
CB_EXPORT int cb_linear_quantized_ring(int kind, const void* rows, long long ldr, const float* row_scale, const void* w,
                                       long long ldw, const void* group_scale, const float* feature_scale,
                                       const float* add, long long lda, void* out, int out_dtype, long long ldo, int M,
                                       int N, int K, int group, int groups, int share, int splits, void* parts,
                                       int* status, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    const int size = kind == FOUR_F32 ? 4 : 2;
    if ((kind != FOUR_BF16 && kind != FOUR_F32) || K <= 0 || K % 256 || K > MOST_K ||
        (((uintptr_t)rows | (uintptr_t)w | (uintptr_t)(ldr * size) | (uintptr_t)ldw) & 15) || (M + 7) / 8 > 65535 ||
        (kind == FOUR_F32 && (M > 5 || parts == nullptr || ((uintptr_t)parts & 15))) || group <= 0 || group % 32 || K % group || splits < 1 || splits > 8)
        return CB_ERR_UNSUPPORTED;
    QuantizedArgs p = {rows, ldr, row_scale, w, ldw, (const uint8_t*)group_scale, feature_scale, add, lda, out, ldo,
                             M, N, K, group, out_dtype == CB_BF16, K / group};
    const uint32_t runs = (uint32_t)group / 32;
    const uint32_t run_magic = (uint32_t)(((1ull << 31) + runs - 1) / runs);
    cudaStream_t s = (cudaStream_t)stream;
    int n_parts = 1;
    if (kind == FOUR_F32) {
        split_rows((const float*)rows, ldr, (__nv_bfloat16*)parts, M, K, s);
        p.rows = parts, p.ldr = K, n_parts = 3;
    }
    return M * n_parts <= 8 ? launch_block<1>(p, groups, share, splits, run_magic, n_parts, status, s)
                            : launch_block<2>(p, groups, share, splits, run_magic, n_parts, status, s);
}
