// out[M,N] = rows[M,K] . W[N,K]^T over quantised weights on the 5th-generation tensor cores, for
// more than a few rows.  128 features of W are the M side of the MMA (lanes of tensor memory) and up
// to 256 rows its N side.
//
//   EIGHT      both operands e4m3, brought by TMA (128 k a stage), tcgen05.mma kind::f8f6f4
//   FOUR_BF16  the codes come in by TMA, 256 k of 128 features a stage; eight warps make bf16 weights
//              of them (exact, see quantized.cuh), 64 k a stage, a feature a thread, and put them into
//              tensor memory, where the MMA takes them from
//   FOUR_F32   the same with three bf16 parts of every row side by side on the MMA's N side, which a
//              kernel before this one has split: their sums lie in tensor memory apart and meet
//              in the epilogue
//
// Few tiles: the blocks (x, y, 0..S-1) form a cluster that splits K.  Each leaves its sums in its own
// shared memory, and each adds up a share of the rows from all of them, in the order of the
// shares: no scratch memory, no atomics, the same sum every time.
//
// fp32 results over 4-bit weights.  The tensor cores cut off what an addition leaves below the sum's last bit, always
// towards zero, and over a long K that adds up (K = 14,336 in one sum: 4.2e-6 of the result's norm; e4m3 products have
// 8 bits and lose nothing to speak of).  So every CHUNK of K the sums come out of tensor memory and are added, rounded, to
// those before them, which stand in the threads' registers and, of 256 rows, half of them in tensor memory beside the
// weights.
//
// Roles: warp 0 sends the copies of the rows (and of 8-bit weights), warp 1 owns tensor memory and
// issues the MMAs, warps 2-9 make weights of codes (two sets of four, 64 k in turn) and then take the sums
// out (two to a quarter of the lanes, 32 rows in turn), warp 10 sends the copies of codes.
#define CB_PDL_BIT 6      // this file's bit in CRUCIBLE_PDL
#include "quantized_tc.cuh"

namespace {

constexpr int FEATURES = 128;
constexpr int THREADS = 352;
constexpr int PACKED_K = 256;           // k of a stage of codes: 128 bytes a feature

// The weights' place is tensor memory, as the MMA's A operand: lane = feature, a column = two neighbouring k, 32 columns
// a stage of 64 k.  (In shared memory they were 16 KB written and 16 KB read a stage beside the rows' and codes' own
// bytes: 64 rows of 4,096 by 28,672 took 41 us, 31 like this.)
constexpr int WEIGHT_STAGES = 4, WEIGHT_COLS = 32;

constexpr int CHUNK = 2048;             // K of one sum where sums are long: a multiple of what a stage of codes holds

template <int KIND, int TOK> struct Sizes {
    static constexpr int PARTS = KIND == FOUR_F32 ? 3 : 1;
    static constexpr int BK = KIND == EIGHT ? 128 : 64;              // 128 bytes a row of either operand
    static constexpr int CODES_BYTES = FEATURES * 128;
    static constexpr int A_BYTES = KIND == EIGHT ? FEATURES * 128 : 0;
    static constexpr int B_BYTES = PARTS * TOK * 128;
    static constexpr int N = PARTS * TOK;
    static constexpr int USED = N + (KIND == EIGHT ? 0 : WEIGHT_STAGES * WEIGHT_COLS);
    static constexpr int TMEM = USED <= 32 ? 32 : (USED <= 64 ? 64 : (USED <= 128 ? 128 : (USED <= 256 ? 256 : 512)));
    // a block of few rows shares its SM with another; one of more has it to itself
    static constexpr int BLOCKS = N <= 96 ? 2 : 1;
    static constexpr int ROOM = BLOCKS == 2 ? 110 * 1024 : 220 * 1024;
    static constexpr int PACKED = KIND == EIGHT ? 0 : (BLOCKS == 2 ? 3 : 4);         // stages of codes
    static constexpr int FIT = (ROOM - PACKED * CODES_BYTES) / (A_BYTES + B_BYTES);
    static constexpr int STAGES = FIT > 8 ? 8 : FIT;
};

template <int KIND, int TOK> struct Storage {
    using S = Sizes<KIND, TOK>;
    alignas(1024) uint8_t b[S::STAGES][S::B_BYTES];
    alignas(1024) uint8_t a[KIND == EIGHT ? S::STAGES : 1][KIND == EIGHT ? S::A_BYTES : 16];
    alignas(1024) uint8_t codes[S::PACKED == 0 ? 1 : S::PACKED][S::PACKED == 0 ? 16 : S::CODES_BYTES];
    alignas(8) uint64_t full[S::STAGES], empty[S::STAGES];            // the copies' ring
    uint64_t made[WEIGHT_STAGES], used[WEIGHT_STAGES];               // the weights' ring in tensor memory
    uint64_t codes_full[4], codes_empty[4], done, drained;
    uint32_t tmem;
    int abort_flag;
};

__device__ __forceinline__ void umma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

template <int KIND, int TOK, bool BF16>
__global__ void __launch_bounds__(THREADS, Sizes<KIND, TOK>::BLOCKS)
linear_tcgen05_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_w,
                      const QuantizedArgs p, int tok, int splits, int* __restrict__ status) {
    using S = Sizes<KIND, TOK>;
    constexpr bool CHUNKED = KIND != EIGHT && !BF16;
    constexpr int CHUNK_STEPS = CHUNK / 64;
    extern __shared__ uint8_t smem_raw[];
    Storage<KIND, TOK>& s = *reinterpret_cast<Storage<KIND, TOK>*>(
        (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * FEATURES, m0 = blockIdx.y * tok;
    const uint32_t rank = splits > 1 ? tc::cluster_rank() : 0u;
    // this block's share of K, in units of what comes in at once; the launcher keeps it from being empty
    constexpr int UNIT = KIND == EIGHT ? S::BK : PACKED_K;
    const int units = (p.K + UNIT - 1) / UNIT, per = (units + splits - 1) / splits;
    const int k_begin = (int)rank * per * UNIT, k_end = min(p.K, k_begin + per * UNIT);
    const int n_kb = (k_end - k_begin + S::BK - 1) / S::BK;
    volatile int* abort_flag = &s.abort_flag;

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::STAGES; ++i) {
            tc::mbar_init(&s.full[i], 1);
            tc::mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < WEIGHT_STAGES; ++i) {
            tc::mbar_init(&s.made[i], 4);                            // (a set of four warps)
            tc::mbar_init(&s.used[i], 1);
        }
        for (int i = 0; i < S::PACKED; ++i) {
            tc::mbar_init(&s.codes_full[i], 1);
            tc::mbar_init(&s.codes_empty[i], 8);
        }
        tc::mbar_init(&s.done, 1);
        tc::mbar_init(&s.drained, 8);
        s.abort_flag = 0;
        tc::fence_barrier_init();
        tc::prefetch_tensormap(&map_rows);
        tc::prefetch_tensormap(&map_w);
    }
    if (warp == 1) {
        tc::tmem_alloc(&s.tmem, S::TMEM);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::tc_fence_after_sync();
    // barriers and tensor memory are ready; what earlier kernels wrote is read from here on
    cb_pdl_wait();
    cb_pdl_trigger();
    const uint32_t tmem = s.tmem, weights = tmem + S::TMEM - WEIGHT_STAGES * WEIGHT_COLS;

    if (warp == 0) {
        if (tc::elect_one()) {
            int st = 0, sent = 0;
            uint32_t parity = 1;
            const uint32_t bytes = (KIND == EIGHT ? S::A_BYTES : 0) + S::PARTS * tok * 128;
            for (int kb = 0; kb < n_kb; ++kb) {
                if (kb >= S::STAGES && !tc::mbar_wait(&s.empty[st], parity, abort_flag)) {
                    tc::give_up(abort_flag, status, tc::ST_PRODUCER_TIMEOUT);
                    break;
                }
                tc::mbar_expect_tx(&s.full[st], bytes);
                const int k = k_begin + kb * S::BK;
                if constexpr (KIND == EIGHT) tc::tma_load_2d(s.a[st], &map_w, &s.full[st], k, n0);
                if constexpr (KIND == FOUR_F32) tc::tma_load_3d(s.b[st], &map_rows, &s.full[st], k, m0, 0);
                else tc::tma_load_2d(s.b[st], &map_rows, &s.full[st], k, m0);
                sent = kb + 1;
                if (++st == S::STAGES) st = 0, parity ^= 1;
            }
            if (*abort_flag) {
                // our own copies land before the block's shared memory goes away
                for (int kb = max(0, sent - S::STAGES); kb < sent; ++kb)
                    for (uint32_t i = 0; i < tc::WAIT_LIMIT; ++i)
                        if (tc::mbar_try_wait(&s.full[kb % S::STAGES], (kb / S::STAGES) & 1)) break;
            }
        }
    } else if (warp == 1) {
        if (tc::elect_one()) {
            const uint32_t idesc = KIND == EIGHT ? instr_desc_e4m3(FEATURES, tok) : tc::instr_desc_bf16(FEATURES, S::PARTS * tok);
            constexpr uint32_t A_STEP = S::A_BYTES >> 4, B_STEP = S::B_BYTES >> 4;
            const uint64_t desc0 = tc::smem_desc_sw128(tc::smem_u32(s.b[0]));
            const uint32_t desc_hi = (uint32_t)(desc0 >> 32), b_lo = (uint32_t)desc0;
            const uint32_t a_lo = (uint32_t)tc::smem_desc_sw128(tc::smem_u32(s.a[0]));
            int st = 0, ws = 0;
            uint32_t parity = 0, made_parity = 0, more = 0;
            bool ok = true;
            uint32_t drained_parity = 0;
            for (int kb = 0; kb < n_kb; ++kb) {
                ok = true;
                if (CHUNKED && kb > 0 && kb % CHUNK_STEPS == 0) {
                    tc::umma_commit(&s.done);
                    ok = tc::mbar_wait(&s.drained, drained_parity, abort_flag);
                    drained_parity ^= 1, more = 0;
                }
                ok = ok && tc::mbar_wait(&s.full[st], parity, abort_flag);
                if (KIND != EIGHT) ok = ok && tc::mbar_wait(&s.made[ws], made_parity, abort_flag);
                if (!ok) {
                    tc::give_up(abort_flag, status, tc::ST_MMA_TIMEOUT);
                    break;
                }
                tc::tc_fence_after_sync();
#pragma unroll
                for (int k = 0; k < 4; ++k) {               // 32 bytes of K an instruction: two descriptor units
                    const uint64_t b = tc::desc_of(b_lo + st * B_STEP + 2 * k, desc_hi);
                    if constexpr (KIND == EIGHT)
                        umma_e4m3(tmem, tc::desc_of(a_lo + st * A_STEP + 2 * k, desc_hi), b, idesc, more);
                    else
                        tc::umma_bf16_ts(tmem, weights + ws * WEIGHT_COLS + 8 * k, b, idesc, more);
                    more = 1;
                }
                tc::umma_commit(&s.empty[st]);
                if (++st == S::STAGES) st = 0, parity ^= 1;
                if (KIND != EIGHT) {
                    tc::umma_commit(&s.used[ws]);
                    if (++ws == WEIGHT_STAGES) ws = 0, made_parity ^= 1;
                }
            }
            if (ok) tc::umma_commit(&s.done);
        }
    } else if (warp == 10) {
        if constexpr (KIND != EIGHT) if (tc::elect_one()) {
            int st = 0, sent = 0;
            uint32_t parity = 1;
            const int n_pk = (k_end - k_begin + PACKED_K - 1) / PACKED_K;
            for (int i = 0; i < n_pk; ++i) {
                if (i >= S::PACKED && !tc::mbar_wait(&s.codes_empty[st], parity, abort_flag)) {
                    tc::give_up(abort_flag, status, tc::ST_PRODUCER_TIMEOUT);
                    break;
                }
                tc::mbar_expect_tx(&s.codes_full[st], S::CODES_BYTES);
                tc::tma_load_2d(s.codes[st], &map_w, &s.codes_full[st], (k_begin + i * PACKED_K) / 2, n0);
                sent = i + 1;
                if (++st == S::PACKED) st = 0, parity ^= 1;
            }
            if (*abort_flag)
                for (int i = max(0, sent - S::PACKED); i < sent; ++i)
                    for (uint32_t j = 0; j < tc::WAIT_LIMIT; ++j)
                        if (tc::mbar_try_wait(&s.codes_full[i % S::PACKED], (i / S::PACKED) & 1)) break;
        }
    } else {
        const int r = (warp & 3) * 32 + lane, set = (warp - 2) >> 2;     // the feature: a lane of tensor memory
        const int n = n0 + r;
        const uint32_t mine = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        bool ok = true;
        // 32 rows' sums of this feature (a last 16 beside something that nobody uses)
        auto load_rows = [&](int c, float (&v)[32]) {
            uint32_t u[32];
            tc::tmem_ld_32x32(mine + (S::PARTS - 1) * tok + c, u);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(u[i]);
#pragma unroll
            for (int j = S::PARTS - 2; j >= 0; --j) {
                tc::tmem_ld_32x32(mine + j * tok + c, u);
                tc::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(u[i]);
            }
        };
        // the sums of the chunks before the last: 32 rows in turn by the two sets
        constexpr int OWN = CHUNKED ? (TOK + 63) / 64 : 1, HELD = OWN < 2 ? OWN : 2;
        static_assert(OWN <= HELD || S::N + (OWN - HELD) * 64 + WEIGHT_STAGES * WEIGHT_COLS <= S::TMEM, "the rest fit in tensor memory");
        float before[HELD][32];
        const uint32_t kept = mine + S::N + set * 32 * (OWN > HELD ? OWN - HELD : 0);
        auto add_before = [&](int o, float (&v)[32]) {
            if (o < HELD) {
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += before[o < HELD ? o : 0][i];
            } else {
                uint32_t u[32];
                tc::tmem_ld_32x32(kept + (o - HELD) * 32, u);
                tc::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] += __uint_as_float(u[i]);
            }
        };
        uint32_t done_parity = 0;
        bool chunks = false;
        if constexpr (KIND != EIGHT) {
            const Scales scales(p, n);
            uint2 sc, next = scales.load(k_begin, k_end);
            const uint32_t my_weights = weights + ((uint32_t)((warp & 3) * 32) << 16);
            int pk = 0;
            uint32_t pk_parity = 0, used_parity = 1;
            for (int kb = 0; kb < n_kb && ok; kb += 4, used_parity ^= 1) {
                ok = tc::mbar_wait(&s.codes_full[pk], pk_parity, abort_flag);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) {
                    tc::give_up(abort_flag, status, tc::ST_EPILOGUE_TIMEOUT);
                    break;
                }
                sc = next;
                next = scales.load(k_begin + (kb + 4) * 64, k_end);
                const uint8_t* packed = s.codes[pk] + r * 128;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (kb + j >= n_kb) break;
                    if ((j & 1) != set) continue;
                    static_assert(WEIGHT_STAGES == 4, "a stage of codes goes once around the weights' ring");
                    uint32_t v[32];
                    make_weights(packed, j, r, scales.of(sc, 2 * j), v);
                    if (kb > 0) {
                        ok = tc::mbar_wait(&s.used[j], used_parity, abort_flag);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) {
                            tc::give_up(abort_flag, status, tc::ST_EPILOGUE_TIMEOUT);
                            break;
                        }
                        tc::tc_fence_after_sync();
                    }
                    tc::tmem_st_32x32(my_weights + j * WEIGHT_COLS, v);
                    tc::tmem_st_wait();
                    tc::tc_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s.made[j]);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&s.codes_empty[pk]);
                if (++pk == S::PACKED) pk = 0, pk_parity ^= 1;
                if constexpr (CHUNKED) {
                    static_assert(CHUNK_STEPS % 4 == 0, "a chunk is whole stages of codes");
                    if (ok && (kb + 4) % CHUNK_STEPS == 0 && kb + 4 < n_kb) {
                        ok = tc::mbar_wait(&s.done, done_parity, abort_flag);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) {
                            tc::give_up(abort_flag, status, tc::ST_EPILOGUE_TIMEOUT);
                            break;
                        }
                        tc::tc_fence_after_sync();
#pragma unroll
                        for (int o = 0; o < OWN; ++o) {
                            if (32 * set + 64 * o >= tok) break;
                            float v[32];
                            load_rows(32 * set + 64 * o, v);
                            if (chunks) add_before(o, v);
                            if (o < HELD) {
#pragma unroll
                                for (int i = 0; i < 32; ++i) before[o < HELD ? o : 0][i] = v[i];
                            } else {
                                uint32_t u[32];
#pragma unroll
                                for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(v[i]);
                                tc::tmem_st_32x32(kept + (o - HELD) * 32, u);
                            }
                        }
                        if (OWN > HELD) tc::tmem_st_wait();
                        tc::tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&s.drained);
                        done_parity ^= 1, chunks = true;
                    }
                }
            }
        }
        // ---- epilogue
        if (ok) {
            ok = tc::mbar_wait(&s.done, done_parity, abort_flag);
            if (!ok && !*abort_flag) tc::give_up(abort_flag, status, tc::ST_EPILOGUE_TIMEOUT);
            ok = __all_sync(0xffffffffu, ok);
        }
        tc::tc_fence_after_sync();
        const float fs = n < p.N ? __ldg(p.feature_scale + n) : 0.f;
        const int m_end = min(p.M, m0 + tok);
        auto whole_rows = [&](int c, int o, float (&v)[32]) {
            load_rows(c, v);
            if (CHUNKED && chunks) add_before(o, v);
        };
        if (splits == 1) {
            if (ok) {
                constexpr int TURNS = CHUNKED ? OWN : 1;            // (registers are indexed by constants)
                for (int c0 = 0; c0 < tok; c0 += 64 * TURNS)
#pragma unroll
                for (int o = 0; o < TURNS; ++o) {
                    const int c = c0 + 64 * o + 32 * set;
                    if (c >= tok) break;
                    float v[32];
                    whole_rows(c, o, v);
                    store_rows<KIND, BF16>(p, v, fs, n, m0 + c, m_end, p.add, p.lda);
                }
            }
        } else {
            float* left = reinterpret_cast<float*>(s.b[0]);           // [row][feature]; the ring is free by now
            if (ok) {
                constexpr int TURNS = CHUNKED ? OWN : 1;
                for (int c0 = 0; c0 < tok; c0 += 64 * TURNS)
#pragma unroll
                for (int o = 0; o < TURNS; ++o) {
                    const int c = c0 + 64 * o + 32 * set;
                    if (c >= tok) break;
                    float v[32];
                    whole_rows(c, o, v);
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        if (c + i < tok) left[(c + i) * FEATURES + r] = v[i];
                }
            }
            tc::cluster_sync_all();
            // this block's share of the rows, 4 at a time by the two sets in turn; what they are added to is asked
            // for ahead of the others' sums
            const int share = (tok / 4 + splits - 1) / splits * 4;
            const uint32_t base = tc::smem_u32(left) + 4 * r;
            const int c_end = min(min(tok, (int)(rank + 1) * share), p.M - m0);
            if (ok && !*abort_flag) {
#pragma unroll 1
                for (int c = (int)rank * share + 4 * set; c < c_end; c += 8) {
                    float a[4], v[4] = {0.f, 0.f, 0.f, 0.f};
                    if (p.add != nullptr) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            a[i] = n < p.N && c + i < c_end ? __ldcg(p.add + (long long)(m0 + c + i) * p.lda + n) : 0.f;
                    }
#pragma unroll 4
                    for (int q = 0; q < splits; ++q) {
                        const uint32_t theirs = tc::cluster_map(base + c * FEATURES * 4, (uint32_t)q);
                        float x[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x[i]) : "r"(theirs + i * FEATURES * 4) : "memory");
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] += x[i];
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int m = m0 + c + i;
                        if (n >= p.N || c + i >= c_end) continue;
                        float y = v[i] * fs;
                        if (KIND == EIGHT) y *= __ldg(p.row_scale + m);
                        if (p.add != nullptr) y += a[i];
                        const long long at = (long long)m * p.ldo + n;
                        if (BF16) static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(y);
                        else static_cast<float*>(p.out)[at] = y;
                    }
                }
            }
        }
        tc::tc_fence_before_sync();
    }
    __syncwarp();
    if (splits > 1) {
        // the other warps' part of the barrier between leaving and reading; then nobody goes while his
        // shared memory is read
        if (warp < 2 || warp == 10) tc::cluster_sync_all();
        tc::cluster_sync_all();
    }
    __syncthreads();
    if (warp == 1) {
        tc::tc_fence_after_sync();
        tc::tmem_dealloc(tmem, S::TMEM);
    }
}

template <int KIND, int TOK, bool BF16>
int launch(const QuantizedArgs& p, const CUtensorMap& rows, const CUtensorMap& w, int tok, int splits, int* status,
           cudaStream_t stream) {
    constexpr int SMEM = (int)sizeof(Storage<KIND, TOK>) + 1024;
    static_assert(SMEM <= 232448, "a block's shared memory");
    static_assert(TOK * FEATURES * 4 <= (int)(sizeof(Storage<KIND, TOK>::a) * (KIND == EIGHT) + sizeof(Storage<KIND, TOK>::b)),
                  "the sums that a block leaves for its cluster must fit in the ring");
    static bool configured[64] = {};
    auto kernel = linear_tcgen05_kernel<KIND, TOK, BF16>;
    const int rc = allow_shared(kernel, SMEM, configured);
    if (rc != 0) return rc;
    cb_launch_cluster(kernel, dim3((p.N + FEATURES - 1) / FEATURES, (p.M + tok - 1) / tok, splits), dim3(THREADS), SMEM, stream,
                      splits, rows, w, p, tok, splits, status);
    return cb_last_error();
}

template <int KIND, bool BF16>
int launch_tok(const QuantizedArgs& p, const CUtensorMap& rows, const CUtensorMap& w, int tok, int splits, int* status,
               cudaStream_t stream) {
    if (tok <= 32) return launch<KIND, 32, BF16>(p, rows, w, tok, splits, status, stream);
    if (tok <= 64) return launch<KIND, 64, BF16>(p, rows, w, tok, splits, status, stream);
    if constexpr (KIND != FOUR_F32) {
        if (tok <= 128) return launch<KIND, 128, BF16>(p, rows, w, tok, splits, status, stream);
        if (tok <= 256) return launch<KIND, 256, BF16>(p, rows, w, tok, splits, status, stream);
    }
    return CB_ERR_UNSUPPORTED;
}

template <int KIND>
int launch_out(const QuantizedArgs& p, const CUtensorMap& rows, const CUtensorMap& w, int tok, int splits, int* status,
               cudaStream_t stream) {
    return p.out_bf16 ? launch_tok<KIND, true>(p, rows, w, tok, splits, status, stream)
                      : launch_tok<KIND, false>(p, rows, w, tok, splits, status, stream);
}

}  // namespace

// `tok`: rows a tile, a multiple of 16 up to 256 (fp32 rows: 64); `splits`: shares of K, 1 to 8 (as many as leave
// none empty); `parts`: bf16 [3, M, K], where fp32 rows are split to.
CB_EXPORT int cb_linear_quantized_tcgen05(int kind, const void* rows, long long ldr, const float* row_scale,
                                          const void* w, long long ldw, const void* group_scale,
                                          const float* feature_scale, const float* add, long long lda, void* out,
                                          int out_dtype, long long ldo, int M, int N, int K, int group, int tok,
                                          int splits, void* parts, int* status, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    const int size = kind == EIGHT ? 1 : (kind == FOUR_F32 ? 4 : 2);
    if (K <= 0 || K > MOST_K || tok < 16 || tok % 16 || tok > (kind == FOUR_F32 ? 64 : 256) || splits < 1 || splits > 8 ||
        (((uintptr_t)rows | (uintptr_t)w | (uintptr_t)(ldr * size) | (uintptr_t)ldw) & 15) ||
        (M + tok - 1) / tok > 65535 || (kind != EIGHT && (group <= 0 || group % 32 || K % group)) ||
        (kind == FOUR_F32 && (parts == nullptr || ((uintptr_t)parts & 15))))
        return CB_ERR_UNSUPPORTED;
    const int unit = kind == EIGHT ? 128 : PACKED_K, units = (K + unit - 1) / unit;
    if (splits > units) splits = units;
    while (splits > 1 && (splits - 1) * ((units + splits - 1) / splits) >= units) --splits;
    const QuantizedArgs p = {rows, ldr, row_scale, w, ldw, (const uint8_t*)group_scale, feature_scale, add, lda, out, ldo,
                             M, N, K, group, out_dtype == CB_BF16, group > 0 ? K / group : 0};
    cudaStream_t st = (cudaStream_t)stream;
    CUtensorMap mr, mw;
    bool ok = quantized_map(&mw, w, false, (uint64_t)N, kind == EIGHT ? (uint64_t)K : (uint64_t)K / 2, (uint64_t)ldw, FEATURES, 1);
    if (kind == FOUR_F32) ok = ok && quantized_map(&mr, parts, true, (uint64_t)M, (uint64_t)K, (uint64_t)K * 2, tok, 3);
    else ok = ok && quantized_map(&mr, rows, kind == FOUR_BF16, (uint64_t)M, (uint64_t)K, (uint64_t)ldr * size, tok, 1);
    if (!ok) return CB_ERR_UNSUPPORTED;
    if (kind == FOUR_F32) {
        split_rows((const float*)rows, ldr, (__nv_bfloat16*)parts, M, K, st);
        return launch_out<FOUR_F32>(p, mr, mw, tok, splits, status, st);
    }
    if (kind == FOUR_BF16) return launch_out<FOUR_BF16>(p, mr, mw, tok, splits, status, st);
    if (kind == EIGHT) return launch_out<EIGHT>(p, mr, mw, tok, splits, status, st);
    return CB_ERR_UNSUPPORTED;
}
