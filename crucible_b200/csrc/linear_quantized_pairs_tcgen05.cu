// out[M,N] = rows[M,K] . W[N,K]^T over quantised weights for many rows (prompts): two SMs on one tile.
//
// A pair of blocks multiplies 256 features by up to 256 rows (tcgen05.mma cta_group::2): each block
// brings 128 of the features and half of the rows, so a block fetches as many bytes for its 128 x 256 sums as
// a lone one would for 256 x 256, and both halves of tensor memory are free to take turns.  Pairs stay on
// their SMs and walk the tiles; while the sums of one leave tensor memory, the other half takes the next.
//
//   EIGHT      both operands e4m3 by TMA, 128 k a stage, kind::f8f6f4
//   FOUR_BF16  the codes by TMA, 256 k a stage; eight warps of each block make bf16 weights of them
//              (exact, see quantized.cuh), 64 k a stage of the MMA's ring, a feature a thread.  (In tensor memory,
//              where lone blocks keep them, they leave room for 192 rows twice, not 256, and what a stage takes
//              is the making: 557 cycles a stage of 192 rows against 656 of 256.)
//
// fp32 results.  The tensor cores cut off what an addition leaves below the sum's last bit, always towards
// zero, and over a long K that adds up (K = 14,336 in one sum: 4.2e-6 of the result's norm).  So a
// tile's K is taken CHUNK at a time, and each chunk's sums are added to what the one before it left in `out`: the
// pair does this under the MMAs of the next chunk.
//
// Roles in each block: warp 0 sends the copies of the rows (and of 8-bit weights), warp 1 owns tensor
// memory (the first block's issues the MMAs), warps 2-9 take the sums out (two to a quarter of the lanes, 32
// rows in turn), warp 10 sends the copies of codes, warps 11-18 make weights of them (two sets of four, 64
// k in turn: between a warp's reading codes and its weights being there lie as long as two stages' MMAs).
#define CB_PDL_BIT 6      // this file's bit in CRUCIBLE_PDL
#include "quantized_tc.cuh"

namespace {

constexpr int MINE = 128;               // features of a block
constexpr int PACKED_K = 256;
constexpr int PACKED = 2;                // (more stages of codes change nothing)
constexpr int TILE_BYTES = MINE * 128;
constexpr int CHUNK = 2048;             // K of one sum, fp32 results

template <int KIND> struct Sizes {
    static constexpr int BK = KIND == EIGHT ? 128 : 64;
    static constexpr int STAGES = KIND == EIGHT ? 6 : 5;
    static constexpr int THREADS = KIND == EIGHT ? 320 : 608;
};

template <int KIND> struct Storage {
    alignas(1024) uint8_t a[Sizes<KIND>::STAGES][TILE_BYTES];
    alignas(1024) uint8_t b[Sizes<KIND>::STAGES][TILE_BYTES];
    alignas(1024) uint8_t codes[KIND == EIGHT ? 1 : PACKED][KIND == EIGHT ? 16 : TILE_BYTES];
    alignas(8) uint64_t full[Sizes<KIND>::STAGES], empty[Sizes<KIND>::STAGES], codes_full[PACKED], codes_empty[PACKED];
    uint64_t done[2], taken[2];         // a half of tensor memory: its sums are whole; they are out of it
    uint32_t tmem;
    int abort_flag;
};

// Both blocks' copies arrive at the first block's barrier (`bar`: its address in the cluster).
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%3, %4}], [%2];"
                 ::"r"(tc::smem_u32(dst)), "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y) : "memory");
}

// An arrival at a barrier of either block.  What it announces lies in this block's shared or tensor memory, where
// the MMAs of the pair read and write it through the async proxy, and a proxy or tcgen05 fence stands ahead of
// the arrival.  So its release has the block as its scope: one of the cluster's waits for every write
// the thread ever made, 1,050 cycles here (a stage's MMAs take 512).
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// One arrival at this barrier of both blocks when the MMAs issued so far have finished.
__device__ __forceinline__ void pair_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(tc::smem_u32(bar)), "h"((uint16_t)3) : "memory");
}

template <int KIND>
__device__ __forceinline__ void pair_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (KIND == EIGHT)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}

// The tiles of a pair in the order in which every role walks them: the rows' tiles of one run of
// features side by side, so that weights are fetched from memory once.
struct Units {
    int tile, tiles, m_tiles, pairs, chunk, chunks, chunk_k, K;
    __device__ Units(const QuantizedArgs& p, int tok, int pair, int pairs_, int chunk_k_)
        : tile(pair), m_tiles((p.M + tok - 1) / tok), pairs(pairs_), chunk(0), chunk_k(chunk_k_), K(p.K) {
        tiles = m_tiles * ((p.N + 2 * MINE - 1) / (2 * MINE));
        chunks = (p.K + chunk_k - 1) / chunk_k;
    }
    __device__ bool more() const { return tile < tiles; }
    __device__ void advance() {
        if (++chunk == chunks) chunk = 0, tile += pairs;
    }
    __device__ int m_tile() const { return tile % m_tiles; }
    __device__ int n_tile() const { return tile / m_tiles; }
    __device__ int k_begin() const { return chunk * chunk_k; }
    __device__ int k_end() const { return min(K, (chunk + 1) * chunk_k); }
};

template <int KIND, bool BF16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Sizes<KIND>::THREADS)
linear_pairs_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_w,
                    const QuantizedArgs p, int tok, int chunk_k, int* __restrict__ status) {
    constexpr int BK = Sizes<KIND>::BK, STAGES = Sizes<KIND>::STAGES;
    extern __shared__ uint8_t smem_raw[];
    Storage<KIND>& s = *reinterpret_cast<Storage<KIND>*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = tc::cluster_rank();
    volatile int* abort_flag = &s.abort_flag;

    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) {
            tc::mbar_init(&s.full[i], KIND == EIGHT ? 1 : 9);        // (the copies, and four warps of each block)
            tc::mbar_init(&s.empty[i], 1);
        }
        for (int i = 0; i < PACKED; ++i) {
            tc::mbar_init(&s.codes_full[i], 1);
            tc::mbar_init(&s.codes_empty[i], 8);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&s.done[i], 1);
            tc::mbar_init(&s.taken[i], 16);                          // (eight warps of each block)
        }
        s.abort_flag = 0;
        tc::fence_barrier_init();
        tc::prefetch_tensormap(&map_rows);
        tc::prefetch_tensormap(&map_w);
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tc::smem_u32(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc::tc_fence_before_sync();
    __syncthreads();
    tc::cluster_sync_all();             // the other block's barriers are ready too
    tc::tc_fence_after_sync();
    // barriers and tensor memory are ready; what earlier kernels wrote is read from here on
    cb_pdl_wait();
    cb_pdl_trigger();
    const uint32_t tmem = s.tmem;
    Units u(p, tok, blockIdx.x >> 1, gridDim.x >> 1, chunk_k);

    if (warp == 0) {
        if (tc::elect_one()) {
            int st = 0;
            long long sent = 0;
            uint32_t parity = 1;
            bool ok = true;
            const uint32_t bytes = (KIND == EIGHT ? 2 * TILE_BYTES : 0) + tok * 128;
            for (; u.more() && ok; u.advance()) {
                const int m0 = u.m_tile() * tok + (int)rank * (tok / 2), n0 = (u.n_tile() * 2 + (int)rank) * MINE;
                for (int k = u.k_begin(), k_end = u.k_end(); k < k_end; k += BK) {
                    if (sent >= STAGES && !tc::mbar_wait(&s.empty[st], parity, abort_flag)) {
                        tc::give_up(abort_flag, status, tc::ST_PRODUCER_TIMEOUT);
                        ok = false;
                        break;
                    }
                    if (rank == 0) tc::mbar_expect_tx(&s.full[st], bytes);
                    const uint32_t bar = tc::cluster_map(tc::smem_u32(&s.full[st]), 0);
                    if constexpr (KIND == EIGHT) pair_load(s.a[st], &map_w, bar, k, n0);
                    pair_load(s.b[st], &map_rows, bar, k, m0);
                    ++sent;
                    if (++st == STAGES) st = 0, parity ^= 1;
                }
            }
            if (*abort_flag && rank == 0) {
                // both blocks' copies land before their shared memory goes away (the barrier of the
                // cluster is behind this).  A stage's barrier may lack arrivals of warps that gave
                // up, so the bound is what ends this wait.
                for (long long i = sent > STAGES ? sent - STAGES : 0; i < sent; ++i)
                    for (uint32_t j = 0; j < tc::WAIT_LIMIT; ++j)
                        if (tc::mbar_try_wait(&s.full[i % STAGES], (uint32_t)(i / STAGES) & 1)) break;
            }
        }
    } else if (warp == 1) {
        if (rank == 0 && tc::elect_one()) {
            const uint32_t idesc = KIND == EIGHT ? instr_desc_e4m3(2 * MINE, tok) : tc::instr_desc_bf16(2 * MINE, tok);
            constexpr uint32_t STEP = TILE_BYTES >> 4;
            const uint64_t desc0 = tc::smem_desc_sw128(tc::smem_u32(s.a[0]));
            const uint32_t desc_hi = (uint32_t)(desc0 >> 32), a_lo = (uint32_t)desc0;
            const uint32_t b_lo = (uint32_t)tc::smem_desc_sw128(tc::smem_u32(s.b[0]));
            int st = 0, at = 0;
            uint32_t parity = 0;
            bool ok = true;
            for (; u.more() && ok; u.advance(), ++at) {
                const int half = at & 1;
                if (at >= 2 && !tc::mbar_wait(&s.taken[half], ((at >> 1) & 1) ^ 1, abort_flag)) {
                    tc::give_up(abort_flag, status, tc::ST_MMA_TIMEOUT);
                    break;
                }
                tc::tc_fence_after_sync();
                const uint32_t d = tmem + half * 256;
                uint32_t more = 0;
                for (int k = u.k_begin(), k_end = u.k_end(); k < k_end; k += BK) {
                    if (!tc::mbar_wait(&s.full[st], parity, abort_flag)) {
                        tc::give_up(abort_flag, status, tc::ST_MMA_TIMEOUT);
                        ok = false;
                        break;
                    }
                    tc::tc_fence_after_sync();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        pair_mma<KIND>(d, tc::desc_of(a_lo + st * STEP + 2 * i, desc_hi),
                                       tc::desc_of(b_lo + st * STEP + 2 * i, desc_hi), idesc, more);
                        more = 1;
                    }
                    pair_commit(&s.empty[st]);
                    if (++st == STAGES) st = 0, parity ^= 1;
                }
                if (ok) pair_commit(&s.done[half]);
            }
        }
    } else if (warp < 10) {
        const int r = (warp & 3) * 32 + lane;
        int at = 0;
        for (; u.more(); u.advance(), ++at) {
            const int half = at & 1;
            bool ok = tc::mbar_wait(&s.done[half], (at >> 1) & 1, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) {
                tc::give_up(abort_flag, status, tc::ST_EPILOGUE_TIMEOUT);
                break;
            }
            tc::tc_fence_after_sync();
            const int n = (u.n_tile() * 2 + (int)rank) * MINE + r, m0 = u.m_tile() * tok;
            const int m_end = min(p.M, m0 + tok);
            const float fs = n < p.N ? __ldg(p.feature_scale + n) : 0.f;
            const bool first = u.chunk == 0;
            const float* add = first ? p.add : static_cast<const float*>(p.out);
            const long long lda = first ? p.lda : p.ldo;
            const uint32_t mine = tmem + half * 256 + ((uint32_t)((warp & 3) * 32) << 16);
#pragma unroll 1
            for (int c = 32 * ((warp - 2) >> 2); c < m_end - m0; c += 64) {
                uint32_t x[32];
                float v[32];
                tc::tmem_ld_32x32(mine + c, x);
                tc::tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(x[i]);
                store_rows<KIND, BF16>(p, v, fs, n, m0 + c, m_end, add, lda);
            }
            tc::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) arrive_at(tc::cluster_map(tc::smem_u32(&s.taken[half]), 0));
        }
    } else if (warp == 10) {
        if constexpr (KIND != EIGHT) if (tc::elect_one()) {
            int st = 0;
            long long sent = 0;
            uint32_t parity = 1;
            bool ok = true;
            for (; u.more() && ok; u.advance()) {
                const int n0 = (u.n_tile() * 2 + (int)rank) * MINE;
                for (int k = u.k_begin(), k_end = u.k_end(); k < k_end; k += PACKED_K) {
                    if (sent >= PACKED && !tc::mbar_wait(&s.codes_empty[st], parity, abort_flag)) {
                        tc::give_up(abort_flag, status, tc::ST_PRODUCER_TIMEOUT);
                        ok = false;
                        break;
                    }
                    tc::mbar_expect_tx(&s.codes_full[st], TILE_BYTES);
                    tc::tma_load_2d(s.codes[st], &map_w, &s.codes_full[st], k / 2, n0);
                    ++sent;
                    if (++st == PACKED) st = 0, parity ^= 1;
                }
            }
            if (*abort_flag)
                for (long long i = sent > PACKED ? sent - PACKED : 0; i < sent; ++i)
                    for (uint32_t j = 0; j < tc::WAIT_LIMIT; ++j)
                        if (tc::mbar_try_wait(&s.codes_full[i % PACKED], (uint32_t)(i / PACKED) & 1)) break;
        }
    } else {
        if constexpr (KIND != EIGHT) {
            const int r = (warp & 3) * 32 + lane, set = (warp - 11) >> 2;
            // (the ring's slots and the stages of codes go on from one unit to the next, and so do the turns)
            int slot = 0, pk = 0;
            long long made = 0;
            uint32_t slot_parity = 1, pk_parity = 0;
            bool ok = true;
            for (; u.more() && ok; u.advance()) {
                const int n = (u.n_tile() * 2 + (int)rank) * MINE + r, k_end = u.k_end();
                const Scales scales(p, n);
                uint2 sc, next = scales.load(u.k_begin(), k_end);
                for (int k = u.k_begin(); k < k_end && ok; k += PACKED_K) {
                    sc = next;
                    next = scales.load(k + PACKED_K, k_end);
                    ok = tc::mbar_wait(&s.codes_full[pk], pk_parity, abort_flag);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (k + 64 * j >= k_end) break;
                        if ((made & 1) == set) {
                            uint32_t v[32];
                            make_weights(s.codes[pk] + r * 128, j, r, scales.of(sc, 2 * j), v);
                            if (made >= STAGES) {
                                ok = tc::mbar_wait(&s.empty[slot], slot_parity, abort_flag);
                                ok = __all_sync(0xffffffffu, ok);
                                if (!ok) break;
                            }
                            uint8_t* to = s.a[slot] + r * 128;
#pragma unroll
                            for (int c = 0; c < 8; ++c)
                                *reinterpret_cast<uint4*>(to + ((c ^ (r & 7)) << 4)) =
                                    make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                            tc::fence_proxy_async();
                            __syncwarp();
                            if (lane == 0) arrive_at(tc::cluster_map(tc::smem_u32(&s.full[slot]), 0));
                        }
                        ++made;
                        if (++slot == STAGES) slot = 0, slot_parity ^= 1;
                    }
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s.codes_empty[pk]);
                    if (++pk == PACKED) pk = 0, pk_parity ^= 1;
                }
            }
            if (!ok) tc::give_up(abort_flag, status, tc::ST_EPILOGUE_TIMEOUT);
        }
    }
    tc::tc_fence_before_sync();
    __syncwarp();
    tc::cluster_sync_all();             // neither block's memory goes while the other's copies, MMAs or arrivals reach it
    if (warp == 1) {
        tc::tc_fence_after_sync();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int KIND, bool BF16>
int launch(const QuantizedArgs& p, const CUtensorMap& rows, const CUtensorMap& w, int tok, int pairs, int* status,
           cudaStream_t stream) {
    constexpr int SMEM = (int)sizeof(Storage<KIND>) + 1024;
    static_assert(SMEM <= 232448, "a block's shared memory");
    static bool configured[64] = {};
    auto kernel = linear_pairs_kernel<KIND, BF16>;
    const int rc = allow_shared(kernel, SMEM, configured);
    if (rc != 0) return rc;
    const int whole = (p.K + PACKED_K - 1) / PACKED_K * PACKED_K;
    cb_launch(kernel, dim3(2 * pairs), dim3(Sizes<KIND>::THREADS), SMEM, stream, rows, w, p, tok,
              BF16 || whole < CHUNK ? whole : CHUNK, status);
    return cb_last_error();
}

}  // namespace

// `tok`: rows a tile, a multiple of 16 up to 256; `pairs`: pairs of SMs to run on.
CB_EXPORT int cb_linear_quantized_pairs(int kind, const void* rows, long long ldr, const float* row_scale, const void* w,
                                        long long ldw, const void* group_scale, const float* feature_scale,
                                        const float* add, long long lda, void* out, int out_dtype, long long ldo, int M,
                                        int N, int K, int group, int tok, int pairs, int* status, void* stream) {
    if (M <= 0 || N <= 0) return 0;
    const int size = kind == EIGHT ? 1 : 2;
    if ((kind != EIGHT && kind != FOUR_BF16) || K <= 0 || K > MOST_K || tok < 16 || tok % 16 || tok > 256 || pairs < 1 ||
        (((uintptr_t)rows | (uintptr_t)w | (uintptr_t)(ldr * size) | (uintptr_t)ldw) & 15) ||
        (kind != EIGHT && (group <= 0 || group % 32 || K % group)))
        return CB_ERR_UNSUPPORTED;
    const QuantizedArgs p = {rows, ldr, row_scale, w, ldw, (const uint8_t*)group_scale, feature_scale, add, lda, out, ldo,
                             M, N, K, group, out_dtype == CB_BF16, group > 0 ? K / group : 0};
    const int tiles = (M + tok - 1) / tok * ((N + 2 * MINE - 1) / (2 * MINE));
    if (pairs > tiles) pairs = tiles;
    CUtensorMap mr, mw;
    if (!quantized_map(&mw, w, false, (uint64_t)N, kind == EIGHT ? (uint64_t)K : (uint64_t)K / 2, (uint64_t)ldw, MINE, 1) ||
        !quantized_map(&mr, rows, kind == FOUR_BF16, (uint64_t)M, (uint64_t)K, (uint64_t)ldr * size, tok / 2, 1))
        return CB_ERR_UNSUPPORTED;
    cudaStream_t st = (cudaStream_t)stream;
    if (kind == EIGHT)
        return p.out_bf16 ? launch<EIGHT, true>(p, mr, mw, tok, pairs, status, st) : launch<EIGHT, false>(p, mr, mw, tok, pairs, status, st);
    return p.out_bf16 ? launch<FOUR_BF16, true>(p, mr, mw, tok, pairs, status, st) : launch<FOUR_BF16, false>(p, mr, mw, tok, pairs, status, st);
}
