// Attention over the paged cache in 4 bits (`cache4.cuh`): scores s_j = q . k_j over the keys that a row sees,
// softmax, o = sum_j p_j v_j, in one pass over the keys with a running maximum.
//
// The codes go to the tensor cores as they are.  With k = step c + low in every group,
//     q . k   = sum_groups step (sum_f q_f c_f) + low (sum_f q_f)
//     o_f     = sum_j (p_j step_j) c_jf + sum_j p_j low_j
// so a tile of 16 keys is two products over codes; steps and lows meet the sums in float32.  A code in the low
// four bits of a half word IS the float16 number code * 2^-24 (a subnormal, which the tensor cores multiply like any
// other), in the next four bits code * 2^-20: taking codes apart is a mask for every two of them and a shift for
// every eight, and 2^-24 and 16 are put right in the scales.  Queries and p step are float16 then: the queries
// of a row are scaled by a power of two so that the largest lies in [2^13, 2^14), which holds bfloat16 numbers
// exactly down to 2^-30 of it; p step is scaled by a power of two that follows the largest step seen, and rounded
// to 11 bits.  float32 rows take two float16 parts of either (22 bits), their sums over keys leave the
// tensor cores tile by tile (these cut off what float32 additions would round), and their codes are made
// normal numbers, code | 1024 less 1032: the tensor cores line the products of subnormals up as if they were
// normal and lose up to ten bits of the sum, which float32 rows showed (3e-5 to 7e-5 off) and bfloat16 ones do not.
//
// Keys are the rows of a tile and queries its columns: eight rows (heads of a group, tokens of a portion) a column
// tile, one or two of them a block, so that no more than that is multiplied for a single token.  S^T comes out with
// keys over lanes; `movmatrix` turns it for the second product, which takes P^T, again eight columns.
//
// A block of four warps takes a row tile's share of the keys, a warp every fourth pair of tiles of 16, each with a
// ring of its own in shared memory that cp.async fills a pair ahead: nothing is waited for but copies of the
// warp itself.  How keys are dealt to blocks:
//   shares   up to eight blocks of a cluster take equal shares of a row tile's keys and put their results together
//            in each other's shared memory;
//   stream   as many blocks as the SMs hold take equal shares of ALL tiles of the launch, wherever one row tile's
//            end and the next one's begin; what a block has of a row tile that it shares with others goes
//            through memory to a second kernel.  For contexts of unlike lengths and for long ones.
//
// 64 tokens of 32 heads of 128 on 8 behind 8,191 keys or fewer, groups of 64: 110 us for 473 MB, 4.3 TB/s (a copy's rate: 72);
// one behind 131,071 41.5 us (22), one of 12 heads of 64 behind 700 6.9 (a launch 2).  No unit is full: shifts and masks
// 56 %, tensor cores 26 %, memory 54 %, but a scheduler has three to four warps, whose every tile is a chain of copy,
// product, maximum, product: without the copies 95 us, without the products 90, without any tiles 24 (beginnings,
// looking for what is whose, putting together).  Without gain: e4m3 codes with k of 32 for the first product (half the
// cycles a product; queries in three parts, 108 -> 122), three blocks an SM with a longer ring, eight warps a block.
// float32 rows take twice the products and more than twice the time.
#pragma once
#include "cache4.cuh"

#include <type_traits>

namespace {

constexpr float A4_LOG2E = 1.4426950408889634f;
constexpr int A4_WARPS = 4;

struct Attn4Params {
    const void* q;
    long long q_stride;
    void* out;
    long long out_stride;
    const uint8_t* codes;
    const uint8_t* scales;
    int n_pages, page_tokens, kv_heads, n_rep;
    const int* row_start;      // requests of consecutive rows ...
    const int* first_pos;
    const int* table;
    int table_stride;
    int requests;
    const int* picks;          // ... or, with picks, every row by itself: [rows][kv heads][count]
    int pick_count;
    const int* row_request;
    const int* positions;
    int rows;
    int page_eights;           // runs of eight keys a page (0: a run may lie in two) ...
    uint32_t page_eights_inverse;     // ... and 2^32 over them, rounded up (0: one run a page)
    int window;                // 0: all earlier keys
    float scale_log2;
    int row_tiles;
    int units;                 // row tiles of all requests (or rows with picks): requests * row_tiles
    int stream;                // blocks that share all tiles, or 0
    float* partial;            // stream: [blocks][2][8 NT][D + 2]
};

// A row tile: rows base .. of a request (row r: token r / n_rep, head r % n_rep of the group), and the tiles of 16 keys
// that they see some of.
struct A4Unit {
    int row0, n_rows, base, first, request, tile_lo, tile_hi;
    __device__ __forceinline__ bool live() const { return base < n_rows; }
    // Its share of the launch's work: rows that see no key are written, too.
    __device__ __forceinline__ int weight() const { return live() ? max(1, tile_hi - tile_lo) : 0; }
};

template <int ROWS>
__device__ __forceinline__ A4Unit a4_unit(const Attn4Params& p, int u) {
    A4Unit v;
    const int x = u / p.row_tiles;
    v.base = (u - x * p.row_tiles) * ROWS;
    v.tile_lo = v.tile_hi = 0;
    if (p.picks != nullptr) {
        v.row0 = x;
        v.request = p.row_request[x];
        v.first = p.positions[x];
        v.n_rows = (v.request >= 0 && v.request < p.requests && v.first >= 0) ? p.n_rep : 0;
        v.tile_hi = p.pick_count * (p.page_eights >> 1);
        return v;
    }
    v.request = x;
    v.row0 = p.row_start[x];
    v.n_rows = v.row0 < 0 ? 0 : (min(p.row_start[x + 1], p.rows) - v.row0) * p.n_rep;
    v.first = p.first_pos[x];
    if (v.live()) {
        if (p.window > 0) v.tile_lo = max(0, v.first + v.base / p.n_rep - p.window + 1) >> 4;
        v.tile_hi = ((v.first + (min(v.n_rows, v.base + ROWS) - 1) / p.n_rep) >> 4) + 1;
        // (what lies beyond the table is not there)
        v.tile_hi = (int)min((long long)v.tile_hi, ((long long)p.table_stride * p.page_tokens + 15) >> 4);
    }
    return v;
}

// Stream: the tiles of all units and kv heads in a row (unit 0 head 0, head 1, .., unit 1 ..), dealt out in equal shares.
// (Counted in 32 bits; the caller has seen to it that they suffice.)
__device__ __forceinline__ uint32_t a4_quota(uint32_t tiles, uint32_t blocks) { return max(8u, (tiles + blocks - 1) / blocks); }

__device__ __forceinline__ uint32_t a4_smem(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void a4_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void a4_copy4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

__device__ __forceinline__ void a4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t a4_turned(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

__device__ __forceinline__ float a4_exp2(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 2^d, d <= 0, as two factors.  Where the scale 2^eps of p step (below) falls from that of values of nothing to that of vast ones,
// 2^d alone is none that float32 holds, but a sum of weights times both is what it was.
struct A4Fall {
    float down, rest;
    __device__ __forceinline__ explicit A4Fall(float d) : down(a4_exp2(fmaxf(d, -100.f))), rest(a4_exp2(fminf(d + 100.f, 0.f))) {}
    __device__ __forceinline__ float whole() const { return down * rest; }
    __device__ __forceinline__ float of(float sum) const { return sum * down * rest; }
};

__device__ __forceinline__ uint32_t a4_half2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ float a4_power(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Two codes a register: from the low four bits of each half (HIGH: from the next four, and 16 times as large).
// In units of 2^-24; or (F32) in units of 1 and less 8, which goes to the lows: terms of both signs, smaller sums.
template <bool F32, bool HIGH>
__device__ __forceinline__ uint32_t a4_codes(uint32_t w) {
    const uint32_t c = w & (HIGH ? 0x00f000f0u : 0x000f000fu);
    if constexpr (!F32) return c;
    const uint32_t m = c | 0x64006400u, k = HIGH ? 0x64806480u : 0x64086408u;       // 1024 + code, 1024 + 8 (or 16 times that)
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&m), *reinterpret_cast<const __half2*>(&k));
    return *reinterpret_cast<const uint32_t*>(&v);
}

// The NG pairs of a key.
template <int NG>
__device__ __forceinline__ void a4_pairs(uint32_t (&out)[NG], const uint8_t* at) {
    if constexpr (NG == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        out[0] = v.x; out[1] = v.y;
    } else if constexpr (NG % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NG / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(at)[i];
            out[4 * i] = v.x; out[4 * i + 1] = v.y; out[4 * i + 2] = v.z; out[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NG; ++i) out[i] = reinterpret_cast<const uint32_t*>(at)[i];
    }
}

template <bool F32>
__device__ __forceinline__ float a4_low(uint32_t pair) {
    return F32 ? fmaf(8.f, c4_step(pair), c4_low(pair)) : c4_low(pair);
}

// Largest over the eight lanes that hold the keys of one column.
__device__ __forceinline__ float a4_over_keys_max(float v) {
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
    v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
    return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
}
__device__ __forceinline__ float a4_over_keys_sum(float v) {
    v += __shfl_xor_sync(0xffffffffu, v, 4);
    v += __shfl_xor_sync(0xffffffffu, v, 8);
    return v + __shfl_xor_sync(0xffffffffu, v, 16);
}

// Shared memory of a block of D features, NG groups, NT column tiles, PARTS float16 parts of a query.
template <int D, int NG, int NT, int PARTS>
struct A4Layout {
    static constexpr int SIDE = 16 * D / 2;                    // codes of a tile's keys, or values
    static constexpr int SCALES = 16 * NG * 4;
    static constexpr int TILE = 2 * SIDE + 2 * SCALES;
    static constexpr int STAGE = 2 * TILE;                     // a pair of tiles
    static constexpr int STAGES = D <= 64 ? 3 : 2;
    static constexpr int PITCH = D + 4;                        // floats of a row of results (lanes of four rows meet other banks)
    static constexpr int RESULT = 8 * NT * PITCH * 4;          // a warp's result takes its ring's place
    static constexpr int RING = STAGE * STAGES > RESULT ? STAGE * STAGES : RESULT;
    static constexpr int Q = (D / 16) * PARTS * NT * 32 * 8;   // queries as the products take them
    static constexpr int ROWS = 8 * NT;
    static constexpr int AT_Q = A4_WARPS * RING;
    static constexpr int AT_SUMS = AT_Q + Q;                   // [ROWS][NG] sums of a row's scaled queries
    static constexpr int AT_FACTOR = AT_SUMS + ROWS * NG * 4;  // [ROWS] what raw scores are multiplied by
    static constexpr int AT_STATE = AT_FACTOR + ROWS * 4;      // [WARPS + 1][ROWS][2]: reference and sum
    static constexpr int TOTAL = AT_STATE + (A4_WARPS + 1) * ROWS * 8;
};

// 16-byte units of a tile's rows change places so that lanes that read rows 2t meet other banks.
template <int D>
__device__ __forceinline__ int a4_place(int r, int unit) {
    constexpr int UNITS = D / 32;
    if constexpr (D == 64) {
        const int u = (r & 3) * 2 + unit;
        return (r >> 2) * 128 + ((u ^ (2 * ((r >> 2) & 1))) << 4);
    } else if constexpr (D == 128) {
        const int u = (r & 1) * 4 + unit;
        return (r >> 1) * 128 + ((u ^ (2 * ((r >> 1) & 3))) << 4);
    } else if constexpr (D == 256) {
        return r * 128 + ((unit ^ (2 * ((r >> 1) & 3)) ^ (r & 1)) << 4);
    } else {
        return (r * UNITS + unit) << 4;
    }
}

// Blocks to an SM, by the registers that a form needs.
template <int D, int NG, int NT, bool F32>
constexpr int A4_BLOCKS = D > 128 || NT > 1 ? 2 : NG * (F32 ? 2 : 1) <= 2 ? 4 : 3;

template <int D, int NG, int NT, bool F32>
__global__ void __launch_bounds__(A4_WARPS * 32, A4_BLOCKS<D, NG, NT, F32>) attention4_kernel(const Attn4Params p) {
    cb_pdl_wait();
    cb_pdl_trigger();              // (after the wait: what puts a stream's results together reads the step's numbers before its own)
    constexpr int PARTS = F32 ? 2 : 1;
    using L = A4Layout<D, NG, NT, PARTS>;
    constexpr int GROUP = D / NG, W = D / 64, KS = D / 16, MT = D / 16;
    constexpr float CODE = F32 ? 1.f : 16777216.f;      // 1 over the unit of the codes
    using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t scan[A4_WARPS], found[3];
    // (the warp's number by way of a shuffle: known to be the same in all lanes, what follows from it lives in uniform registers)
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), g = lane >> 2, t = lane & 3;

    // ---- which rows, which keys ------------------------------------------------
    int index, kv;                      // the unit and its kv head
    uint32_t left = 0;                  // stream: tiles that the block has still to take
    int skip = 0, slot = 0;             // ... tiles of the unit that another block takes, and which partial result comes next
    if (p.stream > 0 && p.units == 1) {
        const uint32_t one = a4_unit<L::ROWS>(p, 0).weight(), tiles = one * p.kv_heads;
        const uint32_t quota = a4_quota(tiles, p.stream), begin = quota * blockIdx.x;
        if (begin >= tiles) return;
        left = min(quota, tiles - begin);
        index = 0;
        kv = begin / one;
        skip = begin - kv * one;
    } else if (p.stream > 0) {
        // all units' tiles (a unit a thread, and the next 128 if there are more), and before each unit
        uint32_t tiles = 0, mine = 0, upto = 0;
        for (int u0 = 0; u0 < p.units; u0 += A4_WARPS * 32) {
            const int u = u0 + threadIdx.x;
            mine = u < p.units ? (uint32_t)a4_unit<L::ROWS>(p, u).weight() * p.kv_heads : 0u;
            upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            if (lane == 31) scan[warp] = upto;
            __syncthreads();
            upto += tiles;
#pragma unroll
            for (int w = 0; w < A4_WARPS; ++w) {
                if (w < warp) upto += scan[w];
                tiles += scan[w];
            }
            __syncthreads();
        }
        const uint32_t quota = a4_quota(tiles, p.stream), begin = quota * blockIdx.x;
        if (begin >= tiles) return;
        left = min(quota, tiles - begin);
        // the unit in which the share begins: among the last 128 looked at, or looked for again
        uint32_t before = 0;
        for (int u0 = 0; u0 < p.units; u0 += A4_WARPS * 32) {
            const int u = u0 + threadIdx.x;
            if (p.units > A4_WARPS * 32) {
                mine = u < p.units ? (uint32_t)a4_unit<L::ROWS>(p, u).weight() * p.kv_heads : 0u;
                upto = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += v;
                }
                if (lane == 31) scan[warp] = upto;
                __syncthreads();
                upto += before;
#pragma unroll
                for (int w = 0; w < A4_WARPS; ++w) {
                    if (w < warp) upto += scan[w];
                    before += scan[w];
                }
            }
            if (begin < upto && begin >= upto - mine) {
                const uint32_t at = begin - (upto - mine), one = mine / p.kv_heads;
                found[0] = u;
                found[1] = at / one;
                found[2] = at - at / one * one;
            }
            __syncthreads();
            if (before > begin) break;
        }
        index = found[0];
        kv = found[1];
        skip = found[2];
    } else {
        index = blockIdx.x / p.kv_heads;
        kv = blockIdx.x - index * p.kv_heads;
    }

    // Where the lane's shares of a tile lie; of keys g (and g + 8), of values 2t and 2t + 1 (and 8 behind these).
    // (kept, not worked out anew for every tile: what the compiler cannot see through it does not take apart again)
    constexpr int EIGHT = 8 * D / 2;                        // eight rows further
    uint32_t k_at = a4_place<D>(g, (t * D / 8) >> 4) + ((t * D / 8) & 15), v_at[2], s_at = 2 * L::SIDE + g * (NG * 4);
    v_at[0] = L::SIDE + a4_place<D>(2 * t, (g * D / 16) >> 4) + ((g * D / 16) & 15);
    v_at[1] = L::SIDE + a4_place<D>(2 * t + 1, (g * D / 16) >> 4) + ((g * D / 16) & 15);
    asm volatile("" : "+r"(k_at), "+r"(v_at[0]), "+r"(v_at[1]), "+r"(s_at));
    const uint32_t ring = a4_smem(smem) + warp * L::RING;
    uint32_t place[D / 64];
#pragma unroll
    for (int j = 0; j < D / 64; ++j) place[j] = ring + a4_place<D>((lane + 32 * j) / (D / 32), (lane + 32 * j) % (D / 32));
    const bool whole = p.page_eights > 0, sixteens = whole && (p.page_eights & 1) == 0;     // eight, sixteen keys lie in one page
    const size_t side_rows = (size_t)p.n_pages * p.kv_heads * p.page_tokens;
    const size_t side_bytes = side_rows * (D / 2);
    const uint32_t page_rows = (uint32_t)p.kv_heads * p.page_tokens;

  for (;;) {
    const A4Unit unit = a4_unit<L::ROWS>(p, index);
    if (p.stream == 0 && !unit.live()) return;           // (all blocks of a cluster together)
    const int weight = unit.weight();
    if (weight == 0) {                                   // (stream: nothing of it is anybody's)
        kv = 0;
        ++index;
        continue;
    }
    const int row0 = unit.row0, n_rows = unit.n_rows, base = unit.base, first = unit.first;
    const int live = min(L::ROWS, n_rows - base);
    const int min_pos = first + base / p.n_rep, max_pos = first + (base + live - 1) / p.n_rep;
    const int lowest = p.window > 0 ? max_pos - p.window : -1;         // a tile that begins here or before needs a look
    const int* table = p.table + (size_t)unit.request * p.table_stride;
    const int* picks = p.picks != nullptr ? p.picks + ((size_t)row0 * p.kv_heads + kv) * p.pick_count : nullptr;
    int tile_lo = unit.tile_lo, tile_hi = unit.tile_hi, taken = weight;
    if (p.stream > 0) {
        taken = min(weight - skip, (int)left);
        tile_lo += skip;
        tile_hi = min(tile_hi, tile_lo + taken);
    } else if (gridDim.z > 1) {
        const int share = (weight + gridDim.z - 1) / gridDim.z;
        tile_lo += blockIdx.z * share;
        tile_hi = min(tile_hi, tile_lo + share);
    }

    // the queries' numbers, asked for before anything else of the unit's
    constexpr int MINE = L::ROWS / A4_WARPS;             // rows a warp prepares
    T query[MINE][D / 32];
#pragma unroll
    for (int j = 0; j < MINE; ++j) {
        const int r = warp + j * A4_WARPS;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) query[j][i] = cb_from_float<T>(0.f);
        if (r < live) {
            const int tok = (base + r) / p.n_rep, head = kv * p.n_rep + (base + r) - tok * p.n_rep;
            const T* src = reinterpret_cast<const T*>(p.q) + (size_t)(row0 + tok) * p.q_stride + (size_t)head * D;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) query[j][i] = src[lane + 32 * i];
        }
    }

    // Sums of a column are kept relative to 2^off, off = m - eps: m the reference of its scores (log2), at most 8 below the
    // largest, and 2^eps the scale of p step in float16 (`limit` is eps + 8); `bound` is the step from which eps is too much.
    float off[NT][2], limit[NT][2], bound[NT][2], sum[NT][2], lows[NT][NG][2], o[MT][NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            off[n][c] = -3.0e38f;
            limit[n][c] = 109.f;
            bound[n][c] = a4_power(-95);
            sum[n][c] = 0.f;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) lows[n][gr][c] = 0.f;
        }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[m][n][i] = 0.f;

    // Codes are 0..15, so that sums over them grow with the keys while results do not: they are differences of these sums and of
    // the lows'.  The tensor cores cut off what they add below a sum's last bit, 0.3 of it a tile on the mean; over 2,048 tiles
    // (equal weights, 131,000 keys by one block) results were off by 0.02 of themselves.  So every 64 tiles the part that the
    // features of a group have in common, taken from the first of them, goes over to the lows, which it nearly cancels: under 0.0005.
    auto settle = [&]() {
        if constexpr (!F32) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int gr = 0; gr < NG; ++gr) {
                        const float x = __shfl_sync(0xffffffffu, o[gr * GROUP / 16][n][c], t);
                        lows[n][gr][c] = fmaf(x, CODE / 8.f, lows[n][gr][c]);      // (eight lanes' are added at the end)
#pragma unroll
                        for (int m = gr * GROUP / 16; m < (gr + 1) * GROUP / 16; ++m) {
                            o[m][n][c] -= x;
                            o[m][n][2 + c] = fmaf(x, -16.f, o[m][n][2 + c]);
                        }
                    }
        }
    };

    // ---- the warp's ring ----------------------------------------------------
    const size_t head_row = (size_t)kv * p.page_tokens;
    const uint8_t* const code_src = p.codes + head_row * (D / 2);
    // (scales: lanes of both sides side by side)
    const uint8_t* const scale_src = p.scales + (head_row + (lane >= 4 * NG ? side_rows : 0)) * (NG * 4) + (lane % (4 * NG)) * 16;
    // The first of eight keys, run i of them, and (whole) its page; -1 where there is none.
    auto key_of = [&](int i, int& page) {
        page = whole ? -1 : 0;
        if (i >= 2 * tile_hi) return -1;
        if (!whole) return i * 8;
        int index = p.page_eights_inverse == 0 ? i : (int)__umulhi((uint32_t)i, p.page_eights_inverse);
        if (index * p.page_eights > i) --index;          // (rounded up, the inverse is at most one too much)
        const int slot = (i - index * p.page_eights) * 8;
        if (picks != nullptr) index = picks[index];
        if ((unsigned)index < (unsigned)p.table_stride) page = table[index];
        if ((unsigned)page >= (unsigned)p.n_pages) page = -1;
        return page < 0 ? -1 : picks != nullptr ? index * p.page_tokens + slot : i * 8;
    };
    // The pairs of tiles to fetch, one after the other; 32 of them are looked up at a time, a lane each: the rows (for head 0)
    // of the four runs of eight keys, and whether some row of the block may not see some key of them.  A run whose
    // page is none is masked whole; what is fetched for it (the pool's first rows) is of no account, as is what lies behind
    // a request's last token.
    int ahead = tile_lo + 2 * warp, looked = 0;
    uint32_t rows_of[4], edges_of;
    auto look = [&]() {
        bool edge = !whole;
        if (whole) {
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                rows_of[u] = 0;
                if (sixteens && (u & 1)) continue;       // (its first half's next rows)
                int page;
                const int key = key_of(2 * (ahead + 2 * A4_WARPS * lane) + u, page);
                if (key >= 0) rows_of[u] = (uint32_t)page * page_rows + (uint32_t)(key % p.page_tokens);
                edge = edge || key < 0 || key + (sixteens ? 15 : 7) > min_pos || key <= lowest;
            }
        }
        edges_of = __ballot_sync(0xffffffffu, edge);
    };
    uint32_t edges = 0;                    // of the pairs in flight, the next to be taken in the lowest bit
    auto fetch = [&](uint32_t stage) {     // `stage`: bytes from the ring's beginning
        if (ahead < tile_hi) {
            if (sixteens) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t row = __shfl_sync(0xffffffffu, rows_of[2 * u], looked);
                    const uint8_t* src = code_src + (size_t)row * (D / 2) + lane * 16;
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        a4_copy16(place[j] + stage + u * L::TILE, src + j * 512);
                        a4_copy16(place[j] + stage + (u * L::TILE + L::SIDE), src + j * 512 + side_bytes);
                    }
                    if constexpr (8 * NG <= 32) {
                        if (lane < 8 * NG)
                            a4_copy16(ring + stage + lane * 16 + (u * L::TILE + 2 * L::SIDE), scale_src + (size_t)row * (NG * 4));
                    } else {
#pragma unroll
                        for (int c = lane; c < 8 * NG; c += 32) {
                            const int side = c / (4 * NG), at = c % (4 * NG);
                            a4_copy16(ring + stage + u * L::TILE + 2 * L::SIDE + c * 16,
                                      p.scales + (head_row + row + side * side_rows) * (NG * 4) + at * 16);
                        }
                    }
                }
            } else if (whole) {
#pragma unroll 1
                for (int u = 0; u < 2; ++u) {
                    const uint32_t lower = __shfl_sync(0xffffffffu, u ? rows_of[2] : rows_of[0], looked);
                    const uint32_t upper = __shfl_sync(0xffffffffu, u ? rows_of[3] : rows_of[1], looked);
                    const uint32_t to = stage + u * L::TILE;
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        const int c = lane + 32 * j, r = c / (D / 32);
                        const uint32_t row = r < 8 ? lower + r : upper + (r - 8);
                        const uint8_t* src = code_src + (size_t)row * (D / 2) + (c % (D / 32)) * 16;
                        a4_copy16(place[j] + to, src);
                        a4_copy16(place[j] + to + L::SIDE, src + side_bytes);
                    }
#pragma unroll
                    for (int c = lane; c < 8 * NG; c += 32) {
                        // 2 NG units of 16 bytes are eight rows' scales
                        const int side = c / (4 * NG), at = c % (4 * NG);
                        const size_t row = (at < 2 * NG ? lower : upper) + head_row + side * side_rows;
                        a4_copy16(ring + to + 2 * L::SIDE + c * 16, p.scales + row * (NG * 4) + (at < 2 * NG ? at : at - 2 * NG) * 16);
                    }
                }
            } else {
                const uint32_t to = ring + stage;
#pragma unroll 1
                for (int c = lane; c < 32 * (D / 32); c += 32) {
                    const int r = c / (D / 32), u = c % (D / 32), key = ahead * 16 + r;
                    const long long one = key <= max_pos
                        ? c4_row(table, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, key) : -1;
                    const size_t row = one >= 0 ? (size_t)one + head_row : 0;
                    const uint8_t* src = p.codes + row * (D / 2) + u * 16;
                    const uint32_t dst = to + (r >> 4) * L::TILE + a4_place<D>(r & 15, u);
                    a4_copy16(dst, src);
                    a4_copy16(dst + L::SIDE, src + side_bytes);
                }
#pragma unroll 1
                for (int c = lane; c < 32 * NG; c += 32) {
                    const int r = c / NG, u = c % NG, key = ahead * 16 + r;
                    const long long one = key <= max_pos
                        ? c4_row(table, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, key) : -1;
                    const size_t row = one >= 0 ? (size_t)one + head_row : 0;
                    const uint8_t* src = p.scales + (row * NG + u) * 4;
                    const uint32_t dst = to + (r >> 4) * L::TILE + 2 * L::SIDE + ((r & 15) * NG + u) * 4;
                    a4_copy4(dst, src);
                    a4_copy4(dst + L::SCALES, src + side_rows * (NG * 4));
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        edges = (edges >> 1) | (edges_of & 1u) << (L::STAGES - 2);
        edges_of >>= 1;
        ahead += 2 * A4_WARPS;
        if (++looked == 32) {
            looked = 0;
            look();
            settle();
        }
    };
    look();
#pragma unroll 1
    for (int s = 0; s < L::STAGES - 1; ++s) fetch(s * L::STAGE);

    // ---- the queries, as columns of the first product --------------------------
    {
        __half* qs = reinterpret_cast<__half*>(smem + L::AT_Q);
        float* sums = reinterpret_cast<float*>(smem + L::AT_SUMS);
        float* factor = reinterpret_cast<float*>(smem + L::AT_FACTOR);
#pragma unroll
        for (int j = 0; j < MINE; ++j) {
            const int r = warp + j * A4_WARPS;
            float v[D / 32];
            float most = 0.f;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) v[i] = cb_to_float(query[j][i]);
#pragma unroll
            for (int i = 0; i < D / 32; ++i) most = fmaxf(most, fabsf(v[i]));
            most = cb_warp_max(most);
            // (100: the factor 2^-e stays far from float32's ends)
            const int e = most > 0.f ? min(13 - ((int)(__float_as_uint(most) >> 23) - 127), 100) : 0;
            const float up = a4_power(e);
            // (never zero, which a masked score, minus infinity, may not meet)
            if (lane == 0) factor[r] = fmaxf(p.scale_log2 * a4_power(-e), __int_as_float(1));
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                v[i] *= up;
                const int f = lane + 32 * i, w = f >> 6, k = (f >> 3) & 7, c8 = f & 7;
                // step (w, k / 4, c8 & 1) of the product, lane (r & 7, c8 / 2), number (0, 2, 1, 3)[k & 3]
                const int ks = (w * 2 + (k >> 2)) * 2 + (c8 & 1), n = ((k & 1) << 1) | ((k >> 1) & 1);
                float y = (k & 1) ? v[i] * 0.0625f : v[i];        // its codes come 16 times too large
#pragma unroll
                for (int part = 0; part < PARTS; ++part) {
                    const __half h = __float2half_rn(y);
                    y -= __half2float(h);
                    qs[(((ks * PARTS + part) * NT + (r >> 3)) * 32 + (r & 7) * 4 + (c8 >> 1)) * 4 + n] = h;
                }
            }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < GROUP / 32; ++i) s += v[gr * (GROUP / 32) + i];
                s = cb_warp_sum(s);
                if (lane == 0) sums[r * NG + gr] = s;
            }
        }
        __syncthreads();
    }
    const uint2* qf = reinterpret_cast<const uint2*>(smem + L::AT_Q) + lane;
    constexpr bool Q_IN_REGS = KS * PARTS * NT <= 8;
    uint2 qr[Q_IN_REGS ? KS * PARTS * NT : 1];
    if constexpr (Q_IN_REGS) {
#pragma unroll
        for (int i = 0; i < KS * PARTS * NT; ++i) qr[i] = qf[i * 32];
    }
    float qsum[NT][NG][2], factor[NT][2];
    int pos[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = n * 8 + 2 * t + c;
            factor[n][c] = reinterpret_cast<const float*>(smem + L::AT_FACTOR)[r];
            pos[n][c] = first + min(base + r, n_rows - 1) / p.n_rep;
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) qsum[n][gr][c] = reinterpret_cast<const float*>(smem + L::AT_SUMS)[r * NG + gr];
        }

    // ---- over the keys -----------------------------------------------------------
    // A pair of tiles.  EDGE: some row may not see some key of it (the four runs' first keys, -1 for none).
    auto pair = [&](auto edge, const uint8_t* at, int key_a, int key_b, int key_c, int key_d) {
        constexpr bool EDGE = decltype(edge)::value;
        float s[2][NT][4];
        uint32_t vsc[2][2][NG];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // S^T = K Q^T, by groups
            const uint8_t* tile = at + u * L::TILE;
            uint32_t kw[2][2 * W], ksc[2][NG];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if constexpr (D == 64 || D == 192) {
#pragma unroll
                    for (int j = 0; j < D / 64; ++j) {
                        const uint2 v = *reinterpret_cast<const uint2*>(tile + k_at + h * EIGHT + j * 8);
                        kw[h][2 * j] = v.x; kw[h][2 * j + 1] = v.y;
                    }
                } else {
                    // (256: the lane's second unit is the first's neighbour, which the places exchange but do not part)
#pragma unroll
                    for (int j = 0; j < D / 128; ++j) {
                        const uint4 v = *reinterpret_cast<const uint4*>(tile + (j == 0 ? k_at : k_at ^ 16) + h * EIGHT);
                        kw[h][4 * j] = v.x; kw[h][4 * j + 1] = v.y; kw[h][4 * j + 2] = v.z; kw[h][4 * j + 3] = v.w;
                    }
                }
                a4_pairs<NG>(ksc[h], tile + s_at + 8 * h * (NG * 4));
                a4_pairs<NG>(vsc[u][h], tile + s_at + L::SCALES + 8 * h * (NG * 4));
            }
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) {
                float acc[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
                for (int b = gr * (GROUP / 32); b < (gr + 1) * (GROUP / 32); ++b) {         // 32 features
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int ks = b * 2 + c, wi = c * W + (b >> 1);
                        const uint32_t wa = (b & 1) ? kw[0][wi] >> 8 : kw[0][wi], wb = (b & 1) ? kw[1][wi] >> 8 : kw[1][wi];
                        const uint32_t a0 = a4_codes<F32, false>(wa), a1 = a4_codes<F32, false>(wb);
                        const uint32_t a2 = a4_codes<F32, true>(wa), a3 = a4_codes<F32, true>(wb);
#pragma unroll
                        for (int part = 0; part < PARTS; ++part)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                uint2 q;
                                if constexpr (Q_IN_REGS) q = qr[(ks * PARTS + part) * NT + n];
                                else q = qf[((ks * PARTS + part) * NT + n) * 32];
                                a4_mma(acc[n], a0, a1, a2, a3, q.x, q.y);
                            }
                    }
                }
                const float sa = c4_step(ksc[0][gr]) * CODE, la = a4_low<F32>(ksc[0][gr]);
                const float sb = c4_step(ksc[1][gr]) * CODE, lb = a4_low<F32>(ksc[1][gr]);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const float wa = gr == 0 ? la * qsum[n][gr][c] : fmaf(la, qsum[n][gr][c], s[u][n][c]);
                        const float wb = gr == 0 ? lb * qsum[n][gr][c] : fmaf(lb, qsum[n][gr][c], s[u][n][2 + c]);
                        s[u][n][c] = fmaf(acc[n][c], sa, wa);
                        s[u][n][2 + c] = fmaf(acc[n][2 + c], sb, wb);
                    }
                }
            }
        }

        // what a row does not see: bits 4 NT u + 4 n + 2 h + c
        uint32_t hidden = 0;
        if constexpr (EDGE) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const int key0 = u == 0 ? (h == 0 ? key_a : key_b) : (h == 0 ? key_c : key_d), key = key0 + g;
                            bool out = key0 < 0 || key > pos[n][c] || (p.window > 0 && key <= pos[n][c] - p.window);
                            if (!whole && !out)
                                out = c4_row(table, p.table_stride, p.page_tokens, p.n_pages, p.kv_heads, key) < 0;
                            if (out) {
                                s[u][n][2 * h + c] = -INFINITY;
                                hidden |= 1u << (4 * NT * u + 4 * n + 2 * h + c);
                            }
                        }
        }

        // the references move only when they have to
        constexpr float LOW = 9.5367431640625e-7f;           // 2^-20
        float most_step[2][2], most_low[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // (a low that is 2^20 steps and more counts, too: 2^eps times it has to be far from float32's end)
                most_step[u][h] = c4_step(vsc[u][h][0]);
                most_low[u][h] = fabsf(__uint_as_float(vsc[u][h][0]));         // (with the step behind it: next to nothing)
#pragma unroll
                for (int gr = 1; gr < NG; ++gr) {
                    most_step[u][h] = fmaxf(most_step[u][h], c4_step(vsc[u][h][gr]));
                    most_low[u][h] = fmaxf(most_low[u][h], fabsf(__uint_as_float(vsc[u][h][gr])));
                }
            }
        bool move = false;
        float top[NT][2], step_top[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                top[n][c] = fmaxf(fmaxf(s[0][n][c], s[0][n][2 + c]), fmaxf(s[1][n][c], s[1][n][2 + c]));
                step_top[n][c] = 0.f;
                if constexpr (EDGE) {
#pragma unroll
                    for (int u = 0; u < 2; ++u)
#pragma unroll
                        for (int h = 0; h < 2; ++h)
                            if (!((hidden >> (4 * NT * u + 4 * n + 2 * h + c)) & 1))
                                step_top[n][c] = fmaxf(step_top[n][c], fmaxf(most_step[u][h], LOW * most_low[u][h]));
                } else {
                    step_top[n][c] = fmaxf(fmaxf(most_step[0][0], most_step[0][1]), fmaxf(most_step[1][0], most_step[1][1]));
                    step_top[n][c] = fmaxf(step_top[n][c], LOW * fmaxf(fmaxf(most_low[0][0], most_low[0][1]), fmaxf(most_low[1][0], most_low[1][1])));
                }
                move = move || fmaf(top[n][c], factor[n][c], -off[n][c]) > limit[n][c] || step_top[n][c] >= bound[n][c];
            }
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const float m = fmaxf(off[n][c] + (limit[n][c] - 8.f), a4_over_keys_max(top[n][c] * factor[n][c]));
                    const float st = a4_over_keys_max(step_top[n][c]);
                    const int e = min(max((int)(__float_as_uint(fmaxf(st, bound[n][c] * 0.5f)) >> 23) - 127, -96), 126);
                    const float e5 = 5.f - (float)e, to = m - e5;
                    const A4Fall fall(off[n][c] - to);
                    const float r = fall.whole();
                    off[n][c] = to;
                    limit[n][c] = e5 + 8.f;
                    bound[n][c] = a4_power(e + 1);
                    sum[n][c] = fall.of(sum[n][c]);
#pragma unroll
                    for (int gr = 0; gr < NG; ++gr) lows[n][gr][c] *= r;
#pragma unroll
                    for (int j = 0; j < MT; ++j) {
                        o[j][n][c] *= r;
                        o[j][n][2 + c] *= r;
                    }
                }
        }

#pragma unroll
        for (int u = 0; u < 2; ++u) {
            // p, and P^T step as columns of the second product
            uint32_t b[NG][PARTS][NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float pr[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    pr[j] = a4_exp2(fmaf(s[u][n][j], factor[n][j & 1], -off[n][j & 1]));
                    sum[n][j & 1] += pr[j];
                }
#pragma unroll
                for (int gr = 0; gr < NG; ++gr) {
                    float w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        w[j] = pr[j] * c4_step(vsc[u][j >> 1][gr]);
                        float low = a4_low<F32>(vsc[u][j >> 1][gr]);
                        if constexpr (EDGE)
                            if ((hidden >> (4 * NT * u + 4 * n + j)) & 1) w[j] = low = 0.f;   // (what nobody wrote may be no number)
                        lows[n][gr][j & 1] = fmaf(pr[j], low, lows[n][gr][j & 1]);
                    }
#pragma unroll
                    for (int part = 0; part < PARTS; ++part) {
                        const uint32_t h0 = a4_half2(w[0], w[1]), h1 = a4_half2(w[2], w[3]);
                        if constexpr (PARTS == 2) {
                            const float2 f0 = __half22float2(*reinterpret_cast<const __half2*>(&h0));
                            const float2 f1 = __half22float2(*reinterpret_cast<const __half2*>(&h1));
                            w[0] -= f0.x; w[1] -= f0.y; w[2] -= f1.x; w[3] -= f1.y;
                        }
                        b[gr][part][n][0] = a4_turned(h0);
                        b[gr][part][n][1] = a4_turned(h1);
                    }
                }
            }

            // O^T += V^T P^T
            uint32_t vw[4][W];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint8_t* from = at + u * L::TILE + v_at[j & 1] + (j >> 1) * EIGHT;
                if constexpr (D == 128) {
                    const uint2 v = *reinterpret_cast<const uint2*>(from);
                    vw[j][0] = v.x; vw[j][1] = v.y;
                } else if constexpr (D == 256) {
                    const uint4 v = *reinterpret_cast<const uint4*>(from);
                    vw[j][0] = v.x; vw[j][1] = v.y; vw[j][2] = v.z; vw[j][3] = v.w;
                } else {
#pragma unroll
                    for (int w = 0; w < W; ++w) vw[j][w] = reinterpret_cast<const uint32_t*>(from)[w];
                }
            }
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    // half words of two keys side by side: features of tiles 4w + half and 4w + 2 + half
                    uint32_t z0 = __byte_perm(vw[0][w], vw[1][w], half ? 0x7632 : 0x5410);
                    uint32_t z1 = __byte_perm(vw[2][w], vw[3][w], half ? 0x7632 : 0x5410);
#pragma unroll
                    for (int v = 0; v < 2; ++v) {
                        const int m = 4 * w + 2 * v + half, gr = m * 16 / GROUP;
                        if (v == 1) { z0 >>= 8; z1 >>= 8; }
                        const uint32_t a0 = a4_codes<F32, false>(z0), a1 = a4_codes<F32, true>(z0);
                        const uint32_t a2 = a4_codes<F32, false>(z1), a3 = a4_codes<F32, true>(z1);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if constexpr (F32) {
                                float part[4] = {0.f, 0.f, 0.f, 0.f};
                                a4_mma(part, a0, a1, a2, a3, b[gr][1][n][0], b[gr][1][n][1]);
                                a4_mma(part, a0, a1, a2, a3, b[gr][0][n][0], b[gr][0][n][1]);
#pragma unroll
                                for (int j = 0; j < 4; ++j) o[m][n][j] += part[j];
                            } else {
                                a4_mma(o[m][n], a0, a1, a2, a3, b[gr][0][n][0], b[gr][0][n][1]);
                            }
                        }
                    }
                }
        }
    };
    // the stage that was read last, to be filled; the next one is to be read
    uint32_t into = (L::STAGES - 1) * L::STAGE;
    auto next = [&]() -> const uint8_t* {
        asm volatile("cp.async.wait_group %0;" ::"n"(L::STAGES - 2) : "memory");
        __syncwarp();
        fetch(into);
        into = into == (L::STAGES - 1) * L::STAGE ? 0 : into + L::STAGE;
        return smem + warp * L::RING + into;
    };
    // (two loops, so that the one over whole tiles is nothing else: one loop that chose between the two forms moved
    // registers about at every turn)
    for (int i = tile_lo + 2 * warp; i < tile_hi; i += 2 * A4_WARPS) {
        while (!(edges & 1)) {
            pair(std::false_type{}, next(), 0, 0, 0, 0);
            i += 2 * A4_WARPS;
            if (i >= tile_hi) break;
        }
        if (i >= tile_hi) break;
        int page;
        const int key_a = key_of(2 * i, page), key_b = key_of(2 * i + 1, page);
        const int key_c = key_of(2 * i + 2, page), key_d = key_of(2 * i + 3, page);
        pair(std::true_type{}, next(), key_a, key_b, key_c, key_d);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the warps' results ------------------------------------------------------
    // A column's result is o over the codes' unit (and over 16 of it where they come 16 times too large) plus its lows,
    // relative to 2^off.
    __syncthreads();
    float* mine = reinterpret_cast<float*>(smem + warp * L::RING);
    float* state = reinterpret_cast<float*>(smem + L::AT_STATE);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const float l = a4_over_keys_sum(sum[n][c]);
            float low[NG];
#pragma unroll
            for (int gr = 0; gr < NG; ++gr) low[gr] = a4_over_keys_sum(lows[n][gr][c]);
            const int r = n * 8 + 2 * t + c;
            if (g == 0) {
                state[(warp * L::ROWS + r) * 2] = off[n][c];
                state[(warp * L::ROWS + r) * 2 + 1] = l;
            }
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                mine[r * L::PITCH + m * 16 + g] = fmaf(o[m][n][c], CODE, low[m * 16 / GROUP]);
                mine[r * L::PITCH + m * 16 + 8 + g] = fmaf(o[m][n][2 + c], CODE / 16.f, low[m * 16 / GROUP]);
            }
        }
    __syncthreads();
    // every row's weights of the warps, and what the block has of it
    float* block_state = state + A4_WARPS * L::ROWS * 2;
    if (threadIdx.x < L::ROWS) {
        const int r = threadIdx.x;
        float top = -3.4e38f, l = 0.f;
#pragma unroll
        for (int w = 0; w < A4_WARPS; ++w) top = fmaxf(top, state[(w * L::ROWS + r) * 2]);
#pragma unroll
        for (int w = 0; w < A4_WARPS; ++w) {
            const A4Fall fall(state[(w * L::ROWS + r) * 2] - top);
            l += fall.of(state[(w * L::ROWS + r) * 2 + 1]);
            state[(w * L::ROWS + r) * 2] = fall.whole();
        }
        block_state[r * 2] = top;
        block_state[r * 2 + 1] = l;
    }
    __syncthreads();
    auto of_block = [&](int i) {
        const int r = i / D;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < A4_WARPS; ++w)
            v = fmaf(reinterpret_cast<const float*>(smem + w * L::RING)[i + r * (L::PITCH - D)], state[(w * L::ROWS + r) * 2], v);
        return v;
    };
    auto store = [&](int i, float v) {
        const int r = i / D, tok = (base + r) / p.n_rep, head = kv * p.n_rep + (base + r) - tok * p.n_rep;
        reinterpret_cast<T*>(p.out)[(size_t)(row0 + tok) * p.out_stride + (size_t)head * D + (i - r * D)] = cb_from_float<T>(v);
    };
    if (p.stream > 0) {
        if (taken < weight) {                            // the other blocks' results of it are needed, too
            float* to = p.partial + ((size_t)blockIdx.x * 2 + slot) * (L::ROWS * (D + 2));
            for (int i = threadIdx.x; i < live * D; i += A4_WARPS * 32) to[2 * L::ROWS + i] = of_block(i);
            if (threadIdx.x < 2 * live) to[threadIdx.x] = block_state[threadIdx.x];
        }
    }
    if (p.stream > 0 ? taken == weight : gridDim.z == 1) {
        for (int i = threadIdx.x; i < live * D; i += A4_WARPS * 32) {
            const float l = block_state[(i / D) * 2 + 1];
            store(i, l == 0.f ? 0.f : of_block(i) / l);          // (a row that sees no key: zeros)
        }
    }
    if (p.stream > 0) {
        left -= taken;
        if (left == 0) return;
        // the next kv head, or unit
        skip = 0;
        slot = 1;                                        // (what follows is shared only if it is the last)
        if (++kv == p.kv_heads) {
            kv = 0;
            ++index;
        }
        __syncthreads();
        continue;
    }
    if (gridDim.z == 1) return;
    // blocks of a cluster: each takes its share of the numbers from all
    for (int i = threadIdx.x; i < live * D; i += A4_WARPS * 32)
        reinterpret_cast<float*>(smem)[i + i / D * (L::PITCH - D)] = of_block(i);      // (over warp 0's, which this thread alone reads)
    __syncthreads();
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const uint32_t result = a4_smem(smem), states = a4_smem(block_state);
    const int shares = gridDim.z;
    const int per = (live * D + shares - 1) / shares;
    for (int i = blockIdx.z * per + threadIdx.x; i < min(live * D, (int)(blockIdx.z + 1) * per); i += A4_WARPS * 32) {
        float top = -3.4e38f, refs[8], ls[8], vals[8];
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            refs[z] = -3.4e38f;
            ls[z] = vals[z] = 0.f;
            if (z < shares) {
                uint32_t there, state_there;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(result + (i + i / D * (L::PITCH - D)) * 4), "r"(z));
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(state_there) : "r"(states + (i / D) * 8), "r"(z));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(vals[z]) : "r"(there));
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(refs[z]), "=f"(ls[z]) : "r"(state_there));
                top = fmaxf(top, refs[z]);
            }
        }
        float v = 0.f, l = 0.f;
#pragma unroll
        for (int z = 0; z < 8; ++z) {
            const A4Fall fall(refs[z] - top);
            v = fmaf(vals[z], fall.whole(), v);
            l += fall.of(ls[z]);
        }
        store(i, l == 0.f ? 0.f : v / l);
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    return;
  }
}

// Stream: a row whose tile several blocks had a share of, a block a row, D / 4 threads a result side by side.  The first of
// these blocks has it as its second result (unless its share begins there), the others as their first.  Who has what
// is worked out while the main kernel still runs; then every thread fetches its share of the results with their
// references at once and keeps a running reference of its own.
template <int D, int NT, bool F32>
__global__ void __launch_bounds__(256) attention4_merge_kernel(const Attn4Params p) {
    constexpr int ROWS = 8 * NT, LANES = D / 4, SETS = 256 / LANES, ONE = ROWS * (D + 2);
    using T = typename std::conditional<F32, float, __nv_bfloat16>::type;
    __shared__ uint32_t counts[2][8];
    __shared__ float refs[SETS][2];
    __shared__ float4 sums[SETS][LANES];
    const int r = blockIdx.y, index = blockIdx.x / p.kv_heads, kv = blockIdx.x - index * p.kv_heads;
    const int tid = threadIdx.x, set = tid / LANES, lane = tid % LANES;
    const A4Unit unit = a4_unit<ROWS>(p, index);
    // (every block waits, one that has nothing to do, too: what is launched behind this kernel waits for it alone)
    if (unit.base + r >= unit.n_rows) {
        cb_pdl_wait();
        return;
    }
    uint32_t tiles = unit.weight(), before = 0;
    if (p.units > 1) {
        tiles = 0;
        for (int u = tid; u < p.units; u += 256) {
            const int w = a4_unit<ROWS>(p, u).weight();
            tiles += w;
            if (u < index) before += w;
        }
        tiles = __reduce_add_sync(0xffffffffu, tiles);
        before = __reduce_add_sync(0xffffffffu, before);
        if ((tid & 31) == 0) {
            counts[0][tid >> 5] = tiles;
            counts[1][tid >> 5] = before;
        }
        __syncthreads();
        tiles = before = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            tiles += counts[0][i];
            before += counts[1][i];
        }
    }
    const uint32_t quota = a4_quota(tiles * p.kv_heads, p.stream), begin = before * p.kv_heads + kv * unit.weight();
    const int from = begin / quota, n = (int)((begin + unit.weight() - 1) / quota) - from + 1;
    const bool second = begin != quota * from;
    cb_pdl_wait();
    cb_pdl_trigger();
    if (n <= 1) return;                          // (its block has written the row)
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -3.4e38f, l = 0.f;
    if (set < SETS) {
#pragma unroll 4
        for (int z = set; z < n; z += SETS) {
            const float* one = p.partial + ((size_t)(from + z) * 2 + (z == 0 && second ? 1 : 0)) * ONE;
            const float2 head = *reinterpret_cast<const float2*>(one + 2 * r);
            const float2 a = *reinterpret_cast<const float2*>(one + 2 * ROWS + r * D + lane * 4);
            const float2 b = *reinterpret_cast<const float2*>(one + 2 * ROWS + r * D + lane * 4 + 2);
            const float most = fmaxf(top, head.x);
            const A4Fall before(top - most), now(head.x - most);
            const float was = before.whole(), w = now.whole();
            v.x = fmaf(a.x, w, v.x * was);
            v.y = fmaf(a.y, w, v.y * was);
            v.z = fmaf(b.x, w, v.z * was);
            v.w = fmaf(b.y, w, v.w * was);
            l = now.of(head.y) + before.of(l);
            top = most;
        }
        sums[set][lane] = v;
        if (lane == 0) {
            refs[set][0] = top;
            refs[set][1] = l;
        }
    }
    __syncthreads();
    if (tid < D) {
        float x = 0.f, most = -3.4e38f;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < SETS; ++i) most = fmaxf(most, refs[i][0]);
#pragma unroll
        for (int i = 0; i < SETS; ++i) {
            const A4Fall fall(refs[i][0] - most);
            x = fmaf(reinterpret_cast<const float*>(sums[i])[tid], fall.whole(), x);
            l += fall.of(refs[i][1]);
        }
        const int tok = (unit.base + r) / p.n_rep, head = kv * p.n_rep + (unit.base + r) - tok * p.n_rep;
        reinterpret_cast<T*>(p.out)[(size_t)(unit.row0 + tok) * p.out_stride + (size_t)head * D + tid] =
            cb_from_float<T>(l == 0.f ? 0.f : x / l);
    }
}

template <int D, int NG, int NT, bool F32>
int attention4_launch(const Attn4Params& p, long long blocks, int shares, cudaStream_t stream) {
    using L = A4Layout<D, NG, NT, F32 ? 2 : 1>;
    static bool ready[64] = {};          // (per device; setting it twice does no harm)
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        const int rc = (int)cudaFuncSetAttribute(attention4_kernel<D, NG, NT, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 L::TOTAL);
        if (rc != 0) return rc;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    const dim3 grid((unsigned)(p.stream > 0 ? p.stream : blocks), 1, (unsigned)(p.stream > 0 ? 1 : shares));
    int rc = cb_launch_cluster(attention4_kernel<D, NG, NT, F32>, grid, dim3(A4_WARPS * 32), L::TOTAL, stream,
                               p.stream > 0 ? 1 : shares, p);
    if (rc == 0 && p.stream > 0)
        rc = cb_launch(attention4_merge_kernel<D, NT, F32>, dim3((unsigned)blocks, 8 * NT), dim3(256), 0, stream, p);
    return rc;
}

template <int D, int NG>
int attention4_of(const Attn4Params& p, int dtype, int column_tiles, long long blocks, int shares, cudaStream_t stream) {
    if (dtype == CB_F32) return attention4_launch<D, NG, 1, true>(p, blocks, shares, stream);
    if (column_tiles == 1) return attention4_launch<D, NG, 1, false>(p, blocks, shares, stream);
    if constexpr (D <= 128) return attention4_launch<D, NG, 2, false>(p, blocks, shares, stream);
    return CB_ERR_UNSUPPORTED;           // (wider heads have no registers for two column tiles)
}

}  // namespace

// One file a head size (D) is built, so that a model compiles only its own.
#define ATTENTION4_ENTRY(D)                                                                                             \
    {                                                                                                                   \
        if (group != 32 && group != 64 && group != 128) return CB_ERR_UNSUPPORTED;                                       \
        if (D % group != 0 || column_tiles < 1 || column_tiles > 2 || shares < 1 || shares > 8) return CB_ERR_UNSUPPORTED; \
        const int rows_a_tile = 8 * column_tiles;                                                                        \
        const int row_tiles = (most_rows * n_rep + rows_a_tile - 1) / rows_a_tile;                                       \
        const long long units = (long long)(picks != nullptr ? rows : requests) * row_tiles, blocks = units * kv_heads;  \
        if (blocks <= 0) return 0;                                                                                       \
        if (blocks >= (1LL << 31)) return CB_ERR_UNSUPPORTED;                                                            \
        const int eights = page_tokens % 8 ? 0 : page_tokens / 8;                                                        \
        const Attn4Params p = {q, q_stride, out, out_stride, reinterpret_cast<const uint8_t*>(codes),                    \
                               reinterpret_cast<const uint8_t*>(scales), n_pages, page_tokens, kv_heads, n_rep,          \
                               row_start, first_pos, table, table_stride, requests, picks, pick_count, row_request,      \
                               positions, rows, eights,                                                                  \
                               eights <= 1 ? 0u : (uint32_t)((1ull << 32) / eights) + 1u, window,                        \
                               scale * A4_LOG2E, row_tiles, (int)units, stream_blocks, partial};                         \
        const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);                                                   \
        int rc = CB_ERR_UNSUPPORTED;                                                                                     \
        if (group == 32) rc = attention4_of<D, D / 32>(p, dtype, column_tiles, blocks, shares, s);                       \
        else if (group == 64) rc = attention4_of<D, D / 64>(p, dtype, column_tiles, blocks, shares, s);                  \
        else if constexpr (D % 128 == 0) rc = attention4_of<D, D / 128>(p, dtype, column_tiles, blocks, shares, s);      \
        if (rc == CB_ERR_UNSUPPORTED) return rc;                                                                         \
        const int last = cb_last_error();                                                                                \
        return rc != 0 ? rc : last;                                                                                      \
    }
