// Which pages a row attends to: for every row and kv head the pages whose bounds allow the largest logits.
//
// A page's bounds are the largest and least of each feature of its keys, in 8 bits with one scale a; a query is
// rounded to 8 bits too, scale b.  No key of the page has a larger q . k than sum_f max(q_f hi_f, q_f lo_f), in 8 bits
//     dot = sum_f max(q_f, 0) hi_f + min(q_f, 0) lo_f,
// two products of whole numbers (below 2^24, so float32 holds them), and a page scores (float) dot * (b a), the
// largest over the heads of the group: every operation is rounded once, so that which pages are picked is defined.
//
// Up to eight blocks of a cluster score a row's pages (four lanes a page, 16 bytes a load, two pages at a time, the
// queries in shared memory) into the first one's shared memory.  That one finds the count-th largest score by its
// bits, eight at a time below the first in which the largest and the least differ (so that the histogram's bins are hit
// evenly; as a rule the second or third decides), and writes the pages out in ascending order, of equal scores
// those that come first.
//
// 16 rows behind 32,767 keys, 8 kv heads of 128 in pages of 64, 64 of 512 pages: 8.5 us, 13.5 MB of bounds (2 at the rate of a
// copy); one row of 4 heads of 64 behind 131,000 keys in pages of 32, 96 of 4,094: 11.7.  Not bounds but the way takes the
// time: a cluster's beginning, the scores' way into one block, then the picking's rounds one behind the other.
#define CB_PDL_BIT 6      // with the other quantised operators
#include "cache4.cuh"

namespace {

constexpr int PICK_THREADS = 512;
constexpr int PICK_ROOM = 220 * 1024;      // bytes of shared memory that scores and queries may take

struct PickParams {
    const void* q;
    long long q_stride;
    const int* positions;
    const int* row_request;
    const int* table;
    int table_stride, n_requests;
    const int8_t* bounds;          // [pages][kv heads][2][D]
    const float* bound_scales;     // [pages][kv heads]
    int n_pages, page_tokens, n_rep, kv_heads, rows;
    int* picks;                    // [rows][kv heads][count]
    int count, first, last;
    int most_pages;                // scores that shared memory holds
};

__device__ __forceinline__ uint32_t order_of(float v) {
    if (!(v == v)) return 0;
    const uint32_t b = __float_as_uint(v + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

template <int D, typename T>
__global__ void __launch_bounds__(PICK_THREADS) pick4_kernel(const PickParams p) {
    cb_pdl_trigger();
    cb_pdl_wait();
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* score = reinterpret_cast<uint32_t*>(smem);                                // [most_pages]
    int4* q8 = reinterpret_cast<int4*>(smem + (size_t)p.most_pages * 4);                // [n_rep][2][D / 16]
    float* q_scale = reinterpret_cast<float*>(q8 + (size_t)p.n_rep * 2 * (D / 16));     // [n_rep]
    __shared__ int histogram[256], found[4], warp_counts[PICK_THREADS / 32];
    __shared__ uint32_t ends[2][PICK_THREADS / 32];
    const int row = blockIdx.x / p.kv_heads, kv = blockIdx.x - row * p.kv_heads;
    const int request = p.row_request[row], pos = p.positions[row];
    if (request < 0 || request >= p.n_requests || pos < 0) return;                      // (all blocks of a cluster)
    const int own = min(pos / p.page_tokens, min(p.table_stride, p.most_pages) - 1), pages = own + 1;
    int* picks = p.picks + ((size_t)row * p.kv_heads + kv) * p.count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (pages <= p.count) {
        if (blockIdx.z == 0)
            for (int i = tid; i < p.count; i += PICK_THREADS) picks[i] = i < pages ? i : -1;
        return;
    }
    // (another block's shared memory may be written once that block runs: arrived here, waited for below)
    if (gridDim.z > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    // pages are scored by four lanes each; the first are asked for before the queries are worked on
    const int* table = p.table + (size_t)request * p.table_stride;
    const int quarter = lane & 3;
    const int stride = gridDim.z * (PICK_THREADS / 4);
    uint32_t there = (uint32_t)__cvta_generic_to_shared(score);
    if (gridDim.z > 1) asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(there) : "r"(there));
    constexpr int WIDE = 2;
    int4 hi[WIDE][D / 64], lo[WIDE][D / 64];
    float a[WIDE];
    int page[WIDE];
    auto load = [&](int at) {
#pragma unroll
        for (int n = 0; n < WIDE; ++n) {
            const int index = at + n * stride + (tid >> 2);
            page[n] = index < pages ? table[index] : -1;
        }
#pragma unroll
        for (int n = 0; n < WIDE; ++n) {
            a[n] = 0.f;
            if ((unsigned)page[n] < (unsigned)p.n_pages) {
                const size_t to = (size_t)page[n] * p.kv_heads + kv;
                const int4* b = reinterpret_cast<const int4*>(p.bounds + to * 2 * D);
#pragma unroll
                for (int j = 0; j < D / 64; ++j) {
                    hi[n][j] = b[quarter + 4 * j];
                    lo[n][j] = b[D / 16 + quarter + 4 * j];
                }
                a[n] = p.bound_scales[to];
            } else {
#pragma unroll
                for (int j = 0; j < D / 64; ++j) hi[n][j] = lo[n][j] = make_int4(0, 0, 0, 0);
            }
        }
    };
    load(blockIdx.z * (PICK_THREADS / 4));
    // the group's queries in 8 bits: a warp a head
    for (int h = warp; h < p.n_rep; h += PICK_THREADS / 32) {
        const T* src = reinterpret_cast<const T*>(p.q) + (size_t)row * p.q_stride + (size_t)(kv * p.n_rep + h) * D;
        float v[D / 32], most = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            v[i] = cb_to_float(src[lane + 32 * i]);
            most = fmaxf(most, fabsf(v[i]));
        }
        const float scale = __fmul_rn(cb_warp_max(most), 1.0f / 127.0f);
        const float inverse = scale > 0.f ? __frcp_rn(scale) : 0.f;
        int8_t* up = reinterpret_cast<int8_t*>(q8 + (size_t)h * 2 * (D / 16));
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int c = (int)fminf(fmaxf(rintf(__fmul_rn(v[i], inverse)), -127.f), 127.f);
            up[lane + 32 * i] = (int8_t)max(c, 0);
            up[D + lane + 32 * i] = (int8_t)min(c, 0);
        }
        if (lane == 0) q_scale[h] = scale;
    }
    __syncthreads();
    if (gridDim.z > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    for (int at = blockIdx.z * (PICK_THREADS / 4); at < pages; at += WIDE * stride) {       // (whole warps: shuffles)
        float best[WIDE];
#pragma unroll
        for (int n = 0; n < WIDE; ++n) best[n] = -INFINITY;
        for (int h = 0; h < p.n_rep; ++h) {
            const int4* up = q8 + (size_t)h * 2 * (D / 16);
            int dot[WIDE] = {};
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
                const int4 u = up[quarter + 4 * j], d = up[D / 16 + quarter + 4 * j];
#pragma unroll
                for (int n = 0; n < WIDE; ++n) {
                    dot[n] = __dp4a(u.x, hi[n][j].x, dot[n]); dot[n] = __dp4a(u.y, hi[n][j].y, dot[n]);
                    dot[n] = __dp4a(u.z, hi[n][j].z, dot[n]); dot[n] = __dp4a(u.w, hi[n][j].w, dot[n]);
                    dot[n] = __dp4a(d.x, lo[n][j].x, dot[n]); dot[n] = __dp4a(d.y, lo[n][j].y, dot[n]);
                    dot[n] = __dp4a(d.z, lo[n][j].z, dot[n]); dot[n] = __dp4a(d.w, lo[n][j].w, dot[n]);
                }
            }
            const float unit = q_scale[h];
#pragma unroll
            for (int n = 0; n < WIDE; ++n) {
                dot[n] += __shfl_xor_sync(0xffffffffu, dot[n], 1);
                dot[n] += __shfl_xor_sync(0xffffffffu, dot[n], 2);
                best[n] = fmaxf(best[n], __fmul_rn((float)dot[n], __fmul_rn(unit, a[n])));
            }
        }
#pragma unroll
        for (int n = 0; n < WIDE; ++n) {
            const int index = at + n * stride + (tid >> 2);
            if (quarter == 0 && index < pages) {
                const uint32_t s = (unsigned)page[n] < (unsigned)p.n_pages ? max(order_of(best[n]), 1u) : 0u;
                if (gridDim.z > 1) asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there + index * 4), "r"(s) : "memory");
                else score[index] = s;
            }
        }
        if (at + WIDE * stride < pages) load(at + WIDE * stride);
    }
    if (gridDim.z > 1) {
        __syncthreads();
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        if (blockIdx.z != 0) return;
    }
    __syncthreads();
    // Pages from `free_lo` to `free_hi` are chosen among; those before and behind them are taken always.
    const int free_lo = p.first, free_hi = own - p.last;
    int wanted = p.count - p.first - p.last;              // (pages > count: there are more than that)
    uint32_t prefix = 0xffffffffu, mask = 0;
    if (wanted > 0) {
        // the ends of the scores: above `shift` + 8 bits they do not differ
        uint32_t least = 0xffffffffu, most = 0;
        for (int i = free_lo + tid; i <= free_hi; i += PICK_THREADS) {
            least = min(least, score[i]);
            most = max(most, score[i]);
        }
        least = __reduce_min_sync(0xffffffffu, least);
        most = __reduce_max_sync(0xffffffffu, most);
        if (lane == 0) ends[0][warp] = least, ends[1][warp] = most;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PICK_THREADS / 32; ++i) {
            least = min(least, ends[0][i]);
            most = max(most, ends[1][i]);
        }
        const int differ = 32 - __clz(least ^ most);      // bits from the lowest on that are not all alike
        mask = differ >= 32 ? 0u : 0xffffffffu << differ;
        prefix = most & mask;
        for (int top = differ; top > 0;) {
            const int shift = max(top - 8, 0);
            const uint32_t bins = (1u << (top - shift)) - 1u;
            if (tid < 256) histogram[tid] = 0;
            __syncthreads();
            for (int i = free_lo + tid; i <= free_hi; i += PICK_THREADS)
                if ((score[i] & mask) == prefix) atomicAdd(&histogram[(score[i] >> shift) & bins], 1);
            __syncthreads();
            if (warp == 0) {
                // lane L sums the bins 8 L .. 8 L + 7; the wanted one is in the first lane from the top that reaches it
                int mine = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) mine += histogram[8 * lane + j];
                int above = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int v = __shfl_down_sync(0xffffffffu, above, o);
                    if (lane + o < 32) above += v;
                }
                above -= mine;                              // scores in higher lanes' bins
                if (above < wanted && above + mine >= wanted) {
                    int b = 7;
                    while (above + histogram[8 * lane + b] < wanted) above += histogram[8 * lane + b--];
                    found[0] = 8 * lane + b;
                    found[1] = wanted - above;
                    found[2] = histogram[8 * lane + b];
                }
            }
            __syncthreads();
            prefix |= (uint32_t)found[0] << shift;
            mask |= bins << shift;
            wanted = found[1];
            if (found[2] == wanted) break;                  // all of the bin: what its lower bits are does not matter
            top = shift;
            __syncthreads();
        }
    }
    // out in ascending order: larger ones, and the first `wanted` equal ones
    int done = 0, equal_done = 0;
    for (int at = 0; at < pages; at += PICK_THREADS) {
        const int i = at + tid;
        const uint32_t s = i < pages ? score[i] & mask : 0;
        const bool always = i < pages && (i < free_lo || i > free_hi);
        const bool equal = i < pages && !always && wanted > 0 && s == prefix;
        const bool larger = always || (i < pages && wanted > 0 && s > prefix);
        const uint32_t equals = __ballot_sync(0xffffffffu, equal), largers = __ballot_sync(0xffffffffu, larger);
        if (lane == 0) warp_counts[warp] = __popc(equals) | (__popc(largers) << 16);
        __syncthreads();
        int before = 0, total = 0;
#pragma unroll
        for (int w = 0; w < PICK_THREADS / 32; ++w) {
            if (w < warp) before += warp_counts[w];
            total += warp_counts[w];
        }
        const uint32_t below = (1u << lane) - 1u;
        const int equal_before = equal_done + (before & 0xffff) + __popc(equals & below);
        const int larger_before = (before >> 16) + __popc(largers & below);
        if (larger || (equal && equal_before < wanted))
            picks[done + larger_before + min(equal_before, wanted) - min(equal_done, wanted)] = i;
        done += (total >> 16) + min(equal_done + (total & 0xffff), wanted) - min(equal_done, wanted);
        equal_done += total & 0xffff;
        __syncthreads();
    }
}

template <int D, typename T>
int pick_launch(const PickParams& p, int shares, cudaStream_t stream) {
    const size_t bytes = (size_t)p.most_pages * 4 + (size_t)p.n_rep * (2 * D + 4);
    // (the limit is the most that any call takes, not this one's: another thread may be between its own and its launch)
    static bool ready[64] = {};          // per device; setting it twice does no harm
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        const int rc = (int)cudaFuncSetAttribute(pick4_kernel<D, T>, cudaFuncAttributeMaxDynamicSharedMemorySize, PICK_ROOM);
        if (rc != 0) return rc;
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    return cb_launch_cluster(pick4_kernel<D, T>, dim3((unsigned)p.rows * p.kv_heads, 1, shares), dim3(PICK_THREADS), bytes,
                             stream, shares, p);
}

}  // namespace

CB_EXPORT int cb_pick4_room() { return PICK_ROOM; }

CB_EXPORT int cb_pick4(const void* q, int dtype, long long q_stride, const int* positions, const int* row_request,
                       const int* table, int table_stride, int n_requests, const void* bounds, const float* bound_scales,
                       int n_pages, int page_tokens, int n_rep, int kv_heads, int head_dim, int rows, int* picks, int count,
                       int first, int last, int most_pages, int shares, void* stream) {
    if (rows <= 0) return 0;
    const int padded = (most_pages + 3) / 4 * 4;
    if ((long long)padded * 4 + (long long)n_rep * (2 * head_dim + 4) > PICK_ROOM || shares < 1 || shares > 8
        || (long long)rows * kv_heads >= (1LL << 31))
        return CB_ERR_UNSUPPORTED;
    const PickParams p = {q, q_stride, positions, row_request, table, table_stride, n_requests,
                          reinterpret_cast<const int8_t*>(bounds), bound_scales, n_pages, page_tokens, n_rep, kv_heads, rows,
                          picks, count, first, last, padded};
    const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    int rc = CB_ERR_UNSUPPORTED;
#define PICK(D)                                                                                                \
    if (head_dim == D) rc = dtype == CB_F32 ? pick_launch<D, float>(p, shares, s) : pick_launch<D, __nv_bfloat16>(p, shares, s);
    PICK(64) PICK(128) PICK(192) PICK(256)
#undef PICK
    if (rc == CB_ERR_UNSUPPORTED) return rc;
    const int last_rc = cb_last_error();
    return rc != 0 ? rc : last_rc;
}
