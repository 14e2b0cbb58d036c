// What the tcgen05 products over quantised weights share: the e4m3 MMA, a row of codes made into
// weights, the way of a tile's sums out of tensor memory, and the tensor maps.
#pragma once
#include "quantized.cuh"
#include "tc_common.cuh"
#include <type_traits>

// kind::f8f6f4 with e4m3 A and B (format 0), K-major, fp32 sums
__device__ __forceinline__ uint32_t instr_desc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// 64 codes of one feature (two runs of 32 k, a scale each) as bf16 weights, two of neighbouring k a register; the codes
// lie in chunks 2j and 2j + 1 of row `r` of a tile of 128-byte rows in the 128-byte swizzle.
__device__ __forceinline__ void make_weights(const uint8_t* codes_row, int j, int r, uint32_t two_scales, uint32_t (&v)[32]) {
    const uint4 c0 = *reinterpret_cast<const uint4*>(codes_row + (((2 * j) ^ (r & 7)) << 4));
    const uint4 c1 = *reinterpret_cast<const uint4*>(codes_row + (((2 * j + 1) ^ (r & 7)) << 4));
    const uint32_t word[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    ScalePair s[2];
    scale_pairs(two_scales, s);
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * c + i] = weight_pair(word[c], i, s[c >> 2]);
}

// The group scales of one feature, 256 k (eight runs of 32) at a time, asked for a stage of codes ahead.  Where 256 k
// are whole groups and a feature's scales begin on a multiple of 8, 4 or 2 bytes, as those 256 k have, one load
// brings them (a load of a byte is 32 lines of memory for a warp, and eight of them for 256 k take the load unit
// as long as the MMAs take); else one of a byte each.
struct Scales {
    const uint8_t* from;
    int sub, lg;                        // runs of 32 k that share a scale, and its logarithm where they come together
    bool together;
    __device__ Scales(const QuantizedArgs& p, int n) : sub(p.group / 32) {
        const int groups = p.groups, per = 8 / sub;
        from = p.group_scale + (long long)min(n, p.N - 1) * groups;
        together = (sub == 1 || sub == 2 || sub == 4) && groups % per == 0 && ((uintptr_t)p.group_scale & (per - 1)) == 0;
        lg = together ? sub >> 1 : 0;
    }
    // The scales of 256 k from k (a multiple of 256; zeros from k_end on), as `of` reads them: nothing here waits for
    // the one load.  (k_end is a multiple of 256, or the whole K, which then is one: all of them are there.)
    __device__ __forceinline__ uint2 load(int k, int k_end) const {
        if (k >= k_end) return make_uint2(0u, 0u);
        if (together) {
            const uint8_t* at = from + (k >> 5 >> lg);
            if (lg == 0) return __ldg(reinterpret_cast<const uint2*>(at));
            if (lg == 1) return make_uint2(__ldg(reinterpret_cast<const uint32_t*>(at)), 0u);
            return make_uint2(__ldg(reinterpret_cast<const uint16_t*>(at)), 0u);
        }
        uint32_t w[2] = {0u, 0u};
        int at = k / 32 / sub, in = k / 32 % sub;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (k + 32 * i < k_end) w[i >> 2] |= (uint32_t)__ldg(from + at) << (8 * (i & 3));
            if (++in == sub) in = 0, ++at;
        }
        return make_uint2(w[0], w[1]);
    }
    // the scales of runs i and i + 1 (i even): the lower two bytes
    __device__ __forceinline__ uint32_t of(uint2 w, int i) const {
        const int b = i >> lg;
        const uint32_t x = (b < 4 ? w.x : w.y) >> (8 * (b & 3));
        return lg == 0 ? x : __byte_perm(x, 0, 0x0000);
    }
};

// 32 rows' sums of feature n, rows m to m + 31 (those below m_end are stored): scales, addition, rounding, store.
// Neighbouring lanes hold neighbouring features, so a row's store is 64 or 128 neighbouring bytes a warp.  Loads go
// out together before anything is stored.  `add`: fp32 with `lda` between rows, or null; it may be the output.
// (WHOLE: nothing to ask per row.  With a question a row, this took 24 instructions a number, which a lone
// warp issues one in five cycles.)
template <int KIND, bool BF16, bool ADD, bool WHOLE>
__device__ __forceinline__ void store_rows_as(const QuantizedArgs& p, const float (&v)[32], float fs, float rs, int n, int m,
                                              int m_end, const float* add, long long lda) {
    const bool here = WHOLE || n < p.N;
    using Out = typename std::conditional<BF16, __nv_bfloat16, float>::type;
    const float* from = ADD ? add + (long long)m * lda + n : nullptr;
    Out* to = static_cast<Out*>(p.out) + ((long long)m * p.ldo + n);
#pragma unroll
    for (int half = 0; half < 32; half += 16) {         // (16 loads on their way; 32 would cost other warps their registers)
        float a[16];
        if (ADD) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                a[i] = WHOLE || (here && m + half + i < m_end) ? __ldcg(from) : 0.f;
                from += lda;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            float x = v[half + i] * fs;
            if (KIND == EIGHT) x *= __shfl_sync(0xffffffffu, rs, half + i);
            if (ADD) x += a[i];
            if (WHOLE || (here && m + half + i < m_end)) *to = cb_from_float<Out>(x);
            to += p.ldo;
        }
    }
}

template <int KIND, bool BF16>
__device__ __forceinline__ void store_rows(const QuantizedArgs& p, const float (&v)[32], float fs, int n, int m, int m_end,
                                           const float* add, long long lda) {
    const int lane = threadIdx.x & 31;
    float rs = 1.f;
    if (KIND == EIGHT) rs = __ldg(p.row_scale + min(m + lane, p.M - 1));
    const bool whole = m + 32 <= m_end && n - lane + 32 <= p.N;
    if (add != nullptr) {
        if (whole) store_rows_as<KIND, BF16, true, true>(p, v, fs, rs, n, m, m_end, add, lda);
        else store_rows_as<KIND, BF16, true, false>(p, v, fs, rs, n, m, m_end, add, lda);
    } else {
        if (whole) store_rows_as<KIND, BF16, false, true>(p, v, fs, rs, n, m, m_end, add, lda);
        else store_rows_as<KIND, BF16, false, false>(p, v, fs, rs, n, m, m_end, add, lda);
    }
}

// A matrix read in boxes of 128 bytes by `box_rows` rows with the 128-byte swizzle; beyond it zeros.  `parts` > 1: so
// many matrices one behind the other, all of them in a box.
static inline bool quantized_map(CUtensorMap* map, const void* base, bool bf16, uint64_t rows, uint64_t cols,
                                 uint64_t row_bytes, uint32_t box_rows, uint32_t parts) {
    tc::EncodeTiledFn fn = tc::encode_fn();
    if (!fn) return false;
    cuuint64_t dims[3] = {cols, rows, parts};
    cuuint64_t strides[2] = {row_bytes, row_bytes * rows};
    cuuint32_t box[3] = {bf16 ? 64u : 128u, box_rows, parts};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8, parts > 1 ? 3 : 2,
              const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
