// What the tcgen05 products over quantised weights share: the e4m3 MMA, a row of codes made into
// weights, the way of a tile's sums out of tensor memory, and the tensor maps.
#pragma once
#include "quantized.cuh"
#include "tc_common.cuh"

// kind::f8f6f4 with e4m3 A and B (format 0), K-major, fp32 sums
__device__ __forceinline__ uint32_t instr_desc_e4m3(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// 64 codes of one feature (two runs of 32 k, a scale each) as bf16 weights in row `r` of a K-major tile of 128-byte
// rows in the 128-byte swizzle; the codes lie in chunks 2j and 2j + 1 of row `r` of such a tile of codes.
__device__ __forceinline__ void make_weights(const uint8_t* codes_row, int j, int r, uint32_t scale0, uint32_t scale1,
                                             uint8_t* weights_row) {
    const uint4 c0 = *reinterpret_cast<const uint4*>(codes_row + (((2 * j) ^ (r & 7)) << 4));
    const uint4 c1 = *reinterpret_cast<const uint4*>(codes_row + (((2 * j + 1) ^ (r & 7)) << 4));
    const uint32_t word[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    uint32_t s2[2], c2[2];
    scale_pairs(scale0, s2[0], c2[0]);
    scale_pairs(scale1, s2[1], c2[1]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
        uint32_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = weight_pair(word[c], i, s2[c >> 2], c2[c >> 2]);
        *reinterpret_cast<uint4*>(weights_row + ((c ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
    }
}

// Walks the group scales of one feature, 256 k at a time.
struct ScaleWalk {
    const uint8_t* scales;
    int sub, at, in;                    // runs of 32 k that share a scale; the present scale; runs it has had
    __device__ ScaleWalk(const QuantizedArgs& p, int n, int k)
        : scales(p.group_scale + (long long)min(n, p.N - 1) * (p.K / p.group)), sub(p.group / 32), at(k / p.group),
          in(k / 32 % (p.group / 32)) {}
    // (`k_end`: zeros from there on)
    __device__ __forceinline__ void next(uint8_t (&sc)[8], int k, int k_end) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            sc[i] = k + 32 * i < k_end ? __ldg(scales + at) : (uint8_t)0;
            if (++in == sub) in = 0, ++at;
        }
    }
};

// 32 rows' sums of feature n, rows m to m + 31 (those below m_end are stored): scales, addition, rounding, store.
// Neighbouring lanes hold neighbouring features, so a row's store is 64 or 128 neighbouring bytes a warp.  Loads go
// out together before anything is stored.  `add`: fp32 with `lda` between rows, or null; it may be the output.
template <int KIND, bool BF16>
__device__ __forceinline__ void store_rows(const QuantizedArgs& p, const float (&v)[32], float fs, int n, int m, int m_end,
                                           const float* add, long long lda) {
    const int lane = threadIdx.x & 31;
    float rs = 1.f;
    if (KIND == EIGHT) rs = __ldg(p.row_scale + min(m + lane, p.M - 1));
    const bool here = n < p.N;
    const bool whole = m + 32 <= m_end;                 // (the same for all threads)
    float a[32];
    if (add != nullptr) {
        const float* from = add + (long long)m * lda + n;
#pragma unroll
        for (int i = 0; i < 32; ++i) a[i] = here && (whole || m + i < m_end) ? __ldcg(from + (long long)i * lda) : 0.f;
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) a[i] = 0.f;
    }
    const long long at = (long long)m * p.ldo + n;
    float* f32 = static_cast<float*>(p.out) + at;
    __nv_bfloat16* bf16 = static_cast<__nv_bfloat16*>(p.out) + at;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
        float x = v[i] * fs;
        if (KIND == EIGHT) x *= __shfl_sync(0xffffffffu, rs, i);
        x += a[i];
        if (here && (whole || m + i < m_end)) {
            if (BF16) bf16[(long long)i * p.ldo] = __float2bfloat16_rn(x);
            else f32[(long long)i * p.ldo] = x;
        }
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

// Shared memory beyond the default, asked for once a kernel and device.
template <typename Kernel>
static inline int allow_shared(Kernel kernel, int bytes, bool (&configured)[64]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64 && configured[dev]) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 64) configured[dev] = true;
    return (int)e;
}
