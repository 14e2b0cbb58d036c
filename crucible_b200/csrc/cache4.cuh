// The key/value cache in 4 bits: how a row lies in memory, and what every kernel over it shares.
//
// A row (one token's key or value of one head, D features, D a multiple of 64 up to 256) is D/2 bytes of
// codes 0..15 and, for every `group` features, a pair of bfloat16 (step, low); feature f stands for
// code * step + low.  Codes lie in int32 words: word (D/64) g + w, 0 <= g < 8, holds the features
// 64 w + 8 k + g, k = 0..7, four bits each, the k of bits 4n..4n+3 being (0, 1, 4, 5, 2, 3, 6, 7)[n].  So
//   - one lane's share of an m16n8k16 tile over 16 features is a run of bits of one word whichever way the
//     tile is turned: as rows of keys (features are multiplied over: lane t of four takes the words of
//     g = 2t, 2t+1) and as columns of values (keys are multiplied over: lane g of eight takes the words of g);
//   - the four codes of a half word are k and k+1 of two 16-feature tiles, and those that a mask takes out of
//     both halves at once lie in one group of 32, so that groups of 32, 64 and 128 all end with a tile.
// Pages: codes [2][pages][kv heads][page tokens][D/2], scales [2][pages][kv heads][page tokens][D/group] words
// (step in the low half), keys first.
#pragma once
#include "common.cuh"

#include <cuda_fp16.h>

// The numbers that are coded are float32, and every operation up to the code is rounded once (no contraction):
// a code is defined to the last bit.
constexpr float C4_LEAST_STEP = 1e-30f;      // a smaller step is none: its reciprocal would leave float32

__device__ __forceinline__ float c4_step(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float c4_low(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// The bits at which feature k (of eight, 8 features apart) lies in its word.
__device__ __forceinline__ int c4_shift(int k) { return 4 * ((k & 1) | ((k & 4) >> 1) | ((k & 2) << 1)); }

// Where a token lies: the number of its row among [pages][kv heads][page tokens] for head 0, or -1 where the
// table names no page of the pool.  (A page the window has passed may be negative or a page of zeros.)
__device__ __forceinline__ long long c4_row(const int* table, int table_stride, int page_tokens, int n_pages, int kv_heads,
                                            int pos) {
    const int index = pos / page_tokens;
    if (pos < 0 || index >= table_stride) return -1;
    const int page = table[index];
    if (page < 0 || page >= n_pages) return -1;
    return (long long)page * kv_heads * page_tokens + (pos - index * page_tokens);
}
