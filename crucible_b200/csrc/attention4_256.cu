// Attention over the cache in 4 bits, heads of 256 features: `attention4.cuh`.
#define CB_PDL_BIT 6      // with the other quantised operators
#include "attention4.cuh"

CB_EXPORT int cb_attention4(const void* q, int dtype, long long q_stride, void* out, long long out_stride, const void* codes,
                            const void* scales, int n_pages, int page_tokens, int kv_heads, int n_rep, int group,
                            const int* row_start, const int* first_pos, const int* table, int table_stride, int requests,
                            const int* picks, int pick_count, const int* row_request, const int* positions, int rows,
                            int most_rows, int window, float scale, int column_tiles, int shares, int stream_blocks,
                            float* partial, void* stream)
ATTENTION4_ENTRY(256)
