// Launchers shared between the attention translation units of libshellcache.
#pragma once
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace sc {

// Merges `rows` rows of `nparts` (out, lse) partials (paged_attention.cu): part s
// of row r has its D values at po[r * o_row + s * o_part + d] and its lse at
// pl[r * l_row + s * l_part]; with ctx_len set only the splits a decode wrote
// are read. Writes bf16 out (+ lse_out) or, with `packed`, fp32 [r][D + 1].
void launch_combine(const float* po, const float* pl, size_t o_row, size_t o_part, size_t l_row,
                    size_t l_part, const int32_t* ctx_len, int Hq, int nparts,
                    int pages_per_split, int D, int rows, uint16_t* out, float* lse_out,
                    float* packed, cudaStream_t s);

// Split-K decode attention over each sequence's pages from f = min(first_page[b],
// ctx / 16) on (D in {64, 128, 256}), partials only: part_out [B, Hq, num_splits, D] and
// part_lse [B, Hq, num_splits] for the splits of ceil(ctx / 16) - f pages. It does
// not wait for the kernel queued before it, except to end after it: that kernel must
// have waited for its own predecessor and must write nothing that this one reads.
int launch_decode_tail(const uint16_t* q, const uint16_t* kv_pool, long long num_pages,
                       const int32_t* block_table, const int32_t* ctx_len,
                       const int32_t* seq_order, const int32_t* first_page, int B, int Hq, int Hkv,
                       int D, int max_pages, int pages_per_split, int num_splits, float scale,
                       float* part_out, float* part_lse, cudaStream_t s);

}  // namespace sc
