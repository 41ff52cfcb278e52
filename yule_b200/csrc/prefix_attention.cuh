// prefix_attention.cuh — what the kernels of the attention behind a shared prefix (prefix_attention.cu, prefix_attention_tc.cu) share.
#pragma once

#include "internal.h"

namespace yule {

struct PrefixParams {
    const float *q, *prefix_k, *prefix_v, *tail_k, *tail_v;
    const uint32_t *tail_lens;
    float *out;
    float2 *part_ml;  // [row][slot]: largest score (in units of ln 2), sum
    float *part_o;    // [row][slot][hd]
    uint32_t hd, n_heads, n_kv_heads, group, prefix_len, n_seqs, n_query, tail_capacity;
    uint32_t prefix_splits, prefix_chunk, prefix_row_tiles, tail_splits, tail_chunk, tail_row_tiles, slots, prefix_items;
    size_t q_stride, out_stride, prefix_stride, tail_stride;
    float scale;  // log2(e) / sqrt(hd)
    int *status;  // of bounded waits
    bool beside;  // prefix_part_kernel: the launch before is prefix_tc_kernel
    bool single;  // prefix_part_kernel: a sequence's whole attention in one CTA, which leaves the output
    bool alone;   // prefix_merge_kernel: there is no launch before it
    bool behind;  // prefix_operands_kernel: the launch before is prefix_part_kernel
};

// The prefix for 128 query rows at a time on tcgen05 (prefix_attention_tc.cu): leaves the parts of slots [0, prefix_splits).  prefix_chunk is a multiple of 64, of at most 512 tiles of
// 64; head_dim 64 or 128; `scratch` on a 128-byte boundary.
constexpr uint32_t kPrefixTcRows = 128, kPrefixTcKeys = 64, kPrefixTcTiles = 512;
bool prefix_tc_supported(uint32_t hd, uint64_t rows);  // rows: query rows of a KV head, as many as a grid takes
size_t prefix_tc_scratch_bytes(const PrefixParams &p);
cudaError_t launch_prefix_tc(const PrefixParams &p, void *scratch, bool pdl, cudaStream_t s, uint64_t *launches);

}  // namespace yule
