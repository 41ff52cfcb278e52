// batch_args.h — what the entry points for a batch served together ask of their arguments: refusals, and the bytes that each buffer has to have.  No CUDA in it.
#pragma once

#include <cstddef>
#include <cstdint>

#include "../../include/yule_cuda.h"

namespace yule {

int32_t fail(int32_t code, const char *fmt, ...);

// Elements from the first of row 0 to the last of row `rows - 1`, rows `stride` apart and `length` long; none for no rows.  Saturates, so that no product
// of arguments comes out small.
inline size_t span(uint64_t rows, uint64_t stride, uint64_t length) {
    if (rows == 0 || length == 0) return 0;
    const unsigned __int128 n = (unsigned __int128)(rows - 1) * stride + length, most = SIZE_MAX / 16;
    return n > most ? (size_t)most : (size_t)n;
}
// For factors below 2^40.
inline uint64_t times(uint64_t a, uint64_t b) {
    const unsigned __int128 n = (unsigned __int128)a * b, most = UINT64_MAX / 16;
    return n > most ? (uint64_t)most : (uint64_t)n;
}

struct PrefixNeeds {
    size_t q, out, prefix, tail, lens;
};
inline int32_t check_prefix_attention(const yule_prefix_attention *shape, PrefixNeeds *need) {
    if (!shape) return fail(YULE_ERR_INVALID_ARGUMENT, "null shape");
    const yule_prefix_attention &s = *shape;
    if (s.n_kv_heads == 0 || s.n_kv_heads > 65535 || s.n_heads == 0 || s.n_heads % s.n_kv_heads || s.n_seqs == 0)
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad attention shape (heads %u, kv heads %u, sequences %u)", s.n_heads, s.n_kv_heads, s.n_seqs);
    if (s.head_dim == 0 || s.head_dim % 4 || s.head_dim > 256) return fail(YULE_ERR_INVALID_ARGUMENT, "head_dim %u must be a multiple of 4 and at most 256", s.head_dim);
    if (s.n_query == 0 || s.n_query > 64) return fail(YULE_ERR_INVALID_ARGUMENT, "%u query tokens per sequence: from 1 to 64", s.n_query);
    if (s.prefix_len > 0x7FFFFFFFu || times(s.n_seqs, s.tail_capacity) > 0x7FFFFFFFu)
        return fail(YULE_ERR_INVALID_ARGUMENT, "at most 2^31 - 1 positions of the prefix, and of all sequences' own caches together");
    const uint64_t heads = (uint64_t)s.n_heads * s.head_dim, kv = (uint64_t)s.n_kv_heads * s.head_dim, tokens = (uint64_t)s.n_seqs * s.n_query;
    if (s.q_stride < heads || s.out_stride < heads || (s.prefix_len && s.prefix_stride < kv) || (s.tail_capacity && s.tail_stride < kv) || s.q_stride % 4 || s.out_stride % 4 ||
        s.prefix_stride % 4 || s.tail_stride % 4)
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad strides (q %u, out %u, prefix %u, tail %u): multiples of 4, at least the heads of a token or position", s.q_stride, s.out_stride,
                    s.prefix_stride, s.tail_stride);
    if (times(tokens, s.n_heads) > 0x7FFFFFFFu) return fail(YULE_ERR_INVALID_ARGUMENT, "more than 2^31 - 1 query rows");
    need->q = 4 * span(tokens, s.q_stride, heads);
    need->out = 4 * span(tokens, s.out_stride, heads);
    need->prefix = 4 * span(s.prefix_len, s.prefix_stride, kv);
    need->tail = 4 * span(times(s.n_seqs, s.tail_capacity), s.tail_stride, kv);
    need->lens = s.tail_capacity ? (size_t)s.n_seqs * 4 : 0;
    return YULE_OK;
}

struct AdapterNeeds {
    size_t down, up, of_adapters, of_rows, input, output;
};
inline int32_t check_adapters(const yule_adapters *shape, AdapterNeeds *need) {
    if (!shape) return fail(YULE_ERR_INVALID_ARGUMENT, "null shape");
    const yule_adapters &s = *shape;
    if (s.gguf_type != YULE_DTYPE_F16 && s.gguf_type != YULE_DTYPE_F32) return fail(YULE_ERR_UNSUPPORTED_DTYPE, "unsupported dtype for adapters: GGUF type %u", s.gguf_type);
    if (s.n_adapters == 0 || s.max_rank == 0 || s.max_rank > 256)
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad adapters (%u of rank %u): at least one, of a rank from 1 to 256", s.n_adapters, s.max_rank);
    if (s.n_cols == 0 || s.n_cols % 4 || s.n_rows == 0 || s.n_rows > (1u << 23))
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad projection (%u rows, %u columns): rows from 1 to 2^23, columns a multiple of 4", s.n_rows, s.n_cols);
    if (s.batch == 0 || s.batch > 0x7FFFFFFFu || s.x_stride < s.n_cols || s.out_stride < s.n_rows || s.x_stride % 4)
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad batch/stride (batch %u, x_stride %u, out_stride %u)", s.batch, s.x_stride, s.out_stride);
    const size_t element = s.gguf_type == YULE_DTYPE_F16 ? 2 : 4;
    need->down = element * span(times(s.n_adapters, s.max_rank), s.n_cols, s.n_cols);
    need->up = element * span(times(s.n_adapters, s.n_rows), s.max_rank, s.max_rank);
    need->of_adapters = (size_t)s.n_adapters * 4;
    need->of_rows = (size_t)s.batch * 4;
    need->input = 4 * span(s.batch, s.x_stride, s.n_cols);
    need->output = 4 * span(s.batch, s.out_stride, s.n_rows);
    return YULE_OK;
}

struct VerifyNeeds {
    size_t target, draft, drafts, places, of_seqs;
};
inline int32_t check_verification(const yule_verification *shape, bool has_draft_logits, VerifyNeeds *need) {
    if (!shape) return fail(YULE_ERR_INVALID_ARGUMENT, "null shape");
    const yule_verification &s = *shape;
    if (s.vocab_size == 0 || s.vocab_size > (1u << 24)) return fail(YULE_ERR_INVALID_ARGUMENT, "vocabulary of %u tokens: from 1 to 2^24", s.vocab_size);
    if (s.n_seqs == 0 || s.n_seqs > 65536 || s.n_draft == 0 || s.n_draft > 256)
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad batch (%u sequences, %u drafts): 1 to 65536 of 1 to 256", s.n_seqs, s.n_draft);
    const bool by_model = has_draft_logits && !s.greedy;
    if (s.target_stride < s.vocab_size || (by_model && s.draft_stride < s.vocab_size))
        return fail(YULE_ERR_INVALID_ARGUMENT, "bad strides (target %u, draft %u): at least the vocabulary", s.target_stride, s.draft_stride);
    if (!s.greedy && !(s.temperature >= 1e-6f && s.temperature <= 1e6f))
        return fail(YULE_ERR_INVALID_ARGUMENT, "temperature %g: from 1e-6 to 1e6 (greedy is an argument of its own)", (double)s.temperature);
    const uint64_t places = (uint64_t)s.n_seqs * (s.n_draft + 1), drafts = (uint64_t)s.n_seqs * s.n_draft;
    need->target = 4 * span(places, s.target_stride, s.vocab_size);
    need->draft = by_model ? 4 * span(drafts, s.draft_stride, s.vocab_size) : 0;
    need->drafts = drafts * 4;
    need->places = places * 4;
    need->of_seqs = (size_t)s.n_seqs * 4;
    return YULE_OK;
}

}  // namespace yule
