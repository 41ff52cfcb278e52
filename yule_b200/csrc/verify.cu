// verify.cu — verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence b has k = min(draft_lens[b], n_draft) drafted tokens x_0 .. x_{k-1}; with p_t the soft-max of its target logits at place t (over the temperature) and q_t that of
// the draft model's (or, without draft logits, all of it on x_t), draft t is accepted while
//     u_t · q_t(x_t) < p_t(x_t).
// At the first that is not, place a, the token comes from w = max(0, p_a − q_a), after k accepted ones from w = p_k: the first i with Σ_{j <= i} w_j > u · Σ w, u the
// last of the sequence's random numbers.  So the tokens are distributed as the target alone would give them.
//
// A pick next to a border has to be the same however the sums are formed, so exponentials and sums are in 64 bits: in 32 the running sum over 128256
// tokens is off by 1e-7 where a token has 8e-6 on average, one pick in a hundred.
//
// Two kernels: largest logit and sum of exponentials of every row's chunks, a CTA each; then a cluster per sequence, which adds those up, compares, and sums w over a slice
// of the vocabulary in each of its CTAs, in tiles, of which the one that holds the pick is gone through once more.

#include <cfloat>

#include <cooperative_groups.h>

#include "internal.h"

namespace yule {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr uint32_t kNothing = 0xFFFFFFFFu;
constexpr uint32_t kCtas = 8;          // of a cluster
constexpr uint32_t kTile = 4 * kThreads;  // tokens of a tile of the second kernel

struct RowPart {
    double sum;   // of exp((logit − most) / temperature)
    float most;   // −infinity: no token is possible
    uint32_t at;  // the highest index of `most`
};
struct VerifyParams {
    const float *target, *draft;
    const uint32_t *drafts, *lens;
    const float *random;
    uint32_t *tokens, *accepted;
    RowPart *parts;  // [sequence][target rows, draft rows][chunk]
    uint32_t vocab, n_seqs, n_draft, chunks;
    size_t target_stride, draft_stride;
    double inv_t;
    bool greedy;
};

// A logit as it counts: NaN as −infinity, +infinity as the largest number.
__device__ __forceinline__ float logit(const float *at) {
    const float x = __ldg(at);
    return x != x ? -INFINITY : fminf(x, FLT_MAX);
}
__device__ __forceinline__ double weight(float x, float most, double inv_t) { return exp(((double)x - (double)most) * inv_t); }
__device__ __forceinline__ uint32_t rows_of(const VerifyParams &p) { return p.draft ? 2 * p.n_draft + 1 : p.n_draft + 1; }
__device__ __forceinline__ uint32_t drafted(const VerifyParams &p, uint32_t b) { return p.lens ? min(__ldg(p.lens + b), p.n_draft) : p.n_draft; }
__device__ __forceinline__ const float *target_row(const VerifyParams &p, uint32_t b, uint32_t t) { return p.target + ((size_t)b * (p.n_draft + 1) + t) * p.target_stride; }
__device__ __forceinline__ const float *draft_row(const VerifyParams &p, uint32_t b, uint32_t t) { return p.draft + ((size_t)b * p.n_draft + t) * p.draft_stride; }

// (most, at) of two: the larger, at equal size the higher index.
__device__ __forceinline__ void take_larger(float &most, uint32_t &at, float other, uint32_t other_at) {
    if (other > most || (other == most && other_at > at)) most = other, at = other_at;
}

template <int N>  // tokens per thread
__global__ void __launch_bounds__(kThreads) verify_rows_kernel(const __grid_constant__ VerifyParams p) {
    __shared__ float s_most[kThreads / 32];
    __shared__ uint32_t s_at[kThreads / 32];
    __shared__ double s_sum[kThreads / 32];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rows = rows_of(p), b = blockIdx.x / rows, r = blockIdx.x % rows, chunk = blockIdx.y, i0 = chunk * kThreads * N;
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    const uint32_t k = drafted(p, b);
    const bool of_target = r <= p.n_draft;
    const uint32_t t = of_target ? r : r - p.n_draft - 1;
    if (of_target ? t > k : t >= k) return;
    const float *row = of_target ? target_row(p, b, t) : draft_row(p, b, t);
    float x[N], most = -INFINITY;
    uint32_t at = 0;
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t j = i0 + i * kThreads + tid;
        x[i] = j < p.vocab ? logit(row + j) : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t j = i0 + i * kThreads + tid;
        if (j < p.vocab) take_larger(most, at, x[i], j);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) take_larger(most, at, __shfl_xor_sync(0xffffffffu, most, d), __shfl_xor_sync(0xffffffffu, at, d));
    if (lane == 0) s_most[warp] = most, s_at[warp] = at;
    __syncthreads();
    most = s_most[0], at = s_at[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; w++) take_larger(most, at, s_most[w], s_at[w]);
    double sum = 0.0;
    if (!p.greedy && most != -INFINITY) {
#pragma unroll
        for (int i = 0; i < N; i++) sum += weight(x[i], most, p.inv_t);
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) s_sum[warp] = sum;
        __syncthreads();
        sum = 0.0;
        for (int w = 0; w < kThreads / 32; w++) sum += s_sum[w];
    }
    if (tid == 0) p.parts[((size_t)b * rows + r) * p.chunks + chunk] = RowPart{sum, most, at};
}

// Sum over the CTA, the same in every thread and every call.
__device__ __forceinline__ double block_sum(double v, double *red) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0;
    for (int w = 0; w < kThreads / 32; w++) v += red[w];
    return v;
}

__global__ void __cluster_dims__(kCtas, 1, 1) __launch_bounds__(kThreads) verify_pick_kernel(const __grid_constant__ VerifyParams p) {
    extern __shared__ __align__(16) unsigned char sm[];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t rank = cluster.block_rank(), b = blockIdx.x / kCtas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rows = rows_of(p);
    RowPart *row = reinterpret_cast<RowPart *>(sm);                 // [rows]
    double *tile_sum = reinterpret_cast<double *>(row + rows);      // [tiles of a slice]
    __shared__ double red[kThreads / 32], s_slice;
    __shared__ uint32_t s_accepted, s_pick, s_last[kThreads / 32];
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    const uint32_t k = drafted(p, b);
    for (uint32_t r = warp; r < rows; r += kThreads / 32) {
        const uint32_t t = r <= p.n_draft ? r : r - p.n_draft - 1;
        if (r <= p.n_draft ? t > k : t >= k) continue;
        const RowPart *part = p.parts + ((size_t)b * rows + r) * p.chunks;
        float most = -INFINITY;
        uint32_t at = 0;
        for (uint32_t c = lane; c < p.chunks; c += 32) take_larger(most, at, __ldcg(&part[c].most), __ldcg(&part[c].at));
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) take_larger(most, at, __shfl_xor_sync(0xffffffffu, most, d), __shfl_xor_sync(0xffffffffu, at, d));
        double sum = 0.0;
        for (uint32_t c = lane; c < p.chunks; c += 32) {
            const float m = __ldcg(&part[c].most);
            if (m != -INFINITY) sum += __ldcg(&part[c].sum) * weight(m, most, p.inv_t);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) row[r] = RowPart{sum, most, at};
    }
    __syncthreads();
    // what is accepted: a lane per draft
    const uint32_t *drafts = p.drafts + (size_t)b * p.n_draft;
    if (warp == 0) {
        uint32_t accepted = 0;
        for (uint32_t t0 = 0; t0 < k; t0 += 32) {
            const uint32_t t = t0 + lane;
            bool fits = true;
            if (t < k) {
                const uint32_t x = __ldg(drafts + t);
                const RowPart pt = row[t];
                if (x >= p.vocab || pt.most == -INFINITY) {
                    fits = false;
                } else if (p.greedy) {
                    fits = pt.at == x;
                } else {
                    const double px = weight(logit(target_row(p, b, t) + x), pt.most, p.inv_t) / pt.sum;
                    double qx = 1.0;
                    if (p.draft) {
                        const RowPart qt = row[p.n_draft + 1 + t];
                        qx = qt.most == -INFINITY ? 0.0 : weight(logit(draft_row(p, b, t) + x), qt.most, p.inv_t) / qt.sum;
                    }
                    fits = (double)__ldg(p.random + (size_t)b * (p.n_draft + 1) + t) * qx < px;
                }
            }
            const uint32_t no = __ballot_sync(0xffffffffu, !fits);
            if (no) {
                accepted = t0 + __ffs(no) - 1;
                break;
            }
            accepted = min(k, t0 + 32);
        }
        if (lane == 0) s_accepted = accepted;
    }
    if (tid == 0) s_pick = kNothing;
    __syncthreads();
    const uint32_t a = s_accepted;
    const RowPart pa = row[a];
    uint32_t *out = p.tokens + (size_t)b * (p.n_draft + 1);
    auto finish = [&](uint32_t pick) {  // by all threads of one CTA
        for (uint32_t t = tid; t <= p.n_draft; t += kThreads) out[t] = t < a ? __ldg(drafts + t) : t == a ? pick : kNothing;
        if (tid == 0) p.accepted[b] = a;
    };
    if (p.greedy || pa.most == -INFINITY) {  // (the same for the whole cluster)
        if (rank == 0) finish(pa.most == -INFINITY ? kNothing : pa.at);
        return;
    }
    // w over this CTA's slice of the vocabulary, tile by tile
    const float *pr = target_row(p, b, a), *qr = p.draft && a < k ? draft_row(p, b, a) : nullptr;
    const RowPart qa = qr ? row[p.n_draft + 1 + a] : RowPart{1.0, -INFINITY, 0};
    const uint32_t without = !p.draft && a < k ? __ldg(drafts + a) : kNothing;
    const double inv_p = 1.0 / pa.sum, inv_q = 1.0 / qa.sum;
    auto w_of = [&](uint32_t i) {
        double w = weight(logit(pr + i), pa.most, p.inv_t) * inv_p;
        if (qr && qa.most != -INFINITY) w -= weight(logit(qr + i), qa.most, p.inv_t) * inv_q;
        return i == without || !(w > 0.0) ? 0.0 : w;
    };
    const uint32_t tiles = (p.vocab + kTile - 1) / kTile, per_cta = (tiles + kCtas - 1) / kCtas, tile0 = min(rank * per_cta, tiles), tile1 = min(tile0 + per_cta, tiles);
    double slice = 0.0;
    for (uint32_t j = tile0; j < tile1; j++) {
        double w = 0.0;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            const uint32_t i = j * kTile + e * kThreads + tid;
            if (i < p.vocab) w += w_of(i);
        }
        w = block_sum(w, red);
        if (tid == 0) tile_sum[j - tile0] = w;
        slice += w;
    }
    if (tid == 0) s_slice = slice;
    cluster.sync();
    double total = 0.0, before = 0.0, mine = 0.0;
    uint32_t owner = kCtas;
    const double u = (double)__ldg(p.random + (size_t)b * (p.n_draft + 1) + p.n_draft);
    double slices[kCtas];
    for (uint32_t c = 0; c < kCtas; c++) total += slices[c] = *cluster.map_shared_rank(&s_slice, c);
    const double goal = u * total;
    for (uint32_t c = 0; c < kCtas; c++) {  // the slice in which the running sum passes the goal, else the last that has anything
        if (!(slices[c] > 0.0)) continue;
        owner = c, before = mine;
        if (mine + slices[c] > goal) break;
        mine += slices[c];
    }
    cluster.sync();  // (nobody leaves while its sum is read)
    if (owner == kCtas) {
        if (rank == 0) finish(kNothing);
        return;
    }
    if (rank != owner) return;
    uint32_t at = tile0;
    double run = before;
    __syncthreads();
    for (uint32_t j = tile0; j < tile1; j++) {
        const double w = tile_sum[j - tile0];
        if (!(w > 0.0)) continue;
        at = j, before = run;
        if (run + w > goal) break;
        run += w;
    }
    // That tile again, four consecutive tokens a thread: the first whose running sum passes the goal, else the last that is possible.
    double w[4], own = 0.0;
    uint32_t last = kNothing;
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
        const uint32_t i = at * kTile + 4 * tid + e;
        w[e] = i < p.vocab ? w_of(i) : 0.0;
        own += w[e];
        if (w[e] > 0.0) last = i;
    }
    double scan = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= (uint32_t)d) scan += x;
    }
    __syncthreads();
    if (lane == 31) red[warp] = scan;
    uint32_t most = last == kNothing ? 0 : last + 1;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
    if (lane == 0) s_last[warp] = most;
    __syncthreads();
    double sum = before + (scan - own);
    for (uint32_t v = 0; v < warp; v++) sum += red[v];
    uint32_t pick = kNothing;
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
        sum += w[e];
        if (pick == kNothing && w[e] > 0.0 && sum > goal) pick = at * kTile + 4 * tid + e;
    }
    if (pick != kNothing) atomicMin(&s_pick, pick);
    __syncthreads();
    if (s_pick == kNothing) {
        pick = 0;
        for (int v = 0; v < kThreads / 32; v++) pick = max(pick, s_last[v]);
        finish(pick - 1);
    } else {
        finish(s_pick);
    }
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }
constexpr int kPerThread = 16;

}  // namespace

size_t verify_scratch_bytes(const VerifyDrafts &a) {
    return (size_t)a.n_seqs * (a.draft ? 2 * a.n_draft + 1 : a.n_draft + 1) * ceil_div(a.vocab, kThreads * kPerThread) * sizeof(RowPart);
}

cudaError_t launch_verify_drafts(const VerifyDrafts &a, cudaStream_t s, uint64_t *launches) {
    VerifyParams p = {};
    p.target = a.target, p.draft = a.draft, p.drafts = a.drafts, p.lens = a.lens, p.random = a.random, p.tokens = a.tokens, p.accepted = a.accepted;
    p.parts = static_cast<RowPart *>(a.scratch);
    p.vocab = a.vocab, p.n_seqs = a.n_seqs, p.n_draft = a.n_draft, p.chunks = ceil_div(a.vocab, kThreads * kPerThread);
    p.target_stride = a.target_stride, p.draft_stride = a.draft_stride, p.inv_t = 1.0 / (double)a.temperature, p.greedy = a.greedy;
    const uint32_t rows = a.draft ? 2 * a.n_draft + 1 : a.n_draft + 1;
    if ((uint64_t)rows * a.n_seqs > 0x7FFFFFFFu || (uint64_t)a.n_seqs * kCtas > 0x7FFFFFFFu || p.chunks > 65535) return cudaErrorInvalidValue;
    cudaError_t e = launch_kernel(verify_rows_kernel<kPerThread>, dim3(rows * a.n_seqs, p.chunks), dim3(kThreads), 0, s, a.pdl, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    const size_t smem = rows * sizeof(RowPart) + ceil_div(ceil_div(a.vocab, kTile), kCtas) * sizeof(double);
    e = launch_kernel(verify_pick_kernel, dim3(a.n_seqs * kCtas), dim3(kThreads), smem, s, true, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace yule
