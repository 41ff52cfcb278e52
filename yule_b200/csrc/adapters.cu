// adapters.cu — low-rank adapters of many requests beside a shared projection.
//
// Row i of the batch has adapter a = row_adapter[i] (none if a >= n_adapters: its output is its base), of rank r = min(ranks[a], max_rank):
//     v_k = Σ_c down[a][k][c] · x[i][c]   (k < r),      out[i][o] = base[i][o] + scales[a] · Σ_k up[a][o][k] · v_k.
// Rows come in tiles; a tile's adapters are its slots, in the order of their first rows.  A slot's rows are the columns of the tensor core's second operand,
// so an adapter is read once per tile whatever the order of the requests.  F16 adapters are tf32 numbers as they are: two products per element (with hi and lo of
// x or v), three for F32 ones.  Sums are added in a fixed order.
//
// Decode steps (tiles of 8): one launch, a cluster of CTAs per slot.  What there is to read is an adapter's 0.1 to 2 MB, so time goes by in latency: a CTA takes
// a share of the columns for all ranks, writes its sums into every other CTA's shared memory, and has its share of the outputs, whose first rows of `up` and of
// base it loads before the barrier.  32 requests of as many adapters of rank 16 beside 4096 × 4096: 7.4 us a call (two launches, with the sums through the scratch:
// 12.2; 8.4 MB at the rate of a copy: 1.3), one token beside 2048 × 2048: 5.8 (7.5), of which the call itself is the most.
//
// Prompts (tiles of 32): two launches, since base and output are most of the traffic and want CTAs of their own.  1501 rows of six requests, rank 64, beside 14336 × 4096:
// 71 us, the first launch 22 of them, the second 51 for 195 MB; both are bound by the instructions around the copies and products, not by memory
// (31 us) or by the tensor core (16).

#include <cuda_fp16.h>

#include <utility>

#include <cooperative_groups.h>

#include "internal.h"
#include "tf32_common.cuh"

namespace yule {

namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 8, kThreads = kWarps * 32;
constexpr uint32_t kStepRows = 8, kTileRows = 32, kPassOuts = kWarps * 32;

struct AdapterParams {
    const void *down, *up;
    const uint32_t *ranks, *row_adapter;
    const float *scales, *x, *base;
    float *out, *sums, *row_scales;  // prompts: sums [row][rank_pitch], scales of rows of halves
    uint32_t n_adapters, max_rank, n_rows, n_cols, batch, cols_per_cta, outs_per_cta, rank_pitch;
    size_t x_stride, out_stride;
    bool whole_ranks, whole_outs;  // rows of `up`, and of out and base, are on the boundaries of vectors of four
};

// (Not by the read-only path: a launch before this one, which this one may have started beside, can have written any input.)
template <typename T>
__device__ __forceinline__ T read(const T *at) {
    return *at;
}

// A tile's rows by adapter: a lane per row, each warp for itself.
struct Tile {
    uint32_t id, same, firsts;  // this row's adapter (~0: none), the rows that share it, the first row of each adapter
};
template <uint32_t ROWS>
__device__ __forceinline__ Tile read_tile(const AdapterParams &p, uint32_t row0) {
    const uint32_t lane = threadIdx.x & 31, row = row0 + lane;
    Tile t;
    t.id = lane < ROWS && row < p.batch ? read(p.row_adapter + row) : ~0u;
    if (t.id >= p.n_adapters) t.id = ~0u;
    t.same = __match_any_sync(0xffffffffu, t.id);
    t.firsts = __ballot_sync(0xffffffffu, t.id != ~0u && (uint32_t)__ffs(t.same) == lane + 1);
    return t;
}
// Adapter and rows of a slot, the rows in `list`, one of the warp's own.
struct Slot {
    uint32_t adapter, n;
};
__device__ __forceinline__ Slot read_slot(const Tile &t, uint32_t slot, uint8_t *list) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t f = t.firsts;
    for (uint32_t i = 0; i < slot; i++) f &= f - 1;
    const int first = __ffs(f) - 1;
    const uint32_t mask = __shfl_sync(0xffffffffu, t.same, first);
    __syncwarp();
    if (mask >> lane & 1u) list[__popc(mask & ((1u << lane) - 1))] = (uint8_t)lane;
    __syncwarp();
    return {__shfl_sync(0xffffffffu, t.id, first), (uint32_t)__popc(mask)};
}
// Rows without an adapter: their base, outputs [o0, o1), four of a thread's pieces under way together.
template <uint32_t ROWS>
__device__ __forceinline__ void copy_base(const AdapterParams &p, const Tile &t, uint32_t row0, uint32_t o0, uint32_t o1, uint8_t *list) {
    const uint32_t lane = threadIdx.x & 31, mask = __ballot_sync(0xffffffffu, t.id == ~0u && lane < ROWS && row0 + lane < p.batch);
    if (p.base == p.out || mask == 0 || o0 >= o1) return;
    if (mask >> lane & 1u) list[__popc(mask & ((1u << lane) - 1))] = (uint8_t)lane;
    __syncwarp();
    auto copy = [&](auto one, uint32_t width) {
        using V = decltype(one);
        const uint32_t per_row = (o1 - o0) / width, n = __popc(mask) * per_row;
        for (uint32_t i = threadIdx.x; i < n; i += 4 * kThreads) {
            V v[4];
            size_t at[4];
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                const uint32_t e = min(i + j * kThreads, n - 1);
                at[j] = (size_t)(row0 + list[e / per_row]) * p.out_stride + o0 + e % per_row * width;
                v[j] = *reinterpret_cast<const V *>(p.base + at[j]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (i + j * kThreads < n) *reinterpret_cast<V *>(p.out + at[j]) = v[j];
        }
    };
    if (p.whole_outs) copy(float4(), 4);
    else copy(float(), 1);
}

// Four elements of an adapter's row from `at` on, of which `n` are there, as they lie and as fp32.
template <typename T>
struct Four;
template <>
struct Four<float> {
    float4 v;
    __device__ __forceinline__ void load(const float *at, int n, bool whole) {
        if (whole && n >= 4) v = read(reinterpret_cast<const float4 *>(at));
        else v = make_float4(n > 0 ? read(at) : 0.f, n > 1 ? read(at + 1) : 0.f, n > 2 ? read(at + 2) : 0.f, n > 3 ? read(at + 3) : 0.f);
    }
    __device__ __forceinline__ float4 get() const { return v; }
};
template <>
struct Four<__half> {
    uint2 v;
    __device__ __forceinline__ void load(const __half *at, int n, bool whole) {
        if (whole && n >= 4) v = read(reinterpret_cast<const uint2 *>(at));
        else {
            const unsigned short *bits = reinterpret_cast<const unsigned short *>(at);
            auto one = [&](int i) -> uint32_t { return n > i ? read(bits + i) : 0u; };
            v = make_uint2(one(0) | one(1) << 16, one(2) | one(3) << 16);
        }
    }
    __device__ __forceinline__ float4 get() const {
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
};

// d += a · b over two steps of eight: this lane's four elements of the operands' rows g (a) and g + 8 (b), and of the second operand's column g.
template <bool EXACT>  // a and b are tf32 numbers
__device__ __forceinline__ void multiply(float (&d)[4], const float4 &a, const float4 &b, const uint4 &hi, const uint4 &lo) {
    uint32_t ah[4] = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(a.z), __float_as_uint(a.w)};
    uint32_t bh[4] = {__float_as_uint(b.x), __float_as_uint(b.y), __float_as_uint(b.z), __float_as_uint(b.w)};
    // (the tensor core truncates what it adds to: the small products have a sum of their own, so that the large ones are cut off twice a step and not six times: error against
    // 64 bits 1.0e-7 to 5.6e-7, 0.7e-7 to 3.2e-7 so)
    float small[4] = {0.f, 0.f, 0.f, 0.f};
    if (!EXACT) {
        uint32_t al[4], bl[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(ah[i]), ah[i], al[i]), split_tf32(__uint_as_float(bh[i]), bh[i], bl[i]);
        mma_tf32(small, al[0], bl[0], al[1], bl[1], hi.x, hi.y);
        mma_tf32(small, al[2], bl[2], al[3], bl[3], hi.z, hi.w);
    }
    mma_tf32(small, ah[0], bh[0], ah[1], bh[1], lo.x, lo.y);
    mma_tf32(small, ah[2], bh[2], ah[3], bh[3], lo.z, lo.w);
    mma_tf32(d, ah[0], bh[0], ah[1], bh[1], hi.x, hi.y);
    mma_tf32(d, ah[2], bh[2], ah[3], bh[3], hi.z, hi.w);
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] += small[i];
}
__device__ __forceinline__ void split4(const float4 &v, uint4 &hi, uint4 &lo) {
    split_tf32(v.x, hi.x, lo.x), split_tf32(v.y, hi.y, lo.y), split_tf32(v.z, hi.z, lo.z), split_tf32(v.w, hi.w, lo.w);
}

__device__ __forceinline__ void store4(const AdapterParams &p, size_t at, uint32_t o, const float4 &b, const float (&d)[4], float scale) {
    const float4 v = make_float4(fmaf(scale, d[0], b.x), fmaf(scale, d[1], b.y), fmaf(scale, d[2], b.z), fmaf(scale, d[3], b.w));
    float *to = p.out + at + o;
    if (p.whole_outs) {
        if (o < p.n_rows) *reinterpret_cast<float4 *>(to) = v;
    } else {
        if (o < p.n_rows) to[0] = v.x;
        if (o + 1 < p.n_rows) to[1] = v.y;
        if (o + 2 < p.n_rows) to[2] = v.z;
        if (o + 3 < p.n_rows) to[3] = v.w;
    }
}
__device__ __forceinline__ float4 load4(const AdapterParams &p, size_t at, uint32_t o, bool there) {  // (not by the read-only path: it can be the output)
    const float *from = p.base + at + o;
    if (p.whole_outs) return there && o < p.n_rows ? *reinterpret_cast<const float4 *>(from) : make_float4(0.f, 0.f, 0.f, 0.f);
    return make_float4(there && o < p.n_rows ? from[0] : 0.f, there && o + 1 < p.n_rows ? from[1] : 0.f, there && o + 2 < p.n_rows ? from[2] : 0.f, there && o + 3 < p.n_rows ? from[3] : 0.f);
}
// Rows o .. o + 3 of `up`, this lane's elements of step j: what the lane has of the first operand, in an order that gives it four consecutive outputs.
template <typename T>
__device__ __forceinline__ void load_up(const AdapterParams &p, const T *up, uint32_t o, uint32_t j, uint32_t rank, Four<T> (&u)[4]) {
    const uint32_t k = 16 * j + 4 * (threadIdx.x & 3);
#pragma unroll
    for (int i = 0; i < 4; i++) u[i].load(up + (size_t)(o + i) * p.max_rank + k, o + i < p.n_rows ? (int)rank - (int)k : 0, p.whole_ranks);
}
// The terms of v lie in rows of so many words: eight lanes of a 16-byte load are in different banks.
__host__ __device__ __forceinline__ uint32_t v_pitch(uint32_t max_rank) { return (max_rank + 31) / 32 * 32 + 16; }

// A decode step's slot: grid x = the cluster, y = slots, z = tiles.
template <typename T, int RANKS>
__global__ void __launch_bounds__(kThreads, 2) adapter_step_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ __align__(16) float got[];  // sums of v: [CTA][row][rank_pitch], then v's terms: hi, lo: [row][pitch]
    __shared__ float meet[kWarps][kStepRows][RANKS * 16 + 1];
    __shared__ uint8_t lists[kWarps][32], none_lists[kWarps][32];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t ctas = gridDim.x, cta = blockIdx.x, row0 = blockIdx.z * kStepRows, slot_at = blockIdx.y;
    const uint32_t out0 = cta * p.outs_per_cta, out1 = min(out0 + p.outs_per_cta, p.n_rows);
    auto started = cluster.barrier_arrive();  // (waited for before anything is written to another CTA)
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    const uint32_t near_rank = lane < p.n_adapters ? read(p.ranks + lane) : 0u;  // (beside the rows' adapters, not behind them)
    const Tile tile = read_tile<kStepRows>(p, row0);
    if (slot_at >= __popc(tile.firsts)) {  // (the same for all the cluster)
        if (slot_at == 0) copy_base<kStepRows>(p, tile, row0, out0, out1, none_lists[warp]);
        cluster.barrier_wait(std::move(started));
        return;
    }
    const uint8_t *rows = lists[warp];
    const Slot slot = read_slot(tile, slot_at, lists[warp]);
    const uint32_t near = __shfl_sync(0xffffffffu, near_rank, slot.adapter & 31), rank = min(slot.adapter < 32 ? near : read(p.ranks + slot.adapter), p.max_rank);
    const float scale = read(p.scales + slot.adapter);
    const T *down = static_cast<const T *>(p.down) + (size_t)slot.adapter * p.max_rank * p.n_cols, *up = static_cast<const T *>(p.up) + (size_t)slot.adapter * p.n_rows * p.max_rank;
    const uint32_t share = p.cols_per_cta / kWarps, col0 = (cta * kWarps + warp) * share, col1 = min(col0 + share, p.n_cols);
    const float *x = p.x + (size_t)(row0 + rows[g < slot.n ? g : 0]) * p.x_stride;
    bool first = true;
    for (uint32_t k0 = 0; k0 < rank; k0 += RANKS * 16) {
        constexpr int kSteps = RANKS == 4 && sizeof(T) == 4 ? 2 : 4;  // steps whose loads are under way together
        float sum[RANKS][4] = {};
        for (uint32_t base = col0; base < col1; base += 16 * kSteps) {
            float4 xv[kSteps];
            Four<T> w[kSteps][RANKS][2];
#pragma unroll
            for (int j = 0; j < kSteps; j++) {
                const uint32_t c = base + 16 * j + 4 * t;
                const bool in = c < col1;
                xv[j] = in && g < slot.n ? read(reinterpret_cast<const float4 *>(x + c)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int r = 0; r < RANKS; r++) {
                    const uint32_t k = k0 + 16 * r + g;
                    w[j][r][0].load(down + (size_t)k * p.n_cols + c, in && k < rank ? 4 : 0, true);
                    w[j][r][1].load(down + (size_t)(k + 8) * p.n_cols + c, in && k + 8 < rank ? 4 : 0, true);
                }
            }
            // (the tensor core truncates what it adds to: sums of 32 or 64 columns, added up in fp32)
            float d[RANKS][4] = {};
#pragma unroll
            for (int j = 0; j < kSteps; j++) {
                uint4 hi, lo;
                split4(xv[j], hi, lo);
#pragma unroll
                for (int r = 0; r < RANKS; r++) multiply<sizeof(T) == 2>(d[r], w[j][r][0].get(), w[j][r][1].get(), hi, lo);
            }
#pragma unroll
            for (int r = 0; r < RANKS; r++)
#pragma unroll
                for (int e = 0; e < 4; e++) sum[r][e] += d[r][e];
        }
        if (k0) __syncthreads();
#pragma unroll
        for (int r = 0; r < RANKS; r++)
#pragma unroll
            for (int e = 0; e < 4; e++) meet[warp][2 * t + (e & 1)][16 * r + g + 8 * (e >> 1)] = sum[r][e];
        __syncthreads();
        if (first) cluster.barrier_wait(std::move(started));
        first = false;
        for (uint32_t i = threadIdx.x; i < slot.n * RANKS * 16 * 4; i += kThreads) {  // four threads per sum, each for a fourth of the CTAs
            const uint32_t row = i / (RANKS * 64), k = i / 4 % (RANKS * 16);
            if (k0 + k >= rank) continue;
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; w++) v += meet[w][row][k];
            for (uint32_t c = i & 3u; c < ctas; c += 4) cluster.map_shared_rank(got, c)[(cta * kStepRows + row) * p.rank_pitch + k0 + k] = v;
        }
    }
    if (first) cluster.barrier_wait(std::move(started));
    auto summed = cluster.barrier_arrive();
    const uint32_t steps = (rank + 15) / 16;
    uint32_t o = out0 + warp * 32 + 4 * g;
    const bool mine[2] = {2 * t < slot.n, 2 * t + 1 < slot.n};
    size_t at[2];
    float4 b[2];
    Four<T> u[4];
    const uint32_t end = out0 + p.outs_per_cta;
#pragma unroll
    for (int c = 0; c < 2; c++) at[c] = (size_t)(row0 + rows[mine[c] ? 2 * t + c : 0]) * p.out_stride, b[c] = load4(p, at[c], o, mine[c] && o < end);
    load_up(p, up, o, 0, o < end ? rank : 0, u);
    if (slot_at == 0) copy_base<kStepRows>(p, tile, row0, out0, out1, none_lists[warp]);
    cluster.barrier_wait(std::move(summed));
    const uint32_t pitch = v_pitch(p.max_rank);
    uint32_t *v_hi = reinterpret_cast<uint32_t *>(got + ctas * kStepRows * p.rank_pitch), *v_lo = v_hi + kStepRows * pitch;
    for (uint32_t i = threadIdx.x; i < slot.n * steps * 16; i += kThreads) {
        const uint32_t r = i / (steps * 16), k = i % (steps * 16);
        float v = 0.f;
        if (k < rank)
            for (uint32_t c = 0; c < ctas; c++) v += got[(c * kStepRows + r) * p.rank_pitch + k];
        split_tf32(v, v_hi[r * pitch + k], v_lo[r * pitch + k]);
    }
    __syncthreads();
    for (; o < end; o += kPassOuts) {
        const uint32_t next = o + kPassOuts;
        float4 bn[2];
#pragma unroll
        for (int c = 0; c < 2; c++) bn[c] = load4(p, at[c], next, mine[c] && next < end);
        float d[2][4] = {};
        for (uint32_t j = 0; j < steps; j++) {
            Four<T> un[4];
            const bool last = j + 1 == steps;
            load_up(p, up, last ? next : o, last ? 0 : j + 1, last && next >= end ? 0 : rank, un);
            uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
            if (g < slot.n) hi = *reinterpret_cast<const uint4 *>(v_hi + g * pitch + 16 * j + 4 * t), lo = *reinterpret_cast<const uint4 *>(v_lo + g * pitch + 16 * j + 4 * t);
            multiply<sizeof(T) == 2>(d[0], u[0].get(), u[1].get(), hi, lo);
            multiply<sizeof(T) == 2>(d[1], u[2].get(), u[3].get(), hi, lo);
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = un[i];
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const float four_of[4] = {d[0][c], d[0][2 + c], d[1][c], d[1][2 + c]};
            if (mine[c]) store4(p, at[c], o, b[c], four_of, scale);
            b[c] = bn[c];
        }
    }
}

// ── prompts ─────────────────────────────────────────────────────────────────────────────────────
// cp.async of W bytes, zeros where there is nothing.
template <int W>
__device__ __forceinline__ void copy_async(uint32_t to, const void *from, bool there) {
    const int bytes = there ? W : 0;
    if (W == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else if (W == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(bytes) : "memory");
}

template <typename T>
struct DownLayout {
    static constexpr uint32_t kCols = 64, kRanks = 64, kStages = 3;
    static constexpr uint32_t kXPitch = (kCols + 16) * 4, kDPitch = (kCols + 16) * sizeof(T);  // bytes: 16- or 8-byte loads of eight rows in different banks
    static constexpr uint32_t kX = kTileRows * kXPitch, kStage = kX + kRanks * kDPitch;
    static constexpr uint32_t kMeet = 4 * kTileRows * (kRanks + 1) * 4, kSum = kTileRows * kRanks * 4;
    static constexpr uint32_t kRing = kStages * kStage, kBytes = (kRing > kMeet ? kRing : kMeet) + kSum;
};

// F16 adapters of ranks to 64 in the second launch: a row of v as fp16 terms, v · 2^e = hi + lo up to 2^-22 of v, with its largest number in [2^14, 2^15): products of fp16 numbers at
// twice the rate of tf32 ones (62 -> 58 us for 1501 rows beside 14336).  Numbers below 2^-16 of the row's largest would lose bits of lo: a row that has such (but not zero), or one that is not finite,
// stays as it is, with 0 as its scale.  `v`: this lane's four numbers of the row that kLanes lanes have; comes back as four hi and four lo, the inverse of 2^e in `scale`.
template <uint32_t LANES>
__device__ __forceinline__ float4 halves_of_row(const float4 &v, float *scale) {
    const float all[4] = {fabsf(v.x), fabsf(v.y), fabsf(v.z), fabsf(v.w)};
    uint32_t most = 0, least = ~0u;  // (of numbers >= 0, as their bits are ordered; NaN is above infinity)
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t bits = __float_as_uint(all[i]);
        most = max(most, bits);
        if (bits) least = min(least, bits);
    }
#pragma unroll
    for (uint32_t m = LANES / 2; m; m /= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, m)), least = min(least, __shfl_xor_sync(0xffffffffu, least, m));
    const bool keep = most >= 0x7F800000u || (most && __uint_as_float(least) < __uint_as_float(most) * 0x1p-16f);
    const int e = max(-113, min(126, 14 - ((int)(most >> 23) - 127)));
    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
    if (scale) *scale = keep ? 0.f : __uint_as_float((uint32_t)(127 - e) << 23);
    if (keep) return v;
    auto terms = [&](float a, float b, uint32_t &hi, uint32_t &lo) {
        const __half2 h = __floats2half2_rn(a * up, b * up);
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(a * up - f.x, b * up - f.y);
        hi = *reinterpret_cast<const uint32_t *>(&h), lo = *reinterpret_cast<const uint32_t *>(&l);
    };
    uint32_t hi[2], lo[2];
    terms(v.x, v.y, hi[0], lo[0]), terms(v.z, v.w, hi[1], lo[1]);
    return make_float4(__uint_as_float(hi[0]), __uint_as_float(hi[1]), __uint_as_float(lo[0]), __uint_as_float(lo[1]));
}
__device__ __forceinline__ float4 row_of_halves(const float4 &v, float scale) {  // and back
    auto two = [&](float hi, float lo) {
        const uint32_t h = __float_as_uint(hi), l = __float_as_uint(lo);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&h)), b = __half22float2(*reinterpret_cast<const __half2 *>(&l));
        return make_float2((a.x + b.x) * scale, (a.y + b.y) * scale);
    };
    const float2 a = two(v.x, v.z), b = two(v.y, v.w);
    return make_float4(a.x, a.y, b.x, b.y);
}
// d += a · b over one step of sixteen, as for tf32: this lane's four elements of rows g (a) and g + 8 (b), and of the second operand's column g.
__device__ __forceinline__ void multiply_f16(float (&d)[4], const uint2 &a, const uint2 &b, float v0, float v1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(b.x), "r"(a.y), "r"(b.y), "r"(__float_as_uint(v0)), "r"(__float_as_uint(v1)));
}

// v of a tile's slots, 64 ranks at a time: grid x = tiles × the cluster (a share of the columns per CTA), y = slots.  A warp has 32 ranks and 16 of each 64 columns.
template <typename T, int W>
__global__ void __launch_bounds__(kThreads, 2) adapter_down_kernel(const __grid_constant__ AdapterParams p) {
    using L = DownLayout<T>;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ uint8_t lists[kWarps][32];
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, part = warp & 3, half = warp >> 2;
    const uint32_t ctas = cluster.num_blocks(), cta = cluster.block_rank(), row0 = blockIdx.x / ctas * kTileRows;
    float *meet = reinterpret_cast<float *>(ring), *mine = reinterpret_cast<float *>(ring + L::kBytes - L::kSum);
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    const Tile tile = read_tile<kTileRows>(p, row0);
    const uint32_t n_slots = __popc(tile.firsts), col0 = cta * p.cols_per_cta, col1 = min(col0 + p.cols_per_cta, p.n_cols), to = (uint32_t)__cvta_generic_to_shared(ring);
    const uint32_t n_stages = col0 < col1 ? (col1 - col0 + L::kCols - 1) / L::kCols : 0;
    const uint8_t *rows = lists[warp];
    for (uint32_t s = blockIdx.y; s < n_slots; s += gridDim.y) {
        const Slot slot = read_slot(tile, s, lists[warp]);
        const uint32_t rank = min(read(p.ranks + slot.adapter), p.max_rank);
        const T *down = static_cast<const T *>(p.down) + (size_t)slot.adapter * p.max_rank * p.n_cols;
        constexpr uint32_t kPerRow = L::kCols * sizeof(T) / W, kCopies = L::kRanks * kPerRow / kThreads;  // copies of a row of `down`, and of a thread
        const uint32_t x_col = threadIdx.x % 16 * 4, x_row = threadIdx.x / 16, w_col = threadIdx.x % kPerRow * (W / sizeof(T)), w_row = threadIdx.x / kPerRow;
        const float *from[2];
#pragma unroll
        for (int i = 0; i < 2; i++) from[i] = p.x + (size_t)(row0 + rows[x_row + 16 * i < slot.n ? x_row + 16 * i : 0]) * p.x_stride + col0 + x_col;
        for (uint32_t k0 = 0; k0 < rank; k0 += L::kRanks) {
            const T *w = down + (size_t)(k0 + w_row) * p.n_cols + col0 + w_col;
            const size_t w_step = (size_t)(kThreads / kPerRow) * p.n_cols;
            auto load = [&](uint32_t i) {
                if (i < n_stages) {
                    const uint32_t stage = to + i % L::kStages * L::kStage, c = i * L::kCols;
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const bool there = x_row + 16 * n < slot.n && col0 + c + x_col < col1;
                        copy_async<16>(stage + (x_row + 16 * n) * L::kXPitch + x_col * 4, there ? from[n] + c : p.x, there);
                    }
#pragma unroll
                    for (uint32_t n = 0; n < kCopies; n++) {
                        const uint32_t k = w_row + n * (kThreads / kPerRow);
                        const bool there = k0 + k < rank && col0 + c + w_col < col1;
                        copy_async<W>(stage + L::kX + k * L::kDPitch + w_col * sizeof(T), there ? w + n * w_step + c : down, there);
                    }
                }
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
            float sum[2][4][4] = {}, d[2][4][4] = {};
            const bool used = k0 + 32 * half < rank;
#pragma unroll
            for (uint32_t i = 0; i + 1 < L::kStages; i++) load(i);
            for (uint32_t i = 0; i < n_stages; i++) {
                asm volatile("cp.async.wait_group %0;" ::"n"(L::kStages - 2) : "memory");
                __syncthreads();  // (the stage is there, and the one before has been read by all)
                load(i + L::kStages - 1);
                const uint8_t *stage = ring + i % L::kStages * L::kStage;
                if (used) {
                    Four<T> w[2][2];
#pragma unroll
                    for (int r = 0; r < 2; r++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
                            w[r][h].v = *reinterpret_cast<const decltype(w[r][h].v) *>(stage + L::kX + (32 * half + 16 * r + 8 * h + g) * L::kDPitch + (16 * part + 4 * t) * sizeof(T));
#pragma unroll
                    for (int n = 0; n < 4; n++) {
                        if (8 * n >= slot.n) break;
                        uint4 hi, lo;
                        split4(*reinterpret_cast<const float4 *>(stage + (8 * n + g) * L::kXPitch + (16 * part + 4 * t) * 4), hi, lo);
#pragma unroll
                        for (int r = 0; r < 2; r++) multiply<sizeof(T) == 2>(d[r][n], w[r][0].get(), w[r][1].get(), hi, lo);
                    }
                    if ((i & 3) == 3 || i + 1 == n_stages) {  // (the tensor core truncates what it adds to: sums of 64 columns, added up in fp32)
#pragma unroll
                        for (int r = 0; r < 2; r++)
#pragma unroll
                            for (int n = 0; n < 4; n++)
#pragma unroll
                                for (int e = 0; e < 4; e++) sum[r][n][e] += d[r][n][e], d[r][n][e] = 0.f;
                    }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 2; r++)
#pragma unroll
                for (int n = 0; n < 4; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) meet[(part * kTileRows + 8 * n + 2 * t + (e & 1)) * (L::kRanks + 1) + 32 * half + 16 * r + g + 8 * (e >> 1)] = sum[r][n][e];
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < slot.n * L::kRanks; i += kThreads) {
                const uint32_t r = i / L::kRanks, k = i % L::kRanks;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < 4; w++) v += meet[(w * kTileRows + r) * (L::kRanks + 1) + k];
                mine[i] = v;
            }
            cluster.sync();
            constexpr uint32_t kLanes = L::kRanks / 4;  // of a row
            for (uint32_t i = cta * kThreads + threadIdx.x; i < (slot.n + 1) / 2 * 2 * kLanes; i += ctas * kThreads) {  // (whole warps: two rows each)
                const uint32_t r = i / kLanes, k = i % kLanes * 4;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (r < slot.n)
                    for (uint32_t c = 0; c < ctas; c++) {
                        const float4 of = *reinterpret_cast<const float4 *>(cluster.map_shared_rank(mine, c) + 4 * i);
                        v.x += of.x, v.y += of.y, v.z += of.z, v.w += of.w;
                    }
                if (p.row_scales) v = halves_of_row<kLanes>(v, r < slot.n && k == 0 ? p.row_scales + row0 + rows[r] : nullptr);
                if (r < slot.n && k0 + k < p.rank_pitch) *reinterpret_cast<float4 *>(p.sums + (size_t)(row0 + rows[r]) * p.rank_pitch + k0 + k) = v;  // (beyond the rank: zeros)
            }
            cluster.sync();  // (the other CTAs have read this one's sums)
        }
        const uint32_t done = (rank + L::kRanks - 1) / L::kRanks * L::kRanks;
        for (uint32_t r = cta; r < slot.n; r += ctas)
            for (uint32_t k = done + threadIdx.x; k < p.rank_pitch; k += kThreads) {
                p.sums[(size_t)(row0 + rows[r]) * p.rank_pitch + k] = 0.f;
                if (k == 0 && p.row_scales) p.row_scales[row0 + rows[r]] = 1.f;
            }
    }
}

// out of all rows, ranks to 64.  A CTA has 128 outputs of one tile after another (its part of all outputs of all tiles), a warp 32 of them, whose rows of `up` it keeps in
// registers while the adapter stays the same.  Rows come in blocks of sixteen of an adapter.  A fifth warp finds them and has their base
// and v copied into shared memory a block ahead (1501 rows beside 14336: 71.1 us in all, two ahead 72.4, three 81.6); named barriers hand the places over and back.
constexpr uint32_t kUpWarps = 4, kPlaces = 4, kAhead = 1, kUpSteps = 4, kNoRow = ~0u - 1, kUpThreads = (kUpWarps + 1) * 32;
__device__ __forceinline__ void barrier_sync(uint32_t id) { asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kUpThreads) : "memory"); }
__device__ __forceinline__ void barrier_arrive(uint32_t id) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kUpThreads) : "memory"); }
template <typename T>
constexpr uint32_t kUpCtas = sizeof(T) == 2 ? 4 : 3;  // of an SM: `up` takes 32 registers, or 64
template <typename T>
__global__ void __launch_bounds__(kUpThreads, kUpCtas<T>) adapter_up_kernel(const __grid_constant__ AdapterParams p) {
    struct Block {
        uint32_t n, adapter, out0, fresh;  // fresh: other rows of `up` than the block before
        uint32_t row[16];
        float row_scale[16];
        uint32_t rank;
        float scale;
    };
    extern __shared__ __align__(16) float4 copies[];  // [place][warp][base of four rows][lane], then [place][pieces of v: of two rows per step][lane]
    __shared__ Block blocks[kPlaces];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, steps = p.rank_pitch / 16;
    float4 *bases = copies + lane, *vs = copies + kPlaces * kUpWarps * 4 * 32 + lane;
    constexpr uint32_t kFull = 1, kEmpty = 1 + kPlaces;  // barriers of the places
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    if (warp == kUpWarps) {
        const uint32_t tiles = (p.batch - 1) / kTileRows + 1;
        const uint64_t items = (uint64_t)tiles * ((p.n_rows + kUpWarps * 32 - 1) / (kUpWarps * 32)), begin = blockIdx.x * items / gridDim.x;
        uint32_t left = (uint32_t)((blockIdx.x + 1) * items / gridDim.x - begin), tile = (uint32_t)(begin % tiles), out0 = (uint32_t)(begin / tiles) * kUpWarps * 32;
        uint32_t firsts = 0, rows = 0, adapter = 0, id = 0, row0 = 0, fresh = 0;
        auto read_id = [&](uint32_t of) { return of * kTileRows + lane < p.batch ? read(p.row_adapter + of * kTileRows + lane) : 0u; };  // (looked at a tile later: nothing waits for it here)
        uint32_t id_next = left ? read_id(tile) : 0u, adapter_before = kNoRow, out_before = 0;
        // The next block, its copies under way (an empty group behind the last one).
        auto fetch = [&](uint32_t place) {
            Block &block = blocks[place];
            while (rows == 0) {
                while (firsts == 0 && left) {
                    left--, row0 = tile * kTileRows, id = row0 + lane >= p.batch ? kNoRow : id_next < p.n_adapters ? id_next : ~0u;
                    const uint32_t same = __match_any_sync(0xffffffffu, id);
                    // (rows without an adapter are blocks like the others where there is something to copy)
                    firsts = __ballot_sync(0xffffffffu, (uint32_t)__ffs(same) == lane + 1 && id != kNoRow && (id != ~0u || p.base != p.out));
                    fresh = out0;
                    if (++tile == tiles) tile = 0, out0 += kUpWarps * 32;
                    if (left) id_next = read_id(tile);
                }
                if (firsts == 0) break;
                adapter = __shfl_sync(0xffffffffu, id, __ffs(firsts) - 1);
                firsts &= firsts - 1;
                rows = __ballot_sync(0xffffffffu, id == adapter);
            }
            const uint32_t before = __popc(rows & ((1u << lane) - 1)), n = min((uint32_t)__popc(rows), 16u), o = fresh + 4 * g;
            const bool taken = (rows >> lane & 1u) && before < 16;
            if (taken) {
                block.row[before] = row0 + lane;
                if (sizeof(T) == 2 && adapter != ~0u) copy_async<4>((uint32_t)__cvta_generic_to_shared(block.row_scale + before), p.row_scales + row0 + lane, true);
            }
            if (lane == 0) block.n = n, block.adapter = adapter, block.out0 = fresh, block.fresh = adapter != adapter_before || fresh != out_before;
            if (n && adapter != ~0u && (adapter != adapter_before || fresh != out_before)) {  // rows of `up` that the compute warps will load
                if (lane == 0) copy_async<4>((uint32_t)__cvta_generic_to_shared(&block.rank), p.ranks + adapter, true), copy_async<4>((uint32_t)__cvta_generic_to_shared(&block.scale), p.scales + adapter, true);
                const char *up = static_cast<const char *>(p.up) + ((size_t)adapter * p.n_rows + fresh) * p.max_rank * sizeof(T);
                const uint32_t bytes = min(kUpWarps * 32, p.n_rows - fresh) * p.max_rank * (uint32_t)sizeof(T);
                for (uint32_t i = lane * 128; i < bytes; i += 32 * 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(up + i));
            }
            adapter_before = adapter, out_before = fresh;
            rows &= ~__ballot_sync(0xffffffffu, taken);
            __syncwarp();
            if (n) {
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(bases + place * kUpWarps * 4 * 32), v_dst = (uint32_t)__cvta_generic_to_shared(vs + place * 2 * steps * 32);
                if (adapter != ~0u)
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++) {
                        if (8 * h >= n) break;
                        const float *v = p.sums + (size_t)block.row[g + 8 * h < n ? g + 8 * h : 0] * p.rank_pitch + 4 * t;
#pragma unroll
                        for (uint32_t j = 0; j < kUpSteps; j++)
                            if (j < steps) copy_async<16>(v_dst + (2 * j + h) * 512, v + 16 * j, true);
                    }
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) {
                    const uint32_t r = c / 2 * 8 + 2 * t + c % 2;
                    if (r >= n) continue;
                    const float *from = p.base + (size_t)block.row[r] * p.out_stride + o;
#pragma unroll
                    for (uint32_t w = 0; w < kUpWarps; w++)
                        if (p.whole_outs) {
                            if (o + 32 * w < p.n_rows) copy_async<16>(dst + (4 * w + c) * 512, from + 32 * w, true);
                        } else {
#pragma unroll
                            for (uint32_t i = 0; i < 4; i++)
                                if (o + 32 * w + i < p.n_rows) copy_async<4>(dst + (4 * w + c) * 512 + 4 * i, from + 32 * w + i, true);
                        }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            return n != 0;
        };
        uint32_t place = 0, of = 0;  // of the next block, and how many have been fetched
        for (bool more = true; more; of++) {
            if (of >= kPlaces) barrier_sync(kEmpty + place);
            more = fetch(place);
            if (of >= kAhead) {
                asm volatile("cp.async.wait_group %0;" ::"n"(kAhead) : "memory");
                barrier_arrive(kFull + (place + kPlaces - kAhead) % kPlaces);
            }
            place = place == kPlaces - 1 ? 0 : place + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        for (uint32_t i = of < kAhead ? of : kAhead; i; i--) barrier_arrive(kFull + (place + kPlaces - i) % kPlaces);
        return;
    }
    uint32_t place = 0;
    float scale = 0.f;
    Four<T> up[kUpSteps][4];
    for (;;) {
        barrier_sync(kFull + place);
        const Block &block = blocks[place];
        const uint32_t n = block.n, of = block.adapter, o = block.out0 + 32 * warp + 4 * g;
        if (n == 0) return;
        scale = of == ~0u ? -0.f : scale;  // (-0 · 0 + base: its bits)
        if (block.fresh && of != ~0u) {
            const uint32_t rank = min(block.rank, p.max_rank);
            scale = block.scale;
            const T *first = static_cast<const T *>(p.up) + (size_t)of * p.n_rows * p.max_rank;
#pragma unroll
            for (uint32_t j = 0; j < kUpSteps; j++) load_up(p, first, o, j, rank, up[j]);
        }
        const float4 *from = bases + (place * kUpWarps + warp) * 4 * 32, *v = vs + place * 2 * steps * 32;
        float d[2][2][4] = {};
        bool halves = false;
        if constexpr (sizeof(T) == 2) {
            const float mine = block.row_scale[lane & 15];
            halves = !__any_sync(0xffffffffu, (lane & 15) < n && mine == 0.f) && of != ~0u;
            if (halves)
#pragma unroll
                for (uint32_t j = 0; j < kUpSteps; j++) {
                    if (j == steps) break;
#pragma unroll
                    for (uint32_t h = 0; h < 2; h++) {
                        const float4 w = v[(2 * j + h) * 32];
                        multiply_f16(d[h][0], up[j][0].v, up[j][1].v, w.z, w.w);
                        multiply_f16(d[h][1], up[j][2].v, up[j][3].v, w.z, w.w);
                        multiply_f16(d[h][0], up[j][0].v, up[j][1].v, w.x, w.y);
                        multiply_f16(d[h][1], up[j][2].v, up[j][3].v, w.x, w.y);
                    }
                }
        }
        if (!halves && of != ~0u)
#pragma unroll
            for (uint32_t j = 0; j < kUpSteps; j++) {
                if (j == steps) break;
                float4 a[4];
#pragma unroll
                for (int i = 0; i < 4; i++) a[i] = up[j][i].get();
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    float4 w = v[(2 * j + h) * 32];
                    if (sizeof(T) == 2 && g + 8 * h < n && block.row_scale[g + 8 * h] != 0.f) w = row_of_halves(w, block.row_scale[g + 8 * h]);
                    uint4 hi, lo;
                    split4(w, hi, lo);
                    multiply<sizeof(T) == 2>(d[h][0], a[0], a[1], hi, lo);
                    multiply<sizeof(T) == 2>(d[h][1], a[2], a[3], hi, lo);
                }
            }
#pragma unroll
        for (uint32_t c = 0; c < 4; c++) {
            const uint32_t r = c / 2 * 8 + 2 * t + c % 2;
            const float(&e)[2][4] = d[c / 2];
            const float back = halves ? block.row_scale[r] : 1.f;
            const float four_of[4] = {e[0][c % 2] * back, e[0][2 + c % 2] * back, e[1][c % 2] * back, e[1][2 + c % 2] * back};
            if (r < n) store4(p, (size_t)block.row[r] * p.out_stride, o, from[c * 32], four_of, scale);
        }
        barrier_arrive(kEmpty + place);
        place = place == kPlaces - 1 ? 0 : place + 1;
    }
}

// out of a tile's slots, larger ranks, a share of the outputs per CTA: grid x = tiles, y = slots, z = shares.  32 outputs a warp and pass.
template <typename T>
__global__ void __launch_bounds__(kThreads, 2) adapter_up_wide_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ __align__(16) uint32_t v_hi[];  // hi, then lo: [row][pitch]
    __shared__ uint8_t lists[kWarps][32];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t row0 = blockIdx.x * kTileRows, out0 = blockIdx.z * p.outs_per_cta, end = min(out0 + p.outs_per_cta, p.n_rows), pitch = v_pitch(p.max_rank);
    uint32_t *v_lo = v_hi + kTileRows * pitch;
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    const Tile tile = read_tile<kTileRows>(p, row0);
    if (blockIdx.y == 0) copy_base<kTileRows>(p, tile, row0, out0, end, lists[warp]);
    const uint32_t n_slots = __popc(tile.firsts);
    const uint8_t *rows = lists[warp];
    for (uint32_t s = blockIdx.y; s < n_slots; s += gridDim.y) {
        const Slot slot = read_slot(tile, s, lists[warp]);
        const uint32_t rank = min(read(p.ranks + slot.adapter), p.max_rank), steps = (rank + 15) / 16;
        const float scale = read(p.scales + slot.adapter);
        const T *up = static_cast<const T *>(p.up) + (size_t)slot.adapter * p.n_rows * p.max_rank;
        __syncthreads();  // (the slot before has read its sums)
        for (uint32_t i = threadIdx.x; i < kTileRows * steps * 16; i += kThreads) {
            const uint32_t r = i / (steps * 16), k = i % (steps * 16);
            const float v = r < slot.n && k < rank ? __ldcg(p.sums + (size_t)(row0 + rows[r]) * p.rank_pitch + k) : 0.f;
            split_tf32(v, v_hi[r * pitch + k], v_lo[r * pitch + k]);
        }
        __syncthreads();
        for (uint32_t o = out0 + warp * 32 + 4 * g; o - 4 * g < end; o += kPassOuts) {
            float4 b[4][2];
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint32_t r = 8 * n + 2 * t + c;
                    b[n][c] = load4(p, (size_t)(row0 + rows[r < slot.n ? r : 0]) * p.out_stride, o, r < slot.n);
                }
            float d[2][4][4] = {};
#pragma unroll 2
            for (uint32_t j = 0; j < steps; j++) {
                Four<T> u[4];
                load_up(p, up, o, j, rank, u);
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    if (8 * n >= slot.n) break;
                    const uint4 hi = *reinterpret_cast<const uint4 *>(v_hi + (8 * n + g) * pitch + 16 * j + 4 * t), lo = *reinterpret_cast<const uint4 *>(v_lo + (8 * n + g) * pitch + 16 * j + 4 * t);
                    multiply<sizeof(T) == 2>(d[0][n], u[0].get(), u[1].get(), hi, lo);
                    multiply<sizeof(T) == 2>(d[1][n], u[2].get(), u[3].get(), hi, lo);
                }
            }
#pragma unroll
            for (int n = 0; n < 4; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const uint32_t r = 8 * n + 2 * t + c;
                    const float four_of[4] = {d[0][n][c], d[0][n][2 + c], d[1][n][c], d[1][n][2 + c]};
                    if (r < slot.n) store4(p, (size_t)(row0 + rows[r]) * p.out_stride, o, b[n][c], four_of, scale);
                }
        }
    }
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }
// 128 rows of 4 (48) adapters of rank 16 and 64 beside 4096 × 4096 take 10.0, 14.3 (14.6, 26.0) us as a step and 18.4, 20.3 (52.6, 61.1) as prompts, 256 rows 15.2,
// 20.5 (21.3, 36.4) and 17.2, 18.8 (33.2, 38.5).
bool is_step(const AdapterBatch &a) { return a.batch <= 128; }
uint32_t rank_pitch(const AdapterBatch &a) { return is_step(a) ? (a.max_rank + 3) / 4 * 4 : (a.max_rank + 15) / 16 * 16; }

cudaError_t launch_cluster(void (*kern)(AdapterParams), dim3 grid, uint32_t ctas, size_t smem, bool pdl, cudaStream_t s, const AdapterParams &p) {
    cudaError_t e;
    if ((ctas > 8 || smem > 24 * 1024) && (e = kernel_opt_in(reinterpret_cast<const void *>(kern), smem, ctas > 8)) != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid, cfg.blockDim = dim3(kThreads), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return launch_config(cfg, kern, p);
}

template <typename T>
cudaError_t launch_step(const AdapterBatch &a, AdapterParams p, cudaStream_t s, uint64_t *launches) {
    const uint32_t tiles = ceil_div(a.batch, kStepRows), slots = a.batch < kStepRows ? a.batch : kStepRows;
    // Sixteen CTAs for a few clusters: one row of rank 64 beside 4096 × 14336 takes 10.2 us with them and 15.7 with eight, beside 2048 × 2048 7.1 and 7.4.  Sixteen clusters (if
    // every row has an adapter of its own) gain from it where adapters are large, 17.9 us against 20.6 (small ones lose, 12.3 against 9.4), more never.
    const uint64_t bytes = (uint64_t)a.max_rank * (a.n_cols + a.n_rows) * sizeof(T);  // of an adapter
    const uint32_t ctas = tiles * slots <= 8 || (tiles * slots <= 16 && bytes >= (1u << 20)) ? 16 : 8;
    p.cols_per_cta = ceil_div(a.n_cols, ctas * kWarps * 16) * kWarps * 16;
    p.outs_per_cta = ceil_div(a.n_rows, ctas * 32) * 32;
    const size_t smem = (size_t)kStepRows * (ctas * p.rank_pitch + 2 * v_pitch(a.max_rank)) * sizeof(float);
    auto kern = a.max_rank <= 16 ? adapter_step_kernel<T, 1> : adapter_step_kernel<T, 4>;
    const cudaError_t e = launch_cluster(kern, dim3(ctas, slots, tiles), ctas, smem, a.pdl, s, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}

template <typename T>
cudaError_t launch_prompts(const AdapterBatch &a, AdapterParams p, int sm_count, cudaStream_t s, uint64_t *launches) {
    using L = DownLayout<T>;
    // Slots: CTAs without one leave at once (33.4 us for 1500 rows of six requests with 4 as with 16), tiles of many adapters are sooner done (1024 rows, 64 of them of 48
    // adapters: 185 us with 4, 162 with 16, 168 with 32).
    const uint32_t tiles = ceil_div(a.batch, kTileRows), slots = a.n_adapters < 16 ? a.n_adapters : 16;
    // As many CTAs per tile as are there at once (1500 rows of 4096 columns: 59.8 us with two, 43.0 with four, 40.0 with the five of this rule, 46.0 with eight; 96 rows of
    // 14336 columns: 66, 44, and 27 with eight).
    uint32_t ctas = 8;
    while (ctas > 1 && ((ctas - 1) * L::kCols >= a.n_cols || (uint64_t)tiles * ctas > 7 * (uint64_t)sm_count / 4)) ctas--;
    p.cols_per_cta = ceil_div(a.n_cols, ctas * L::kCols) * L::kCols;
    auto down = adapter_down_kernel<T, 16>;
    if constexpr (sizeof(T) == 2)
        if (a.n_cols % 8) down = adapter_down_kernel<T, 8>;
    cudaError_t e = launch_cluster(down, dim3(tiles * ctas, slots), ctas, L::kBytes, a.pdl, s, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (a.max_rank <= 16 * kUpSteps) {
        const uint64_t items = (uint64_t)tiles * ceil_div(a.n_rows, kUpWarps * 32), at_once = kUpCtas<T> * (uint64_t)sm_count;
        const size_t smem = (size_t)kPlaces * (kUpWarps * 4 + p.rank_pitch / 8) * 512;
        auto up = adapter_up_kernel<T>;
        if ((e = kernel_opt_in(reinterpret_cast<const void *>(up), smem, false)) != cudaSuccess) return e;
        e = launch_kernel(up, dim3((uint32_t)(items < at_once ? items : at_once)), dim3(kUpThreads), smem, s, true, p);
    } else {
        p.outs_per_cta = 2 * kPassOuts;
        const size_t smem = (size_t)2 * kTileRows * v_pitch(a.max_rank) * 4;
        auto up = adapter_up_wide_kernel<T>;
        if ((e = kernel_opt_in(reinterpret_cast<const void *>(up), smem, false)) != cudaSuccess) return e;
        e = launch_kernel(up, dim3(tiles, slots, ceil_div(a.n_rows, p.outs_per_cta)), dim3(kThreads), smem, s, true, p);
    }
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace

size_t adapter_scratch_bytes(const AdapterBatch &a) { return is_step(a) ? 0 : (size_t)a.batch * (rank_pitch(a) + 1) * sizeof(float); }

cudaError_t launch_adapters(const AdapterBatch &a, int sm_count, cudaStream_t s, uint64_t *launches) {
    AdapterParams p = {};
    p.down = a.down, p.up = a.up, p.ranks = a.ranks, p.row_adapter = a.row_adapter, p.scales = a.scales, p.x = a.x, p.base = a.base, p.out = a.out;
    p.sums = static_cast<float *>(a.scratch);
    p.n_adapters = a.n_adapters, p.max_rank = a.max_rank, p.n_rows = a.n_rows, p.n_cols = a.n_cols, p.batch = a.batch;
    p.x_stride = a.x_stride, p.out_stride = a.out_stride;
    p.rank_pitch = rank_pitch(a);
    p.row_scales = a.type == YULE_DTYPE_F16 && a.max_rank <= 16 * kUpSteps ? p.sums + (size_t)a.batch * p.rank_pitch : nullptr;
    p.whole_ranks = a.max_rank % 4 == 0;
    p.whole_outs = a.n_rows % 4 == 0 && a.out_stride % 4 == 0;
    if (is_step(a)) return a.type == YULE_DTYPE_F16 ? launch_step<__half>(a, p, s, launches) : launch_step<float>(a, p, s, launches);
    return a.type == YULE_DTYPE_F16 ? launch_prompts<__half>(a, p, sm_count, s, launches) : launch_prompts<float>(a, p, sm_count, s, launches);
}

}  // namespace yule
