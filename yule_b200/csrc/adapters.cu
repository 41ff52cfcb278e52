// adapters.cu — low-rank adapters of many requests beside a shared projection.
//
// Row i of the batch has adapter a = row_adapter[i] (none if a >= n_adapters: its output is its base), of rank r = min(ranks[a], max_rank):
//     v_k = Σ_c down[a][k][c] · x[i][c]   (k < r),      out[i][o] = base[i][o] + scales[a] · Σ_k up[a][o][k] · v_k.
// Two kernels.  The first leaves the sums v of each chunk of columns in the scratch, the second adds the chunks up and multiplies with `up`.  Rows come in tiles; a tile's
// adapters are its slots: a CTA takes one of them with all the rows of the tile that have it as the columns of the tensor core's second operand, so an
// adapter is read once per tile whatever the order of the requests, and rows of other adapters are zeros there.  F16 adapters are tf32 numbers as they are: two products
// per element (of hi and lo of x or v), three for F32 ones.  Sums are added in a fixed order.

#include <cuda_fp16.h>

#include "internal.h"
#include "tf32_common.cuh"

namespace yule {

namespace {

constexpr int kWarps = 4;

struct AdapterParams {
    const void *down, *up;
    const uint32_t *ranks, *row_adapter;
    const float *scales, *x, *base;
    float *out, *sums;  // sums: [row][split][rank_pitch]
    uint32_t n_adapters, max_rank, n_rows, n_cols, batch, splits, cols_per_split, rank_pitch, slots;
    size_t x_stride, out_stride;
    bool whole_ranks, whole_outs;  // rows of `up`, and of out and base, are on the boundaries of vectors of four
};

// The rows of a tile and who is first of its adapter.
template <int ROWS>
struct Tile {
    uint32_t id[ROWS];     // adapter of each row, ~0 for none
    uint32_t first[ROWS];  // adapters in the order of their first rows
    uint32_t n;
};
template <int ROWS>
__device__ __forceinline__ void read_tile(const AdapterParams &p, uint32_t row0, Tile<ROWS> &tile) {
    static_assert(ROWS <= 32, "a lane per row");
    if (threadIdx.x < 32) {
        const uint32_t lane = threadIdx.x, row = row0 + lane;
        uint32_t id = lane < ROWS && row < p.batch ? __ldg(p.row_adapter + row) : ~0u;
        if (id >= p.n_adapters) id = ~0u;
        const uint32_t same = __match_any_sync(0xffffffffu, id), firsts = __ballot_sync(0xffffffffu, id != ~0u && (uint32_t)__ffs(same) == lane + 1);
        if (lane < ROWS) tile.id[lane] = id;
        if (firsts >> lane & 1u) tile.first[__popc(firsts & ((1u << lane) - 1))] = id;
        if (lane == 0) tile.n = __popc(firsts);
    }
    __syncthreads();
}

// Four elements of an adapter's row from `at` on, of which `n` are there, as fp32.
template <typename T>
__device__ __forceinline__ float4 four(const T *at, int n, bool whole);
template <>
__device__ __forceinline__ float4 four<float>(const float *at, int n, bool whole) {
    if (whole && n >= 4) return __ldg(reinterpret_cast<const float4 *>(at));
    return make_float4(n > 0 ? __ldg(at) : 0.f, n > 1 ? __ldg(at + 1) : 0.f, n > 2 ? __ldg(at + 2) : 0.f, n > 3 ? __ldg(at + 3) : 0.f);
}
template <>
__device__ __forceinline__ float4 four<__half>(const __half *at, int n, bool whole) {
    if (whole && n >= 4) {
        const uint2 v = __ldg(reinterpret_cast<const uint2 *>(at));
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    auto one = [&](int i) { return n > i ? __half2float(__ldg(at + i)) : 0.f; };
    return make_float4(one(0), one(1), one(2), one(3));
}

// d += a · b over two steps of eight: this lane's four elements of the operands' rows g (a) and g + 8 (b), and of the second operand's column g.
template <bool EXACT>  // a and b are tf32 numbers
__device__ __forceinline__ void multiply(float (&d)[4], const float4 &a, const float4 &b, const uint4 &hi, const uint4 &lo) {
    uint32_t ah[4] = {__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(a.z), __float_as_uint(a.w)};
    uint32_t bh[4] = {__float_as_uint(b.x), __float_as_uint(b.y), __float_as_uint(b.z), __float_as_uint(b.w)};
    if (!EXACT) {
        uint32_t al[4], bl[4];
#pragma unroll
        for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(ah[i]), ah[i], al[i]), split_tf32(__uint_as_float(bh[i]), bh[i], bl[i]);
        mma_tf32(d, al[0], bl[0], al[1], bl[1], hi.x, hi.y);
        mma_tf32(d, al[2], bl[2], al[3], bl[3], hi.z, hi.w);
    }
    mma_tf32(d, ah[0], bh[0], ah[1], bh[1], lo.x, lo.y);
    mma_tf32(d, ah[2], bh[2], ah[3], bh[3], lo.z, lo.w);
    mma_tf32(d, ah[0], bh[0], ah[1], bh[1], hi.x, hi.y);
    mma_tf32(d, ah[2], bh[2], ah[3], bh[3], hi.z, hi.w);
}
__device__ __forceinline__ void split4(const float4 &v, uint4 &hi, uint4 &lo) {
    split_tf32(v.x, hi.x, lo.x), split_tf32(v.y, hi.y, lo.y), split_tf32(v.z, hi.z, lo.z), split_tf32(v.w, hi.w, lo.w);
}

// v of a tile's rows over a chunk of columns: 16·RANKS rows of `down` at a time, rows of x in eights as columns.  A warp takes 64 columns in turn with the others.
template <typename T, int ROWS, int RANKS>
__global__ void __launch_bounds__(kWarps * 32) adapter_down_kernel(const __grid_constant__ AdapterParams p) {
    __shared__ Tile<ROWS * 8> tile;
    __shared__ float meet[kWarps][ROWS * 8][RANKS * 16 + 1];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t row0 = blockIdx.x * ROWS * 8, split = blockIdx.z;
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    read_tile(p, row0, tile);
    const uint32_t col0 = split * p.cols_per_split, col1 = min(col0 + p.cols_per_split, p.n_cols);
    for (uint32_t slot = blockIdx.y; slot < tile.n; slot += p.slots) {
        const uint32_t a = tile.first[slot], rank = min(__ldg(p.ranks + a), p.max_rank);
        const T *down = static_cast<const T *>(p.down) + (size_t)a * p.max_rank * p.n_cols;
        bool mine[ROWS];
#pragma unroll
        for (int n = 0; n < ROWS; n++) mine[n] = tile.id[8 * n + g] == a;
        for (uint32_t k0 = 0; k0 < rank; k0 += RANKS * 16) {
            float sum[RANKS][ROWS][4];
#pragma unroll
            for (int r = 0; r < RANKS; r++)
#pragma unroll
                for (int n = 0; n < ROWS; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) sum[r][n][e] = 0.f;
            for (uint32_t base = col0 + warp * 64; base < col1; base += kWarps * 64) {
                // (the tensor core truncates what it adds to: sums of 64 columns, added up in fp32)
                float d[RANKS][ROWS][4];
#pragma unroll
                for (int r = 0; r < RANKS; r++)
#pragma unroll
                    for (int n = 0; n < ROWS; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) d[r][n][e] = 0.f;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) {
                    const uint32_t c = base + 16 * j + 4 * t;
                    const bool in = c < col1;
                    uint4 hi[ROWS], lo[ROWS];
#pragma unroll
                    for (int n = 0; n < ROWS; n++)
                        split4(in && mine[n] ? __ldg(reinterpret_cast<const float4 *>(p.x + (size_t)(row0 + 8 * n + g) * p.x_stride + c)) : make_float4(0.f, 0.f, 0.f, 0.f), hi[n], lo[n]);
#pragma unroll
                    for (int r = 0; r < RANKS; r++) {
                        const uint32_t k = k0 + 16 * r + g;
                        const float4 u = four(down + (size_t)k * p.n_cols + c, in && k < rank ? 4 : 0, true), v = four(down + (size_t)(k + 8) * p.n_cols + c, in && k + 8 < rank ? 4 : 0, true);
#pragma unroll
                        for (int n = 0; n < ROWS; n++) multiply<sizeof(T) == 2>(d[r][n], u, v, hi[n], lo[n]);
                    }
                }
#pragma unroll
                for (int r = 0; r < RANKS; r++)
#pragma unroll
                    for (int n = 0; n < ROWS; n++)
#pragma unroll
                        for (int e = 0; e < 4; e++) sum[r][n][e] += d[r][n][e];
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < RANKS; r++)
#pragma unroll
                for (int n = 0; n < ROWS; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) meet[warp][8 * n + 2 * t + (e & 1)][16 * r + g + 8 * (e >> 1)] = sum[r][n][e];
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < ROWS * 8 * RANKS * 16; i += kWarps * 32) {
                const uint32_t row = i / (RANKS * 16), k = i % (RANKS * 16);
                if (tile.id[row] != a || k0 + k >= rank) continue;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWarps; w++) v += meet[w][row][k];
                p.sums[((size_t)(row0 + row) * p.splits + split) * p.rank_pitch + k0 + k] = v;
            }
        }
    }
}

// out of a tile's rows for 32 outputs a warp: rows of `up` as rows of the first operand, in an order that gives a lane four consecutive outputs.
template <typename T, int ROWS>
__global__ void __launch_bounds__(kWarps * 32) adapter_up_kernel(const __grid_constant__ AdapterParams p) {
    extern __shared__ __align__(16) uint32_t v_terms[];  // hi, then lo: [row][pitch]
    __shared__ Tile<ROWS * 8> tile;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t row0 = blockIdx.x * ROWS * 8, pitch = (p.max_rank + 31) / 32 * 32 + 16, o = (blockIdx.z * kWarps + warp) * 32 + 4 * g;
    uint32_t *v_hi = v_terms, *v_lo = v_terms + ROWS * 8 * pitch;
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    read_tile(p, row0, tile);
    auto store = [&](uint32_t row, const float (&d)[4], float scale) {
        const float *from = p.base + (size_t)row * p.out_stride + o;
        float *to = p.out + (size_t)row * p.out_stride + o;
        if (p.whole_outs) {
            if (o >= p.n_rows) return;
            const float4 b = *reinterpret_cast<const float4 *>(from);
            *reinterpret_cast<float4 *>(to) = make_float4(fmaf(scale, d[0], b.x), fmaf(scale, d[1], b.y), fmaf(scale, d[2], b.z), fmaf(scale, d[3], b.w));
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (o + i < p.n_rows) to[i] = fmaf(scale, d[i], from[i]);
        }
    };
    // rows without an adapter: their base
    if (blockIdx.y == 0 && p.base != p.out)
#pragma unroll
        for (int n = 0; n < ROWS; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const uint32_t r = 8 * n + 2 * t + c;
                const float none[4] = {0.f, 0.f, 0.f, 0.f};
                if (tile.id[r] == ~0u && row0 + r < p.batch) store(row0 + r, none, 0.f);
            }
    for (uint32_t slot = blockIdx.y; slot < tile.n; slot += p.slots) {
        const uint32_t a = tile.first[slot], rank = min(__ldg(p.ranks + a), p.max_rank), steps = (rank + 15) / 16;
        const float scale = __ldg(p.scales + a);
        const T *up = static_cast<const T *>(p.up) + (size_t)a * p.n_rows * p.max_rank;
        __syncthreads();  // (the slot before has read its sums)
        for (uint32_t i = threadIdx.x; i < ROWS * 8 * steps * 16; i += kWarps * 32) {
            const uint32_t r = i / (steps * 16), k = i % (steps * 16);
            float v = 0.f;
            if (tile.id[r] == a && k < rank)
                for (uint32_t s = 0; s < p.splits; s++) v += __ldcg(p.sums + ((size_t)(row0 + r) * p.splits + s) * p.rank_pitch + k);
            split_tf32(v, v_hi[r * pitch + k], v_lo[r * pitch + k]);
        }
        __syncthreads();
        float d[2][ROWS][4];
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) d[c][n][e] = 0.f;
#pragma unroll 2
        for (uint32_t j = 0; j < steps; j++) {
            const uint32_t k = 16 * j + 4 * t;
            const int there = (int)rank - (int)k;
            float4 u[4];
#pragma unroll
            for (int i = 0; i < 4; i++) u[i] = four(up + (size_t)(o + i) * p.max_rank + k, o + i < p.n_rows ? there : 0, p.whole_ranks);
#pragma unroll
            for (int n = 0; n < ROWS; n++) {
                const uint4 hi = *reinterpret_cast<const uint4 *>(v_hi + (8 * n + g) * pitch + k), lo = *reinterpret_cast<const uint4 *>(v_lo + (8 * n + g) * pitch + k);
                multiply<sizeof(T) == 2>(d[0][n], u[0], u[1], hi, lo);
                multiply<sizeof(T) == 2>(d[1][n], u[2], u[3], hi, lo);
            }
        }
#pragma unroll
        for (int n = 0; n < ROWS; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const uint32_t r = 8 * n + 2 * t + c;
                const float four_of[4] = {d[0][n][c], d[0][n][2 + c], d[1][n][c], d[1][n][2 + c]};
                if (tile.id[r] == a) store(row0 + r, four_of, scale);
            }
    }
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// Tiles of 32 rows for prompts, of 8 with a slot per row for decode steps.
uint32_t tile_rows(const AdapterBatch &a) { return a.batch > 64 ? 32 : 8; }
uint32_t splits_of(const AdapterBatch &a, int sm_count) {
    const uint32_t slots = tile_rows(a) == 8 ? a.batch : ceil_div(a.batch, 32);
    const uint32_t want = ceil_div(3 * (uint64_t)sm_count, slots), most = ceil_div(a.n_cols, kWarps * 64);
    return want < most ? want : most;
}

template <typename T>
cudaError_t launch_typed(const AdapterBatch &a, AdapterParams p, cudaStream_t s, uint64_t *launches) {
    const uint32_t rows = tile_rows(a), tiles = ceil_div(a.batch, rows);
    const dim3 block(kWarps * 32), down(tiles, p.slots, p.splits), up(tiles, p.slots, ceil_div(a.n_rows, kWarps * 32));
    if (up.z > 65535) return cudaErrorInvalidValue;
    cudaError_t e;
    if (rows == 8)
        e = a.max_rank <= 16 ? launch_kernel(adapter_down_kernel<T, 1, 1>, down, block, 0, s, a.pdl, p) : launch_kernel(adapter_down_kernel<T, 1, 4>, down, block, 0, s, a.pdl, p);
    else
        e = a.max_rank <= 16 ? launch_kernel(adapter_down_kernel<T, 4, 1>, down, block, 0, s, a.pdl, p) : launch_kernel(adapter_down_kernel<T, 4, 4>, down, block, 0, s, a.pdl, p);
    if (e != cudaSuccess) return e;
    ++*launches;
    const size_t smem = (size_t)2 * rows * ((a.max_rank + 31) / 32 * 32 + 16) * 4;
    auto kern = rows == 8 ? adapter_up_kernel<T, 1> : adapter_up_kernel<T, 4>;
    if (smem > 40 * 1024 && (e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem)) != cudaSuccess) return e;
    e = launch_kernel(kern, up, block, smem, s, true, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace

size_t adapter_scratch_bytes(const AdapterBatch &a, int sm_count) { return (size_t)a.batch * splits_of(a, sm_count) * ((a.max_rank + 3) / 4 * 4) * sizeof(float); }

cudaError_t launch_adapters(const AdapterBatch &a, int sm_count, cudaStream_t s, uint64_t *launches) {
    AdapterParams p = {};
    p.down = a.down, p.up = a.up, p.ranks = a.ranks, p.row_adapter = a.row_adapter, p.scales = a.scales, p.x = a.x, p.base = a.base, p.out = a.out;
    p.sums = static_cast<float *>(a.scratch);
    p.n_adapters = a.n_adapters, p.max_rank = a.max_rank, p.n_rows = a.n_rows, p.n_cols = a.n_cols, p.batch = a.batch;
    p.x_stride = a.x_stride, p.out_stride = a.out_stride;
    p.splits = splits_of(a, sm_count);
    p.cols_per_split = ceil_div(ceil_div(a.n_cols, p.splits), 64) * 64;
    p.splits = ceil_div(a.n_cols, p.cols_per_split);
    p.rank_pitch = (a.max_rank + 3) / 4 * 4;
    p.slots = tile_rows(a) == 8 ? (a.batch < 8 ? a.batch : 8) : 1;
    p.whole_ranks = a.max_rank % 4 == 0;
    p.whole_outs = a.n_rows % 4 == 0 && a.out_stride % 4 == 0;
    return a.type == YULE_DTYPE_F16 ? launch_typed<__half>(a, p, s, launches) : launch_typed<float>(a, p, s, launches);
}

}  // namespace yule
