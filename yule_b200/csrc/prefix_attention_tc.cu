// prefix_attention_tc.cu — the shared prefix of a batch for 128 query rows at a time, on tcgen05.
//
// A first kernel writes the prefix's K and V as the tensor core reads them, once for all query rows.  Then a CTA has 128 query rows of one KV head (query tokens of all sequences one
// after the other, the heads of the group within a token) and a chunk of the prefix, of which every row sees every position; it leaves (m, Σ, o) of each row, which
// prefix_merge_kernel adds to the other parts.
//
// Precision.  The tensor core multiplies fp16 and truncates what it adds to.  A query row, and the K and V of a tile of 64 positions, are scaled by powers of two so that their largest
// element is 2^13 to 2^14, and split into hi + lo (22 bits; what is 2^-14 of the largest loses the lower ones).  A score, and an output of a tile, is the small products first,
// then hi·hi; outputs of tiles are added up in fp32, with the mean of what truncation takes given back.  A value that is not finite makes every row's output not
// finite: every row sees it.
//
// Roles (512 threads): eight warps do the soft-max (a thread per row and half a tile's positions), four add the output up (a thread per row), two issue the MMAs of scores and of
// output (one that does both waits for either 2900 clocks a tile), two the bulk copies of K and of V.  The query rows are in tensor memory; K has three buffers, V, scores and probabilities have two, and the scores of a tile are issued two tiles ahead of its output,
// which comes in parts of 64 dimensions: one is added up while the next is multiplied.  (Converting K and V where they are used took 5000 to 7400 clocks a tile and CTA, by
// the soft-max warps or by eight more: the MMAs take 1536.)

#include <cfloat>
#include <mutex>
#include <type_traits>

#include <cuda_fp16.h>

#include "prefix_attention.cuh"
#include "qgemm_common.cuh"

namespace yule {

namespace {

constexpr int kRows = (int)kPrefixTcRows;  // query rows per CTA = TMEM lanes
constexpr int kKeys = (int)kPrefixTcKeys;  // positions per tile
constexpr int kThreads = 512;
constexpr uint32_t kSumWarp = 8, kMmaWarp = 12, kKeyWarp = 13, kOutputWarp = 14, kValueWarp = 15;  // the first of each; soft-max from 0 on
constexpr int kLaunchRegs = 96;  // registers per thread that 512 threads are launched with (the build checks that the kernels get them)
constexpr int kSoftRegs = 96, kSumRegs = 168, kIssueRegs = 24;
static_assert(2 * kSoftRegs + kSumRegs + kIssueRegs <= 4 * kLaunchRegs, "register split");
constexpr uint32_t kMostTiles = kPrefixTcTiles;  // of a chunk
constexpr float kTruncation = 0.8e-7f;  // what truncation takes of a sum on average, as a fraction (four additions at full size): given back
constexpr float kProbBits = 12.f;       // probabilities are stored 2^12 as large, clear of fp16's subnormals

// (a, b) → packed fp16 pairs hi and lo
__device__ __forceinline__ void split2(uint64_t ab, uint32_t &hi, uint32_t &lo) {
    const float2 x = unpair(ab);
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 f = __half22float2(h), rest = unpair(fma2(pair(f.x, f.y), pair(-1.f, -1.f), ab));
    const __half2 l = __floats2half2_rn(rest.x, rest.y);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = *reinterpret_cast<const uint32_t *>(&l);
}
// 2^e with m·2^e in [2^13, 2^14) and its inverse; m == 0, inf and NaN give 1 and 1 (they stay what they are)
__device__ __forceinline__ void pow2_scale(float m, float &scale, float &inv) {
    const int eb = (int)((__float_as_uint(m) >> 23) & 0xFFu);
    int se = (m == 0.f || eb == 0xFF) ? 127 : 127 + 13 - (eb - 127);
    se = se < 1 ? 1 : (se > 253 ? 253 : se);
    scale = __uint_as_float((uint32_t)se << 23);
    inv = __uint_as_float((uint32_t)(254 - se) << 23);
}
__device__ __forceinline__ float power(float x) {  // of two, to 2^-22; subnormal ones are nothing
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int HD>
struct Layout {
    // Operands in the no-swizzle core-matrix layout (8 rows x 16 bytes; core matrices of one step of eight contiguous along the rows): K rows by
    // dimension, V transposed: dimensions by position.  In memory a tile is K hi, K lo, V hi, V lo.
    static constexpr uint32_t kPlane = kKeys * HD * 2, kTile = 4 * kPlane;
    static constexpr uint32_t kOffK = 0, kOffV = 6 * kPlane, kOffRows = 10 * kPlane;  // three buffers of K, two of V
    // per row: alpha (two tiles), largest score of either half (two tiles), sums of either half, last largest score, score factor; then inverse scales of K and V of the chunk's
    // tiles; then barriers
    static constexpr uint32_t kOffScales = kOffRows + 10 * kRows * 4, kOffBars = kOffScales + kMostTiles * 8, kBars = 24;
    static constexpr uint32_t kSmem = kOffBars + kBars * 8 + 16;
    // before the first tile the query rows as packed words (where the last K and V will be), behind the last one the output, a row after the other
    static constexpr uint32_t kPitch = HD + 4, kOffQ = 4 * kPlane;
    static_assert(kOffQ + kRows * kPitch * 4 <= kOffRows, "query rows beside the first two K");
    // tensor memory columns: two buffers of scores, output, two buffers of probabilities (hi, lo), query rows (hi, lo)
    static constexpr uint32_t kS = 0, kO = 128, kP = 256, kQ = 384;
    static_assert(kSmem <= 227 * 1024 && kOffBars % 8 == 0, "shared memory");
};

// A tile of K (z = 0) or of V as the tensor core reads it, and its inverse scale.  Bound by memory: 16 bytes of each pair of elements (8192 positions of 8 heads of
// 128, 134 MB, 22 us).  (A CTA for both K and V has half as many on their way: 2048 positions 10.4 us, 8.2 so.)
template <int HD>
__global__ void __launch_bounds__(256) prefix_operands_kernel(const __grid_constant__ PrefixParams p, unsigned char *tiles, float2 *scales, uint32_t tile0) {
    using L = Layout<HD>;
    constexpr int N = HD / 32;  // pieces of eight elements per thread
    __shared__ uint32_t most_of[8];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y, at = (tile0 + blockIdx.x) * kKeys, keys = p.prefix_len - at;
    const bool of_k = blockIdx.z == 0;
    const size_t slot = (size_t)kvh * gridDim.x + blockIdx.x;
    const float *from = (of_k ? p.prefix_k : p.prefix_v) + (size_t)at * p.prefix_stride + (size_t)kvh * HD;
    // (behind the sequences' own positions, which it runs beside: they let it start when what came before them was over, and only one CTA's end waits for theirs)
    const bool waits = blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;
    if (!p.behind) yule_pdl_wait();
    yule_pdl_launch_dependents();
    // K: eight dimensions of a position; eight neighbouring lanes take eight positions (whole rows of core matrices), the four groups of a warp four steps of eight dimensions.
    // V: eight positions of a dimension; neighbouring lanes take neighbouring dimensions.
    const uint32_t key = warp * 8 + (lane & 7u), dim = tid % HD, first = tid / HD * 8;
    float x[N][8], most = 0.f;
    if (of_k) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) {
            const float4 *src = reinterpret_cast<const float4 *>(from + (size_t)key * p.prefix_stride + 32 * i + 8 * (lane >> 3));
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (key < keys) a = __ldcg(src), b = __ldcg(src + 1);
            x[i][0] = a.x, x[i][1] = a.y, x[i][2] = a.z, x[i][3] = a.w, x[i][4] = b.x, x[i][5] = b.y, x[i][6] = b.z, x[i][7] = b.w;
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < N; i++)
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) {
                const uint32_t j = first + i * (256 / HD) * 8 + e;
                x[i][e] = j < keys ? __ldcg(from + (size_t)j * p.prefix_stride + dim) : 0.f;
            }
    }
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int e = 0; e < 8; e++) most = fmaxf(most, fabsf(x[i][e]));
    const uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    if (lane == 0) most_of[warp] = all;
    __syncthreads();
    float scale, inv;
    pow2_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, most_of[lane & 7u])), scale, inv);
    if (tid == 0) (of_k ? scales[slot].x : scales[slot].y) = inv;
    unsigned char *to = tiles + slot * L::kTile + (of_k ? 0 : 2 * L::kPlane);
    const uint64_t two = pair(scale, scale);
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) split2(mul2(pair(x[i][2 * e], x[i][2 * e + 1]), two), hi[e], lo[e]);
        unsigned char *d = to + (of_k ? (4 * i + (lane >> 3)) * (kKeys * 16) + key * 16 : (i * 256 + tid) * 16);
        *reinterpret_cast<uint4 *>(d) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4 *>(d + L::kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
    if (p.behind && waits) yule_pdl_wait();
}

template <int HD>
__global__ void __launch_bounds__(640, 1) prefix_tc_kernel(  // (so many threads would leave each of them kLaunchRegs)
    const __grid_constant__ PrefixParams p, const unsigned char *tiles, const float2 *scales, uint32_t slot0, uint32_t tiles_in_memory) {
    using L = Layout<HD>;
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int KS = HD / 16;           // k16 steps of a score
    constexpr uint32_t kParts = HD / 64;  // of the output
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t slot = slot0 + blockIdx.x, row0 = blockIdx.y * kRows, kvh = blockIdx.z, n_rows = p.n_seqs * p.n_query * p.group;
    const uint32_t key0 = slot * p.prefix_chunk, keys = min(p.prefix_chunk, p.prefix_len - key0), n_tiles = (keys + kKeys - 1) / kKeys;
    const size_t tile0 = (size_t)kvh * tiles_in_memory + blockIdx.x * (p.prefix_chunk / kKeys);

    float *alpha_row = reinterpret_cast<float *>(smem + L::kOffRows), *most_row = alpha_row + 2 * kRows, *sum_row = most_row + 4 * kRows, *last_row = sum_row + 2 * kRows,
          *factor_row = last_row + kRows;
    float2 *inverse = reinterpret_cast<float2 *>(smem + L::kOffScales);  // of K and V, by tile
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    const uint32_t bar0 = smem_u32(bars);
    // pairs by tile parity: V there, free (and the probabilities used); scores there, free; probabilities there; alpha free; three: K there, free; by part: output there, free; else one: sums there
    const uint32_t v_full = bar0, v_empty = bar0 + 16, s_full = bar0 + 32, s_empty = bar0 + 48, p_full = bar0 + 64, a_empty = bar0 + 80, k_full = bar0 + 96, k_empty = bar0 + 120,
                   o_full = bar0 + 144, o_empty = bar0 + 160, l_full = bar0 + 176;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    if (tid == 0) {
        for (uint32_t b = 0; b < 3; b++) {
            mbar_init(k_full + 8 * b, 1);   // the loader's expect_tx
            mbar_init(k_empty + 8 * b, 1);  // tcgen05.commit
        }
        for (uint32_t b = 0; b < 2; b++) {
            mbar_init(v_full + 8 * b, 1);
            mbar_init(v_empty + 8 * b, 1);
            mbar_init(s_full + 8 * b, 1);
            mbar_init(s_empty + 8 * b, 8);
            mbar_init(p_full + 8 * b, 8);
            mbar_init(a_empty + 8 * b, 4);
            mbar_init(o_full + 8 * b, 2);  // tcgen05.commit, and the thread that saw the probabilities (and with them alpha) arrive
            mbar_init(o_empty + 8 * b, 4);
        }
        mbar_init(l_full, 8);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // What came before prefix_operands_kernel is over, or this kernel could not have started; only what reads that kernel's results waits for it.
    yule_pdl_launch_dependents();

    auto load = [&](uint32_t j, uint32_t to, uint32_t full, uint32_t from) {  // by one thread: two planes of tile j
        mbar_arrive_expect_tx(full, 2 * L::kPlane);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(smem + to)), "l"(tiles + (tile0 + j) * L::kTile + from),
                     "r"(2 * L::kPlane), "r"(full)
                     : "memory");
    };
    // The query rows, a warp after the other: loaded as they lie, scaled and split; then, a thread per row, into tensor memory.
    const uint32_t quarter = warp & 3u, r = quarter * 32 + lane, lanes = quarter << 21;
    uint32_t *q_words = reinterpret_cast<uint32_t *>(smem + L::kOffQ);  // [row][hi, lo]
    constexpr int kEach = kRows / (kThreads / 32), kPer = HD / 32;      // rows of a warp, elements of a lane
    float x[kEach][kPer];
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        uint32_t row = row0 + warp * kEach + i;
        row = row < n_rows ? row : n_rows - 1;
        const float *qp = p.q + (size_t)(row / p.group) * p.q_stride + (size_t)(kvh * p.group + row % p.group) * HD + lane * kPer;
        if constexpr (HD == 128) {
            const float4 v = __ldcg(reinterpret_cast<const float4 *>(qp));
            x[i][0] = v.x, x[i][1] = v.y, x[i][2] = v.z, x[i][3] = v.w;
        } else {
            const float2 v = __ldcg(reinterpret_cast<const float2 *>(qp));
            x[i][0] = v.x, x[i][1] = v.y;
        }
    }
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        float most = 0.f, scale, inv;
#pragma unroll
        for (int e = 0; e < kPer; e++) most = fmaxf(most, fabsf(x[i][e]));
        pow2_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(most))), scale, inv);
        uint32_t *to = q_words + (warp * kEach + i) * L::kPitch + lane * (kPer / 2);
#pragma unroll
        for (int e = 0; e < kPer; e += 2) split2(pair(x[i][e] * scale, x[i][e + 1] * scale), to[e / 2], to[HD / 2 + e / 2]);
        if (lane == 0) factor_row[warp * kEach + i] = inv * p.scale;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    if (warp == kKeyWarp || warp == kValueWarp) yule_pdl_wait();
    if (warp == kKeyWarp && lane == 0)  // (beside the query rows)
        for (uint32_t j = 0; j < 2 && j < n_tiles; j++) load(j, L::kOffK + j * 2 * L::kPlane, k_full + 8 * j, 0);
    if (warp < 4) {
        const uint4 *from = reinterpret_cast<const uint4 *>(q_words + r * L::kPitch);
#pragma unroll
        for (int i = 0; i < HD; i += 8) tmem_st8(tmem_base + lanes + L::kQ + i, from[i / 4], from[i / 4 + 1]);
        tmem_st_wait();
    } else if (warp < kMmaWarp) {
        yule_pdl_wait();
        for (uint32_t j = tid - 128; j < n_tiles; j += 256) inverse[j] = __ldcg(scales + tile0 + j);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp >= kMmaWarp) {
        move_registers<true, kIssueRegs, kLaunchRegs>();
        constexpr uint32_t idesc = (1u << 4) | (64u >> 3 << 17) | ((uint32_t)(kRows >> 4) << 24);  // fp16 × fp16 → fp32, K-major, M = 128, N = 64 positions, or dimensions of a part
        constexpr uint64_t plane = L::kPlane >> 4;
        static_assert(kKeys == 64, "N");
        bool ok = true;
        auto await = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_wait(bar, parity, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            return ok;
        };
        const uint32_t base = smem_u32(smem);
        if (warp == kMmaWarp) {
            RingPos kr;
            for (uint32_t j = 0; j < n_tiles; j++, kr.advance(3)) {
                const uint32_t b = j & 1u;
                if (!await(k_full + 8 * kr.s, kr.ph) || !await(s_empty + 8 * b, ((j >> 1) & 1u) ^ 1u)) break;
                const uint32_t d = tmem_base + L::kS + b * 64, q_hi = tmem_base + L::kQ, q_lo = q_hi + HD / 2;
                const uint64_t kd = smem_desc(base + L::kOffK + kr.s * 2 * L::kPlane, kKeys * 16, 128);
                constexpr uint64_t step = (2 * kKeys * 16) >> 4;
                if (elect_one()) {
                    mma_steps<0, KS>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<(i != 0)>(d, q_lo + 8 * i, kd + i * step, idesc);
                        umma_f16_ts<1>(d, q_hi + 8 * i, kd + i * step + plane, idesc);
                    });
                    mma_steps<0, KS>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<1>(d, q_hi + 8 * i, kd + i * step, idesc);
                    });
                    umma_commit(k_empty + 8 * kr.s);
                    umma_commit(s_full + 8 * b);
                }
                __syncwarp();
            }
        } else if (warp == kOutputWarp) {
            for (uint32_t j = 0; j < n_tiles && ok; j++) {
                const uint32_t b = j & 1u, ph = (j >> 1) & 1u;
                if (!await(v_full + 8 * b, ph) || !await(p_full + 8 * b, ph)) break;
                const uint64_t vd = smem_desc(base + L::kOffV + b * 2 * L::kPlane, HD * 16, 128);
                constexpr uint64_t step = (2 * HD * 16) >> 4;
                const uint32_t hi = tmem_base + L::kP + b * 64, lo = hi + 32;
                mma_steps<0, kParts>([&](auto pc) {
                    constexpr uint32_t part = decltype(pc)::value;
                    constexpr uint64_t dims = (part * 64 * 16) >> 4;
                    if (!ok || !await(o_empty + 8 * part, (j & 1u) ^ 1u)) return;
                    const uint32_t d = tmem_base + L::kO + 64 * part;
                    if (elect_one()) {
                        mma_steps<0, 4>([&](auto ic) {
                            constexpr uint32_t i = decltype(ic)::value;
                            umma_f16_ts<(i != 0)>(d, lo + 8 * i, vd + i * step + dims, idesc);
                            umma_f16_ts<1>(d, hi + 8 * i, vd + i * step + dims + plane, idesc);
                        });
                        mma_steps<0, 4>([&](auto ic) {
                            constexpr uint32_t i = decltype(ic)::value;
                            umma_f16_ts<1>(d, hi + 8 * i, vd + i * step + dims, idesc);
                        });
                        if (part + 1 == kParts) umma_commit(v_empty + 8 * b);
                        umma_commit(o_full + 8 * part);  // (the last of all: what waits for the last tile's knows that nothing is under way)
                        mbar_arrive(o_full + 8 * part);
                    }
                    __syncwarp();
                });
            }
        } else if (warp == kKeyWarp && lane == 0) {
            RingPos kr;
            kr.advance(3), kr.advance(3);
            for (uint32_t j = 2; j < n_tiles && ok; j++, kr.advance(3)) {
                ok = mbar_wait(k_empty + 8 * kr.s, kr.ph ^ 1u, abort_flag, p.status);
                if (ok) load(j, L::kOffK + kr.s * 2 * L::kPlane, k_full + 8 * kr.s, 0);
            }
        } else if (warp == kValueWarp && lane == 0) {
            for (uint32_t j = 0; j < n_tiles && ok; j++) {
                const uint32_t b = j & 1u;
                ok = mbar_wait(v_empty + 8 * b, ((j >> 1) & 1u) ^ 1u, abort_flag, p.status);
                if (ok) load(j, L::kOffV + b * 2 * L::kPlane, v_full + 8 * b, 2 * L::kPlane);
            }
        }
    } else if (warp < kSumWarp) {
        const uint32_t half = warp >> 2, col0 = half * (kKeys / 2);
        const float row_factor = factor_row[r];
        float m = -FLT_MAX, l = 0.f;
        bool ok = true;
        // (A warp that gives up goes on to meet the other half at the barrier of every tile, which has no bound.)
        auto await = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_wait(bar, parity, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
        };
        for (uint32_t j = 0; j < n_tiles; j++) {
            const uint32_t b = j & 1u, ph = (j >> 1) & 1u;
            const float f = fmaxf(row_factor * inverse[j].x, FLT_MIN);  // (never 0: a position that is not there has a score of −infinity)
            await(a_empty + 8 * b, ph ^ 1u);  // alpha of the tile before the last has been read, behind its output: its probabilities have been used
            await(s_full + 8 * b, ph);
            tc_fence_after();
            uint32_t a[32];
            float mx4[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};
            if (ok) {
                tmem_ld32_issue(tmem_base + lanes + L::kS + b * 64 + col0, a);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty + 8 * b);
                const uint32_t seen = keys - min(keys, j * kKeys + col0);  // positions of this half that are there (or more)
                if (seen < kKeys / 2)
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) a[i] = i < seen ? a[i] : 0xFF800000u;
#pragma unroll
                for (uint32_t i = 0; i < 32; i++) mx4[i & 3] = fmaxf(mx4[i & 3], __uint_as_float(a[i]));
            }
            // The row's largest score, from both halves.  (Words by tile parity: who writes a tile's has met the other half behind its reading of the tile before the last.)
            const float most = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            most_row[(b * 2 + half) * kRows + r] = most;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
            const float mx = fmaxf(most, most_row[(b * 2 + (half ^ 1u)) * kRows + r]);
            const float mn = fmaxf(m, mx * f);
            const float alpha = power(m - mn);
            m = mn;
            if (ok) {
                if (half == 0) alpha_row[b * kRows + r] = alpha;
                const uint64_t f2 = pair(f, f), less2 = pair(kProbBits - mn, kProbBits - mn);
                uint64_t sum2 = 0;
                const uint32_t to = tmem_base + lanes + L::kP + b * 64 + col0 / 2;
#pragma unroll
                for (uint32_t c0 = 0; c0 < kKeys / 2; c0 += 16) {
                    uint32_t hi[8], lo[8];
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) {
                        const float2 e = unpair(fma2(pair_bits(a[c0 + 2 * i], a[c0 + 2 * i + 1]), f2, less2));
                        const uint64_t w = pair(power(e.x), power(e.y));
                        sum2 = add2(sum2, w);
                        split2(w, hi[i], lo[i]);
                    }
                    tmem_st8(to + c0 / 2, make_uint4(hi[0], hi[1], hi[2], hi[3]), make_uint4(hi[4], hi[5], hi[6], hi[7]));
                    tmem_st8(to + 32 + c0 / 2, make_uint4(lo[0], lo[1], lo[2], lo[3]), make_uint4(lo[4], lo[5], lo[6], lo[7]));
                }
                const float2 sums = unpair(sum2);
                l = fmaf(l, alpha, sums.x + sums.y);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * b);
            }
        }
        sum_row[half * kRows + r] = l;
        if (half == 0) last_row[r] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(l_full);
    } else {
        // output sums: this thread's row
        move_registers<true, kSumRegs, kLaunchRegs>();
        uint64_t o[HD / 2];
#pragma unroll
        for (int i = 0; i < HD / 2; i++) o[i] = 0;
        bool ok = true;
        for (uint32_t j = 0; j < n_tiles && ok; j++) {
            float alpha = 0.f;
            const float vi = inverse[j].y;
#pragma unroll
            for (uint32_t part = 0; part < kParts; part++) {
                ok = ok && mbar_wait(o_full + 8 * part, j & 1u, abort_flag, p.status);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                if (part == 0) alpha = alpha_row[(j & 1u) * kRows + r];
                if (part + 1 == kParts) {  // (all of the tile has been multiplied: its probabilities may be overwritten too)
                    __syncwarp();
                    if (lane == 0) mbar_arrive(a_empty + 8 * (j & 1u));
                }
                const uint64_t alpha2 = pair(alpha, alpha), vi2 = pair(vi, vi);
#pragma unroll
                for (uint32_t c0 = 64 * part; c0 < 64 * part + 64; c0 += 16) {
                    uint32_t y[16];
                    tmem_ld16_issue(tmem_base + lanes + L::kO + c0, y);
                    tmem_ld_wait();
                    if (c0 + 16 == 64 * part + 64) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(o_empty + 8 * part);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 16; i += 2) o[(c0 + i) / 2] = fma2(o[(c0 + i) / 2], alpha2, mul2(pair_bits(y[i], y[i + 1]), vi2));
                }
            }
        }
        ok = ok && mbar_wait(l_full, 0, abort_flag, p.status);
        ok = __all_sync(0xffffffffu, ok);
        if (ok) {
            // (the last MMAs and copies are over: K and V are done with)  A row per thread into shared memory
            float *mine = reinterpret_cast<float *>(smem) + r * L::kPitch;
            const uint64_t lost = pair(kTruncation, kTruncation);
#pragma unroll
            for (uint32_t i = 0; i < HD; i += 4) {
                const float2 u = unpair(fma2(o[i / 2], lost, o[i / 2])), w = unpair(fma2(o[i / 2 + 1], lost, o[i / 2 + 1]));
                *reinterpret_cast<float4 *>(mine + i) = make_float4(u.x, u.y, w.x, w.y);
            }
        }
    }

    // nothing of this CTA may still be in flight when its TMEM and shared memory go
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (!*abort_flag && warp < kSumWarp) {
        // the rows as they lie in memory, sixteen per soft-max warp (which have the registers that the kernel was compiled to)
        static_assert(kSoftRegs >= kLaunchRegs, "registers");
        constexpr uint32_t kMine = kRows / kSumWarp;
        constexpr uint32_t kLanes = HD / 4, kStep = 32 / kLanes;  // lanes per row, rows at a time
        const float *rows = reinterpret_cast<const float *>(smem);
        uint32_t at = warp * kMine + lane / kLanes, row = row0 + at, token = row / p.group, head = row - token * p.group;
        const uint32_t d = lane % kLanes * 4;
#pragma unroll 8
        for (uint32_t i = 0; i < kMine / kStep; i++, at += kStep, row += kStep) {
            if (row < n_rows) {
                const size_t part = ((size_t)token * p.n_heads + kvh * p.group + head) * p.slots + slot;
                *reinterpret_cast<float4 *>(p.part_o + part * HD + d) = *reinterpret_cast<const float4 *>(rows + at * L::kPitch + d);
                if (d == 0) p.part_ml[part] = make_float2(last_row[at] - kProbBits, sum_row[at] + sum_row[kRows + at]);
            }
            for (head += kStep; head >= p.group; head -= p.group) token++;
        }
    }

    if (*abort_flag) {
        // gave up: let MMAs and copies that were already issued drain before the resources are freed
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {
        }
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
    }
}

// Chunks of the prefix whose operands are in memory at a time.
uint32_t chunks_at_a_time(const PrefixParams &p) {
    constexpr size_t kMostBytes = (size_t)512 << 20;
    const size_t chunk = (size_t)p.prefix_chunk * p.n_kv_heads * p.hd * 8;
    return chunk >= kMostBytes ? 1 : (uint32_t)(kMostBytes / chunk);
}

template <int HD>
cudaError_t launch_variant(PrefixParams p, void *scratch, bool pdl, cudaStream_t s, uint64_t *launches) {
    auto kern = prefix_tc_kernel<HD>;
    static bool attr_done[64] = {};  // the opt-in for large dynamic shared memory belongs to the device
    static std::mutex mu;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    {
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 0 || dev >= 64 || !attr_done[dev]) {
            cudaFuncAttributes fa;  // the split of the registers counts on what the launch brings: a library that was not built by build.py must not hang
            e = cudaFuncGetAttributes(&fa, kern);
            if (e == cudaSuccess && fa.numRegs < kLaunchRegs) e = cudaErrorInvalidValue;
            if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Layout<HD>::kSmem);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) attr_done[dev] = true;
        }
    }
    const uint32_t at_a_time = chunks_at_a_time(p), per_chunk = p.prefix_chunk / kKeys, all = (p.prefix_len + kKeys - 1) / kKeys;
    for (uint32_t slot0 = 0; slot0 < p.prefix_splits; slot0 += at_a_time) {
        const uint32_t chunks = p.prefix_splits - slot0 < at_a_time ? p.prefix_splits - slot0 : at_a_time, tile0 = slot0 * per_chunk;
        const uint32_t n = all - tile0 < chunks * per_chunk ? all - tile0 : chunks * per_chunk;
        unsigned char *tiles = static_cast<unsigned char *>(scratch);
        float2 *scales = reinterpret_cast<float2 *>(tiles + (size_t)n * p.n_kv_heads * Layout<HD>::kTile);
        e = launch_kernel(prefix_operands_kernel<HD>, dim3(n, p.n_kv_heads, 2), dim3(256), 0, s, pdl || slot0 > 0, p, tiles, scales, tile0);
        if (e == cudaSuccess)
            e = launch_kernel(kern, dim3(chunks, p.prefix_row_tiles, p.n_kv_heads), dim3(kThreads), Layout<HD>::kSmem, s, true, p, static_cast<const unsigned char *>(tiles),
                              static_cast<const float2 *>(scales), slot0, n);
        if (e != cudaSuccess) return e;
        *launches += 2;
        p.behind = false;
    }
    return cudaSuccess;
}

}  // namespace

bool prefix_tc_supported(uint32_t hd, uint64_t rows) { return (hd == 64 || hd == 128) && rows <= 65535ull * kPrefixTcRows; }

size_t prefix_tc_scratch_bytes(const PrefixParams &p) {
    const size_t tiles = (size_t)(p.prefix_len + kKeys - 1) / kKeys, most = (size_t)chunks_at_a_time(p) * (p.prefix_chunk / kKeys);
    return (tiles < most ? tiles : most) * p.n_kv_heads * ((size_t)kKeys * p.hd * 8 + sizeof(float2)) + 256;
}

cudaError_t launch_prefix_tc(const PrefixParams &p, void *scratch, bool pdl, cudaStream_t s, uint64_t *launches) {
    if (p.prefix_chunk % kPrefixTcKeys || p.prefix_chunk / kPrefixTcKeys > kMostTiles || p.prefix_row_tiles > 65535 || p.n_kv_heads > 65535 || !p.status) return cudaErrorInvalidValue;
    return p.hd == 64 ? launch_variant<64>(p, scratch, pdl, s, launches) : p.hd == 128 ? launch_variant<128>(p, scratch, pdl, s, launches) : cudaErrorInvalidValue;
}

}  // namespace yule
