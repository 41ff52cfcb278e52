// prefix_attention_tc.cu — the shared prefix of a batch for 128 query rows at a time, on tcgen05.
//
// A CTA has 128 query rows of one KV head (query tokens of all sequences one after the other, the heads of the group within a token) and a chunk of the prefix, of which
// every row sees every position; it leaves (m, Σ, o) of each row, which prefix_merge_kernel adds to the other parts.
//
// Precision.  The tensor core multiplies fp16 and truncates what it adds to.  A query row, and the K and V of a tile of 64 positions, are scaled by powers of two so that their largest
// element is 2^13 to 2^14, and split into hi + lo (22 bits; what is 2^-14 of the largest loses the lower ones).  A score, and an output of a tile, is the small products first,
// then hi·hi; outputs of tiles are added up in fp32, with the mean of what truncation takes given back.  A value that is not finite makes every row's output not
// finite: every row sees it.
//
// Roles (512 threads): eight warps convert and do the soft-max (a thread per row and half a tile's positions), four add the output up (a thread per row), one issues the MMAs, one
// the copies.  The fp32 K and V of the next tile come to shared memory by tiled bulk copies (asked for into registers instead, they were waited for with the next load
// from tensor memory: 7400 clocks a tile).  The query rows are in tensor memory.  K has one buffer of operands (the next tile's is written when this one's scores are there, and multiplied under
// this one's soft-max), V, scores and probabilities have two.

#include <cfloat>
#include <mutex>
#include <type_traits>

#include <cuda.h>
#include <cuda_fp16.h>

#include "prefix_attention.cuh"
#include "qgemm_common.cuh"

namespace yule {

namespace {

constexpr int kRows = (int)kPrefixTcRows;  // query rows per CTA = TMEM lanes
constexpr int kKeys = (int)kPrefixTcKeys;  // positions per tile
constexpr int kThreads = 512, kWorkers = 256, kMmaWarp = 12, kLoadWarp = 13;
constexpr int kLaunchRegs = 128;  // registers per thread that 512 threads are launched with (the build checks that the kernels get them)
constexpr int kWorkRegs = 152, kSumRegs = 168, kIssueRegs = 40;
static_assert(2 * kWorkRegs + kSumRegs + kIssueRegs <= 4 * kLaunchRegs, "register split");
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

struct PrefixMaps {
    CUtensorMap k, v;  // rows of the prefix in boxes of 64 positions by 32 dimensions, swizzled within 128 bytes
};

template <int HD>
struct Layout {
    // K and V of a tile as they come: per 32 dimensions a box of 64 rows of 128 bytes, whose eight 16-byte pieces are exchanged by the row's number.
    static constexpr uint32_t kRaw = kKeys * HD * 4, kOffRawK = 0, kOffRawV = kRaw;
    // Operands in the no-swizzle core-matrix layout (8 rows x 16 bytes; core matrices of one step of eight contiguous along the rows): K rows by
    // dimension, V transposed: dimensions by position.
    static constexpr uint32_t kPlane = kKeys * HD * 2, kOffK = 2 * kRaw, kOffV = kOffK + 2 * kPlane, kOffRows = kOffV + 2 * 2 * kPlane;  // two buffers of V
    // per row: alpha (two tiles), largest score of either half (two tiles; before them, largest elements of the query row's quarters), sums of either half, last largest score;
    // then the warps' largest elements of K and V (two tiles), inverse scales of V (four tiles); then barriers
    static constexpr uint32_t kOffMost = kOffRows + 9 * kRows * 4, kOffBars = kOffMost + (32 + 4) * 4, kBars = 20;
    static constexpr uint32_t kSmem = kOffBars + kBars * 8 + 16;
    // tensor memory columns: two buffers of scores, output, two buffers of probabilities (hi, lo), query rows (hi, lo)
    static constexpr uint32_t kS = 0, kO = 128, kP = 256, kQ = 384;
    static_assert(kSmem <= 227 * 1024 && kOffBars % 8 == 0, "shared memory");
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) prefix_tc_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ PrefixMaps maps) {
    using L = Layout<HD>;
    extern __shared__ __align__(1024) unsigned char smem[];
    constexpr int KS = HD / 16;  // k16 steps of a score
    constexpr int N = HD / 32;   // pieces of eight elements of K, and of V, per worker and tile
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t slot = blockIdx.x, row0 = blockIdx.y * kRows, kvh = blockIdx.z, n_rows = p.n_seqs * p.n_query * p.group;
    const uint32_t key0 = slot * p.prefix_chunk, keys = min(p.prefix_chunk, p.prefix_len - key0), n_tiles = (keys + kKeys - 1) / kKeys;

    float *alpha_row = reinterpret_cast<float *>(smem + L::kOffRows), *most_row = alpha_row + 2 * kRows, *sum_row = most_row + 4 * kRows, *last_row = sum_row + 2 * kRows;
    uint32_t *most_of = reinterpret_cast<uint32_t *>(smem + L::kOffMost);  // [K, V][tile parity][worker warp]
    float *v_inv = reinterpret_cast<float *>(most_of + 32);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    const uint32_t bar0 = smem_u32(bars);
    // pairs by tile parity: V there; scores there, free; probabilities there; probabilities and V used; alpha free; else one: K there; output there, free; sums there; raw K there, free,
    // raw V there, free
    const uint32_t v_full = bar0, s_full = bar0 + 16, s_empty = bar0 + 32, p_full = bar0 + 48, pv_done = bar0 + 64, a_empty = bar0 + 80, k_full = bar0 + 96, o_full = bar0 + 104,
                   o_empty = bar0 + 112, l_full = bar0 + 120, rk_full = bar0 + 128, rk_empty = bar0 + 136, rv_full = bar0 + 144, rv_empty = bar0 + 152;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + L::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    if (tid == 0) {
        for (uint32_t b = 0; b < 2; b++) {
            mbar_init(v_full + 8 * b, 8);
            mbar_init(s_full + 8 * b, 1);  // tcgen05.commit
            mbar_init(s_empty + 8 * b, 8);
            mbar_init(p_full + 8 * b, 8);
            mbar_init(pv_done + 8 * b, 1);  // tcgen05.commit
            mbar_init(a_empty + 8 * b, 4);
        }
        mbar_init(k_full, 8);
        mbar_init(o_full, 2);  // tcgen05.commit, and the thread that saw the probabilities (and with them alpha) arrive
        mbar_init(o_empty, 4);
        mbar_init(l_full, 8);
        mbar_init(rk_full, 1);  // the loader's expect_tx
        mbar_init(rk_empty, 8);
        mbar_init(rv_full, 1);
        mbar_init(rv_empty, 8);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
    }
    if (warp == kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    yule_pdl_wait();
    yule_pdl_launch_dependents();  // (what comes behind may start: all that this kernel waits for is over)

    auto load = [&](uint32_t j, bool is_k) {  // by one thread
        const uint32_t full = is_k ? rk_full : rv_full, to = smem_u32(smem + (is_k ? L::kOffRawK : L::kOffRawV));
        mbar_arrive_expect_tx(full, L::kRaw);
#pragma unroll
        for (uint32_t i = 0; i < N; i++)  // (elements of eight bytes)
            asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(to + i * (kKeys * 128)),
                         "l"(reinterpret_cast<uint64_t>(is_k ? &maps.k : &maps.v)), "r"(full), "r"(kvh * (HD / 2) + 16 * i), "r"(key0 + j * kKeys)
                         : "memory");
    };
    // The query rows: a thread of four warps each, a quarter of the dimensions.
    const uint32_t quarter = warp & 3u, r = quarter * 32 + lane, lanes = quarter << 21;
    float4 x[HD / 16];
    float row_max = 0.f, row_scale, row_factor;
    {
        uint32_t row = row0 + r;
        row = row < n_rows ? row : n_rows - 1;
        const float *qp = p.q + (size_t)(row / p.group) * p.q_stride + (size_t)(kvh * p.group + row % p.group) * HD + (warp >> 2) * (HD / 4);
#pragma unroll
        for (int i = 0; i < HD / 16; i++) x[i] = __ldcg(reinterpret_cast<const float4 *>(qp) + i);
#pragma unroll
        for (int i = 0; i < HD / 16; i++) row_max = fmaxf(fmaxf(row_max, fmaxf(fabsf(x[i].x), fabsf(x[i].y))), fmaxf(fabsf(x[i].z), fabsf(x[i].w)));
        most_row[(warp >> 2) * kRows + r] = row_max;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    if (warp == kLoadWarp && lane == 0) load(0, true), load(0, false);
    {
#pragma unroll
        for (int i = 0; i < 4; i++) row_max = fmaxf(row_max, most_row[i * kRows + r]);
        float inv;
        pow2_scale(row_max, row_scale, inv);
        row_factor = inv * p.scale;
        const uint64_t scale2 = pair(row_scale, row_scale);
        uint32_t hi[HD / 8], lo[HD / 8];
#pragma unroll
        for (int i = 0; i < HD / 16; i++) {
            split2(mul2(pair(x[i].x, x[i].y), scale2), hi[2 * i], lo[2 * i]);
            split2(mul2(pair(x[i].z, x[i].w), scale2), hi[2 * i + 1], lo[2 * i + 1]);
        }
        const uint32_t to = tmem_base + lanes + L::kQ + (warp >> 2) * (HD / 8);
#pragma unroll
        for (int i = 0; i < HD / 8; i += 8) {
            tmem_st8(to + i, make_uint4(hi[i], hi[i + 1], hi[i + 2], hi[i + 3]), make_uint4(hi[i + 4], hi[i + 5], hi[i + 6], hi[i + 7]));
            tmem_st8(to + HD / 2 + i, make_uint4(lo[i], lo[i + 1], lo[i + 2], lo[i + 3]), make_uint4(lo[i + 4], lo[i + 5], lo[i + 6], lo[i + 7]));
        }
        tmem_st_wait();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp >= 12) {
        move_registers<true, kIssueRegs, kLaunchRegs>();
        if (warp == kMmaWarp) {
            constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);  // fp16 × fp16 → fp32, K-major, M = 128, N = 64
            constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);     // N = head_dim
            constexpr uint64_t plane = L::kPlane >> 4;
            bool ok = true;
            auto await = [&](uint32_t bar, uint32_t parity) {
                ok = ok && mbar_wait(bar, parity, abort_flag, p.status);
                ok = __all_sync(0xffffffffu, ok);
                tc_fence_after();
                return ok;
            };
            const uint32_t base = smem_u32(smem);
            auto scores = [&](uint32_t j) {
                const uint32_t b = j & 1u;
                if (!await(s_empty + 8 * b, ((j >> 1) & 1u) ^ 1u) || !await(k_full, j & 1u)) return;
                const uint32_t d = tmem_base + L::kS + b * 64, q_hi = tmem_base + L::kQ, q_lo = q_hi + HD / 2;
                const uint64_t kd = smem_desc(base + L::kOffK, kKeys * 16, 128);
                constexpr uint64_t step = (2 * kKeys * 16) >> 4;
                if (elect_one()) {
                    mma_steps<0, KS>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<(i != 0)>(d, q_lo + 8 * i, kd + i * step, idesc_s);
                        umma_f16_ts<1>(d, q_hi + 8 * i, kd + i * step + plane, idesc_s);
                    });
                    mma_steps<0, KS>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<1>(d, q_hi + 8 * i, kd + i * step, idesc_s);
                    });
                    umma_commit(s_full + 8 * b);
                }
                __syncwarp();
            };
            scores(0);
            for (uint32_t j = 0; j < n_tiles && ok; j++) {
                if (j + 1 < n_tiles) scores(j + 1);
                if (!ok) break;
                const uint32_t b = j & 1u, ph = (j >> 1) & 1u;
                if (!await(v_full + 8 * b, ph) || !await(o_empty, (j & 1u) ^ 1u) || !await(p_full + 8 * b, ph)) break;
                const uint64_t vd = smem_desc(base + L::kOffV + b * 2 * L::kPlane, HD * 16, 128);
                constexpr uint64_t step = (2 * HD * 16) >> 4;
                const uint32_t d = tmem_base + L::kO, hi = tmem_base + L::kP + b * 64, lo = hi + 32;
                if (elect_one()) {
                    mma_steps<0, 4>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<(i != 0)>(d, lo + 8 * i, vd + i * step, idesc_o);
                        umma_f16_ts<1>(d, hi + 8 * i, vd + i * step + plane, idesc_o);
                    });
                    mma_steps<0, 4>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<1>(d, hi + 8 * i, vd + i * step, idesc_o);
                    });
                    umma_commit(o_full);
                    umma_commit(pv_done + 8 * b);
                    mbar_arrive(o_full);
                }
                __syncwarp();
            }
        } else if (warp == kLoadWarp && lane == 0) {
            for (uint32_t j = 1; j < n_tiles; j++) {
                if (!mbar_wait(rk_empty, (j & 1u) ^ 1u, abort_flag, p.status)) break;
                load(j, true);
                if (!mbar_wait(rv_empty, (j & 1u) ^ 1u, abort_flag, p.status)) break;
                load(j, false);
            }
        }
    } else if (warp < 8) {
        const uint32_t half = warp >> 2, col0 = half * (kKeys / 2);
        float m = -FLT_MAX, l = 0.f, k_inv, k_inv_next, k_scale = 0.f;
        float4 k[N][2];
        bool ok = true;
        // (A warp that gives up goes on to meet the others at the barriers of every tile, which have no bound.)
        auto await = [&](uint32_t bar, uint32_t parity) {
            ok = ok && mbar_wait(bar, parity, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
        };
        // The largest element of a tile, of all workers.  (Two words per warp, by tile parity: who writes a tile's has met everybody behind the reading of the tile before the last.)
        auto largest = [&](float most, uint32_t which, uint32_t j) {
            const uint32_t all = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
            uint32_t *words = most_of + (which * 2 + (j & 1u)) * 8;
            if (lane == 0) words[warp] = all;
            asm volatile("bar.sync %0, %1;" ::"r"(5 + which), "n"(kWorkers) : "memory");
            return __uint_as_float(__reduce_max_sync(0xffffffffu, words[lane & 7u]));
        };
        // K: eight dimensions of a position; eight neighbouring lanes take eight positions (whole rows of core matrices), the four groups of a warp four steps.
        auto place = [&](uint32_t i, uint32_t &key, uint32_t &step) {
            const uint32_t unit = i * 8 + warp;
            key = (unit & 7u) * 8 + (lane & 7u), step = (unit >> 3) * 4 + (lane >> 3);
        };
        auto read_k = [&](uint32_t j) {
            await(rk_full, j & 1u);
            float most = 0.f;
            if (ok) {
#pragma unroll
                for (uint32_t i = 0; i < N; i++) {
                    uint32_t key, step;
                    place(i, key, step);
                    const unsigned char *from = smem + L::kOffRawK + (step >> 2) * (kKeys * 128) + key * 128;
#pragma unroll
                    for (uint32_t e = 0; e < 2; e++) {
                        k[i][e] = *reinterpret_cast<const float4 *>(from + ((((step & 3u) * 2 + e) ^ (key & 7u)) << 4));
                        most = fmaxf(fmaxf(most, fmaxf(fabsf(k[i][e].x), fabsf(k[i][e].y))), fmaxf(fabsf(k[i][e].z), fabsf(k[i][e].w)));
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(rk_empty);
            }
            pow2_scale(largest(most, 0, j), k_scale, k_inv_next);
        };
        auto store_k = [&] {
            if (!ok) return;
            const uint64_t scale2 = pair(k_scale, k_scale);
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                uint32_t key, step, hi[4], lo[4];
                place(i, key, step);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    split2(mul2(pair(k[i][e].x, k[i][e].y), scale2), hi[2 * e], lo[2 * e]);
                    split2(mul2(pair(k[i][e].z, k[i][e].w), scale2), hi[2 * e + 1], lo[2 * e + 1]);
                }
                unsigned char *to = smem + L::kOffK + step * (kKeys * 16) + key * 16;
                *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(to + L::kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full);
        };
        // V: eight positions of a dimension; neighbouring lanes take neighbouring dimensions.
        auto convert_v = [&](uint32_t j) {
            await(rv_full, j & 1u);
            float v[N][8], most = 0.f, scale, inv;
            if (ok) {
#pragma unroll
                for (uint32_t i = 0; i < N; i++) {
                    const uint32_t unit = i * kWorkers + tid, dim = unit % HD, key = unit / HD * 8;
                    const unsigned char *from = smem + L::kOffRawV + (dim >> 5) * (kKeys * 128) + key * 128 + (dim & 3u) * 4;
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) {
                        v[i][e] = *reinterpret_cast<const float *>(from + e * 128 + ((((dim & 31u) >> 2) ^ e) << 4));
                        most = fmaxf(most, fabsf(v[i][e]));
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(rv_empty);
            }
            pow2_scale(largest(most, 1, j), scale, inv);
            await(pv_done + 8 * (j & 1u), ((j >> 1) & 1u) ^ 1u);  // the tile that had this buffer has been multiplied (and its probabilities used)
            if (!ok) return;
            const uint64_t scale2 = pair(scale, scale);
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int e = 0; e < 4; e++) split2(mul2(pair(v[i][2 * e], v[i][2 * e + 1]), scale2), hi[e], lo[e]);
                unsigned char *to = smem + L::kOffV + (j & 1u) * 2 * L::kPlane + (i * kWorkers + tid) * 16;
                *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                *reinterpret_cast<uint4 *>(to + L::kPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            }
            if (tid == 0) v_inv[j & 3u] = inv;
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full + 8 * (j & 1u));
        };
        move_registers<true, kWorkRegs, kLaunchRegs>();
        read_k(0);
        store_k();
        k_inv = k_inv_next;
        convert_v(0);
        for (uint32_t j = 0; j < n_tiles; j++) {
            const uint32_t b = j & 1u, ph = (j >> 1) & 1u;
            if (j + 1 < n_tiles) read_k(j + 1);
            await(s_full + 8 * b, ph);
            tc_fence_after();
            if (j + 1 < n_tiles) store_k();  // this tile's K has been multiplied: the next one's takes its place
            const float f = fmaxf(row_factor * k_inv, FLT_MIN);  // (never 0: a position that is not there has a score of −infinity)
            k_inv = k_inv_next;
            const uint32_t seen = keys - min(keys, j * kKeys + col0);  // positions of this half that are there (or more)
            uint32_t a[32];
            float mx4[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};
            if (ok) {
                tmem_ld32_issue(tmem_base + lanes + L::kS + b * 64 + col0, a);
                tmem_ld_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty + 8 * b);
                if (seen < kKeys / 2)
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) a[i] = i < seen ? a[i] : 0xFF800000u;  // −infinity: no probability
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
            await(a_empty + 8 * b, ph ^ 1u);
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
            if (j + 1 < n_tiles) convert_v(j + 1);
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
        for (uint32_t j = 0; j < n_tiles; j++) {
            ok = mbar_wait(o_full, j & 1u, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const float alpha = alpha_row[(j & 1u) * kRows + r], vi = v_inv[j & 3u];
            __syncwarp();
            if (lane == 0) mbar_arrive(a_empty + 8 * (j & 1u));
            const uint64_t alpha2 = pair(alpha, alpha), vi2 = pair(vi, vi);
#pragma unroll
            for (uint32_t c0 = 0; c0 < HD; c0 += 32) {
                uint32_t y[32];
                tmem_ld32_issue(tmem_base + lanes + L::kO + c0, y);
                tmem_ld_wait();
                if (c0 + 32 == HD) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_empty);
                }
#pragma unroll
                for (uint32_t i = 0; i < 32; i += 2) o[(c0 + i) / 2] = fma2(o[(c0 + i) / 2], alpha2, mul2(pair_bits(y[i], y[i + 1]), vi2));
            }
        }
        if (ok) ok = mbar_wait(l_full, 0, abort_flag, p.status);
        const uint32_t row = row0 + r;
        if (ok && row < n_rows) {
            const size_t part = ((size_t)(row / p.group) * p.n_heads + kvh * p.group + row % p.group) * p.slots + slot;
            p.part_ml[part] = make_float2(last_row[r] - kProbBits, sum_row[r] + sum_row[kRows + r]);
            float *to = p.part_o + part * HD;
            const uint64_t lost = pair(kTruncation, kTruncation);
#pragma unroll
            for (uint32_t i = 0; i < HD; i += 4) {
                const float2 u = unpair(fma2(o[i / 2], lost, o[i / 2])), w = unpair(fma2(o[i / 2 + 1], lost, o[i / 2 + 1]));
                *reinterpret_cast<float4 *>(to + i) = make_float4(u.x, u.y, w.x, w.y);
            }
        }
    }

    // common exit: nothing of this CTA may still be in flight when its TMEM and shared memory go
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
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

template <int HD>
cudaError_t launch_variant(const PrefixParams &p, bool pdl, cudaStream_t s) {
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
    alignas(64) PrefixMaps maps;
    e = cached_tensor_map_2d(p.prefix_k, 8, (uint64_t)p.n_kv_heads * HD / 2, p.prefix_len, p.prefix_stride * 4, 16, kKeys, &maps.k, 128);
    if (e == cudaSuccess) e = cached_tensor_map_2d(p.prefix_v, 8, (uint64_t)p.n_kv_heads * HD / 2, p.prefix_len, p.prefix_stride * 4, 16, kKeys, &maps.v, 128);
    if (e != cudaSuccess) return e;
    return launch_kernel(kern, dim3(p.prefix_splits, p.prefix_row_tiles, p.n_kv_heads), dim3(kThreads), Layout<HD>::kSmem, s, pdl, p, maps);
}

}  // namespace

bool prefix_tc_supported(uint32_t hd) { return hd == 64 || hd == 128; }

cudaError_t launch_prefix_tc(const PrefixParams &p, bool pdl, cudaStream_t s, uint64_t *launches) {
    if (p.prefix_chunk % kPrefixTcKeys || p.prefix_row_tiles > 65535 || p.n_kv_heads > 65535 || !p.status) return cudaErrorInvalidValue;
    const cudaError_t e = p.hd == 64 ? launch_variant<64>(p, pdl, s) : p.hd == 128 ? launch_variant<128>(p, pdl, s) : cudaErrorInvalidValue;
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace yule
