// prefix_attention_tc.cu — the shared prefix of a batch for 128 query rows at a time, on tcgen05.
//
// A CTA has 128 query rows of one KV head (query tokens of all sequences one after the other, the heads of the group within a token) and a chunk of the prefix, of which
// every row sees every position; it leaves (m, Σ, o) of each row, which prefix_merge_kernel adds to the other parts.
//
// Precision.  The tensor core multiplies fp16 and truncates what it adds to.  A query row, and the K and V of a tile of 64 positions, are scaled by powers of two so that their largest
// element is 2^13 to 2^14, and split into hi + lo (22 bits; what is 2^-14 of the largest loses the lower ones).  A score is hi·hi in one accumulator and hi·lo + lo·hi in another,
// added in fp32; the output of a tile is the small products first, then hi·hi, in an accumulator of its own, added up in fp32 with the mean of what
// truncation takes given back.  A value that is not finite makes every row's output not finite: every row sees it.
//
// Roles (512 threads): eight warps convert and do the soft-max (a thread per row and half a tile's positions), four add the output up (a thread per row), one issues
// the MMAs.  The K and V of the next tiles are asked for into registers while this one is computed; K has one buffer of operands (the next tile's is written when this one's scores
// are there, and multiplied under this one's soft-max), V, scores and probabilities have two.

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
constexpr int kThreads = 512, kWorkers = 256, kMmaWarp = 12;
constexpr int kLaunchRegs = 128;  // registers per thread that 512 threads are launched with (the build checks that the kernels get them)
constexpr int kWorkRegs = 152, kSumRegs = 168, kIssueRegs = 40;
static_assert(2 * kWorkRegs + kSumRegs + kIssueRegs <= 4 * kLaunchRegs, "register split");
constexpr float kTruncation = 0.8e-7f;  // what truncation takes of a sum on average, as a fraction (four additions at full size): given back
constexpr float kProbBits = 12.f;       // probabilities are stored 2^12 as large, clear of fp16's subnormals

// (a, b) → packed fp16 pairs hi and lo
__device__ __forceinline__ void split2(uint64_t ab, uint32_t &hi, uint32_t &lo) {
    const float2 x = unpair(ab);
    const __half2 h = __floats2half2_rn(x.x, x.y);
    const float2 f = __half22float2(h), rest = unpair(add2(ab, pair(-f.x, -f.y)));
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
    // Operands in the no-swizzle core-matrix layout (8 rows x 16 bytes; core matrices of one step of eight contiguous along the rows): Q and K rows by
    // dimension, V transposed: dimensions by position.
    static constexpr uint32_t kQPlane = kRows * HD * 2, kKPlane = kKeys * HD * 2, kVPlane = kKeys * HD * 2;
    static constexpr uint32_t kOffK = 2 * kQPlane, kOffV = kOffK + 2 * kKPlane, kOffRows = kOffV + 2 * 2 * kVPlane;  // two buffers of V
    // per row: alpha (two tiles), largest score of either half (two tiles), sums of either half, last largest score, score factor; then the warps' largest elements of K and V
    // (two tiles), inverse scales of V (four tiles); then barriers
    static constexpr uint32_t kOffMost = kOffRows + 10 * kRows * 4, kOffBars = kOffMost + (32 + 4) * 4;
    static constexpr uint32_t kSmem = kOffBars + 18 * 8 + 16;
    // tensor memory columns: two buffers of scores (hi·hi | the others), output, two buffers of probabilities (hi, lo)
    static constexpr uint32_t kS = 0, kO = 256, kP = 384;
    static_assert(kSmem <= 227 * 1024 && kOffBars % 8 == 0, "shared memory");
};

template <int HD>
__global__ void __launch_bounds__(kThreads, 1) prefix_tc_kernel(const __grid_constant__ PrefixParams p) {
    using L = Layout<HD>;
    extern __shared__ __align__(128) unsigned char smem[];
    constexpr int KS = HD / 16;  // k16 steps of a score
    constexpr int N = HD / 32;   // pieces of eight elements of K, and of V, per worker and tile
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t slot = blockIdx.x, row0 = blockIdx.y * kRows, kvh = blockIdx.z, n_rows = p.n_seqs * p.n_query * p.group;
    const uint32_t key0 = slot * p.prefix_chunk, keys = min(p.prefix_chunk, p.prefix_len - key0), n_tiles = (keys + kKeys - 1) / kKeys;

    float *alpha_row = reinterpret_cast<float *>(smem + L::kOffRows), *most_row = alpha_row + 2 * kRows, *sum_row = most_row + 4 * kRows, *last_row = sum_row + 2 * kRows,
          *factor_row = last_row + kRows;
    uint32_t *most_of = reinterpret_cast<uint32_t *>(smem + L::kOffMost);  // [K, V][tile parity][worker warp]
    float *v_inv = reinterpret_cast<float *>(most_of + 32);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + L::kOffBars);
    const uint32_t bar0 = smem_u32(bars);
    // pairs by tile parity: V there; scores there, free; probabilities there; probabilities and V used; alpha free; else one: K there; output there, free; sums there
    const uint32_t v_full = bar0, s_full = bar0 + 16, s_empty = bar0 + 32, p_full = bar0 + 48, pv_done = bar0 + 64, a_empty = bar0 + 80, k_full = bar0 + 96, o_full = bar0 + 104,
                   o_empty = bar0 + 112, l_full = bar0 + 120;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 18);
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

    // K: eight dimensions of a position; eight neighbouring lanes take eight positions (whole rows of core matrices), the four groups of a warp four steps (whole lines).
    // V: eight positions of a dimension; neighbouring lanes take neighbouring dimensions.
    uint64_t k[N][4], v[N][4];
    const float *kc = p.prefix_k + (size_t)key0 * p.prefix_stride + (size_t)kvh * HD, *vc = p.prefix_v + (size_t)key0 * p.prefix_stride + (size_t)kvh * HD;
    auto place = [&](uint32_t i, uint32_t &key, uint32_t &step) {
        const uint32_t unit = i * 8 + (tid >> 5);
        key = (unit & 7u) * 8 + (tid & 7u), step = (unit >> 3) * 4 + ((tid >> 3) & 3u);
    };
    auto load_k = [&](uint32_t j) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) {
            uint32_t key, step;
            place(i, key, step);
            key += j * kKeys;
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (key < keys) {
                const float4 *src = reinterpret_cast<const float4 *>(kc + (size_t)key * p.prefix_stride + 8 * step);
                a = __ldcg(src), b = __ldcg(src + 1);
            }
            k[i][0] = pair(a.x, a.y), k[i][1] = pair(a.z, a.w), k[i][2] = pair(b.x, b.y), k[i][3] = pair(b.z, b.w);
        }
    };
    auto load_v = [&](uint32_t j) {
#pragma unroll
        for (uint32_t i = 0; i < N; i++) {
            const uint32_t unit = i * kWorkers + tid, dim = unit % HD, key = j * kKeys + unit / HD * 8;
            const float *src = vc + (size_t)key * p.prefix_stride + dim;
            float x[8];
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) x[e] = key + e < keys ? __ldcg(src + (size_t)e * p.prefix_stride) : 0.f;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) v[i][e] = pair(x[2 * e], x[2 * e + 1]);
        }
    };
    // The largest element of a tile, of all workers.  (Two words per warp, by tile parity: who writes a tile's has met everybody behind the reading of the tile before the last.)
    auto largest = [&](const uint64_t (&x)[N][4], uint32_t which, uint32_t j) {
        uint32_t most = 0;  // ordered like |x|; an infinity or NaN wins
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 f = unpair(x[i][e]);
                most = max(most, max(__float_as_uint(f.x) & 0x7FFFFFFFu, __float_as_uint(f.y) & 0x7FFFFFFFu));
            }
        most = __reduce_max_sync(0xffffffffu, most);
        uint32_t *words = most_of + (which * 2 + (j & 1u)) * 8;
        if (lane == 0) words[warp] = most;
        asm volatile("bar.sync %0, %1;" ::"r"(5 + which), "n"(kWorkers) : "memory");
        return __uint_as_float(__reduce_max_sync(0xffffffffu, words[lane & 7u]));
    };
    if (warp < 8) load_k(0), load_v(0);

    // The query rows: four threads a row, each with the largest of all four.
    {
        static_assert(kThreads == 4 * kRows, "query rows");
        const uint32_t r = tid >> 2, part = tid & 3;
        uint32_t row = row0 + r;
        row = row < n_rows ? row : n_rows - 1;
        const float *qp = p.q + (size_t)(row / p.group) * p.q_stride + (size_t)(kvh * p.group + row % p.group) * HD;
        float4 x[N][2];
        float mx = 0.f, sc, inv;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                x[i][e] = __ldcg(reinterpret_cast<const float4 *>(qp + (4 * i + part) * 8 + 4 * e));
                mx = fmaxf(fmaxf(mx, fmaxf(fabsf(x[i][e].x), fabsf(x[i][e].y))), fmaxf(fabsf(x[i][e].z), fabsf(x[i][e].w)));
            }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        pow2_scale(mx, sc, inv);
#pragma unroll
        for (int i = 0; i < N; i++) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                split2(pair(x[i][e].x * sc, x[i][e].y * sc), hi[2 * e], lo[2 * e]);
                split2(pair(x[i][e].z * sc, x[i][e].w * sc), hi[2 * e + 1], lo[2 * e + 1]);
            }
            unsigned char *to = smem + (4 * i + part) * (kRows * 16) + r * 16;
            *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4 *>(to + L::kQPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        if (part == 0) factor_row[r] = inv * p.scale;
        fence_async_smem();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    if (warp >= 12) {
        move_registers<true, kIssueRegs, kLaunchRegs>();
        if (warp == kMmaWarp) {
            constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t)(kKeys >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);  // fp16 × fp16 → fp32, K-major, M = 128, N = 64
            constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(kRows >> 4) << 24);     // N = head_dim
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
                const uint32_t d = tmem_base + L::kS + b * 128;
                const uint64_t q = smem_desc(base, kRows * 16, 128), kd = smem_desc(base + L::kOffK, kKeys * 16, 128);
                constexpr uint32_t q_plane = L::kQPlane >> 4, k_plane = L::kKPlane >> 4, q_step = (2 * kRows * 16) >> 4, k_step = (2 * kKeys * 16) >> 4;
                const uint32_t q_lo = (uint32_t)q, q_hi = (uint32_t)(q >> 32), k_lo = (uint32_t)kd, k_hi = (uint32_t)(kd >> 32);
                if (elect_one()) {
                    mma_steps<0, KS>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ss<(i != 0)>(d, q_lo + i * q_step, q_hi, k_lo + i * k_step, k_hi, idesc_s);
                        umma_f16_ss<(i != 0)>(d + 64, q_lo + i * q_step + q_plane, q_hi, k_lo + i * k_step, k_hi, idesc_s);
                        umma_f16_ss<1>(d + 64, q_lo + i * q_step, q_hi, k_lo + i * k_step + k_plane, k_hi, idesc_s);
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
                const uint64_t vd = smem_desc(base + L::kOffV + b * 2 * L::kVPlane, HD * 16, 128);
                constexpr uint64_t v_plane = L::kVPlane >> 4, v_step = (2 * HD * 16) >> 4;
                const uint32_t d = tmem_base + L::kO, hi = tmem_base + L::kP + b * 64, lo = hi + 32;
                if (elect_one()) {
                    mma_steps<0, 4>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<(i != 0)>(d, lo + 8 * i, vd + i * v_step, idesc_o);
                        umma_f16_ts<1>(d, hi + 8 * i, vd + i * v_step + v_plane, idesc_o);
                    });
                    mma_steps<0, 4>([&](auto ic) {
                        constexpr uint32_t i = decltype(ic)::value;
                        umma_f16_ts<1>(d, hi + 8 * i, vd + i * v_step, idesc_o);
                    });
                    umma_commit(o_full);
                    umma_commit(pv_done + 8 * b);
                    mbar_arrive(o_full);
                }
                __syncwarp();
            }
        }
    } else if (warp < 8) {
        move_registers<true, kWorkRegs, kLaunchRegs>();
        const uint32_t quarter = warp & 3u, r = quarter * 32 + lane, lanes = quarter << 21, half = warp >> 2, col0 = half * (kKeys / 2);
        const float row_factor = factor_row[r];
        float m = -FLT_MAX, l = 0.f, k_inv = 0.f, k_inv_next;
        bool ok = true;
        // (A warp that gives up goes on to meet the others at the barriers of every tile, which have no bound.)
        auto convert_k = [&](uint32_t j) {
            float scale;
            pow2_scale(largest(k, 0, j), scale, k_inv_next);
            if (ok) {
                const uint64_t scale2 = pair(scale, scale);
#pragma unroll
                for (uint32_t i = 0; i < N; i++) {
                    uint32_t key, step, hi[4], lo[4];
                    place(i, key, step);
#pragma unroll
                    for (int e = 0; e < 4; e++) split2(mul2(k[i][e], scale2), hi[e], lo[e]);
                    unsigned char *to = smem + L::kOffK + step * (kKeys * 16) + key * 16;
                    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4 *>(to + L::kKPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(k_full);
            }
        };
        auto convert_v = [&](uint32_t j) {
            float scale, inv;
            pow2_scale(largest(v, 1, j), scale, inv);
            // the tile that had this buffer has been multiplied (and its probabilities used)
            ok = ok && mbar_wait(pv_done + 8 * (j & 1u), ((j >> 1) & 1u) ^ 1u, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                const uint64_t scale2 = pair(scale, scale);
#pragma unroll
                for (uint32_t i = 0; i < N; i++) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) split2(mul2(v[i][e], scale2), hi[e], lo[e]);
                    unsigned char *to = smem + L::kOffV + (j & 1u) * 2 * L::kVPlane + (i * kWorkers + tid) * 16;
                    *reinterpret_cast<uint4 *>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                    *reinterpret_cast<uint4 *>(to + L::kVPlane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                }
                if (tid == 0) v_inv[j & 3u] = inv;
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_full + 8 * (j & 1u));
            }
        };
        convert_k(0);
        k_inv = k_inv_next;
        if (n_tiles > 1) load_k(1);
        convert_v(0);
        if (n_tiles > 1) load_v(1);
        for (uint32_t j = 0; j < n_tiles; j++) {
            const uint32_t b = j & 1u, ph = (j >> 1) & 1u;
            ok = ok && mbar_wait(s_full + 8 * b, ph, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
            if (j + 1 < n_tiles) {  // this tile's K has been multiplied: the next one's takes its place
                convert_k(j + 1);
                if (j + 2 < n_tiles) load_k(j + 2);
            }
            const float f = row_factor * k_inv;
            k_inv = k_inv_next;
            const uint32_t at = tmem_base + lanes + L::kS + b * 128 + col0;
            const uint32_t seen = keys - min(keys, j * kKeys + col0);  // positions of this half that are there (or more)
            const bool edge = seen < kKeys / 2;
            float mx4[4] = {-FLT_MAX, -FLT_MAX, -FLT_MAX, -FLT_MAX};
            if (ok) {
#pragma unroll
                for (uint32_t c0 = 0; c0 < kKeys / 2; c0 += 16) {
                    uint32_t a[16], c[16];
                    tmem_ld16_issue(at + c0, a);
                    tmem_ld16_issue(at + 64 + c0, c);
                    tmem_ld_wait();
#pragma unroll
                    for (uint32_t i = 0; i < 16; i += 2) {
                        float2 s = unpair(add2(pair_bits(a[i], a[i + 1]), pair_bits(c[i], c[i + 1])));
                        if (edge) s.x = c0 + i < seen ? s.x : -FLT_MAX, s.y = c0 + i + 1 < seen ? s.y : -FLT_MAX;
                        mx4[i & 2] = fmaxf(mx4[i & 2], s.x);
                        mx4[(i & 2) + 1] = fmaxf(mx4[(i & 2) + 1], s.y);
                    }
                }
            }
            // The row's largest score, from both halves.  (Words by tile parity: who writes a tile's has met the other half behind its reading of the tile before the last.)
            const float most = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
            most_row[(b * 2 + half) * kRows + r] = most;
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
            const float mx = fmaxf(most, most_row[(b * 2 + (half ^ 1u)) * kRows + r]);
            const float mn = mx < -3e38f ? m : fmaxf(m, mx * f);
            const float alpha = power(m - mn);
            m = mn;
            ok = ok && mbar_wait(a_empty + 8 * b, ph ^ 1u, abort_flag, p.status);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
                if (half == 0) alpha_row[b * kRows + r] = alpha;
                const uint64_t f2 = pair(f, f), less2 = pair(kProbBits - mn, kProbBits - mn);
                uint64_t sum2 = 0;
#pragma unroll
                for (uint32_t c0 = 0; c0 < kKeys / 2; c0 += 16) {
                    uint32_t a[16], c[16], hi[8], lo[8];
                    tmem_ld16_issue(at + c0, a);
                    tmem_ld16_issue(at + 64 + c0, c);
                    tmem_ld_wait();
                    if (c0 + 16 == kKeys / 2) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(s_empty + 8 * b);
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 8; i++) {
                        const float2 e = unpair(fma2(add2(pair_bits(a[2 * i], a[2 * i + 1]), pair_bits(c[2 * i], c[2 * i + 1])), f2, less2));
                        float2 w = make_float2(power(e.x), power(e.y));
                        if (edge) w.x = c0 + 2 * i < seen ? w.x : 0.f, w.y = c0 + 2 * i + 1 < seen ? w.y : 0.f;
                        const uint64_t w2 = pair(w.x, w.y);
                        sum2 = add2(sum2, w2);
                        split2(w2, hi[i], lo[i]);
                    }
                    const uint32_t to = tmem_base + lanes + L::kP + b * 64 + (col0 + c0) / 2;
                    tmem_st8(to, make_uint4(hi[0], hi[1], hi[2], hi[3]), make_uint4(hi[4], hi[5], hi[6], hi[7]));
                    tmem_st8(to + 32, make_uint4(lo[0], lo[1], lo[2], lo[3]), make_uint4(lo[4], lo[5], lo[6], lo[7]));
                }
                const float2 sums = unpair(sum2);
                l = fmaf(l, alpha, sums.x + sums.y);
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + 8 * b);
            }
            if (j + 1 < n_tiles) {
                convert_v(j + 1);
                if (j + 2 < n_tiles) load_v(j + 2);
            }
        }
        sum_row[half * kRows + r] = l;
        if (half == 0) last_row[r] = m;
        __syncwarp();
        if (lane == 0) mbar_arrive(l_full);
    } else {
        // output sums: this thread's row
        move_registers<true, kSumRegs, kLaunchRegs>();
        const uint32_t r = (warp & 3u) * 32 + lane, lanes = (warp & 3u) << 21;
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
            const uint64_t alpha2 = pair(alpha, alpha), vi2 = pair(vi, vi), lost = pair(kTruncation, kTruncation);
#pragma unroll
            for (uint32_t c0 = 0; c0 < HD; c0 += 16) {
                uint32_t x[16];
                tmem_ld16_issue(tmem_base + lanes + L::kO + c0, x);
                tmem_ld_wait();
                if (c0 + 16 == HD) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(o_empty);
                }
#pragma unroll
                for (uint32_t i = 0; i < 16; i += 2) {
                    const uint64_t y = pair_bits(x[i], x[i + 1]);
                    o[(c0 + i) / 2] = fma2(o[(c0 + i) / 2], alpha2, mul2(fma2(y, lost, y), vi2));
                }
            }
        }
        if (ok) ok = mbar_wait(l_full, 0, abort_flag, p.status);
        const uint32_t row = row0 + r;
        if (ok && row < n_rows) {
            const size_t part = ((size_t)(row / p.group) * p.n_heads + kvh * p.group + row % p.group) * p.slots + slot;
            p.part_ml[part] = make_float2(last_row[r] - kProbBits, sum_row[r] + sum_row[kRows + r]);
            float *to = p.part_o + part * HD;
#pragma unroll
            for (uint32_t i = 0; i < HD; i += 4) {
                const float2 x = unpair(o[i / 2]), y = unpair(o[i / 2 + 1]);
                *reinterpret_cast<float4 *>(to + i) = make_float4(x.x, x.y, y.x, y.y);
            }
        }
    }

    // common exit: nothing of this CTA may still be in flight when its TMEM and shared memory go
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (*abort_flag) {
        // gave up: let MMAs that were already issued drain before the resources are freed
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
    return launch_kernel(kern, dim3(p.prefix_splits, p.prefix_row_tiles, p.n_kv_heads), dim3(kThreads), Layout<HD>::kSmem, s, pdl, p);
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
