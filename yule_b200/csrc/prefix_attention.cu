// prefix_attention.cu — decode attention of a batch whose sequences share a long prefix: the prefix is read once for all of them.
//
// For query token t of sequence b, head h with KV head g = h / (n_heads / n_kv_heads):
//     s_j = q · k_j / sqrt(hd),   o = Σ_j exp(s_j − m) v_j / Σ_j exp(s_j − m),
// j over the prefix, then over the sequence's own positions below min(len_b, capacity) − (n_query − 1 − t): the newest n_query positions are those of the
// query tokens, each of which sees itself and what came before it.  A row that sees nothing is zero.
//
// The positions that all of a sequence's query tokens see are cut into chunks; a CTA takes a chunk of the prefix for some query rows of one KV head, or a chunk of a
// sequence's own positions for that sequence's rows, and leaves (m, Σ, o) of each row in the scratch.  A last kernel, a warp per row, adds the parts up, and
// with them the at most n_query − 1 newest positions that not all query tokens see, one by one in fp32 (so that what is hidden from a row is not read for it).
// Parts are added in a fixed order: the same call gives the same bits.

#include <cuda.h>

#include <cfloat>

#include "prefix_attention.cuh"
#include "qgemm_common.cuh"
#include "tf32_common.cuh"

namespace yule {

namespace {

constexpr int kWarps = 2, kKeys = 16;  // a warp takes tiles of 16 positions in turn with the CTA's other
constexpr uint32_t kTileKeys = kWarps * kKeys;

struct PartMaps {
    CUtensorMap m[4];  // prefix K and V, own K and V: rows in boxes of 16 positions by 32 dimensions, swizzled within 128 bytes
};

// Positions of sequence b's own caches (without capacity there are no lengths either).
__device__ __forceinline__ uint32_t own_len(const PrefixParams &p, uint32_t b) { return p.tail_capacity ? min(__ldcg(p.tail_lens + b), p.tail_capacity) : 0; }
// Positions of sequence b that all its query tokens see.
__device__ __forceinline__ uint32_t common_len(const PrefixParams &p, uint32_t b) {
    const uint32_t n = own_len(p, b);
    return n > p.n_query - 1 ? n - (p.n_query - 1) : 0;
}
__device__ __forceinline__ float4 load4(const float *at, bool there) { return there ? __ldcg(reinterpret_cast<const float4 *>(at)) : make_float4(0.f, 0.f, 0.f, 0.f); }

// A warp per tile of 16 positions, the positions as rows of the tensor core's first operand and the query rows as the eight columns of its second, so that a CTA with few
// query rows multiplies few zeros.  K and V of a tile come to the warp's own shared memory by tiled bulk copies: the next tile's K is asked for when this one's scores are there, its V
// when its output is.  (Loaded into registers they take as much of L1 while they are on their way, and beside prefix_tc_kernel there is none: 114 us for 64
// sequences of 64 heads behind 8192 positions where copies took 104.)  They are split where they are used; which position and which dimensions a lane has is chosen so that its loads are 16 bytes and meet no others' banks.
// HD: head_dim rounded up, or head_dim itself (EXACT); ROWS: query rows in eights; SINGLE: all positions of a sequence (prefix, then its own), whose output the CTA leaves.
template <int HD, int ROWS, bool EXACT, bool SINGLE>
__global__ void __launch_bounds__(kWarps * 32) prefix_part_kernel(const __grid_constant__ PrefixParams p, const __grid_constant__ PartMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    constexpr int kPitch = HD + 16;  // floats of a query row: lanes of two rows meet in different banks
    constexpr int kRows = ROWS * 8;
    constexpr uint32_t kHalf = kKeys * HD * 4;  // K or V of a tile: per 32 dimensions 16 rows of 128 bytes, whose 16-byte pieces are exchanged by the row's number
    __shared__ uint64_t bars[kWarps][2];
    __shared__ int gave_up;
    float *sm = reinterpret_cast<float *>(smem + kWarps * 2 * kHalf);
    uint32_t *q_hi = reinterpret_cast<uint32_t *>(sm), *q_lo = q_hi + kRows * kPitch;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t turned = (g >> 1) | ((g & 1u) << 2);  // g with its lowest bit as its highest: two neighbours are four rows, or pieces, apart
    // Behind the prefix on the tensor core nothing here depends on it, and what came before it is over (it waited, and let this kernel start): only one CTA's end waits, so that who
    // waits for this kernel has waited for that one.
    const bool waits = !p.beside || (blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1);
    if (!p.beside) yule_pdl_wait();
    yule_pdl_launch_dependents();  // (behind the wait: prefix_operands_kernel counts on it)

    // which positions, for which rows: x the rows (of the prefix's first), y the KV head, z the chunk
    const uint32_t kvh = blockIdx.y, split = blockIdx.z;
    uint32_t row0, n_rows, key0, key1, slot = split, line = 0;
    const bool of_prefix = blockIdx.x < p.prefix_items;
    if (of_prefix) {
        row0 = blockIdx.x * kRows;
        n_rows = p.n_seqs * p.n_query * p.group;
        key0 = split * p.prefix_chunk;
        key1 = split < p.prefix_splits ? min(key0 + p.prefix_chunk, p.prefix_len) : key0;
    } else {
        const uint32_t i = blockIdx.x - p.prefix_items, b = p.tail_row_tiles == 1 ? i : i / p.tail_row_tiles, first = b * p.n_query * p.group;
        row0 = first + (i - b * p.tail_row_tiles) * kRows;
        n_rows = first + p.n_query * p.group;
        key0 = split * p.tail_chunk;
        const uint32_t seen = common_len(p, b);
        key1 = split < p.tail_splits && key0 < seen ? min(key0 + p.tail_chunk, seen) : key0;
        slot += p.prefix_splits;
        line = b * p.tail_capacity;  // the sequence's first row
    }
    // The query rows, all under way together and beside the length (one after the other: 8 sequences of five tokens took 30.9 us in all, 27.8 so).
    constexpr int kEach = kRows * (HD / 4) / (kWarps * 32);
    static_assert(kRows * (HD / 4) % (kWarps * 32) == 0, "pieces of the query rows");
    float4 query[kEach];
    {
        uint32_t r = tid / (HD / 4), token = (row0 + r) / p.group, head = (row0 + r) % p.group;
#pragma unroll
        for (int i = 0; i < kEach; i++) {
            const uint32_t e = tid + i * kWarps * 32, next = e / (HD / 4), d = e % (HD / 4) * 4;
            for (head += next - r, r = next; head >= p.group; token++) head -= p.group;
            query[i] = load4(p.q + (size_t)token * p.q_stride + (size_t)(kvh * p.group + head) * p.hd + d, row0 + r < n_rows && d < p.hd);
        }
    }
    // The tiles: of the chunk, or of the prefix and behind them those of the sequence's own positions.
    const uint32_t of_it = SINGLE ? (p.prefix_len + kKeys - 1) / kKeys : 0, n_tiles = of_it + (key1 > key0 ? (key1 - key0 + kKeys - 1) / kKeys : 0);
    if (n_tiles == 0 && !SINGLE) {
        if (waits) yule_pdl_wait();
        return;
    }
    const uint32_t ring = smem_u32(smem) + warp * 2 * kHalf, bar = smem_u32(&bars[warp][0]);
    const unsigned char *mine = smem + warp * 2 * kHalf;
    auto copy = [&](uint32_t tile, uint32_t which) {  // by one lane: K (0) or V of the tile
        const bool prefix = SINGLE ? tile < of_it : of_prefix;
        const uint32_t at = SINGLE && prefix ? tile * kKeys : line + key0 + (tile - of_it) * kKeys;
        const uint64_t map = reinterpret_cast<uint64_t>(&maps.m[(prefix ? 0 : 2) + which]);
        mbar_arrive_expect_tx(bar + 8 * which, kHalf);
#pragma unroll
        for (uint32_t i = 0; i < HD / 32; i++)  // (elements of eight bytes)
            asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(ring + which * kHalf + i * (kKeys * 128)), "l"(map),
                         "r"(bar + 8 * which), "r"(kvh * (p.hd / 2) + 16 * i), "r"(at)
                         : "memory");
    };
    if (lane == 0) {
        mbar_init(bar, 1);
        mbar_init(bar + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
        if (tid == 0) gave_up = 0;
        if (warp < n_tiles) copy(warp, 0), copy(warp, 1);
    }
    // query rows, in units of ln 2, as two terms
#pragma unroll
    for (int i = 0; i < kEach; i++) {
        const uint32_t e = tid + i * kWarps * 32, r = e / (HD / 4), d = e % (HD / 4) * 4;
        uint4 hi, lo;
        split_tf32(query[i].x * p.scale, hi.x, lo.x);
        split_tf32(query[i].y * p.scale, hi.y, lo.y);
        split_tf32(query[i].z * p.scale, hi.z, lo.z);
        split_tf32(query[i].w * p.scale, hi.w, lo.w);
        *reinterpret_cast<uint4 *>(q_hi + r * kPitch + d) = hi;
        *reinterpret_cast<uint4 *>(q_lo + r * kPitch + d) = lo;
    }
    __syncthreads();

    // Per lane the rows 8n + 2t, 8n + 2t + 1, and of them the dimensions 32i + 4·turned on.
    float o[ROWS][HD / 32][2][4], m[ROWS][2], l[ROWS][2];
#pragma unroll
    for (int n = 0; n < ROWS; n++) {
        m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 32; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][i][0][e] = o[n][i][1][e] = 0.f;
    }
    uint32_t phase = 0;
    bool ok = true;
    auto await = [&](uint32_t which) {
        ok = mbar_wait(bar + 8 * which, phase, &gave_up, p.status);
        ok = __all_sync(0xffffffffu, ok);
        return ok;
    };
    const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
    for (uint32_t tile = warp; tile < n_tiles; tile += kWarps, phase ^= 1u) {
        const uint32_t there = SINGLE && tile < of_it ? p.prefix_len - tile * kKeys : key1 - key0 - (tile - of_it) * kKeys;  // positions from the tile's first on (what lies behind, in the tile or the row, may be anything)
        const bool whole = there >= (uint32_t)kKeys, in0 = turned < there, in1 = turned + 8 < there;
        // Scores of positions base + turned and base + turned + 8.  The tensor core truncates what it adds to, so the large products of four steps at a time have sums of their own.
        // (With few query rows a sum of all small products would be a chain of as many steps as there are products: four sums.)
        constexpr int kSums = ROWS == 1 ? 4 : 1;
        float s[ROWS][4], small[ROWS][kSums][4];
#pragma unroll
        for (int n = 0; n < ROWS; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                s[n][e] = 0.f;
#pragma unroll
                for (int c = 0; c < kSums; c++) small[n][c][e] = 0.f;
            }
        if (!await(0)) break;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            float big[ROWS][4];
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) big[n][e] = 0.f;
#pragma unroll
            for (int j = 2 * i; j < 2 * i + 2; j++) {
                const unsigned char *at = mine + i * (kKeys * 128) + turned * 128 + ((((j & 1) * 4 + t) ^ turned) << 4);
                float4 a = *reinterpret_cast<const float4 *>(at), b = *reinterpret_cast<const float4 *>(at + 8 * 128);
                if (!EXACT && 16 * j + 4 * t >= p.hd) a = b = zero;
                uint32_t ah[4], al[4], bh[4], bl[4];
                split_tf32(a.x, ah[0], al[0]), split_tf32(a.y, ah[1], al[1]), split_tf32(a.z, ah[2], al[2]), split_tf32(a.w, ah[3], al[3]);
                split_tf32(b.x, bh[0], bl[0]), split_tf32(b.y, bh[1], bl[1]), split_tf32(b.z, bh[2], bl[2]), split_tf32(b.w, bh[3], bl[3]);
#pragma unroll
                for (int n = 0; n < ROWS; n++) {
                    const uint4 qh = *reinterpret_cast<const uint4 *>(q_hi + (8 * n + g) * kPitch + 16 * j + 4 * t);
                    const uint4 ql = *reinterpret_cast<const uint4 *>(q_lo + (8 * n + g) * kPitch + 16 * j + 4 * t);
                    mma_tf32(small[n][0], al[0], bl[0], al[1], bl[1], qh.x, qh.y);
                    mma_tf32(small[n][1 % kSums], ah[0], bh[0], ah[1], bh[1], ql.x, ql.y);
                    mma_tf32(big[n], ah[0], bh[0], ah[1], bh[1], qh.x, qh.y);
                    mma_tf32(small[n][2 % kSums], al[2], bl[2], al[3], bl[3], qh.z, qh.w);
                    mma_tf32(small[n][3 % kSums], ah[2], bh[2], ah[3], bh[3], ql.z, ql.w);
                    mma_tf32(big[n], ah[2], bh[2], ah[3], bh[3], qh.z, qh.w);
                }
            }
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] += big[n][e];
        }
        __syncwarp();
        if (lane == 0 && tile + kWarps < n_tiles) copy(tile + kWarps, 0);
        // Soft-max of s[0], s[1] (the first position) and s[2], s[3] (the second) in rows 8n + 2t and 8n + 2t + 1.
        uint32_t ph[ROWS][4], pl[ROWS][4];
        float alpha[ROWS][2];
#pragma unroll
        for (int n = 0; n < ROWS; n++) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float rest = small[n][0][e];
                if (kSums == 4) rest = (rest + small[n][1 % kSums][e]) + (small[n][2 % kSums][e] + small[n][3 % kSums][e]);
                s[n][e] = (e < 2 ? in0 : in1) ? s[n][e] + rest : -INFINITY;
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float mx = fmaxf(s[n][c], s[n][c + 2]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                mx = fmaxf(mx, m[n][c]);
                const float from = mx == -INFINITY ? 0.f : mx;  // (scores of −infinity alone)
                alpha[n][c] = exp2f(m[n][c] - from);
                m[n][c] = mx;
                s[n][c] = exp2f(s[n][c] - from);
                s[n][c + 2] = exp2f(s[n][c + 2] - from);
                l[n][c] = fmaf(l[n][c], alpha[n][c], s[n][c] + s[n][c + 2]);
            }
            // as the second operand of the output's products: row (position) t or t + 4 of each eight, column (query row) g; position k of eight is the turned number of 2·(k % 4) + k / 4
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int src = (2 * (int)t + (e & 1)) * 4 + (int)(g >> 1), up = e >> 1;  // e: positions t, t + 4, t + 8, t + 12
                const float even = __shfl_sync(0xffffffffu, s[n][2 * up], src), odd = __shfl_sync(0xffffffffu, s[n][2 * up + 1], src);
                split_tf32(g & 1 ? odd : even, ph[n][e], pl[n][e]);
            }
        }
        // Output: positions t and t + 4 of each eight of this lane.
        if (!await(1)) break;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            float fresh[ROWS][2][4];
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) fresh[n][0][e] = fresh[n][1][e] = 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const unsigned char *at = mine + kHalf + i * (kKeys * 128) + (8 * u + t) * 128;
                float4 a = *reinterpret_cast<const float4 *>(at + ((turned ^ t) << 4)), b = *reinterpret_cast<const float4 *>(at + 4 * 128 + ((turned ^ (t + 4)) << 4));
                if (!EXACT && 32 * i + 4 * turned >= p.hd) a = b = zero;
                if (!whole) {
                    if (8 * u + t >= there) a = zero;
                    if (8 * u + t + 4 >= there) b = zero;
                }
                uint32_t ah[4], al[4], bh[4], bl[4];
                split_tf32(a.x, ah[0], al[0]), split_tf32(a.y, ah[1], al[1]), split_tf32(a.z, ah[2], al[2]), split_tf32(a.w, ah[3], al[3]);
                split_tf32(b.x, bh[0], bl[0]), split_tf32(b.y, bh[1], bl[1]), split_tf32(b.z, bh[2], bl[2]), split_tf32(b.w, bh[3], bl[3]);
#pragma unroll
                for (int n = 0; n < ROWS; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {  // dimensions 32i + 4·turned + 2c and the next one
                        mma_tf32(fresh[n][c], al[2 * c], al[2 * c + 1], bl[2 * c], bl[2 * c + 1], ph[n][2 * u], ph[n][2 * u + 1]);
                        mma_tf32(fresh[n][c], ah[2 * c], ah[2 * c + 1], bh[2 * c], bh[2 * c + 1], pl[n][2 * u], pl[n][2 * u + 1]);
                        mma_tf32(fresh[n][c], ah[2 * c], ah[2 * c + 1], bh[2 * c], bh[2 * c + 1], ph[n][2 * u], ph[n][2 * u + 1]);
                    }
            }
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int c = 0; c < 2; c++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[n][i][c][e] = fmaf(o[n][i][c][e], alpha[n][e & 1], fresh[n][c][e]);
        }
        __syncwarp();
        if (lane == 0 && tile + kWarps < n_tiles) copy(tile + kWarps, 1);
    }
    if (!ok) {  // gave up: the copies that are on their way have a moment to arrive (the status word says that nothing here counts)
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {
        }
    }

    // the warps' parts of a row, in the order of the warps
    __syncthreads();  // (the query rows are done with: their memory is the meeting place)
    float *part = sm, *ml = sm + kWarps * kRows * HD;
#pragma unroll
    for (int n = 0; n < ROWS; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float sum = l[n][c];
            sum += __shfl_xor_sync(0xffffffffu, sum, 4);
            sum += __shfl_xor_sync(0xffffffffu, sum, 8);
            sum += __shfl_xor_sync(0xffffffffu, sum, 16);
            const uint32_t r = warp * kRows + 8 * n + 2 * t + c;
            if (g == 0) ml[2 * r] = m[n][c], ml[2 * r + 1] = sum;
#pragma unroll
            for (int i = 0; i < HD / 32; i++)
                *reinterpret_cast<float4 *>(part + r * HD + 32 * i + 4 * turned) = make_float4(o[n][i][0][c], o[n][i][0][2 + c], o[n][i][1][c], o[n][i][1][2 + c]);
        }
    __syncthreads();
    uint32_t r = tid / (HD / 4), token = (row0 + r) / p.group, head = (row0 + r) % p.group;
#pragma unroll 2
    for (uint32_t e = tid; e < kRows * (HD / 4); e += kWarps * 32) {
        const uint32_t next = e / (HD / 4), d = e % (HD / 4) * 4;
        for (head += next - r, r = next; head >= p.group; token++) head -= p.group;
        if (row0 + r >= n_rows || d >= p.hd) continue;
        float mx = -INFINITY, sum = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; w++) mx = fmaxf(mx, ml[2 * (w * kRows + r)]);
#pragma unroll
        for (int w = 0; w < kWarps; w++) {
            const float f = exp2f(ml[2 * (w * kRows + r)] - (mx == -INFINITY ? 0.f : mx));
            const float4 x = *reinterpret_cast<const float4 *>(part + (w * kRows + r) * HD + d);
            sum = fmaf(f, ml[2 * (w * kRows + r) + 1], sum);
            acc.x = fmaf(f, x.x, acc.x), acc.y = fmaf(f, x.y, acc.y), acc.z = fmaf(f, x.z, acc.z), acc.w = fmaf(f, x.w, acc.w);
        }
        if constexpr (SINGLE) {
            const float inv = n_tiles ? 1.0f / sum : 0.f;
            *reinterpret_cast<float4 *>(p.out + (size_t)token * p.out_stride + (size_t)(kvh * p.group + head) * p.hd + d) = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
            continue;
        }
        const size_t at = ((size_t)token * p.n_heads + kvh * p.group + head) * p.slots + slot;
        if (d == 0) p.part_ml[at] = make_float2(mx, sum);
        *reinterpret_cast<float4 *>(p.part_o + at * p.hd + d) = acc;
    }
    if (waits) yule_pdl_wait();
}

// A warp per (token, head): the newest positions one by one, while the parts are on their way (8 sequences of five tokens: 32.1 -> 30.9 us), then the parts in the order of
// their slots.
template <int N>  // float4 of a row per lane
__global__ void __launch_bounds__(128, 3) prefix_merge_kernel(const __grid_constant__ PrefixParams p) {
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (p.alone) yule_pdl_wait();  // (else what came before the parts is over, or the kernel that leaves them had not let this one start)
    yule_pdl_launch_dependents();
    if (row >= p.n_seqs * p.n_query * p.n_heads) {
        yule_pdl_wait();
        return;
    }
    const uint32_t token = row / p.n_heads, head = row % p.n_heads, b = token / p.n_query, kvh = head / p.group;
    const uint32_t len = own_len(p, b), common = common_len(p, b), back = p.n_query - 1 - token % p.n_query;
    const uint32_t seen = len > back ? len - back : 0, slots = p.prefix_splits + (common + p.tail_chunk - 1) / p.tail_chunk;
    const float2 *ml = p.part_ml + (size_t)row * p.slots;
    const float *po = p.part_o + (size_t)row * p.slots * p.hd;
    float m = -INFINITY, l = 0.f;
    float4 o[N];
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    // the newest positions, while the parts are on their way
    if (common < seen) {
        const float *qp = p.q + (size_t)token * p.q_stride + (size_t)head * p.hd;
        const size_t cache = ((size_t)b * p.tail_capacity) * p.tail_stride + (size_t)kvh * p.hd;
        float4 q[N];
#pragma unroll
        for (int i = 0; i < N; i++) q[i] = load4(qp + 4 * (lane + 32 * i), 4 * (lane + 32 * i) < p.hd);
        for (uint32_t j = common; j < seen; j++) {
            const float *kr = p.tail_k + cache + j * p.tail_stride, *vr = p.tail_v + cache + j * p.tail_stride;
            float s = 0.f, finite = 0.f;  // (or NaN: an infinite score of either sign is one, as in the parts, where the terms of an infinity are)
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float4 k = load4(kr + 4 * (lane + 32 * i), 4 * (lane + 32 * i) < p.hd);
                s = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, fmaf(q[i].z, k.z, fmaf(q[i].w, k.w, s))));
                finite = fmaf(0.f, k.x, fmaf(0.f, k.y, fmaf(0.f, k.z, fmaf(0.f, k.w, finite))));
            }
            s += finite;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            s *= p.scale;
            const float mn = fmaxf(m, s), f0 = mn == -INFINITY ? 0.f : mn, alpha = exp2f(m - f0), e = exp2f(s - f0);
            m = mn;
            l = fmaf(l, alpha, e);
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float4 v = load4(vr + 4 * (lane + 32 * i), 4 * (lane + 32 * i) < p.hd);
                o[i].x = fmaf(o[i].x, alpha, e * v.x), o[i].y = fmaf(o[i].y, alpha, e * v.y), o[i].z = fmaf(o[i].z, alpha, e * v.z), o[i].w = fmaf(o[i].w, alpha, e * v.w);
            }
        }
    }
    yule_pdl_wait();
    // the parts of sixteen slots at a time on their way (of eight with two vectors of four a lane), added in the order of the slots
    constexpr int kParts = 16 / N;
    for (uint32_t s0 = 0; s0 < slots; s0 += kParts) {
        float4 v[kParts][N];
        const float2 x = lane < kParts && s0 + lane < slots ? __ldcg(ml + s0 + lane) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int e = 0; e < kParts; e++)
#pragma unroll
            for (int i = 0; i < N; i++) v[e][i] = load4(po + (size_t)(s0 + e) * p.hd + 4 * (lane + 32 * i), s0 + e < slots && 4 * (lane + 32 * i) < p.hd);
        float most = x.x;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
        most = fmaxf(most, m);
        const float from = most == -INFINITY ? 0.f : most, alpha = exp2f(m - from), f = exp2f(x.x - from);
        m = most;
        float sum = f * x.y;
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        l = fmaf(l, alpha, sum);
#pragma unroll
        for (int i = 0; i < N; i++) o[i].x *= alpha, o[i].y *= alpha, o[i].z *= alpha, o[i].w *= alpha;
#pragma unroll
        for (int e = 0; e < kParts; e++) {
            const float w = __shfl_sync(0xffffffffu, f, e);
#pragma unroll
            for (int i = 0; i < N; i++) o[i].x = fmaf(w, v[e][i].x, o[i].x), o[i].y = fmaf(w, v[e][i].y, o[i].y), o[i].z = fmaf(w, v[e][i].z, o[i].z), o[i].w = fmaf(w, v[e][i].w, o[i].w);
        }
    }
    const float inv = p.prefix_len == 0 && seen == 0 ? 0.f : 1.0f / l;
    float *to = p.out + (size_t)token * p.out_stride + (size_t)head * p.hd;
#pragma unroll
    for (int i = 0; i < N; i++)
        if (4 * (lane + 32 * i) < p.hd) *reinterpret_cast<float4 *>(to + 4 * (lane + 32 * i)) = make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv);
}

template <int HD, int ROWS, bool EXACT, bool SINGLE = false>
cudaError_t launch_part(const PrefixParams &p, const PartMaps &maps, dim3 items, bool pdl, cudaStream_t s) {
    constexpr size_t query = (size_t)2 * ROWS * 8 * (HD + 16) * 4, meeting = (size_t)kWarps * ROWS * 8 * (HD + 2) * 4;
    constexpr size_t smem = (size_t)kWarps * 2 * kKeys * HD * 4 + (query > meeting ? query : meeting);
    auto kern = prefix_part_kernel<HD, ROWS, EXACT, SINGLE>;
    if (smem > 47 * 1024) {  // (beside a kilobyte of its own)
        const cudaError_t e = kernel_opt_in(reinterpret_cast<const void *>(kern), smem, false);
        if (e != cudaSuccess) return e;
    }
    return launch_kernel(kern, items, dim3(kWarps * 32), smem, s, pdl, p, maps);
}
template <int HD, bool EXACT>
cudaError_t launch_rows(const PrefixParams &p, const PartMaps &maps, uint32_t rows, dim3 items, bool pdl, cudaStream_t s) {
    if (p.single) return launch_part<HD, 1, EXACT, true>(p, maps, items, pdl, s);
    if constexpr (HD <= 128) {
        if (rows == 2) return launch_part<HD, 2, EXACT>(p, maps, items, pdl, s);
        if (rows == 3) return launch_part<HD, 3, EXACT>(p, maps, items, pdl, s);
    }
    return launch_part<HD, 1, EXACT>(p, maps, items, pdl, s);
}
template <int HD>
cudaError_t launch_dims(const PrefixParams &p, const PartMaps &maps, uint32_t rows, dim3 items, bool pdl, cudaStream_t s) {
    return p.hd == HD ? launch_rows<HD, true>(p, maps, rows, items, pdl, s) : launch_rows<HD, false>(p, maps, rows, items, pdl, s);
}

uint32_t ceil_div(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

// The cut of the work.
struct Cut {
    bool tc;        // the prefix goes to the kernel for 128 rows at a time
    uint32_t rows;  // query rows of a CTA of the other one, in eights
};
Cut shape_of(const PrefixAttention &a, int sm_count, PrefixParams *p) {
    const uint32_t group = a.n_heads / a.n_kv_heads, mine = a.n_query * group, all = a.n_seqs * mine;
    Cut cut;
    // The tensor core's accumulators take 128 rows whatever there is of them, and the copies of K and V in its form a launch: 4 to 5 us that have to be won back.
    // Without it and with it, 32 heads of 128 (8 KV heads): 32 rows of 1024 positions 18.0 and 19.2 us, of 4096 33.5 and 28.2; 128 rows of 256 17.8 and 17.4, of 4096
    // 85 and 33; 16 rows of 4096 24.6 and 27.9.  32 heads of 64 (4 KV heads): 128 rows of 1024 13.1 and 12.7, 256 rows of 4096 43 and 18.
    cut.tc = prefix_tc_supported(a.hd, all) && all >= 32 && (uint64_t)all * a.prefix_len * a.n_kv_heads * a.hd >= (1u << 25);
    if (const char *e = knob("YULE_PREFIX_TC")) cut.tc = prefix_tc_supported(a.hd, all) && a.prefix_len > 0 && atoi(e) != 0;
    // (24 rows take 1.43 times as long as 16: 172 and 120 us for 64 sequences of eight tokens of 32 heads)
    cut.rows = a.hd > 128 || mine <= 8 ? 1 : mine <= 16 || 1.43 * ceil_div(mine, 24) > ceil_div(mine, 16) ? 2 : 3;
    p->group = group;
    // Few positions: all of a sequence in one CTA, and nothing to be added up.  A launch less, but 32 positions at a time: 4 sequences of 32 heads of 64, 92 positions 9.2 and 6.6 us,
    // 124 9.2 and 8.3, 192 9.0 and 9.3; of 128, 32 positions 9.3 and 6.7, 92 9.4 and 8.2, 124 9.1 and 11.3.
    const bool can = !cut.tc && a.n_query == 1 && mine <= 8;
    p->single = can && ((uint64_t)a.prefix_len + a.tail_capacity) * a.hd <= 10240;
    if (const char *e = knob("YULE_PREFIX_SINGLE")) p->single = can && atoi(e) != 0;
    if (p->single) {
        p->prefix_row_tiles = p->prefix_splits = p->slots = 0;
        p->tail_row_tiles = p->tail_splits = 1;
        p->tail_chunk = a.tail_capacity, p->prefix_chunk = a.prefix_len;
        return cut;
    }
    // Chunks such that there are eight CTAs per SM, of at least one tile for every warp: 32 own caches of to 1000 positions behind a prefix of 64 take 72.8 us with one per SM,
    // 49.6 with two, 40.4 with four, 36.5 with eight, 35.3 with sixteen, one of 4000 22.0, 18.8, 16.1, 19.7 and 19.8.
    const uint32_t want = 8 * sm_count;
    auto chunk = [&](uint64_t units, uint32_t len) {
        const uint64_t per = units ? (want + units - 1) / units : 1;
        const uint64_t c = ((len + per - 1) / per + kTileKeys - 1) / kTileKeys * kTileKeys;
        return (uint32_t)(c < kTileKeys ? kTileKeys : c);
    };
    if (cut.tc) {
        // One CTA per SM: rounds of them times the tiles of each, and what a round and a part to be added up cost.
        p->prefix_row_tiles = ceil_div(all, kPrefixTcRows);
        const uint64_t units = (uint64_t)a.n_kv_heads * p->prefix_row_tiles;
        const uint32_t tiles = ceil_div(a.prefix_len, kPrefixTcKeys);
        double least = 1e30;
        for (uint32_t s = ceil_div(tiles, kPrefixTcTiles), most = s + 63; s <= tiles && s <= most; s++) {
            const uint32_t each = ceil_div(tiles, s);
            const double rounds = (double)((units * ceil_div(tiles, each) + sm_count - 1) / sm_count), cost = rounds * (4.0 + each) + 0.05 * s;
            if (cost < least) least = cost, p->prefix_chunk = each * kPrefixTcKeys;
        }
    } else {
        p->prefix_row_tiles = ceil_div(all, cut.rows * 8);
        p->prefix_chunk = chunk((uint64_t)a.n_kv_heads * p->prefix_row_tiles, a.prefix_len);
    }
    p->prefix_splits = ceil_div(a.prefix_len, p->prefix_chunk);
    p->tail_row_tiles = ceil_div(mine, cut.rows * 8);
    const uint32_t common = a.tail_capacity > a.n_query - 1 ? a.tail_capacity - (a.n_query - 1) : 0;
    p->tail_chunk = chunk((uint64_t)a.n_kv_heads * a.n_seqs * p->tail_row_tiles, common);
    p->tail_splits = ceil_div(common, p->tail_chunk);
    p->slots = p->prefix_splits + p->tail_splits;
    return cut;
}

size_t parts_bytes(const PrefixAttention &a, const PrefixParams &p) {
    const size_t parts = (size_t)a.n_seqs * a.n_query * a.n_heads * p.slots;
    return (parts * (sizeof(float2) + (size_t)a.hd * sizeof(float)) + 127) / 128 * 128;
}

}  // namespace

size_t prefix_attention_scratch_bytes(const PrefixAttention &a, int sm_count) {
    PrefixParams p = {};
    const Cut cut = shape_of(a, sm_count, &p);
    p.prefix_len = a.prefix_len, p.n_kv_heads = a.n_kv_heads, p.hd = a.hd;
    return parts_bytes(a, p) + (cut.tc ? prefix_tc_scratch_bytes(p) : 0);
}

cudaError_t launch_prefix_attention(const PrefixAttention &a, int sm_count, cudaStream_t s, uint64_t *launches) {
    PrefixParams p = {};
    const Cut cut = shape_of(a, sm_count, &p);
    p.q = a.q, p.prefix_k = a.prefix_k, p.prefix_v = a.prefix_v, p.tail_k = a.tail_k, p.tail_v = a.tail_v, p.tail_lens = a.tail_lens, p.out = a.out;
    p.hd = a.hd, p.n_heads = a.n_heads, p.n_kv_heads = a.n_kv_heads, p.prefix_len = a.prefix_len, p.n_seqs = a.n_seqs, p.n_query = a.n_query, p.tail_capacity = a.tail_capacity;
    p.q_stride = a.q_stride, p.out_stride = a.out_stride, p.prefix_stride = a.prefix_stride, p.tail_stride = a.tail_stride;
    p.scale = (float)(1.4426950408889634 / sqrt((double)a.hd));
    const size_t parts = (size_t)a.n_seqs * a.n_query * a.n_heads * p.slots;
    p.part_o = static_cast<float *>(a.scratch);
    p.part_ml = reinterpret_cast<float2 *>(p.part_o + parts * a.hd);
    p.status = a.status;
    const uint64_t out_rows = (uint64_t)a.n_seqs * a.n_query * a.n_heads;
    p.alone = !cut.tc && p.prefix_splits == 0 && p.tail_splits == 0;
    p.prefix_items = cut.tc ? 0 : p.prefix_splits ? p.prefix_row_tiles : 0;
    const uint64_t items = p.prefix_items + (p.tail_splits ? (uint64_t)a.n_seqs * p.tail_row_tiles : 0);
    const uint32_t splits = !cut.tc && p.prefix_splits > p.tail_splits ? p.prefix_splits : p.tail_splits;
    if (items > 0x7FFFFFFFu || out_rows > 0x7FFFFFFFu || a.n_kv_heads > 65535 || splits > 65535) return cudaErrorInvalidValue;
    cudaError_t e = cudaSuccess;
    bool pdl = a.pdl;
    auto own = [&]() -> cudaError_t {
        alignas(64) PartMaps maps = {};
        auto map = [&](const float *at, uint64_t rows, size_t stride, CUtensorMap *to) {
            return cached_tensor_map_2d(at, 8, (uint64_t)a.n_kv_heads * a.hd / 2, rows, stride * 4, 16, kKeys, to, 128);
        };
        if (p.prefix_items || (p.single && a.prefix_len)) {
            e = map(a.prefix_k, a.prefix_len, p.prefix_stride, &maps.m[0]);
            if (e == cudaSuccess) e = map(a.prefix_v, a.prefix_len, p.prefix_stride, &maps.m[1]);
        }
        if (p.tail_splits && a.tail_capacity && e == cudaSuccess) {
            const uint64_t rows = (uint64_t)a.n_seqs * a.tail_capacity;
            e = map(a.tail_k, rows, p.tail_stride, &maps.m[2]);
            if (e == cudaSuccess) e = map(a.tail_v, rows, p.tail_stride, &maps.m[3]);
        }
        if (e != cudaSuccess) return e;
        const dim3 n((uint32_t)items, a.n_kv_heads, splits);
        e = a.hd <= 64    ? launch_dims<64>(p, maps, cut.rows, n, pdl, s)
            : a.hd <= 96  ? launch_dims<96>(p, maps, cut.rows, n, pdl, s)
            : a.hd <= 128 ? launch_dims<128>(p, maps, cut.rows, n, pdl, s)
                          : launch_rows<256, false>(p, maps, cut.rows, n, pdl, s);
        ++*launches;
        pdl = true;
        return e;
    };
    // What comes first?  A sequence's own positions fill the GPU at once and leave when their memory is read, and K and V are converted beside them; behind the prefix they run beside the
    // tensor core, a CTA per SM.  First and last, us: 32 sequences of 32 heads of 128 behind 1024 positions, 30 of their own 23.0 and 25.7, 1000 46.2 and 51.5, behind
    // 2048 26.3 and 27.8, 51.7 and 54.4, with 300 35.5 and 35.3; behind 8192 (67 MB) 52.6 and 49.3, with 1000 75.5 and 77.0; 64 of 64 heads behind 8192 82.3 and 74.3, 127.8 and 122.2;
    // 64 of 32 heads of 64 behind 2048 (4 MB), 300 of their own, 23.6 and 26.9.
    bool own_first = items && cut.tc && (uint64_t)a.prefix_len * a.n_kv_heads * a.hd * 8 <= 24u << 20;
    if (const char *x = knob("YULE_PREFIX_OWN_FIRST")) own_first = items && cut.tc && atoi(x) != 0;
    p.beside = cut.tc && !own_first, p.behind = own_first;
    if (own_first && (e = own()) != cudaSuccess) return e;
    if (cut.tc) {
        if ((e = launch_prefix_tc(p, static_cast<unsigned char *>(a.scratch) + parts_bytes(a, p), pdl, s, launches)) != cudaSuccess) return e;
        pdl = true;
    }
    if (items && !own_first && (e = own()) != cudaSuccess) return e;
    if (p.single) return cudaSuccess;
    const dim3 grid(ceil_div(out_rows, 4));
    e = a.hd <= 128 ? launch_kernel(prefix_merge_kernel<1>, grid, dim3(128), 0, s, pdl, p) : launch_kernel(prefix_merge_kernel<2>, grid, dim3(128), 0, s, pdl, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace yule
