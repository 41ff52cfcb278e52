// prefix_attention.cu — decode attention of a batch whose sequences share a long prefix: the prefix is read once for all of them.
//
// For query token t of sequence b, head h with KV head g = h / (n_heads / n_kv_heads):
//     s_j = q · k_j / sqrt(hd),   o = Σ_j exp(s_j − m) v_j / Σ_j exp(s_j − m),
// j over the prefix, then over the sequence's own positions below min(len_b, capacity) − (n_query − 1 − t): the newest n_query positions are those of the
// query tokens, each of which sees itself and what came before it.  A row that sees nothing is zero.
//
// The positions that all of a sequence's query tokens see are cut into chunks; a CTA takes a chunk of the prefix for some query rows of one KV head, or a chunk of a
// sequence's own positions for that sequence's rows, and leaves (m, Σ, o) of each row in the scratch.  A second kernel, a warp per row, adds the parts up, and
// with them the at most n_query − 1 newest positions that not all query tokens see, one by one in fp32 (so that what is hidden from a row is not read for it).
// Parts are added in a fixed order: the same call gives the same bits.

#include <cfloat>

#include "prefix_attention.cuh"
#include "tf32_common.cuh"

namespace yule {

namespace {

constexpr int kWarps = 4, kKeys = 16;  // a warp takes tiles of 16 positions in turn with the CTA's others
constexpr uint32_t kTileKeys = kWarps * kKeys;

// Positions of sequence b's own caches (without capacity there are no lengths either).
__device__ __forceinline__ uint32_t own_len(const PrefixParams &p, uint32_t b) { return p.tail_capacity ? min(__ldg(p.tail_lens + b), p.tail_capacity) : 0; }
// Positions of sequence b that all its query tokens see.
__device__ __forceinline__ uint32_t common_len(const PrefixParams &p, uint32_t b) {
    const uint32_t n = own_len(p, b);
    return n > p.n_query - 1 ? n - (p.n_query - 1) : 0;
}
__device__ __forceinline__ float4 load4(const float *at, bool there) { return there ? __ldcg(reinterpret_cast<const float4 *>(at)) : make_float4(0.f, 0.f, 0.f, 0.f); }

// A warp per tile of 16 positions, the positions as rows of the tensor core's first operand and the query rows as the eight columns of its second, so that a CTA with few
// query rows multiplies few zeros.  K and V go from memory to registers (every element belongs to one lane) and are split there; the order of dimensions and
// positions within a product is chosen so that a lane's elements are 16 consecutive bytes.  HD: head_dim rounded up; ROWS: query rows in eights.
template <int HD, int ROWS>
__global__ void __launch_bounds__(kWarps * 32) prefix_part_kernel(const __grid_constant__ PrefixParams p) {
    extern __shared__ __align__(16) float sm[];
    constexpr int kPitch = HD + 16;  // floats: lanes of two rows meet in different banks
    constexpr int kRows = ROWS * 8;
    uint32_t *q_hi = reinterpret_cast<uint32_t *>(sm), *q_lo = q_hi + kRows * kPitch;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    yule_pdl_launch_dependents();
    yule_pdl_wait();

    // which positions, for which rows
    uint32_t item = blockIdx.x, kvh, row0, n_rows, key0, key1, slot;
    const float *kc, *vc;
    size_t stride;
    if (item < p.prefix_items) {
        slot = item % p.prefix_splits;
        item /= p.prefix_splits;
        kvh = item % p.n_kv_heads;
        row0 = item / p.n_kv_heads * kRows;
        n_rows = p.n_seqs * p.n_query * p.group;
        key0 = slot * p.prefix_chunk;
        key1 = min(key0 + p.prefix_chunk, p.prefix_len);
        kc = p.prefix_k, vc = p.prefix_v, stride = p.prefix_stride;
    } else {
        item -= p.prefix_items;
        const uint32_t split = item % p.tail_splits;
        item /= p.tail_splits;
        kvh = item % p.n_kv_heads;
        item /= p.n_kv_heads;
        const uint32_t b = item / p.tail_row_tiles, first = b * p.n_query * p.group;
        row0 = first + item % p.tail_row_tiles * kRows;
        n_rows = first + p.n_query * p.group;
        key0 = split * p.tail_chunk;
        const uint32_t seen = common_len(p, b);
        if (key0 >= seen) return;
        key1 = min(key0 + p.tail_chunk, seen);
        slot = p.prefix_splits + split;
        kc = p.tail_k + (size_t)b * p.tail_capacity * p.tail_stride, vc = p.tail_v + (size_t)b * p.tail_capacity * p.tail_stride, stride = p.tail_stride;
    }
    kc += (size_t)kvh * p.hd, vc += (size_t)kvh * p.hd;

    // query rows, in units of ln 2, as two terms
    for (uint32_t i = tid; i < kRows * (HD / 4); i += kWarps * 32) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4, row = row0 + r;
        const float4 v = load4(p.q + (size_t)(row / p.group) * p.q_stride + (size_t)(kvh * p.group + row % p.group) * p.hd + d, row < n_rows && d < p.hd);
        uint4 hi, lo;
        split_tf32(v.x * p.scale, hi.x, lo.x);
        split_tf32(v.y * p.scale, hi.y, lo.y);
        split_tf32(v.z * p.scale, hi.z, lo.z);
        split_tf32(v.w * p.scale, hi.w, lo.w);
        *reinterpret_cast<uint4 *>(q_hi + r * kPitch + d) = hi;
        *reinterpret_cast<uint4 *>(q_lo + r * kPitch + d) = lo;
    }
    __syncthreads();

    // Per lane the rows 8n + 2t, 8n + 2t + 1, and of them the dimensions 32i + 4g .. 32i + 4g + 3.
    float o[ROWS][HD / 32][2][4], m[ROWS][2], l[ROWS][2];
#pragma unroll
    for (int n = 0; n < ROWS; n++) {
        m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 32; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[n][i][0][e] = o[n][i][1][e] = 0.f;
    }
    for (uint32_t base = key0 + warp * kKeys; base < key1; base += kTileKeys) {
        const bool in0 = base + g < key1, in1 = base + g + 8 < key1;
        const float *k0 = kc + (size_t)(base + g) * stride + 4 * t, *k1 = k0 + 8 * stride;
        // Scores.  The tensor core truncates what it adds to, so the large products of four steps at a time have sums of their own.
        float s[ROWS][4], small[ROWS][4];
#pragma unroll
        for (int n = 0; n < ROWS; n++)
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] = small[n][e] = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            float big[ROWS][4];
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) big[n][e] = 0.f;
#pragma unroll
            for (int j = 2 * i; j < 2 * i + 2; j++) {
                const bool dims = 16 * j + 4 * t < p.hd;
                const float4 a = load4(k0 + 16 * j, in0 && dims), b = load4(k1 + 16 * j, in1 && dims);
                uint32_t ah[4], al[4], bh[4], bl[4];
                split_tf32(a.x, ah[0], al[0]), split_tf32(a.y, ah[1], al[1]), split_tf32(a.z, ah[2], al[2]), split_tf32(a.w, ah[3], al[3]);
                split_tf32(b.x, bh[0], bl[0]), split_tf32(b.y, bh[1], bl[1]), split_tf32(b.z, bh[2], bl[2]), split_tf32(b.w, bh[3], bl[3]);
#pragma unroll
                for (int n = 0; n < ROWS; n++) {
                    const uint4 qh = *reinterpret_cast<const uint4 *>(q_hi + (8 * n + g) * kPitch + 16 * j + 4 * t);
                    const uint4 ql = *reinterpret_cast<const uint4 *>(q_lo + (8 * n + g) * kPitch + 16 * j + 4 * t);
                    mma_tf32(small[n], al[0], bl[0], al[1], bl[1], qh.x, qh.y);
                    mma_tf32(small[n], ah[0], bh[0], ah[1], bh[1], ql.x, ql.y);
                    mma_tf32(big[n], ah[0], bh[0], ah[1], bh[1], qh.x, qh.y);
                    mma_tf32(small[n], al[2], bl[2], al[3], bl[3], qh.z, qh.w);
                    mma_tf32(small[n], ah[2], bh[2], ah[3], bh[3], ql.z, ql.w);
                    mma_tf32(big[n], ah[2], bh[2], ah[3], bh[3], qh.z, qh.w);
                }
            }
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) s[n][e] += big[n][e];
        }
        // Soft-max: positions base + g (s[0], s[1]) and base + g + 8 (s[2], s[3]) of rows 8n + 2t and 8n + 2t + 1.
        uint32_t ph[ROWS][4], pl[ROWS][4];
        float alpha[ROWS][2];
#pragma unroll
        for (int n = 0; n < ROWS; n++) {
#pragma unroll
            for (int e = 0; e < 4; e++) s[n][e] = (e < 2 ? in0 : in1) ? s[n][e] + small[n][e] : -INFINITY;
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
            // as the second operand of the output's products: row (position) t or t + 4 of each eight, column (query row) g
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int key = (e & 1) * 4 + t, src = key * 4 + (int)(g >> 1), up = e >> 1;  // e: positions 0.., 4.., 8.., 12..
                const float even = __shfl_sync(0xffffffffu, s[n][2 * up], src), odd = __shfl_sync(0xffffffffu, s[n][2 * up + 1], src);
                split_tf32(g & 1 ? odd : even, ph[n][e], pl[n][e]);
            }
        }
        // Output.  Position 8u + t and 8u + t + 4 of this lane, dimensions 32i + 4g on.
        const float *v0 = vc + (size_t)(base + t) * stride + 4 * g;
#pragma unroll
        for (int i = 0; i < HD / 32; i++) {
            float fresh[ROWS][2][4];
#pragma unroll
            for (int n = 0; n < ROWS; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) fresh[n][0][e] = fresh[n][1][e] = 0.f;
            const bool dims = 32 * i + 4 * g < p.hd;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const float4 a = load4(v0 + 32 * i + (size_t)(8 * u) * stride, dims && base + 8 * u + t < key1), b = load4(v0 + 32 * i + (size_t)(8 * u + 4) * stride, dims && base + 8 * u + t + 4 < key1);
                uint32_t ah[4], al[4], bh[4], bl[4];
                split_tf32(a.x, ah[0], al[0]), split_tf32(a.y, ah[1], al[1]), split_tf32(a.z, ah[2], al[2]), split_tf32(a.w, ah[3], al[3]);
                split_tf32(b.x, bh[0], bl[0]), split_tf32(b.y, bh[1], bl[1]), split_tf32(b.z, bh[2], bl[2]), split_tf32(b.w, bh[3], bl[3]);
#pragma unroll
                for (int n = 0; n < ROWS; n++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {  // dimensions 32i + 4g + 2c and the next one
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
                *reinterpret_cast<float4 *>(part + r * HD + 32 * i + 4 * g) = make_float4(o[n][i][0][c], o[n][i][0][2 + c], o[n][i][1][c], o[n][i][1][2 + c]);
        }
    __syncthreads();
    for (uint32_t i = tid; i < kRows * (HD / 4); i += kWarps * 32) {
        const uint32_t r = i / (HD / 4), d = i % (HD / 4) * 4, row = row0 + r;
        if (row >= n_rows || d >= p.hd) continue;
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
        const size_t at = ((size_t)(row / p.group) * p.n_heads + kvh * p.group + row % p.group) * p.slots + slot;
        if (d == 0) p.part_ml[at] = make_float2(mx, sum);
        *reinterpret_cast<float4 *>(p.part_o + at * p.hd + d) = acc;
    }
}

// A warp per (token, head): the parts in the order of their slots, then the newest positions one by one.
template <int N>  // float4 of a row per lane
__global__ void __launch_bounds__(128) prefix_merge_kernel(const __grid_constant__ PrefixParams p) {
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    if (row >= p.n_seqs * p.n_query * p.n_heads) return;
    const uint32_t token = row / p.n_heads, head = row % p.n_heads, b = token / p.n_query, kvh = head / p.group;
    const uint32_t len = own_len(p, b), common = common_len(p, b), back = p.n_query - 1 - token % p.n_query;
    const uint32_t seen = len > back ? len - back : 0, slots = p.prefix_splits + (common + p.tail_chunk - 1) / p.tail_chunk;
    const float2 *ml = p.part_ml + (size_t)row * p.slots;
    const float *po = p.part_o + (size_t)row * p.slots * p.hd;
    float m = -INFINITY, l = 0.f;
    for (uint32_t s = lane; s < slots; s += 32) m = fmaxf(m, __ldcg(&ml[s].x));
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    float4 o[N];
#pragma unroll
    for (int i = 0; i < N; i++) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float from = m == -INFINITY ? 0.f : m;
#pragma unroll 4
    for (uint32_t s = 0; s < slots; s++) {
        const float2 x = __ldcg(ml + s);
        const float f = exp2f(x.x - from);
        l = fmaf(f, x.y, l);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float4 v = load4(po + (size_t)s * p.hd + 4 * (lane + 32 * i), 4 * (lane + 32 * i) < p.hd);
            o[i].x = fmaf(f, v.x, o[i].x), o[i].y = fmaf(f, v.y, o[i].y), o[i].z = fmaf(f, v.z, o[i].z), o[i].w = fmaf(f, v.w, o[i].w);
        }
    }
    if (common < seen) {
        const float *qp = p.q + (size_t)token * p.q_stride + (size_t)head * p.hd;
        const size_t cache = ((size_t)b * p.tail_capacity) * p.tail_stride + (size_t)kvh * p.hd;
        float4 q[N];
#pragma unroll
        for (int i = 0; i < N; i++) q[i] = load4(qp + 4 * (lane + 32 * i), 4 * (lane + 32 * i) < p.hd);
        for (uint32_t j = common; j < seen; j++) {
            const float *kr = p.tail_k + cache + j * p.tail_stride, *vr = p.tail_v + cache + j * p.tail_stride;
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < N; i++) {
                const float4 k = load4(kr + 4 * (lane + 32 * i), 4 * (lane + 32 * i) < p.hd);
                s = fmaf(q[i].x, k.x, fmaf(q[i].y, k.y, fmaf(q[i].z, k.z, fmaf(q[i].w, k.w, s))));
            }
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
    const float inv = p.prefix_len == 0 && seen == 0 ? 0.f : 1.0f / l;
    float *to = p.out + (size_t)token * p.out_stride + (size_t)head * p.hd;
#pragma unroll
    for (int i = 0; i < N; i++)
        if (4 * (lane + 32 * i) < p.hd) *reinterpret_cast<float4 *>(to + 4 * (lane + 32 * i)) = make_float4(o[i].x * inv, o[i].y * inv, o[i].z * inv, o[i].w * inv);
}

template <int HD, int ROWS>
cudaError_t launch_part(const PrefixParams &p, uint32_t items, bool pdl, cudaStream_t s, uint64_t *launches) {
    constexpr size_t query = (size_t)2 * ROWS * 8 * (HD + 16) * 4, meeting = (size_t)kWarps * ROWS * 8 * (HD + 2) * 4, smem = query > meeting ? query : meeting;
    auto kern = prefix_part_kernel<HD, ROWS>;
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);  // (of the current device)
        if (e != cudaSuccess) return e;
    }
    const cudaError_t e = launch_kernel(kern, dim3(items), dim3(kWarps * 32), smem, s, pdl, p);
    if (e == cudaSuccess) ++*launches;
    return e;
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
    cut.tc = prefix_tc_supported(a.hd) && all >= 32 && a.prefix_len >= 64;
    if (const char *e = knob("YULE_PREFIX_TC")) cut.tc = prefix_tc_supported(a.hd) && atoi(e) != 0 && a.prefix_len > 0;
    cut.rows = mine > 8 && a.hd <= 128 ? 2 : 1;
    p->group = group;
    // Chunks such that the CTAs are a few per SM, of at least one tile for every warp.
    const uint32_t want = 4 * sm_count;
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
        for (uint32_t s = 1; s <= tiles && s <= 64; s++) {
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

}  // namespace

size_t prefix_attention_scratch_bytes(const PrefixAttention &a, int sm_count) {
    PrefixParams p = {};
    shape_of(a, sm_count, &p);
    const size_t parts = (size_t)a.n_seqs * a.n_query * a.n_heads * p.slots;
    return parts * (sizeof(float2) + (size_t)a.hd * sizeof(float)) + 256;
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
    uint64_t items = (uint64_t)a.n_seqs * p.n_kv_heads * p.tail_row_tiles * p.tail_splits;
    if (!cut.tc) items += (uint64_t)p.n_kv_heads * p.prefix_row_tiles * p.prefix_splits;
    if (items > 0x7FFFFFFFu || out_rows > 0x7FFFFFFFu) return cudaErrorInvalidValue;
    cudaError_t e = cudaSuccess;
    bool pdl = a.pdl;
    if (cut.tc) {
        if ((e = launch_prefix_tc(p, pdl, s, launches)) != cudaSuccess) return e;
        pdl = true;
    }
    p.prefix_items = cut.tc ? 0 : p.n_kv_heads * p.prefix_row_tiles * p.prefix_splits;
    if (items) {
#define YULE_PART(H) e = cut.rows == 1 ? launch_part<H, 1>(p, (uint32_t)items, pdl, s, launches) : launch_part<H, 2>(p, (uint32_t)items, pdl, s, launches)
        if (a.hd <= 64) YULE_PART(64);
        else if (a.hd <= 96) YULE_PART(96);
        else if (a.hd <= 128) YULE_PART(128);
        else e = launch_part<256, 1>(p, (uint32_t)items, pdl, s, launches);
#undef YULE_PART
        if (e != cudaSuccess) return e;
        pdl = true;
    }
    const dim3 grid(ceil_div(out_rows, 4));
    e = a.hd <= 128 ? launch_kernel(prefix_merge_kernel<1>, grid, dim3(128), 0, s, pdl, p) : launch_kernel(prefix_merge_kernel<2>, grid, dim3(128), 0, s, pdl, p);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace yule
