// verify.cu — verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Sequence b has k = min(draft_lens[b], n_draft) drafted tokens x_0 .. x_{k-1}; with p_t the soft-max of its target logits at place t (over the temperature) and q_t that of
// the draft model's (or, without draft logits, all of it on x_t), draft t is accepted while
//     u_t · q_t(x_t) < p_t(x_t).
// At the first that is not, place a, the token comes from w = max(0, p_a − q_a), after k accepted ones from w = p_k: the first i with Σ_{j <= i} w_j > u · Σ w, u the
// last of the sequence's random numbers.  So the tokens are distributed as the target alone would give them.
//
// One launch, a cluster of CTAs per sequence, a slice of the vocabulary per CTA.  Places come in groups, each a pass over its rows of logits, one barrier of the
// cluster and comparisons that all CTAs make alike: in a large batch the rows of a group behind the first rejected draft are not read and other sequences'
// rows are on their way while one picks; in a small one all places are one group.
//
// A pick next to a border has to be the same however the sums are formed: in 32 bits the running sum over 128256 tokens is off by 1e-7 where a token has 8e-6 on
// average, one pick in a hundred.  So w and its sums are in 64 bits (exponentials to 2^-34, see Weight), for the two rows that the token is drawn from.  The
// comparisons before it are in 32 bits, good to 2^-16, and made again in 64 where the two sides are nearer than 2^-13 of one another, or both below 2^-100.
//
// w takes one pass over its two rows, although it needs the sums of both first: with the ratio of the sums known to 2^-16, tokens with p > q are told from the others,
// and Σ w over them is Σ exp_p − ratio · Σ exp_q with the ratio known by then.  A token on the wrong side has |p − q| below 2^-16 of p, so with the mass of all
// tokens that near at most 2^-14 of Σ w, w is good to 2^-30; with more (models that are as good as the same) a second pass knows the ratio and adds w itself up,
// which a difference of sums near 1 would lose below 2^-53.  Where w is nothing at all the token comes from p.  The share of the vocabulary that holds the pick is gone through again with w itself.

#include <cfloat>
#include <utility>

#include <cooperative_groups.h>

#include "internal.h"

namespace yule {

namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kNothing = 0xFFFFFFFFu;
constexpr int kBatch = 16;           // logits of a row that a thread has on their way
constexpr int kAhead = 4;            // and of the rows that it draws from
constexpr float kNear = 0x1p-13f;
constexpr float kFewBits = 0x1p-100f;  // less, and a product or quotient on the way can have been subnormal

__device__ __forceinline__ uint64_t pair(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

struct VerifyParams {
    const float *target, *draft;
    const uint32_t *drafts, *lens;
    const float *random;
    uint32_t *tokens, *accepted;
    uint32_t vocab, n_draft, group;
    size_t target_stride, draft_stride;
    double per_bit;  // log2(e) / temperature
};

// (Not by the read-only path: a launch before this one, which this one may have started beside, can have written any input.)
template <typename T>
__device__ __forceinline__ T read(const T *at) {
    return *at;
}

// A logit as it counts: NaN as −infinity, +infinity as the largest number.
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX); }
__device__ __forceinline__ float power(float x) {  // of two, to 2^-22; subnormal ones are nothing
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 2^((x − most) · per_bit) in 64 bits, for a logit x (clean or not) and the largest of its row, up to 2^-34 of itself; less than 2^-1022 is nothing.  Argument n + f, n rounded in 32 bits, |f| <= 0.501: 2^f by a polynomial of
// degree 7 (interpolating at Chebyshev points), n into the exponent.  Nine operations in 64 bits, whose pipe bounds a pass over w.
struct Weight {
    double per_bit;
    float most, per32, floor;  // floor: what lies below is nothing, and too far off to be rounded (rounded up: at most 1100 bits, or `most` itself)
    __device__ __forceinline__ Weight(float m, double per) : per_bit(per), most(m), per32((float)per) { floor = __fsub_ru(m, (float)(1100.0 / per)); }
    __device__ __forceinline__ double operator()(float x) const {
        constexpr float kRound = 12582912.f;  // 1.5 · 2^23
        const float c = fminf(fmaxf(x, floor), most), z = fmaf(c - most, per32, kRound);
        const int n = __float_as_int(z) - 0x4B400000;
        const double f = fma((double)c - (double)most, per_bit, -(double)(z - kRound));
        double e = 1.530390509058455e-05;
        e = fma(e, f, 0.0001546999476270236);
        e = fma(e, f, 0.0013333477833756698);
        e = fma(e, f, 0.009618024781872923);
        e = fma(e, f, 0.05550410906806735);
        e = fma(e, f, 0.24022651219745797);
        e = fma(e, f, 0.6931471805567823);
        e = fma(e, f, 0.9999999999589098);
        const double w = __hiloint2double(__double2hiint(e) + (n << 20), __double2loint(e));
        return !(x >= floor) || n < -1021 ? 0.0 : w;
    }
};

// (most, at) of two: the larger, at equal size the higher index.
__device__ __forceinline__ void take_larger(float &most, uint32_t &at, float other, uint32_t other_at) {
    if (other > most || (other == most && other_at > at)) most = other, at = other_at;
}
// A number's bits in an order that integers have.
__device__ __forceinline__ int ordered(float x) {
    const int i = __float_as_int(x);
    return i ^ ((i >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float from_ordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7FFFFFFF)); }
// (most, sum of 2^((x − most) · per_bit)) of a warp's lanes.
__device__ __forceinline__ void join(float &most, float &sum, float per_bit) {
    const float m = from_ordered(__reduce_max_sync(0xffffffffu, ordered(most)));
    sum *= power((most - (m == -INFINITY ? 0.f : m)) * per_bit);
    most = m;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
}

// Over the lower sixteen lanes of a warp.
__device__ __forceinline__ double sum16(double v) {
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    return v;
}
// Of sixteen parts in the lower lanes of a warp, the one in which the running sum (from `run` on) passes the goal, else the last that has anything (16: none); run: what is before it.
__device__ __forceinline__ uint32_t part_of(double part, double goal, double &run) {
    const uint32_t lane = threadIdx.x & 31;
    part = lane < 16 && part > 0.0 ? part : 0.0;
    double scan = part;
#pragma unroll
    for (int d = 1; d < 16; d <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= (uint32_t)d) scan += x;
    }
    const uint32_t any = __ballot_sync(0xffffffffu, part > 0.0), past = __ballot_sync(0xffffffffu, part > 0.0 && run + scan > goal);
    if (!any) return 16;
    const uint32_t at = past ? __ffs(past) - 1 : 31 - __clz(any);
    run += __shfl_sync(0xffffffffu, scan - part, at);
    return at;
}

constexpr uint32_t kMostDrafts = 256;  // of a sequence (the entry point's limit)
constexpr uint32_t kMostRows = 16;     // of a group

struct Shared {
    float2 row[2][16][kWarps];  // by parity of the group, CTA: what the warps have of their rows, written by them; greedy: (most, its index)
    float2 whole[kMostRows];    // of the whole rows
    uint32_t drafts[kMostDrafts];
    float random[kMostDrafts], last_random, target_at[kMostDrafts], draft_at[kMostDrafts];  // logits of the drafts themselves; −infinity outside the vocabulary
    double exact[2][5][16], warp_exact[5][kWarps];  // Σ exp_p, Σ exp_q; the same over tokens with p > q; Σ exp_p where the two are near; of the slices by parity of the pass
    double warp_scan[kWarps];
    uint32_t pick, last[kWarps];
};

template <int CTAS, bool GREEDY>
__global__ void __launch_bounds__(kThreads, 2) verify_kernel(const __grid_constant__ VerifyParams p) {
    __shared__ Shared sh;
    cg::cluster_group cluster = cg::this_cluster();
    auto started = cluster.barrier_arrive();  // (waited for before anything is written to another CTA)
    const uint32_t rank = blockIdx.x % CTAS, b = blockIdx.x / CTAS, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // a CTA's slice, and of it a warp's share
    const uint32_t share = ((p.vocab + CTAS * kWarps - 1) / (CTAS * kWarps) + 3) & ~3u, lo = min(rank * kWarps * share, p.vocab), hi = min(lo + kWarps * share, p.vocab);
    const float per_bit = (float)p.per_bit;
    yule_pdl_launch_dependents();
    yule_pdl_wait();
    const uint32_t k = p.lens ? min(read(p.lens + b), p.n_draft) : p.n_draft;
    const float *target = p.target + (size_t)b * (p.n_draft + 1) * p.target_stride, *draft = !GREEDY && p.draft ? p.draft + (size_t)b * p.n_draft * p.draft_stride : nullptr;
    for (uint32_t t = tid; t < k; t += kThreads) {
        if (!GREEDY) sh.random[t] = read(p.random + (size_t)b * (p.n_draft + 1) + t);
        const uint32_t x = read(p.drafts + (size_t)b * p.n_draft + t);
        const bool in = x < p.vocab;
        sh.drafts[t] = x;
        sh.target_at[t] = in ? clean(read(target + (size_t)t * p.target_stride + x)) : -INFINITY;
        sh.draft_at[t] = in && draft ? clean(read(draft + (size_t)t * p.draft_stride + x)) : -INFINITY;
    }
    if (tid == 0) {
        sh.pick = kNothing;
        if (!GREEDY) sh.last_random = read(p.random + (size_t)b * (p.n_draft + 1) + p.n_draft);
    }
    cluster.barrier_wait(std::move(started));

    // Rows of a group are shared out to the warps: per_row of them a row, the target's rows of all places, then the draft model's.
    const uint32_t kinds = draft ? 2 : 1, per_row = kWarps / (kinds * p.group), my_row = warp / per_row, place = my_row % p.group, kind = my_row / p.group;
    const uint32_t first = (warp % per_row) * 32 + lane, step = per_row * 32;  // (of fours of logits, or of single ones)
    uint32_t a = 0, g = p.group;  // the place in question, and which of its group it is
    uint32_t t0 = 0u - p.group, parity = 0, pass = 0;
    double z[5], ratio, less;  // Σ w = z[2] − less · z[3]
    bool alone = false;        // the token comes from p
    float pm, qm;
    const float *pr, *qr;
    uint32_t *out = p.tokens + (size_t)b * (p.n_draft + 1);
    auto finish = [&](uint32_t pick) {  // by all threads of one CTA
        for (uint32_t t = tid; t <= p.n_draft; t += kThreads) out[t] = t < a ? sh.drafts[t] : t == a ? pick : kNothing;
        if (tid == 0) p.accepted[b] = a;
    };
    for (;;) {
        if (g == p.group) {
            // The next group of places: largest logit and sum of exponentials of each row, in 32 bits.
            t0 += p.group, g = 0, parity ^= 1u;
            const uint32_t t = t0 + place;
            float most = -INFINITY, sum = 0.f;
            uint32_t at = 0;
            if (kind == 0 ? t <= k : t < k) {
                const float *row = kind == 0 ? target + (size_t)t * p.target_stride : draft + (size_t)t * p.draft_stride;
                auto add = [&](float (&v)[kBatch], auto index) {
                    if (GREEDY) {
#pragma unroll
                        for (int j = 0; j < kBatch; j++)
                            if (index(j) < hi) take_larger(most, at, clean(v[j]), index(j));
                        return;
                    }
                    float m = most;
#pragma unroll
                    for (int j = 0; j < kBatch; j++) m = fmaxf(m, v[j]);
                    float from = m == -INFINITY ? 0.f : m;
                    const uint64_t per2 = pair(per_bit, per_bit), from2 = pair(-from, -from);
                    uint64_t sums2 = 0;
#pragma unroll
                    for (int j = 0; j < kBatch; j += 2) {
                        const float2 e = unpair(mul2(add2(pair(v[j], v[j + 1]), from2), per2));
                        sums2 = add2(sums2, pair(power(e.x), power(e.y)));
                    }
                    const float2 two = unpair(sums2);
                    float s = fmaf(sum, power((most - from) * per_bit), two.x + two.y);
                    if (!(s < INFINITY) || m == INFINITY) {  // NaN or infinity among them: once more, as they count
                        m = most;
#pragma unroll
                        for (int j = 0; j < kBatch; j++) m = fmaxf(m, v[j] = clean(v[j]));
                        from = m == -INFINITY ? 0.f : m;
                        s = sum * power((most - from) * per_bit);
                        for (int j = 0; j < kBatch; j++) s += power((v[j] - from) * per_bit);
                    }
                    most = m, sum = s;
                };
                float v[kBatch];
                const uint32_t head = min((4u - (uint32_t)((uintptr_t)(row + lo) / 4 & 3u)) & 3u, hi - lo);  // ahead of the first 16-byte boundary
                if (head && warp % per_row == 0) {
#pragma unroll
                    for (int j = 0; j < kBatch; j++) v[j] = -INFINITY;
                    if (lane < head) v[0] = read(row + lo + lane);
                    add(v, [&](int j) { return j == 0 && lane < head ? lo + lane : hi; });
                }
                uint32_t i = lo + head + 4 * first;
                for (; i + (kBatch - 4) * step + 4 <= hi; i += kBatch * step) {
#pragma unroll
                    for (int j = 0; j < kBatch; j += 4) {
                        const float4 x = read(reinterpret_cast<const float4 *>(row + i + j * step));
                        v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
                    }
                    add(v, [&](int j) { return i + (j & 3) + (j & ~3) * step; });
                }
                if (i < hi) {  // what is left
                    auto index = [&](int j) { return i + (j & 3) + (j & ~3) * step; };
#pragma unroll
                    for (int j = 0; j < kBatch; j++) v[j] = index(j) < hi ? read(row + index(j)) : -INFINITY;
                    add(v, index);
                }
            }
            if (GREEDY) {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) take_larger(most, at, __shfl_xor_sync(0xffffffffu, most, d), __shfl_xor_sync(0xffffffffu, at, d));
                sum = __uint_as_float(at);
            } else {
                join(most, sum, per_bit);
            }
            if (lane < CTAS) cluster.map_shared_rank(&sh, lane)->row[parity][rank][warp] = make_float2(most, sum);
            cluster.sync();
            // a warp per row
            if (warp < kinds * p.group) {
                most = -INFINITY, sum = 0.f, at = 0;
                for (uint32_t i = lane; i < per_row * CTAS; i += 32) {
                    const float2 o = sh.row[parity][i / per_row][warp * per_row + i % per_row];
                    if (GREEDY) {
                        take_larger(most, at, o.x, __float_as_uint(o.y));
                    } else {
                        const float m = fmaxf(most, o.x), from = m == -INFINITY ? 0.f : m;
                        sum = sum * power((most - from) * per_bit) + o.y * power((o.x - from) * per_bit);
                        most = m;
                    }
                }
                if (GREEDY) {
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) take_larger(most, at, __shfl_xor_sync(0xffffffffu, most, d), __shfl_xor_sync(0xffffffffu, at, d));
                    sum = __uint_as_float(at);
                } else {
                    join(most, sum, per_bit);
                }
                if (lane == 0) sh.whole[warp] = make_float2(most, sum);
            }
            __syncthreads();
        }
        // Place t0 + g, by all threads alike.
        a = t0 + g;
        const float2 of_p = sh.whole[g], of_q = draft ? sh.whole[p.group + g] : make_float2(-INFINITY, 1.f);
        pm = of_p.x, qm = of_q.x;
        bool unsure = false;
        if (a < k) {
            bool fits = pm != -INFINITY && sh.target_at[a] != -INFINITY;
            if (GREEDY) {
                fits = fits && __float_as_uint(of_p.y) == sh.drafts[a];
            } else if (fits) {
                const float px = exp2f((sh.target_at[a] - pm) * per_bit) / of_p.y;
                float ux = sh.random[a];
                if (draft) ux *= qm == -INFINITY ? 0.f : exp2f((sh.draft_at[a] - qm) * per_bit) / of_q.y;
                const bool few_bits = fmaxf(px, ux) < kFewBits;
                fits = !few_bits && ux < px * (1.f - kNear);
                unsure = few_bits || (!fits && !(ux > px * (1.f + kNear)));
            }
            if (fits) {
                g++;
                continue;
            }
        }
        if (GREEDY || pm == -INFINITY) {
            if (rank == 0) finish(pm == -INFINITY ? kNothing : __float_as_uint(of_p.y));
            return;
        }
        // Not accepted, or too near to say, or the token behind the last draft: sums in 64 bits.
        pr = target + (size_t)a * p.target_stride, qr = draft && a < k && qm != -INFINITY && !alone ? draft + (size_t)a * p.draft_stride : nullptr;
        const uint32_t without = !draft && a < k ? sh.drafts[a] : kNothing;
        ratio = qr ? (double)of_p.y / (double)of_q.y : 0.0;
        bool known = !qr;
        for (;;) {
            const Weight wp(pm, p.per_bit), wq(qr ? qm : 0.f, p.per_bit);
            double s0 = 0.0, s1 = 0.0, a0 = 0.0, a1 = 0.0, near = 0.0;
            const uint32_t i1 = min(lo + (warp + 1) * share, hi);
            float x[kAhead], y[kAhead];
            auto load = [&](uint32_t i0) {
#pragma unroll
                for (int j = 0; j < kAhead; j++) {
                    const uint32_t i = i0 + j * 32;
                    x[j] = i < i1 ? read(pr + i) : -INFINITY;
                    y[j] = qr && i < i1 ? read(qr + i) : -INFINITY;
                }
            };
            load(lo + warp * share + lane);
            for (uint32_t i0 = lo + warp * share + lane; i0 - lane < i1; i0 += kAhead * 32) {
                float xs[kAhead], ys[kAhead];
#pragma unroll
                for (int j = 0; j < kAhead; j++) xs[j] = x[j], ys[j] = y[j];
                load(i0 + kAhead * 32);
#pragma unroll
                for (int j = 0; j < kAhead; j++) {
                    const double e = wp(xs[j]);
                    s0 += e;
                    if (qr) {
                        const double f = wq(ys[j]), d = fma(-ratio, f, e);
                        s1 += f;
                        const int of_d = __double2hiint(d);
                        if (of_d >= 0) a0 += known ? d : e, a1 += f;  // (a difference of zero adds nothing)
                        if ((of_d & 0x7FF00000) <= (__double2hiint(e) & 0x7FF00000) - (15 << 20)) near += e;  // |d| < 2^-14 e, and all below 2^-16
                    } else if (i0 + j * 32 != without) {
                        a0 += e;
                    }
                }
            }
            double of[5] = {s0, s1, a0, a1, near};
#pragma unroll
            for (int d = 16; d > 0; d >>= 1)
#pragma unroll
                for (int i = 0; i < 5; i++) of[i] += __shfl_xor_sync(0xffffffffu, of[i], d);
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < 5; i++) sh.warp_exact[i][warp] = of[i];
            __syncthreads();
            pass++;
            if (warp < 5) {
                const double s = sum16(lane < kWarps ? sh.warp_exact[warp][lane] : 0.0);
                if (lane < CTAS) cluster.map_shared_rank(&sh, lane)->exact[pass & 1u][warp][rank] = s;
            }
            cluster.sync();
#pragma unroll
            for (int i = 0; i < 5; i++) z[i] = __shfl_sync(0xffffffffu, sum16(lane < CTAS ? sh.exact[pass & 1u][i][lane] : 0.0), 0);
            if (qr) ratio = z[0] / z[1];
            if (known || !(z[4] > 0x1p-14 * (z[2] - ratio * z[3]))) break;
            known = true;
        }
        if (unsure && !alone) {
            const double px = Weight(pm, p.per_bit)(sh.target_at[a]) / z[0], qx = !draft ? 1.0 : qr ? Weight(qm, p.per_bit)(sh.draft_at[a]) / z[1] : 0.0;
            if ((double)sh.random[a] * qx < px) {
                g++;
                continue;
            }
        }
        less = known ? 0.0 : ratio;
        if (!qr || z[2] - less * z[3] > 0.0) break;
        alone = true;  // nothing of w: p and q are the same, and a draft cannot be in either
    }

    // The token: the slice of the vocabulary in which the running sum passes the goal, and in it the warp's share (every warp for itself).
    const uint32_t without = !draft && a < k ? sh.drafts[a] : kNothing;
    const double goal = (double)sh.last_random * (z[2] - less * z[3]);
    double run = 0.0;
    const uint32_t owner = part_of(lane < CTAS ? sh.exact[pass & 1u][2][lane] - less * sh.exact[pass & 1u][3][lane] : 0.0, goal, run);
    if (owner == 16) {
        if (rank == 0) finish(kNothing);
        return;
    }
    if (rank != owner) return;
    const uint32_t of_warp = part_of(lane < kWarps ? sh.warp_exact[2][lane] - less * sh.warp_exact[3][lane] : 0.0, goal, run) & 15u;
    // That share again, some consecutive tokens a thread: the first whose running sum passes the goal, else the last that is possible.
    const Weight wp(pm, p.per_bit), wq(qr ? qm : 0.f, p.per_bit);
    auto w_of = [&](uint32_t i) {
        double w = wp(read(pr + i));
        if (qr) w = fma(-wq(read(qr + i)), ratio, w);
        return i == without || !(w > 0.0) ? 0.0 : w;
    };
    const uint32_t each = (share + kThreads - 1) / kThreads, s0 = min(lo + of_warp * share, hi), s1 = min(s0 + share, hi), i0 = min(s0 + tid * each, s1), i1 = min(i0 + each, s1);
    double own = 0.0;
    uint32_t last = 0;  // one more than its index
    for (uint32_t i = i0; i < i1; i++) {
        const double w = w_of(i);
        own += w;
        if (w > 0.0) last = i + 1;
    }
    double scan = own;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, scan, d);
        if (lane >= (uint32_t)d) scan += x;
    }
    last = __reduce_max_sync(0xffffffffu, last);
    if (lane == 31) sh.warp_scan[warp] = scan;
    if (lane == 0) sh.last[warp] = last;
    __syncthreads();
    run += __shfl_sync(0xffffffffu, sum16(lane < warp ? sh.warp_scan[lane] : 0.0), 0) + (scan - own);
    if (run + own > goal)
        for (uint32_t i = i0; i < i1; i++) {
            const double w = w_of(i);
            run += w;
            if (w > 0.0 && run > goal) {
                atomicMin(&sh.pick, i);
                break;
            }
        }
    __syncthreads();
    last = __reduce_max_sync(0xffffffffu, lane < kWarps ? sh.last[lane] : 0u);
    finish(sh.pick != kNothing ? sh.pick : last - 1);
}

template <int CTAS, bool GREEDY>
cudaError_t launch_variant(const VerifyParams &p, uint32_t n_seqs, bool pdl, cudaStream_t s) {
    auto kern = verify_kernel<CTAS, GREEDY>;
    if (CTAS > 8) {
        const cudaError_t e = kernel_opt_in(reinterpret_cast<const void *>(kern), 0, true);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_seqs * CTAS);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CTAS;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl ? 2 : 1;
    return launch_config(cfg, kern, p);
}

}  // namespace

cudaError_t launch_verify_drafts(const VerifyDrafts &a, int sm_count, cudaStream_t s, uint64_t *launches) {
    VerifyParams p = {};
    p.target = a.target, p.draft = a.draft, p.drafts = a.drafts, p.lens = a.lens, p.random = a.random, p.tokens = a.tokens, p.accepted = a.accepted;
    p.vocab = a.vocab, p.n_draft = a.n_draft, p.target_stride = a.target_stride, p.draft_stride = a.draft_stride;
    p.per_bit = 1.4426950408889634 / (double)a.temperature;
    // Sixteen CTAs per sequence while all have an SM and a half: 13 sequences with four drafts over 128256 tokens take 35.7 us with sixteen and 54.4 with eight, 18 58 and
    // 65, 24 64 and 65, 32 77 and 69; over 32000 tokens 13 take 17.1 and 21.8, 32 42 and 29.
    const bool few = (uint64_t)a.n_seqs * 16 <= 2 * (uint64_t)sm_count;
    const uint32_t slice = a.vocab / (few ? 16 : 8) * 4 + 1, most = a.draft ? 8 : 16;
    // Places of a group: few logits per CTA go by in latency and want all their places at once (one sequence over 32000 tokens: 16.2 us one by one, 13.6 by twos, 12.0
    // by fours; greedy ones of 24 sequences 16.0, 11.9, 10.7, 8.7 by eights), many in bandwidth, where rows behind a rejected draft are better not read (32 sequences over
    // 128256: 69, 71, 76, 84).
    p.group = 1;
    while (p.group < most && p.group * 2 * slice <= 65536 && p.group <= a.n_draft) p.group *= 2;
    cudaError_t e;
    if (few) e = a.greedy ? launch_variant<16, true>(p, a.n_seqs, a.pdl, s) : launch_variant<16, false>(p, a.n_seqs, a.pdl, s);
    else e = a.greedy ? launch_variant<8, true>(p, a.n_seqs, a.pdl, s) : launch_variant<8, false>(p, a.n_seqs, a.pdl, s);
    if (e == cudaSuccess) ++*launches;
    return e;
}

}  // namespace yule
