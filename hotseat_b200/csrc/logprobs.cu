// Scores of logit rows: log probabilities of given tokens, entropy, rank and
// the top alternatives, in one pass over the logits.
//
// A row is cut into up to 8 contiguous shares, taken by a cluster of as many
// CTAs or, where there are many rows, by fewer in turn (down to one: 2,048 rows
// of 151,936 in bf16, all outputs, top 5: 400 us; one CTA a row instead of
// eight, so fewer starts, joins and first bounds, was 790 -> 521 of that). The
// 512 threads of a CTA hold a share in registers, so the logits are read once
// (but for the candidates): the maximum, then sum exp(x - m) and
// sum exp(x - m)(x - m) (for the entropy ln l - t / l), the tokens before the
// given one, and the top candidates all come from the registers, while the
// next share is on its way to the L2. The CTAs' results meet in distributed
// shared memory; nothing is kept in global memory between them, so calls on
// several streams share nothing. Shares' sums are joined in one order, whoever
// took them.
//
// Top candidates: the order's key of a token is unique, so the `top`-th
// largest of the largest keys of 32 or 64 thread groups is a bound that all of
// a CTA's top tokens reach, and few others: these are collected and each
// placed by counting the larger ones. After a CTA's first share its top tokens
// so far are such a bound. Where more tokens reach it than there is room for
// (logits in order, say), the bound is taken from the threads' own largest
// keys, which leaves at most 64 x 40. The cluster's first CTA merges the CTAs'
// lists the same way.
//
// A share that is longer than a CTA holds (20,480 logits) goes through the
// registers in strips, their results joined in turn. A strip costs the same
// whatever is in it, so a row costs its strips: 2,048 rows in bf16, all outputs,
// top 5, take 400 us at 151,936, 128,256, 102,400 and 32,000 tokens, 453 at
// 50,257, whose rows are not aligned, and 733 at 256,000, where every share has two.
//
// Bound by the instructions of a logit (about a dozen) and the barriers of a
// strip: 2,048 rows of 151,936 in bf16: entropy alone 294 us (2.1 TB/s), with
// log probability, rank and 20 alternatives 443. One f32 row: 7.6 and 12.9 us.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "common.h"
#include "device.cuh"
#include "kernels.h"
#include "kv_region.h"

namespace cg = cooperative_groups;

namespace hs {
namespace {

constexpr uint32_t kThreads = 512, kPer = 40;       // logits a thread holds
constexpr uint32_t kStrip = kThreads * kPer;        // logits a CTA holds
constexpr uint32_t kCluster = 8;
constexpr uint32_t kCand = kLogprobTop * kPer + kLogprobTop;  // candidates at most, and the strips' so far
constexpr float kLog2e = 1.44269504088896341f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
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

template <int DT>
__device__ __forceinline__ float logit(const void* p, uint64_t e) {
    if constexpr (DT == HS_F32) return __ldg(static_cast<const float*>(p) + e);
    else if constexpr (DT == HS_F16) return __half2float(static_cast<const __half*>(p)[e]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[e]);
}

// The order of logits as unsigned numbers (NaN first, -0 equal to 0), and the
// key of a token: larger for one that comes earlier (logit descending, id
// ascending). Never 0 for a token.
__device__ __forceinline__ uint32_t order(float x) {
    uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    return isnan(x) ? 0xffffffffu : b;
}
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) { return ((uint64_t)order(x) << 32) | (0xffffffffu - id); }
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return 0xffffffffu - (uint32_t)k; }

// sum exp(x - m) and sum exp(x - m)(x - m) of some logits with maximum m, and
// how many come before the given token.
struct Sums {
    double l = 0.0, t = 0.0;
    float m = -INFINITY;
    uint32_t before = 0;
};
// Two disjoint sets of logits as one. A NaN in either stays.
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    r.before = a.before + b.before;
    auto add = [&](const Sums& x) {
        if (isnan(x.l) || isnan(x.t)) {
            r.l = r.t = __longlong_as_double(0x7ff8000000000000ll);
        } else if (x.l != 0.0) {
            // d <= 0 and the weight in f32: off by 2^-22 at d = 0 (where it is 1), less
            // of the whole the further below
            const float d = fmaxf(__fsub_rn(x.m, r.m), -200.0f);
            const double w = d == 0.0f ? 1.0 : (double)ex2(__fmul_rn(d, kLog2e));
            r.l += x.l * w;
            r.t += (x.t + x.l * (double)d) * w;
        }
    };
    add(a);
    add(b);
    return r;
}

// Lanes 0 .. n - 1's (n a power of two) as one, pairs first: in lane 0.
__device__ __forceinline__ Sums join_lanes(Sums x, uint32_t n) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t o = 1; o < n; o <<= 1) {
        Sums y;
        y.l = __shfl_xor_sync(0xffffffffu, x.l, o);
        y.t = __shfl_xor_sync(0xffffffffu, x.t, o);
        y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
        y.before = __shfl_xor_sync(0xffffffffu, x.before, o);
        x = lane & o ? join(y, x) : join(x, y);
    }
    return x;
}

struct Shared {
    double l[2][16], t[2][16];     // the warps' sums, of every other strip
    float m[2][16];
    uint32_t before[2][16], n_cand[2];
    float row_m, row_lz;
    uint64_t bound;
    uint64_t group[64];            // largest key of a thread group
    uint64_t best[kThreads];       // ... of a thread (the second way)
    uint64_t cand[kCand];
    uint64_t all[kCluster * kLogprobTop];
    uint64_t top[2][kLogprobTop];  // the top tokens so far, in order (0: none), and the next ones
    Sums sums[kCluster];           // the shares' sums; the first CTA's: everyone's, and top tokens in `all`
};

// Logit i = (j * 512 + tid) * V + e of a strip is this thread's number V j + e.
template <int V>
__device__ __forceinline__ uint32_t place(uint32_t k) {
    return ((k / V) * kThreads + threadIdx.x) * V + k % V;
}

template <int DT, int V>
__global__ void __launch_bounds__(kThreads, 2) k_logprobs(const LogprobArgs a, uint32_t shares, uint32_t share) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared& s = *reinterpret_cast<Shared*>(smem);
    constexpr uint32_t EB = DT == HS_F32 ? 4 : 2;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    cg::cluster_group cl = cg::this_cluster();
    const uint32_t rank = blockIdx.x, ctas = gridDim.x;
    const uint64_t r = blockIdx.y + (uint64_t)blockIdx.z * gridDim.y;
    if (r >= a.rows) return;  // the whole cluster
    const uint8_t* row = static_cast<const uint8_t*>(a.logits) + r * a.row_stride * EB;
    const uint32_t id = a.ids ? __ldg(a.ids + r) : 0xffffffffu;
    const float xt = id < a.vocab ? logit<DT>(row, id) : __int_as_float(0x7fc00000);
    // every CTA of the cluster is there before one writes to the first
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    if (tid < kLogprobTop) s.top[0][tid] = 0;
    if (tid == 0) s.n_cand[0] = s.n_cand[1] = 0, s.bound = 0;
    uint32_t cur = 0, strip = 0;  // of s.top and s.n_cand; strips so far

    for (uint32_t v = rank; v < shares; v += ctas) {
    const uint32_t begin = min(v * share, a.vocab), end = min(begin + share, a.vocab);
    if (begin == end && tid == 0) s.sums[v] = Sums();
    for (uint32_t from = begin; from < end; from += kStrip, strip++) {
        const uint32_t n = min(kStrip, end - from), par = strip & 1;
        const uint8_t* mine = row + (uint64_t)from * EB;
        // the strip, -inf behind its end
        float x[kPer];
#pragma unroll
        for (uint32_t j = 0; j < kPer / V; j++) {
            const uint32_t i = (j * kThreads + tid) * V;
            if (V > 1 && i + V <= n) {
                const uint4 w = __ldg(reinterpret_cast<const uint4*>(mine + (uint64_t)i * EB));
                const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    if constexpr (DT == HS_F32) {
                        x[V * j + e % V] = __uint_as_float(u[e]);
                    } else if constexpr (DT == HS_F16) {
                        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[e]));
                        x[V * j + 2 * e % V] = f.x, x[V * j + (2 * e + 1) % V] = f.y;
                    } else {
                        x[V * j + 2 * e % V] = __uint_as_float(u[e] << 16), x[V * j + (2 * e + 1) % V] = __uint_as_float(u[e] & 0xffff0000u);
                    }
                }
            } else {
#pragma unroll
                for (uint32_t e = 0; e < V; e++) x[V * j + e] = i + e < n ? logit<DT>(mine, i + e) : -INFINITY;
            }
        }
        {   // the next strip on its way to the L2
            const uint32_t f = from + kStrip < end ? from + kStrip : min((v + ctas) * share, a.vocab);
            const uint32_t g = v + ctas < shares || f < end ? min(f + min(kStrip, share), a.vocab) : f;
            for (uint64_t b = tid * 128ull; b < (uint64_t)(g - f) * EB; b += kThreads * 128ull)
                asm volatile("prefetch.global.L2 [%0];" ::"l"(row + (uint64_t)f * EB + b));
        }
        // the warp's maximum (NaN skipped: it shows in the sums), under which its sums stand
        float m = -INFINITY;
#pragma unroll
        for (uint32_t k = 0; k < kPer; k++) m = fmaxf(m, x[k]);
        const float mine_top = m;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));

        // Sums over eight logits in f32, over more in f64. A logit 200 below the
        // maximum has no weight, and its distance is cut there: 0 times -inf is not.
        double l = 0.0, t = 0.0;
        const float shift = m == -INFINITY ? 0.0f : -m;
        const uint64_t shift2 = pack2(shift, shift), log2e2 = pack2(kLog2e, kLog2e);
#pragma unroll
        for (uint32_t k = 0; k < kPer; k += 8) {
            uint64_t lp[4], tp[4];
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint64_t d2 = add2(pack2(x[k + 2 * e], x[k + 2 * e + 1]), shift2);
                float d0, d1, y0, y1;
                unpack2(d2, &d0, &d1);
                unpack2(mul2(d2, log2e2), &y0, &y1);
                lp[e] = pack2(ex2(y0), ex2(y1));
                tp[e] = mul2(lp[e], pack2(fmaxf(d0, -200.0f), fmaxf(d1, -200.0f)));
            }
            const uint64_t ls = add2(add2(lp[0], lp[1]), add2(lp[2], lp[3])), ts = add2(add2(tp[0], tp[1]), add2(tp[2], tp[3]));
            float l0, l1, t0, t1;
            unpack2(ls, &l0, &l1);
            unpack2(ts, &t0, &t1);
            l += (double)(l0 + l1), t += (double)(t0 + t1);
        }
        const bool nan = isnan(l);  // one of the thread's logits is, or +inf among them
        uint32_t before = 0;
        if (a.rank && id < a.vocab) {
            if (isnan(xt)) {  // before it: NaNs of lower ids
#pragma unroll
                for (uint32_t k = 0; k < kPer; k++) before += isnan(x[k]) && from + place<V>(k) < id ? 1 : 0;
            } else {
                // greater or NaN, or equal with a lower id: not below, by ids, a
                // bound of xt or of the number just under it (none under -inf: NaN)
                float under = xt == 0.0f ? __int_as_float(0x80000001u) : __int_as_float(__float_as_int(xt) + (xt < 0.0f ? 1 : -1));
                if (xt == -INFINITY) under = __int_as_float(0x7fc00000);
                // V logits at once lie on one side of the id, but for the V that hold it
#pragma unroll
                for (uint32_t j = 0; j < kPer / V; j++) {
                    const uint32_t p = place<V>(V * j), first = from + p;
                    const float limit = first + V <= id ? under : xt;
#pragma unroll
                    for (uint32_t e = 0; e < V; e++) before += !(x[V * j + e] <= limit) ? 1 : 0;
                    if (first < id && id < first + V) {
#pragma unroll
                        for (uint32_t e = 0; e < V; e++) before += x[V * j + e] == xt && first + e < id ? 1 : 0;
                    }
                }
                // the strip's filling, -inf, is before nothing; but `under` is NaN for a token of -inf
                if (xt == -INFINITY) {
#pragma unroll
                    for (uint32_t j = 0; j < kPer / V; j++)
#pragma unroll
                        for (uint32_t e = 0; e < V; e++)
                            if (place<V>(V * j + e) >= n && from + place<V>(V * j) + V <= id) before--;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
            t += __shfl_xor_sync(0xffffffffu, t, o);
            before += __shfl_xor_sync(0xffffffffu, before, o);
        }
        if (lane == 0) s.l[par][warp] = l, s.t[par][warp] = t, s.m[par][warp] = m, s.before[par][warp] = before;

        bool all = a.top && strip == 0;  // the same for every thread, as what follows from barriers
        // Candidates from `bound` on, of the threads that may hold any: few, so that
        // their warp reads their logits again, eight lanes a thread's (a thread over
        // its own registers is 40 steps of code that the others wait for).
        auto collect = [&](bool holds, uint64_t bound) {
            const uint32_t all_of = __ballot_sync(0xffffffffu, holds);
            for (uint32_t who = all_of; who;) {
                uint32_t one = who;  // without its first lane / 8
#pragma unroll
                for (uint32_t i = 0; i < 4; i++) {
                    if (i < lane / 8) one &= one - 1;
                    who &= who - 1;
                }
                if (!one) continue;
                const uint32_t t = warp * 32 + __ffs(one) - 1;
#pragma unroll
                for (uint32_t i = 0; i < kPer / 8; i++) {
                    const uint32_t k = 8 * i + lane % 8, p = (k / V * kThreads + t) * V + k % V;
                    if (p >= n) continue;
                    const uint64_t key = order_key(logit<DT>(mine, p), from + p);
                    if (key >= bound) {
                        const uint32_t c = atomicAdd(&s.n_cand[cur], 1u);
                        if (c < kCand) s.cand[c] = key;
                    }
                }
            }
            return all_of != 0;
        };
        if (a.top && strip > 0) {
            // the top tokens so far are a bound already (the first strip held as many)
            const uint64_t bound = s.top[cur][a.top - 1];
            if (__syncthreads_or(collect(nan || order_key(mine_top, from + place<V>(0)) >= bound, bound))) {
                const uint32_t nc = s.n_cand[cur];
                if (nc > kCand) {
                    all = true;
                } else {
                    for (uint32_t i = tid; i < nc + a.top; i += kThreads) {
                        const uint64_t key = i < nc ? s.cand[i] : s.top[cur][i - nc];
                        uint32_t above = i < nc ? 0 : i - nc;
                        for (uint32_t j = 0; j < nc; j++) above += s.cand[j] > key ? 1 : 0;
                        if (i < nc)
                            for (uint32_t j = 0; j < a.top; j++) above += s.top[cur][j] > key ? 1 : 0;
                        if (above < a.top) s.top[cur ^ 1][above] = key;
                    }
                    if (tid == 0) s.n_cand[cur ^ 1] = 0;
                    __syncthreads();
                    cur ^= 1;
                }
            }
        }
        if (all) {
            // the thread's largest key: a NaN, else its largest logit, the first of equal ones
            uint32_t at = 0;
#pragma unroll
            for (uint32_t i = 0; i < kPer; i++) {
                const uint32_t k = kPer - 1 - i;
                if (x[k] == mine_top) at = k;
            }
            uint64_t best = place<V>(at) < n ? order_key(mine_top, from + place<V>(at)) : 0;
            if (nan) {
#pragma unroll 1
                for (uint32_t k = 0; k < kPer; k++) {
                    if (place<V>(k) >= n) continue;
                    const uint64_t key = order_key(logit<DT>(mine, place<V>(k)), from + place<V>(k));
                    if (key > best) best = key;
                }
            }
            // groups of 16 threads, of 8 for more than 16 tokens; the bound is the
            // key that top - 1 of theirs are above (0 if fewer hold any)
            const uint32_t size = a.top <= 16 ? 16 : 8, groups = kThreads / size;
            uint64_t g = best;
            for (uint32_t o = size / 2; o > 0; o >>= 1) {
                const uint64_t other = __shfl_xor_sync(0xffffffffu, g, o);
                g = other > g ? other : g;
            }
            if (tid % size == 0) s.group[tid / size] = g;
            __syncthreads();
            // the strips' top tokens so far stand with this one's
            const uint32_t held = strip > 0 ? a.top : 0;
            if (tid == 0) s.n_cand[cur] = held, s.bound = 0;
            if (tid < held) s.cand[tid] = s.top[cur][tid];
            __syncthreads();
            if (tid < groups) {
                const uint64_t key = s.group[tid];
                uint32_t above = 0;
#pragma unroll 16
                for (uint32_t i = 0; i < groups; i++) above += s.group[i] > key ? 1 : 0;
                if (key && above == a.top - 1) s.bound = key;
            }
            __syncthreads();
            collect(best && best >= s.bound, s.bound);
            __syncthreads();
            if (s.n_cand[cur] > kCand) {  // the same for every thread
                s.best[tid] = best;
                __syncthreads();
                if (tid == 0) s.n_cand[cur] = held, s.bound = 0;
                __syncthreads();
                uint32_t above = 0;
                for (uint32_t i = 0; i < kThreads; i++) above += s.best[i] > best ? 1 : 0;
                if (best && above == a.top - 1) s.bound = best;
                __syncthreads();
                collect(best && best >= s.bound, s.bound);
                __syncthreads();
            }
            const uint32_t nc = s.n_cand[cur];
            if (tid < a.top) s.top[cur ^ 1][tid] = 0;
            __syncthreads();
            for (uint32_t i = tid; i < nc; i += kThreads) {
                const uint64_t key = s.cand[i];
                uint32_t above = 0;
                for (uint32_t j = 0; j < nc; j++) above += s.cand[j] > key ? 1 : 0;
                if (above < a.top) s.top[cur ^ 1][above] = key;
            }
            if (tid == 0) s.n_cand[cur ^ 1] = 0;
            __syncthreads();
            cur ^= 1;
        }
        if (!a.top) __syncthreads();
        // The warps' sums as the strip's, by one of them: lanes 0 .. 15, pairs
        // first. (Their places are taken anew two strips on, behind a barrier.)
        if (warp == strip % (kThreads / 32)) {
            Sums part;
            if (lane < 16) {
                part.l = s.l[par][lane], part.t = s.t[par][lane], part.m = s.m[par][lane], part.before = s.before[par][lane];
                if (part.m == -INFINITY && !isnan(part.l)) part.l = part.t = 0.0;
            }
            part = join_lanes(part, 16);
            if (lane == 0) s.sums[v] = from == begin ? part : join(s.sums[v], part);
        }
    }
    }
    __syncthreads();
    // results go to the cluster's first CTA; the others are done then
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    Shared& to = *cl.map_shared_rank(&s, 0);
    const uint32_t nk = ctas * a.top;
    if (rank > 0 && tid < shares && tid % ctas == rank) to.sums[tid] = s.sums[tid];
    if (tid < a.top) to.all[rank * a.top + tid] = s.top[cur][tid];
    __syncwarp();  // the barrier takes a warp as one
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (rank != 0) return;
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp == 0) {
        Sums sums;
        if (lane < shares) sums = s.sums[lane];
        sums = join_lanes(sums, shares);
        // nothing but -inf, or +inf: no distribution
        if (sums.m == -INFINITY || sums.m == INFINITY) sums.l = sums.t = __longlong_as_double(0x7ff8000000000000ll);
        const double lz = log(sums.l);
        if (lane == 0) {
            s.row_m = sums.m;
            s.row_lz = (float)lz;
            if (a.logp) a.logp[r] = (xt - sums.m) - (float)lz;
            if (a.entropy) a.entropy[r] = (float)(lz - sums.t / sums.l);
            if (a.rank) a.rank[r] = id < a.vocab ? sums.before : 0xffffffffu;
        }
    }
    __syncthreads();
    for (uint32_t i = tid; i < nk; i += kThreads) {
        const uint64_t key = s.all[i];
        if (!key) continue;
        uint32_t above = 0;
#pragma unroll 8
        for (uint32_t j = 0; j < nk; j++) above += s.all[j] > key ? 1 : 0;
        if (above < a.top) {
            const uint32_t tok = key_id(key);
            if (a.top_ids) a.top_ids[r * a.top + above] = tok;
            if (a.top_logp) a.top_logp[r * a.top + above] = (logit<DT>(row, tok) - s.row_m) - s.row_lz;
        }
    }
}

template <int DT>
cudaError_t launch_dt(const LogprobArgs& a, cudaStream_t st) {
    // Shares of a multiple of 8 logits, so that they start as aligned as the row
    // does; a short row's are 4,096 logits at least.
    constexpr int V = DT == HS_F32 ? 4 : 8;
    uint32_t shares = 1;
    while (shares < kCluster && shares * 4096u < a.vocab) shares *= 2;
    const uint32_t share = ((a.vocab + shares - 1) / shares + 7) / 8 * 8;
    // Few rows: a CTA a share. Rows that fill the GPU's 296 places twice without
    // that: fewer CTAs a row, which take its shares in turn, with the same sums.
    uint32_t ctas = 1;
    while (ctas < shares && (uint64_t)a.rows * ctas < 4 * 148) ctas *= 2;
    const uint64_t bytes = DT == HS_F32 ? 4 : 2;
    const bool vec = reinterpret_cast<uintptr_t>(a.logits) % 16 == 0 && a.row_stride * bytes % 16 == 0;
    cudaLaunchConfig_t cfg = {};
    const uint32_t ry = a.rows < 65535 ? a.rows : 65535;
    cfg.gridDim = dim3(ctas, ry, (a.rows + ry - 1) / ry);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = st;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = ctas;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return vec ? cudaLaunchKernelEx(&cfg, k_logprobs<DT, V>, a, shares, share) : cudaLaunchKernelEx(&cfg, k_logprobs<DT, 1>, a, shares, share);
}

}  // namespace

cudaError_t launch_logprobs(const LogprobArgs& a, cudaStream_t st) {
    if (!a.rows) return cudaSuccess;
    return a.dtype == HS_F32 ? launch_dt<HS_F32>(a, st) : a.dtype == HS_F16 ? launch_dt<HS_F16>(a, st) : launch_dt<HS_BF16>(a, st);
}

int check_logprobs(uint32_t rows, uint32_t vocab, const void* ids, uint32_t top, const void* logp, const void* rank,
                   const void* top_ids, const void* top_logp) {
    if (!vocab || vocab > (1u << 24)) return fail(HS_E_ARG, "vocab must be 1..2^24");
    if (rows > (1u << 24)) return fail(HS_E_ARG, "more than 2^24 rows");
    if (top > kLogprobTop || top > vocab) return fail(HS_E_ARG, "top must be at most 64 and at most vocab");
    if (!ids && (logp || rank)) return fail(HS_E_ARG, "logp and rank need ids");
    if (!top && (top_ids || top_logp)) return fail(HS_E_ARG, "top outputs with top = 0");
    return HS_OK;
}

}  // namespace hs

extern "C" int hs_logprobs(int device, const void* logits, uint32_t dtype, uint64_t row_stride, uint32_t rows,
                           uint32_t vocab, const uint32_t* ids, uint32_t top, float* logp, float* entropy,
                           uint32_t* rank, uint32_t* top_ids, float* top_logp, void* stream) {
    using namespace hs;
    int rc = check_logprobs(rows, vocab, ids, top, logp, rank, top_ids, top_logp);
    if (rc) return rc;
    if (dtype > HS_BF16) return fail(HS_E_ARG, "unknown element type");
    if (!rows) return HS_OK;
    if (!logits) return fail(HS_E_ARG, "null logits");
    if (reinterpret_cast<uintptr_t>(logits) % (dtype == HS_F32 ? 4 : 2))
        return fail(HS_E_ARG, "logits are not aligned to their element type");
    DeviceGuard g(device);
    HS_CUDA_TRY(g.err);
    LogprobArgs a{logits, row_stride, dtype, rows, vocab, ids, top, logp, entropy, rank, top_ids, top_logp};
    cudaError_t e = launch_logprobs(a, static_cast<cudaStream_t>(stream));
    return e == cudaSuccess ? HS_OK : fail(HS_E_CUDA, std::string("logprobs launch: ") + cudaGetErrorString(e));
}
