// Attention over the 8-bit KV cache.
//
// Codes are integers of at most 127, which f16 holds exactly, so both
// products run on the tensor cores with the codes as one operand and no loss:
// the scales are taken outside, on the scores (K) and on the weights (V). The
// other operand, f32 rows' q and every type's weights, is an f16 pair hi + lo
// (22 bits; q of 16 bits is exact in one f16), after scaling by powers of two that
// keep it in f16's range:
//   q:       its largest element to [2^13, 2^14)
//   weights: w = exp(S - m) s_v 2^(10 - e), 2^e at or above the largest s_v that
//            the row has seen so far, so that weights down to 2^-34 of the largest
//            still count, and what a row does not see does not matter
// Scores, statistics and sums are f32.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "common.h"
#include "device.cuh"
#include "kernels.h"
#include "kv8.h"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

namespace hs {
namespace {

template <int DT>
__device__ __forceinline__ float load1(const void* p, uint64_t e) {
    if constexpr (DT == HS_F32) return static_cast<const float*>(p)[e];
    else if constexpr (DT == HS_F16) return __half2float(static_cast<const __half*>(p)[e]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[e]);
}
template <int DT>
__device__ __forceinline__ void store1(void* p, uint64_t e, float x) {
    if constexpr (DT == HS_F32) static_cast<float*>(p)[e] = x;
    else if constexpr (DT == HS_F16) static_cast<__half*>(p)[e] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(p)[e] = __float2bfloat16_rn(x);
}

// Four consecutive elements; `vec`: at once, where base and strides allow it.
template <int DT>
__device__ __forceinline__ void load4(const void* p, uint64_t e, bool vec, float* x) {
    if (!vec) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = load1<DT>(p, e + i);
    } else if constexpr (DT == HS_F32) {
        const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + e);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const uint16_t*>(p) + e);
        const uint32_t w[2] = {v.x, v.y};
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if constexpr (DT == HS_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}
template <int DT>
__device__ __forceinline__ void store4(void* p, uint64_t e, bool vec, float4 v) {
    if (!vec) {
        store1<DT>(p, e, v.x), store1<DT>(p, e + 1, v.y), store1<DT>(p, e + 2, v.z), store1<DT>(p, e + 3, v.w);
    } else if constexpr (DT == HS_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + e) = v;
    } else if constexpr (DT == HS_F16) {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + e) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p) + e) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

// ------------------------------------------------------------- single rows

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// f16 of the signed bytes 0 and 2 (or 1 and 3) of w: a byte b with its sign
// bit flipped, under the exponent of 1024, is 1152 + b, exactly.
__device__ __forceinline__ uint32_t sub1152(uint32_t x) {
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&x), __floats2half2_rn(1152.0f, 1152.0f));
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t even_bytes(uint32_t w) { return sub1152((w & 0x00ff00ffu) ^ 0x64806480u); }
__device__ __forceinline__ uint32_t odd_bytes(uint32_t w) { return sub1152(((w >> 8) & 0x00ff00ffu) ^ 0x64806480u); }

// f16 pair of (x, y): hi, and what hi leaves
__device__ __forceinline__ void pair16(float x, float y, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    *hi = *reinterpret_cast<const uint32_t*>(&h);
    *lo = *reinterpret_cast<const uint32_t*>(&l);
}

// The power of two that takes amax into [2^13, 2^14), and its inverse; 1 for
// zeros and what is not finite.
__device__ __forceinline__ float fit_f16(float amax, float* inverse) {
    const int e = (int)(__float_as_uint(amax) >> 23) - 127;
    const bool ok = amax > 0.0f && e < 128;
    // both factors stay normal: e + 114 and 140 - e are at most 254 for e >= -114
    const int k = ok ? 13 - max(e, -113) : 0;
    *inverse = __uint_as_float((uint32_t)(127 - k) << 23);
    return __uint_as_float((uint32_t)(127 + k) << 23);
}

constexpr float kLog2e = 1.44269504088896341f;
// The running maximum of scores (in powers of two) is raised once a score
// passes it by more than this: weights stay below 2^4, and most blocks skip
// the reduction over the warp and the rescaling.
constexpr float kSlack = 4.0f;

__device__ __forceinline__ void cp_async4(void* dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(src)) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// A single row per slot. One CTA takes a split of the positions of one (slot,
// KV head), its warps blocks of BP positions in turn. A warp computes
// S^T = K q^T (16 positions by 8 query heads an instruction; the codes are
// the operand of 16 rows, so a group of up to 8 heads wastes none of it) and
// O^T += V^T w^T, with K's and V's codes loaded straight into the operand
// layout: a lane's 16 bytes of a K row are its share of four k-steps (a dot
// product does not mind which), its bytes of four V rows its share of the
// m-tiles. Blocks arrive by cp.async in a ring of each warp's own, so that a
// warp waits for its own copies only; with loads into registers instead, one
// block ahead, the same kernel took 56 us (46) for 64 sequences of 8,192
// positions, 14/2 heads of 64.
//
// The splits are joined in two levels: those of a cluster (up to 8) through
// distributed shared memory, each CTA a share of the outputs; where a row has
// more, each share's last cluster joins the clusters' records in order.
//
// Bound by issue and by chains of dependent instructions: about 515 a warp for
// a block's 4 KB of codes, four fifths of all at 64 x 8,192 positions, where the
// schedulers issue in 48 % of their clocks and the first stalls are fixed
// latencies and the CTA's barriers; below ~2,000 positions by the CTA's start and
// joins. The grid has every split that the region's max_ctx allows, and CTAs
// without one leave at once. 64 rows of 14/2 heads of 64, f32, up to 2,048
// positions: 17.5 us, 3.6 at the memory's rate; 8,192 positions each: 46 us
// (3.1 TB/s); one row: 6.2 us at 2,048 positions, 15.5 at 32,768 (12/2 heads of
// 128, f16).
template <int HD, int DT, int NT>
struct DecGeom {
    static constexpr uint32_t BP = HD == 64 ? 32 : 16;  // positions of a block: 4 KB of codes either way
    static constexpr uint32_t MB = BP / 16;
    static constexpr uint32_t KS = HD / 16;             // k-steps of the scores, m-tiles of the output
    static constexpr uint32_t NC = 8 * NT;
    static constexpr uint32_t W = 4, THREADS = 32 * W;
    // A warp's ring of blocks: K rows; V rows, padded so that the rows a lane
    // group reads together fall into different banks; K and V scales.
    static constexpr uint32_t STAGES = 2, VP = HD + 16, V_AT = BP * HD, S_AT = V_AT + BP * VP, STAGE = S_AT + 8 * BP;
    static constexpr uint32_t RING = W * STAGES * STAGE;
    static constexpr uint32_t OS = HD + 4;  // row stride of the outputs, which take the ring's space
    static_assert(RING >= W * NC * OS * 4, "the outputs fit in the ring");
    // f32 rows keep q as pairs; q of 16 bits is exact in one f16. Weights are
    // pairs for every type: one f16 moves a result by 2^-12 of the largest value
    // under it, which a sum of values that cancel shows in bf16 too.
    static constexpr bool QPAIR = DT == HS_F32;
};

template <int HD, int DT, int NT>
__global__ void __launch_bounds__(DecGeom<HD, DT, NT>::THREADS, NT == 1 ? 4 : 2) k_kv8_single(const Kv8AttendArgs a) {
    using G = DecGeom<HD, DT, NT>;
    constexpr uint32_t BP = G::BP, MB = G::MB, KS = G::KS, NC = G::NC, W = G::W, THREADS = G::THREADS;
    constexpr uint32_t OS = G::OS;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ uint32_t sm_q[2][NT][KS][2][32];  // q as operand words [hi, lo][k-step][2][lane]
    __shared__ float sm_m[W][NC], sm_l[W][NC], sm_cf[NC], cta_m[NC], cta_l[NC];
    __shared__ uint32_t sm_last;
    float(*sm_o)[NC][OS] = reinterpret_cast<float(*)[NC][OS]>(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    // KV heads of a position run side by side: with rows [pos][head] they share lines of the L2
    const uint32_t slot = blockIdx.z, split = blockIdx.y, cs = a.cluster, first = split & ~(cs - 1);
    const uint32_t kvh = a.chunks == 1 ? blockIdx.x : blockIdx.x / a.chunks, chunk = blockIdx.x - kvh * a.chunks;
    const uint32_t h0 = kvh * a.group + chunk * NC, cols = min(NC, a.group - chunk * NC);
    const uint32_t item = slot * gridDim.x + blockIdx.x;
    const uint32_t pos = __ldg(a.rows.pos + slot);
    const uint8_t* base = reinterpret_cast<const uint8_t*>(__ldg(reinterpret_cast<const unsigned long long*>(a.kv.base + slot)));
    if (pos >= a.kv.max_ctx) {  // the whole cluster leaves here
        if (split == 0) {
            if (pos != kPosNone && tid == 0) atomicOr(a.rows.err, ERR_POS);
            for (uint32_t i = tid; i < cols * HD; i += THREADS)
                store1<DT>(const_cast<void*>(a.out.p), slot * a.out.row + (h0 + i / HD) * a.out.head + i % HD, 0.0f);
        }
        return;
    }
    const uint32_t n = pos + 1;
    const uint32_t len = kv8_split_len(n, HD, a.max_splits), splits = (n + len - 1) / len;
    // and here: no split for this CTA, in a cluster that has none or that joins
    // without it (a thread that has left is not waited for at a cluster's barrier)
    if (split >= splits && (first >= splits || splits <= cs)) return;
    const uint32_t from = min(split * len, n), to = min(n, from + len);

    const uint64_t ps = a.kv.pos_stride;
    const float* ksp = reinterpret_cast<const float*>(base + a.kv.scale_off(0, kvh, 0));
    const float* vsp = reinterpret_cast<const float*>(base + a.kv.scale_off(1, kvh, 0));
    constexpr uint32_t LPR = HD / 16, RPI = 32 / LPR;  // lanes a row, rows a warp copies at once
    const uint32_t lr = lane / LPR, lc = lane % LPR * 16;
    const uint8_t* kp = base + a.kv.code_off(0, kvh, 0) + lc;
    const uint8_t* vp = base + a.kv.code_off(1, kvh, 0) + lc;
    uint8_t* ring = smem + warp * (G::STAGES * G::STAGE);

    // Copies the block at p0 into a stage. Positions past the split are read
    // as its last one and get no weight. One group a call, empty past the end.
    auto fetch = [&](uint32_t p0, uint8_t* st) {
        if (p0 < to) {
            const uint64_t sp = (uint64_t)(min(p0 + lane % BP, to - 1) >> a.kv.block_shift) * a.kv.sblk_stride;
            if (HD == 64 || lane < 16) cp_async4(st + G::S_AT + 4 * (lane % BP), ksp + sp);
            if (HD == 64 || lane >= 16) cp_async4(st + G::S_AT + 4 * BP + 4 * (lane % BP), vsp + sp);
            uint8_t *dk = st + lr * HD + lc, *dv = st + G::V_AT + lr * G::VP + lc;
            if (p0 + BP <= to) {
                const uint64_t at = (p0 + lr) * ps, step = RPI * ps;
                const uint8_t *k = kp + at, *v = vp + at;
#pragma unroll
                for (uint32_t i = 0; i < BP / RPI; i++, k += step, v += step) {
                    cp_async16(dk + i * RPI * HD, k);
                    cp_async16(dv + i * RPI * G::VP, v);
                }
            } else {
#pragma unroll
                for (uint32_t i = 0; i < BP / RPI; i++) {
                    const uint64_t at = min(p0 + lr + i * RPI, to - 1) * ps;
                    cp_async16(dk + i * RPI * HD, kp + at);
                    cp_async16(dv + i * RPI * G::VP, vp + at);
                }
            }
        }
        cp_async_commit();
    };
    uint32_t p0 = from + warp * BP, st_in = 0, st_out = 0;
#pragma unroll
    for (uint32_t i = 0; i < G::STAGES - 1; i++) fetch(p0 + i * W * BP, ring + i * G::STAGE);
    st_in = G::STAGES - 1;

    // q as the second operand, prepared once for the CTA: column c of n-tile
    // c / 8 is head h0 + c, its element d = 64 i + 16 t + 4 j + e goes to k-step
    // 4 i + j of lane 4 (c % 8) + t: word e % 2, half e / 2
#pragma unroll
    for (uint32_t i = 0; i < NC / W; i++) {
        const uint32_t c = warp * (NC / W) + i;
        float x[HD / 32], top = 0.0f;
#pragma unroll
        for (uint32_t e = 0; e < HD / 32; e++) {
            x[e] = c < cols ? load1<DT>(a.q.p, slot * a.q.row + (uint64_t)(h0 + c) * a.q.head + lane + 32 * e) : 0.0f;
            top = fmaxf(top, fabsf(x[e]));
        }
#pragma unroll
        for (uint32_t d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        float inv;
        const float fit = fit_f16(top, &inv);
        if (lane == 0) sm_cf[c] = (a.scale * kLog2e) * inv;
#pragma unroll
        for (uint32_t e = 0; e < HD / 32; e++) {
            const uint32_t d = lane + 32 * e, k = d / 64 * 4 + d % 16 / 4, to_lane = 4 * (c % 8) + d % 64 / 16;
            const __half hi = __float2half_rn(x[e] * fit);
            reinterpret_cast<__half*>(&sm_q[0][c / 8][k][d & 1][to_lane])[(d & 2) / 2] = hi;
            if constexpr (G::QPAIR)
                reinterpret_cast<__half*>(&sm_q[1][c / 8][k][d & 1][to_lane])[(d & 2) / 2] =
                    __float2half_rn(x[e] * fit - __half2float(hi));
        }
    }
    __syncthreads();
    uint32_t qh[NT][KS][2], ql[G::QPAIR ? NT : 1][G::QPAIR ? KS : 1][2];
    float cf[NT][2];  // columns 2t, 2t + 1: softmax scale x log2(e) x what q was scaled by
#pragma unroll
    for (uint32_t nt = 0; nt < NT; nt++) {
        cf[nt][0] = sm_cf[8 * nt + 2 * t], cf[nt][1] = sm_cf[8 * nt + 2 * t + 1];
#pragma unroll
        for (uint32_t j = 0; j < KS; j++)
#pragma unroll
            for (uint32_t w = 0; w < 2; w++) {
                qh[nt][j][w] = sm_q[0][nt][j][w][lane];
                if constexpr (G::QPAIR) ql[nt][j][w] = sm_q[1][nt][j][w][lane];
            }
    }

    float o[NT][KS][4] = {}, m[NT][2], l[NT][2] = {}, vmax = 0.0f, vfit = 0.0f;
#pragma unroll
    for (uint32_t nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -INFINITY;

    auto block = [&](auto tail) {
        constexpr bool TAIL = decltype(tail)::value;
        cp_async_wait<G::STAGES - 2>();
        __syncwarp();
        const uint8_t* st = ring + st_out * G::STAGE;
        st_out = st_out + 1 == G::STAGES ? 0 : st_out + 1;
        // the stage before this one was read to its end: its space takes the next block
        fetch(p0 + (G::STAGES - 1) * W * BP, ring + st_in * G::STAGE);
        st_in = st_in + 1 == G::STAGES ? 0 : st_in + 1;
        // scores: rows g and g + 8 of each 16 positions, columns 2t and 2t + 1
        float s[NT][MB][4] = {};
#pragma unroll
        for (uint32_t b = 0; b < MB; b++)
#pragma unroll
            for (uint32_t j = 0; j < KS; j++) {
                const uint4 w0 = *reinterpret_cast<const uint4*>(st + (16 * b + g) * HD + j / 4 * 64 + 16 * t);
                const uint4 w1 = *reinterpret_cast<const uint4*>(st + (16 * b + 8 + g) * HD + j / 4 * 64 + 16 * t);
                const uint32_t u = j % 4 == 0 ? w0.x : j % 4 == 1 ? w0.y : j % 4 == 2 ? w0.z : w0.w;
                const uint32_t v = j % 4 == 0 ? w1.x : j % 4 == 1 ? w1.y : j % 4 == 2 ? w1.z : w1.w;
                const uint32_t f[4] = {even_bytes(u), even_bytes(v), odd_bytes(u), odd_bytes(v)};
#pragma unroll
                for (uint32_t nt = 0; nt < NT; nt++) {
                    if constexpr (G::QPAIR) mma16816(s[nt][b], f, ql[nt][j][0], ql[nt][j][1]);
                    mma16816(s[nt][b], f, qh[nt][j][0], qh[nt][j][1]);
                }
            }
        float vs[MB][2], top[NT][2];
        bool grew = false, vgrew = false;
#pragma unroll
        for (uint32_t nt = 0; nt < NT; nt++) top[nt][0] = top[nt][1] = -INFINITY;
#pragma unroll
        for (uint32_t b = 0; b < MB; b++)
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) {
                const uint32_t at = 16 * b + 8 * r + g;
                const bool in = !TAIL || p0 + at < to;
                const float ks = reinterpret_cast<const float*>(st + G::S_AT)[at];
                vs[b][r] = in ? reinterpret_cast<const float*>(st + G::S_AT)[BP + at] : 0.0f;
                vgrew |= vs[b][r] > vmax;
#pragma unroll
                for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
                    for (uint32_t c = 0; c < 2; c++) {
                        float& x = s[nt][b][2 * r + c];
                        x = in ? x * (ks * cf[nt][c]) : -INFINITY;
                        top[nt][c] = fmaxf(top[nt][c], x);
                    }
            }
        uint32_t va[MB][KS][4];  // V^T: (row 2i or 2i + 1 of the lane's bytes) by position pairs
#pragma unroll
        for (uint32_t b = 0; b < MB; b++)
#pragma unroll
            for (uint32_t h = 0; h < 2; h++) {
                const uint8_t* v0 = st + G::V_AT + (16 * b + 8 * h + 2 * t) * G::VP + (HD / 8) * g;
                uint32_t w[2][HD / 32];
#pragma unroll
                for (uint32_t r = 0; r < 2; r++) {
                    if constexpr (HD == 64) {
                        const uint2 x = *reinterpret_cast<const uint2*>(v0 + r * G::VP);
                        w[r][0] = x.x, w[r][1] = x.y;
                    } else {
                        const uint4 x = *reinterpret_cast<const uint4*>(v0 + r * G::VP);
                        w[r][0] = x.x, w[r][1] = x.y, w[r][2] = x.z, w[r][3] = x.w;
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < KS / 2; i++) {
                    const uint32_t lo = __byte_perm(w[0][i], w[1][i], 0x5410), hi = __byte_perm(w[0][i], w[1][i], 0x7632);
                    va[b][2 * i][2 * h] = even_bytes(lo), va[b][2 * i][2 * h + 1] = odd_bytes(lo);
                    va[b][2 * i + 1][2 * h] = even_bytes(hi), va[b][2 * i + 1][2 * h + 1] = odd_bytes(hi);
                }
            }

#pragma unroll
        for (uint32_t nt = 0; nt < NT; nt++) grew |= top[nt][0] > m[nt][0] + kSlack || top[nt][1] > m[nt][1] + kSlack;
        if (__any_sync(0xffffffffu, grew || vgrew)) {
            // new maxima for the warp (over the 8 row groups), older sums scaled to them
            float vnew = vmax;
#pragma unroll
            for (uint32_t b = 0; b < MB; b++) vnew = fmaxf(vnew, fmaxf(vs[b][0], vs[b][1]));
#pragma unroll
            for (uint32_t d = 4; d < 32; d <<= 1) vnew = fmaxf(vnew, __shfl_xor_sync(0xffffffffu, vnew, d));
            float vback = 1.0f;
            if (vnew > vmax) {  // the power of two above vnew
                const uint32_t e = min((__float_as_uint(vnew) >> 23) + 1, 254u);
                const float fit = __uint_as_float(min(264u - e, 254u) << 23);  // 2^10 for a weight of 1
                vback = vfit > 0.0f ? fit / vfit : 1.0f;
                vfit = fit;
                vmax = __uint_as_float(e << 23);
            }
#pragma unroll
            for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
                for (uint32_t c = 0; c < 2; c++) {
                    float x = fmaxf(m[nt][c], top[nt][c]);
#pragma unroll
                    for (uint32_t d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    const float f = x == m[nt][c] ? 1.0f : ex2(m[nt][c] - x);
                    m[nt][c] = x;
                    l[nt][c] *= f;
#pragma unroll
                    for (uint32_t i = 0; i < KS; i++) {
                        o[nt][i][c] *= f * vback;
                        o[nt][i][2 + c] *= f * vback;
                    }
                }
        }
#pragma unroll
        for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
            for (uint32_t b = 0; b < MB; b++) {
                float w[4];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    const float p = ex2(s[nt][b][e] - m[nt][e & 1]);
                    l[nt][e & 1] += p;
                    w[e] = p * (vs[b][e >> 1] * vfit);
                }
                uint32_t w0, w1, x0, x1;
                pair16(w[0], w[1], &w0, &x0);
                pair16(w[2], w[3], &w1, &x1);
                w0 = transpose8x8(w0), w1 = transpose8x8(w1);
                x0 = transpose8x8(x0), x1 = transpose8x8(x1);
#pragma unroll
                for (uint32_t i = 0; i < KS; i++) {
                    mma16816(o[nt][i], va[b][i], x0, x1);
                    mma16816(o[nt][i], va[b][i], w0, w1);
                }
            }
    };
    for (; p0 + BP <= to; p0 += W * BP) block(std::false_type{});
    if (p0 < to) block(std::true_type{});
    cp_async_wait<0>();
    __syncthreads();  // every warp's ring is free for the outputs

    // the warps' records: outputs [column][d], maxima and sums (a warp without a block: -inf, 0, 0)
    const float vinv = vfit > 0.0f ? 1.0f / vfit : 0.0f;
#pragma unroll
    for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
        for (uint32_t c = 0; c < 2; c++) {
            float x = l[nt][c];
#pragma unroll
            for (uint32_t d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
            const uint32_t col = 8 * nt + 2 * t + c;
            if (g == 0) sm_m[warp][col] = m[nt][c], sm_l[warp][col] = x;
            float* to_o = &sm_o[warp][col][(HD / 8) * g];
#pragma unroll
            for (uint32_t i = 0; i < KS; i += 2)
                *reinterpret_cast<float4*>(to_o + 2 * i) = make_float4(o[nt][i][c] * vinv, o[nt][i][2 + c] * vinv,
                                                                       o[nt][i + 1][c] * vinv, o[nt][i + 1][2 + c] * vinv);
        }
    __syncthreads();
    // the CTA's record, in the first warp's place: a float4 of a column a thread
    for (uint32_t i = tid; i < cols * (HD / 4); i += THREADS) {
        const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
        float mm = -INFINITY, ll = 0.0f, f[W];
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (uint32_t w = 0; w < W; w++) mm = fmaxf(mm, sm_m[w][col]);
#pragma unroll
        for (uint32_t w = 0; w < W; w++) {
            f[w] = from + w * BP < to ? ex2(sm_m[w][col] - mm) : 0.0f;
            ll = fmaf(sm_l[w][col], f[w], ll);
            const float4 x = *reinterpret_cast<const float4*>(&sm_o[w][col][d]);
            acc.x = fmaf(x.x, f[w], acc.x), acc.y = fmaf(x.y, f[w], acc.y);
            acc.z = fmaf(x.z, f[w], acc.z), acc.w = fmaf(x.w, f[w], acc.w);
        }
        *reinterpret_cast<float4*>(&sm_o[0][col][d]) = acc;
        if (d == 0) cta_m[col] = mm, cta_l[col] = ll;
    }
    auto store = [&](uint32_t col, uint32_t d, float4 acc, float ll) {
        const uint64_t at = slot * a.out.row + (uint64_t)(h0 + col) * a.out.head + d;
        const float inv = __frcp_rn(ll);
        store4<DT>(const_cast<void*>(a.out.p), at, a.out_vec, make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
    };
    if (splits == 1) {
        __syncthreads();
        for (uint32_t i = tid; i < cols * (HD / 4); i += THREADS) {
            const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
            store(col, d, *reinterpret_cast<const float4*>(&sm_o[0][col][d]), cta_l[col]);
        }
        return;
    }

    // a cluster's splits: CTA `rank` joins its share of the outputs (the lanes'
    // loops before a cluster's barrier differ in length, and a warp meets it as one)
    cg::cluster_group cl = cg::this_cluster();
    __syncwarp();
    cl.sync();
    const uint32_t rank = split - first, held = min(cs, splits - first);
    const uint32_t shares = splits <= cs ? splits : cs;
    const uint32_t per = (cols * (HD / 4) + shares - 1) / shares, i0 = rank * per, i1 = min(cols * (HD / 4), i0 + per);
    const uint32_t n_cl = (splits + cs - 1) / cs;
    constexpr uint32_t REC = kv8_record(HD, NC);  // outputs, then each share's copy of maxima and sums
    float* rec0 = a.part + (uint64_t)item * a.max_clusters * REC;
    float* rec = rec0 + first / cs * REC;
    const uint32_t stats = NC * HD + rank * 2 * NC;
    for (uint32_t i = i0 + tid; i < i1; i += THREADS) {
        const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
        float mm = -INFINITY, ll = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float mr[8];
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) {
            mr[r] = r < held ? *cl.map_shared_rank(&cta_m[col], r) : -INFINITY;
            mm = fmaxf(mm, mr[r]);
        }
#pragma unroll
        for (uint32_t r = 0; r < 8; r++) {
            if (r >= held) continue;
            const float f = ex2(mr[r] - mm);
            ll = fmaf(*cl.map_shared_rank(&cta_l[col], r), f, ll);
            const float4 x = *reinterpret_cast<const float4*>(cl.map_shared_rank(&sm_o[0][col][d], r));
            acc.x = fmaf(x.x, f, acc.x), acc.y = fmaf(x.y, f, acc.y);
            acc.z = fmaf(x.z, f, acc.z), acc.w = fmaf(x.w, f, acc.w);
        }
        if (n_cl == 1) {
            store(col, d, acc, ll);
        } else {
            *reinterpret_cast<float4*>(rec + 4 * i) = acc;
            if (d == 0 || i == i0) rec[stats + col] = mm, rec[stats + NC + col] = ll;
        }
    }
    // no CTA leaves while others read its record: their reads lie before the barrier
    __syncwarp();
    cluster_sync();
    if (n_cl == 1) return;

    // more clusters: the last one to finish this share joins their records in order
    __threadfence();
    __syncthreads();
    uint32_t* counter = a.counters + item * 8 + rank;
    if (tid == 0) sm_last = atomicAdd(counter, 1u);
    __syncthreads();
    if (sm_last != n_cl - 1) return;
    __threadfence();
    if (tid == 0) *counter = 0;
    for (uint32_t i = i0 + tid; i < i1; i += THREADS) {
        const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
        float mm = -INFINITY, ll = 0.0f;
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (uint32_t c = 0; c < n_cl; c++) {
            const float* r = rec0 + c * REC;
            const float mc = __ldcg(r + stats + col), lc = __ldcg(r + stats + NC + col);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(r + 4 * i));
            const float up = fmaxf(mm, mc), f = up == mm ? 1.0f : ex2(mm - up), fc = ex2(mc - up);
            mm = up;
            ll = fmaf(lc, fc, ll * f);
            acc.x = fmaf(x.x, fc, acc.x * f), acc.y = fmaf(x.y, fc, acc.y * f);
            acc.z = fmaf(x.z, fc, acc.z * f), acc.w = fmaf(x.w, fc, acc.w * f);
        }
        store(col, d, acc, ll);
    }
}

// ------------------------------------------------------------------- chunks

// Rows of prompts and chunks of them, on the fifth-generation tensor cores.
// A CTA takes 256 of the (row, head of the group) pairs of one (slot, KV
// head) and walks the positions in tiles of 128:
//
//   warps 0-3, 4-7  one 128-row tile each, a thread a row: scores from TMEM,
//                   softmax, weights back to TMEM over the scores they came
//                   from, the tile's outputs from TMEM into f32 registers;
//                   the first thread issues the tile's MMAs
//   warps 8-15      codes from the cache to f16 tiles in shared memory, 16
//                   positions a warp (f32 rows: warps 8-11, 32 positions): K as
//                   it lies, V transposed. A warp loads a tile's codes into
//                   registers as it writes the one before, and waits for no
//                   other warp.
//
//   S = Q K^T    A = Q (shared), B = K (shared), 128 x 128
//   O' = W V     A = W (TMEM),   B = V^T (shared), 128 x head_dim
//
// While one row tile's threads are at their softmax the other's products run;
// a tile's own follow one another, as its next scores take its weights' place.
//
// SPLIT: few rows over many positions (kv8_chunk_shared), which would leave
// most SMs idle. A cluster's CTAs take the positions in equal runs of steps,
// leave outputs, maxima and sums in shared memory, and each joins a share of
// the rows.
//
// Bound by the row warps' softmax (exponentials, pairs, TMEM round trips), not by
// the products: a step of 256 x 128 scores takes 4.1 us at head_dim 64 and 4.9 at
// 128 in 16 bits, 4.3 and 6.2 in f32. A CTA's start, masked step and end take 16
// to 21 us (TMEM, q, the first codes; the outputs through shared memory).
// 12/2 heads of 128, 2,048 rows a slot: 8 slots in bf16 281 us (367 TFLOP/s of
// the 1,630 measured, each product of pairs counted once); 4 in f32 184 us (280).
template <int HD, int DT>
struct ChunkGeom {
    static constexpr bool QPAIR = DT == HS_F32;
    static constexpr uint32_t KT = 128, ROWS = 256;
    // f32 rows take each tile's O' out of TMEM and sum it in registers, rounded
    // to nearest: left to grow there, 2,048 positions were 1.7e-6 off (the
    // tensor cores' sums truncate), so 7.5e-7. Their row warps get 192 registers a
    // thread, and four code warps, of 120, do with the rest.
    static constexpr bool OREG = DT == HS_F32;
    static constexpr uint32_t CW = OREG ? 4 : 8, THREADS = 256 + 32 * CW, SUB = 8 / CW;
    static constexpr uint32_t SLAB = 128 * 128;            // 128 rows of 64 f16
    static constexpr uint32_t Q_BYTES = HD / 64 * SLAB;    // one row tile, hi or lo
    static constexpr uint32_t K_BYTES = HD / 64 * SLAB, V_BYTES = 2 * HD * 128;
    static constexpr uint32_t NB = HD == 128 && QPAIR ? 1 : 2;  // K and V buffers
    static constexpr uint32_t Q_AT = 0, K_AT = Q_AT + 2 * (QPAIR ? 2 : 1) * Q_BYTES, V_AT = K_AT + NB * K_BYTES;
    static constexpr uint32_t SC_AT = V_AT + NB * V_BYTES;  // scales: [NB][K 128 | V 128 | units 8]
    static constexpr uint32_t SC = 2 * KT + KT / 16;        // floats of a buffer's scales, with V's unit for each 16
    static constexpr uint32_t BYTES = SC_AT + NB * SC * 4 + 1024;
    static_assert(SC_AT >= ROWS * HD * 4, "the outputs fit where the operands were");
    static constexpr uint32_t S_COL = 0, O_COL = 256;       // TMEM columns: S of both tiles, O' of both
    // V's scales stand in shared memory in units of 2^e, e for 16 positions, the
    // largest of them just under 2^VEXP
    static constexpr int VEXP = 10, UNIT_MIN = -126;
};

constexpr uint32_t kChunkLimit = 1u << 22;
// Registers a thread of the row warps and of the code warps where they are
// dealt out anew: two of the first and one of the second are what the launch
// of 384 threads holds, 168 a thread.
constexpr int kChunkRegsRow = 192, kChunkRegsCode = 120;

// Two f32 at once (each rounded on its own).
__device__ __forceinline__ void mul2(float* x, float a, float b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(x[0], x[1])), "l"(pack2(a, b)));
    unpack2(r, x, x + 1);
}
__device__ __forceinline__ void fma2(float* x, float a, float b) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pack2(x[0], x[1])), "l"(pack2(a, a)), "l"(pack2(b, b)));
    unpack2(r, x, x + 1);
}
__device__ __forceinline__ void add2(float* x, float a, float b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pack2(x[0], x[1])), "l"(pack2(a, b)));
    unpack2(r, x, x + 1);
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <uint32_t N = 128>
__device__ __forceinline__ void bar_sync(uint32_t id) {
    asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(N) : "memory");
}

template <int HD, int DT, bool SPLIT>
__global__ void __launch_bounds__(ChunkGeom<HD, DT>::THREADS, 1) k_kv8_chunk(const Kv8AttendArgs a) {
    using G = ChunkGeom<HD, DT>;
    constexpr uint32_t KT = G::KT, NB = G::NB;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t kfull[NB], kempty[NB], vfull[NB], vempty[NB], s_done[2], o_done[2];
    __shared__ uint32_t tmem_slot;
    __shared__ float row_cf[G::ROWS];
    __shared__ uint64_t row_q[G::ROWS], row_out[G::ROWS];  // element offsets of the tile's rows
    __shared__ float row_m[SPLIT ? G::ROWS : 1], row_l[SPLIT ? G::ROWS : 1];
    // the warp's number as a value that is the same for its lanes
    const uint32_t tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const uint32_t group = a.group;

    // the tile: slot, its rows' first pair, its last position. Tiles of slot i
    // start at row_start[i] * group / 256 + i, room for all that it can have.
    const uint32_t part = SPLIT ? blockIdx.x % kKv8ChunkSplits : 0, at = SPLIT ? blockIdx.x / kKv8ChunkSplits : blockIdx.x;
    const uint32_t n_at = SPLIT ? gridDim.x / kKv8ChunkSplits : gridDim.x;
    const uint32_t bt = n_at / a.kv.nkv - 1 - at / a.kv.nkv;  // long ones first
    uint32_t slot, kvh = at % a.kv.nkv;
    uint64_t f0 = 0;
    if (SPLIT && a.slot_clusters) {
        slot = at / a.slot_clusters;
        kvh = at % a.slot_clusters % a.kv.nkv;
        f0 = (uint64_t)(at % a.slot_clusters / a.kv.nkv) * G::ROWS;
    } else {
        uint32_t lo = 0, hi = a.rows.n_slots;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if ((uint64_t)__ldg(a.rows.row_start + mid) * group / G::ROWS + mid <= bt)
                lo = mid + 1;
            else
                hi = mid;
        }
        if (lo == 0) return;
        slot = lo - 1;
        f0 = (bt - ((uint64_t)__ldg(a.rows.row_start + slot) * group / G::ROWS + slot)) * G::ROWS;
    }
    const uint32_t r0 = __ldg(a.rows.row_start + slot);
    const uint32_t r1 = min(__ldg(a.rows.row_start + slot + 1), a.rows.n_rows), m = r1 > r0 ? r1 - r0 : 0;
    const uint64_t pairs = (uint64_t)m * group;
    const uint32_t pos0 = __ldg(a.rows.pos + slot);
    if (SPLIT != (pos0 < a.kv.max_ctx && kv8_chunk_shared((pairs + G::ROWS - 1) / G::ROWS, pos0, a.kv.nkv))) return;
    if (f0 >= pairs) return;
    const uint32_t live = (uint32_t)min((uint64_t)G::ROWS, pairs - f0);  // pairs of this CTA
    const uint32_t jlast = (uint32_t)((f0 + live - 1) / group);          // its last row
    if (pos0 == kPosNone || (uint64_t)pos0 + (uint32_t)(f0 / group) >= a.kv.max_ctx) {  // nothing to see
        if (pos0 != kPosNone && tid == 0) atomicOr(a.rows.err, ERR_POS);
        for (uint32_t i = tid; i < live * HD; i += G::THREADS) {
            const uint64_t f = f0 + i / HD;
            store1<DT>(const_cast<void*>(a.out.p), (r0 + f / group) * a.out.row + (kvh * group + f % group) * a.out.head + i % HD, 0.0f);
        }
        return;
    }
    const uint64_t plast = (uint64_t)pos0 + jlast;
    if (plast >= a.kv.max_ctx && tid == 0) atomicOr(a.rows.err, ERR_POS);
    const uint32_t seen = (uint32_t)min(plast + 1, (uint64_t)a.kv.max_ctx);  // positions [0, seen)
    // this CTA's positions: [first, first + end), whole tiles but for the last
    const uint32_t all = (seen + KT - 1) / KT, first = SPLIT ? all * part / kKv8ChunkSplits * KT : 0;
    const uint32_t end = (SPLIT ? min(seen, all * (part + 1) / kKv8ChunkSplits * KT) : seen) - first;
    const uint32_t tiles = (end + KT - 1) / KT;
    const uint32_t users = live > 128 ? 2 : 1;  // row tiles at work

    if (tid == 0) {
        for (uint32_t i = 0; i < NB; i++) {
            mbar_init(&kfull[i], G::CW);  // a warp's arrival each
            mbar_init(&vfull[i], G::CW);
            mbar_init(&kempty[i], users);
            mbar_init(&vempty[i], users);
        }
        for (uint32_t i = 0; i < 2; i++) {
            mbar_init(&s_done[i], 1);
            mbar_init(&o_done[i], 1);
        }
        mbar_init_fence();
    }
    if (warp == 0) {
        tc5::alloc(&tmem_slot, 512);
        tc5::relinquish();
    }
    const uint8_t* base = reinterpret_cast<const uint8_t*>(a.kv.base[slot]);
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    const uint32_t tmem = tmem_slot;
    float* sc = reinterpret_cast<float*>(smem + G::SC_AT);  // [NB][G::SC]
    // A wait that runs out marks the call and no longer waits: every thread
    // still passes every barrier, and the CTA ends.
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !mbar_wait_bounded(bar, parity, kChunkLimit)) {
            dead = true;
            atomicOr(a.rows.err, ERR_TIMEOUT);
        }
        __syncwarp();  // lanes leave the loop apart, and warp-wide instructions follow
    };

    if (warp >= 8) {
        // ---------------------------------------------------- codes to f16
        if constexpr (G::OREG) tc5::setmaxnreg_dec<kChunkRegsCode>();
        // this warp's positions of a tile: 16 of each 128 / SUB, from 16 cw on
        const uint32_t cw = warp - 8;
        constexpr uint32_t SP = KT / G::SUB;
        const uint64_t ps = a.kv.pos_stride;
        // K: a lane takes 16 codes of rows kr, kr + RPP, ...
        constexpr uint32_t CPR = HD / 16, RPP = 32 / CPR, KP = 16 / RPP;
        const uint32_t kc = lane % CPR, kr = lane / CPR;
        const float* ksp = reinterpret_cast<const float*>(base + a.kv.scale_off(0, kvh, first >> a.kv.block_shift));
        // V: four codes of each of eight positions (a 16-byte piece of a
        // transposed row), of position group vg, then vg + 1 where HD = 128.
        // Element d = 4 dw + e goes to row e * HD / 4 + dw, so that the lanes'
        // pieces fall into different banks; the outputs' columns follow.
        constexpr uint32_t DW = HD / 4, VP = HD / 64;
        const uint32_t dw = lane % DW, vg = 2 * cw + lane / DW;
        const uint8_t* kp = base + a.kv.code_off(0, kvh, first) + 16 * kc;
        const uint8_t* vp = base + a.kv.code_off(1, kvh, first) + 4 * dw;
        uint4 kw[G::SUB][KP];
        uint32_t vw[G::SUB][VP][8];
        float ks[G::SUB], vs[G::SUB];
        auto load_k = [&](uint32_t t, uint32_t u) {
            const uint32_t p0 = t * KT + u * SP + 16 * cw + kr;
            if ((t + 1) * KT <= end) {
                const uint8_t* q = kp + p0 * ps;
#pragma unroll
                for (uint32_t i = 0; i < KP; i++, q += RPP * ps) kw[u][i] = __ldg(reinterpret_cast<const uint4*>(q));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < KP; i++)
                    kw[u][i] = __ldg(reinterpret_cast<const uint4*>(kp + min(p0 + i * RPP, end - 1) * ps));
            }
        };
        auto load_v = [&](uint32_t t, uint32_t u) {
            const uint32_t p0 = t * KT + u * SP + 8 * vg;
            if ((t + 1) * KT <= end) {
                const uint8_t* q = vp + p0 * ps;
#pragma unroll
                for (uint32_t i = 0; i < VP * 8; i++, q += ps) vw[u][i / 8][i % 8] = __ldg(reinterpret_cast<const uint32_t*>(q));
            } else {
#pragma unroll
                for (uint32_t i = 0; i < VP * 8; i++)
                    vw[u][i / 8][i % 8] = __ldg(reinterpret_cast<const uint32_t*>(vp + min(p0 + i, end - 1) * ps));
            }
        };
        auto load_s = [&](uint32_t t, uint32_t u) {  // the position of lane % 16; behind the end: 0
            const uint32_t p = t * KT + u * SP + 16 * cw + lane % 16;
            const float* at = ksp + (uint64_t)(min(p, end - 1) >> a.kv.block_shift) * a.kv.sblk_stride;
            ks[u] = p < end ? __ldg(at) : 0.0f;
            vs[u] = p < end ? __ldg(at + a.kv.splane / 4) : 0.0f;
        };
        // places in the tiles of buffer 0: of a chunk's first half (the second
        // lies beside it), of the pieces' row dw (the others DW rows on)
        const uint32_t to_k = smem_u32(smem + G::K_AT) + kc / 4 * G::SLAB + (16 * cw + kr) * 128 + ((2 * kc % 8) ^ (kr & 7)) * 16;
        const uint32_t to_v = smem_u32(smem + G::V_AT) + vg / 8 * (HD * 128) + dw * 128 + ((vg % 8) ^ (dw & 7)) * 16;
#pragma unroll
        for (uint32_t u = 0; u < G::SUB; u++) load_s(0, u), load_k(0, u), load_v(0, u);
        for (uint32_t t = 0; t < tiles; t++) {
            const uint32_t b = t % NB, use = t / NB;
            float ks_now[G::SUB], vs_now[G::SUB];
#pragma unroll
            for (uint32_t u = 0; u < G::SUB; u++) {
                ks_now[u] = ks[u], vs_now[u] = vs[u];
                if (t + 1 < tiles) load_s(t + 1, u);
            }
            if (use > 0) wait(&kempty[b], (use - 1) & 1);
#pragma unroll
            for (uint32_t u = 0; u < G::SUB; u++) {
#pragma unroll
                for (uint32_t i = 0; i < KP; i++) {
                    const uint4 w = kw[u][i];
                    // codes 0, 2, 1, 3 of every four, as q's elements lie
                    const uint4 x = make_uint4(even_bytes(w.x), odd_bytes(w.x), even_bytes(w.y), odd_bytes(w.y));
                    const uint4 y = make_uint4(even_bytes(w.z), odd_bytes(w.z), even_bytes(w.w), odd_bytes(w.w));
                    // rows RPP apart: their places' swizzle is the same where RPP is 8, else it flips bit 2
                    const uint32_t row = b * G::K_BYTES + (u * SP + i * RPP) * 128, flip = RPP == 4 && (i & 1) ? 64 : 0;
                    sts128((to_k ^ flip) + row, x);
                    sts128((to_k ^ flip ^ 16) + row, y);
                }
                if (t + 1 < tiles) load_k(t + 1, u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&kfull[b]);

            if (use > 0) wait(&vempty[b], (use - 1) & 1);
#pragma unroll
            for (uint32_t u = 0; u < G::SUB; u++) {
                // scales go with V: they are read until the weights are written
                float top = fmaxf(vs_now[u], 0.0f);  // (a NaN is skipped)
#pragma unroll
                for (uint32_t d = 8; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                const int unit = max((int)(__float_as_uint(top) >> 23) - 126 - G::VEXP, G::UNIT_MIN);  // at most 128 - VEXP + 1
                float* to_s = sc + b * G::SC + u * SP + 16 * cw;
                if (lane < 16) to_s[lane] = ks_now[u], to_s[KT + lane] = vs_now[u] * __uint_as_float((127u - unit) << 23);
                if (lane == 0) sc[b * G::SC + 2 * KT + u * (SP / 16) + cw] = (float)unit;
#pragma unroll
                for (uint32_t v = 0; v < VP; v++) {
                    // elements d, d + 1, then d + 2, d + 3, by position pairs; group
                    // vg + 1's pieces lie beside group vg's: vg is even there
                    const uint32_t to = (to_v ^ (16 * v)) + b * G::V_BYTES + u * (SP / 64 * HD * 128);
#pragma unroll
                    for (uint32_t e = 0; e < 4; e += 2) {
                        uint32_t f[2][4];
#pragma unroll
                        for (uint32_t p = 0; p < 4; p++) {
                            const uint32_t x = __byte_perm(vw[u][v][2 * p], vw[u][v][2 * p + 1], e == 0 ? 0x5410 : 0x7632);
                            f[0][p] = even_bytes(x), f[1][p] = odd_bytes(x);
                        }
                        sts128(to + e * (DW * 128), make_uint4(f[0][0], f[0][1], f[0][2], f[0][3]));
                        sts128(to + (e + 1) * (DW * 128), make_uint4(f[1][0], f[1][1], f[1][2], f[1][3]));
                    }
                }
                if (t + 1 < tiles) load_v(t + 1, u);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&vfull[b]);
        }
        if constexpr (SPLIT) {  // the row warps join; what they do in registers these may not have stays theirs
            __syncthreads();
            cluster_sync();
            cluster_sync();
            __syncthreads();
            return;
        }
    } else {
        // ---------------------------------------------------- one row tile
        if constexpr (G::OREG) tc5::setmaxnreg_inc<kChunkRegsRow>();
        const uint32_t w = warp / 4, th = tid % 128, row = w * 128 + th;
        if (w < users) {
            const bool on = row < live;
            const uint64_t f = f0 + (on ? row : 0);
            const uint32_t j = (uint32_t)(f / group), h = kvh * group + (uint32_t)(f - (uint64_t)j * group);
            const uint64_t p = (uint64_t)pos0 + j;
            // the last position this row sees, of this CTA's (none: negative)
            const int lim = on && p < a.kv.max_ctx ? (int)p - (int)first : -1;
            row_q[row] = (r0 + (uint64_t)j) * a.q.row + (uint64_t)h * a.q.head;
            row_out[row] = (r0 + (uint64_t)j) * a.out.row + (uint64_t)h * a.out.head;
            __syncwarp();
            uint8_t* qt = smem + G::Q_AT + w * G::Q_BYTES;
            // q to f16 rows of 64, elements 0, 2, 1, 3 of every four as K's codes
            // lie; HD / 8 lanes take a row, eight elements each
            constexpr uint32_t LPR = HD / 8, RPW = 32 / LPR, AT_ONCE = 8;
            const uint32_t qc = lane % LPR;
#pragma unroll 1
            for (uint32_t i0 = 0; i0 < LPR; i0 += AT_ONCE) {
                float x[AT_ONCE][8];
#pragma unroll
                for (uint32_t i = 0; i < AT_ONCE; i++) {
                    const uint64_t at = row_q[w * 128 + th / 32 * 32 + (i0 + i) * RPW + lane / LPR] + 8 * qc;
                    load4<DT>(a.q.p, at, a.q_vec, x[i]);
                    load4<DT>(a.q.p, at + 4, a.q_vec, x[i] + 4);
                }
#pragma unroll
                for (uint32_t i = 0; i < AT_ONCE; i++) {
                    const uint32_t r = th / 32 * 32 + (i0 + i) * RPW + lane / LPR;
                    float top = 0.0f;
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) top = fmaxf(top, fabsf(x[i][e]));
#pragma unroll
                    for (uint32_t d = LPR / 2; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    float inv;
                    const float fit = fit_f16(top, &inv);
                    if (qc == 0) row_cf[w * 128 + r] = (a.scale * kLog2e) * inv;
                    uint32_t hi4[4], lo4[4];
#pragma unroll
                    for (uint32_t e = 0; e < 2; e++) {
                        pair16(x[i][4 * e] * fit, x[i][4 * e + 2] * fit, &hi4[2 * e], &lo4[2 * e]);
                        pair16(x[i][4 * e + 1] * fit, x[i][4 * e + 3] * fit, &hi4[2 * e + 1], &lo4[2 * e + 1]);
                    }
                    uint8_t* to = qt + qc / 8 * G::SLAB + r * 128 + ((qc % 8) ^ (r & 7)) * 16;
                    *reinterpret_cast<uint4*>(to) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
                    if constexpr (G::QPAIR) *reinterpret_cast<uint4*>(to + 2 * G::Q_BYTES) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
                }
            }
            __syncwarp();
            const float cf = row_cf[row];
            fence_proxy_async_smem();
            bar_sync(1 + w);

            const uint32_t scol = tmem + G::S_COL + w * KT, ocol = tmem + G::O_COL + w * HD;
            const uint32_t lanes = (warp % 4 * 32) << 16;
            // the tile's operands, as descriptors
            const uint64_t q_desc = tc5::sw128_desc(smem_u32(qt)), k_desc = tc5::sw128_desc(smem_u32(smem + G::K_AT)),
                           v_desc = tc5::sw128_desc(smem_u32(smem + G::V_AT));
            auto issue_s = [&](uint32_t t) {
                const uint32_t b = t % NB;
                wait(&kfull[b], t / NB & 1);
                tc5::fence_after();
                if (tc5::elect()) {
                    const uint64_t kd = k_desc + b * (G::K_BYTES / 16);
#pragma unroll
                    for (uint32_t k = 0; k < HD / 16; k++) {
                        const uint32_t at = k / 4 * (G::SLAB / 16) + 2 * (k % 4);
                        if constexpr (G::QPAIR) tc5::mma_ss(scol, q_desc + 2 * G::Q_BYTES / 16 + at, kd + at, tc5::idesc_f16(128, KT), k > 0);
                        tc5::mma_ss(scol, q_desc + at, kd + at, tc5::idesc_f16(128, KT), G::QPAIR || k > 0);
                    }
                    tc5::commit(&s_done[w]);
                    tc5::commit(&kempty[b]);
                }
                __syncwarp();
            };
            auto issue_o = [&](uint32_t t) {
                const uint32_t b = t % NB;
                tc5::fence_after();
                if (tc5::elect()) {
                    const uint64_t vd = v_desc + b * (G::V_BYTES / 16);
                    const bool more = !G::OREG && t > 0;
#pragma unroll
                    for (uint32_t k = 0; k < KT / 16; k++) {
                        const uint32_t at = k / 4 * (HD * 128 / 16) + 2 * (k % 4);
                        tc5::mma_ts(ocol, scol + k * 16 + 8, vd + at, tc5::idesc_f16(128, HD), k > 0 || more);
                        tc5::mma_ts(ocol, scol + k * 16, vd + at, tc5::idesc_f16(128, HD), true);
                    }
                    tc5::commit(&o_done[w]);
                    tc5::commit(&vempty[b]);
                }
                __syncwarp();
            };
            const bool issuer = warp % 4 == 0;
            if (issuer) issue_s(0);

            // The running maximum in powers of two (a whole number, so that it and the
            // units add up exactly), the sum of weights, the unit of the outputs.
            float mx = -INFINITY, l = 0.0f, un = G::UNIT_MIN;
            auto pow2f = [](float e) {  // a whole number -127 (gives 0) .. 127
                return __uint_as_float((__float_as_uint(12582912.0f + e) + 127u) << 23);
            };
            // Columns 16 c.. of the scores, under K's scales.
            auto scaled = [&](const float* ks, uint32_t c, float* x) {
#pragma unroll
                for (uint32_t i = 0; i < 16; i += 4) {
                    const float4 k4 = *reinterpret_cast<const float4*>(ks + 16 * c + i);
                    mul2(x + i, k4.x, k4.y);
                    mul2(x + i + 2, k4.z, k4.w);
                }
            };
            auto largest = [&](auto masked, uint32_t c, const float* x, float top, int left) {
#pragma unroll
                for (uint32_t i = 0; i < 16; i++) {
                    if constexpr (decltype(masked)::value) {
                        if ((int)(16 * c + i) <= left) top = fmaxf(top, x[i]);
                    } else {
                        top = fmaxf(top, x[i]);
                    }
                }
                return top;
            };
            // The largest unit that this row sees of a tile; of a group of 16 that it sees
            // in part, by the scales that it does see.
            auto largest_unit = [&](auto masked, const float* vs, int left) {
                const float* us = vs + KT;
                float u = G::UNIT_MIN;
                if constexpr (decltype(masked)::value) {
                    const int whole = (left + 1) >> 4, part = (left + 1) & 15;
#pragma unroll
                    for (int c = 0; c < 8; c++)
                        if (c < whole) u = fmaxf(u, us[c]);
                    if (left >= 0 && left < (int)KT - 1 && part) {
                        float top = 0.0f;
#pragma unroll 1
                        for (int i = 0; i < part; i++) top = fmaxf(top, vs[16 * whole + i]);
                        if (top > 0.0f) u = fmaxf(u, us[whole] + (float)((int)(__float_as_uint(top) >> 23) - 126 - G::VEXP));
                    }
                } else {
                    const float4 a4 = *reinterpret_cast<const float4*>(us), b4 = *reinterpret_cast<const float4*>(us + 4);
                    u = fmaxf(fmaxf(fmaxf(a4.x, a4.y), fmaxf(a4.z, a4.w)), fmaxf(fmaxf(b4.x, b4.y), fmaxf(b4.z, b4.w)));
                }
                return u;
            };
            // Weights of columns 16 c.. into TMEM over their scores (hi in the first
            // eight columns, lo in the others); adds their sum. A weight is formed times
            // 2^d, d its group's unit over the outputs' (0 or less where the group is seen
            // whole), and summed without it. Far below, where the group adds nothing,
            // d is cut; so it is far above, where a group's other values, 2^100 times
            // larger, are hidden. The masked form also takes scores whose product with cf
            // has to be rounded as their maximum was, lest the two part by whole powers of two.
            auto weights = [&](auto masked, const float* vs, uint32_t c, float* x, float off, int left, float* total) {
                uint32_t wh[8], wl[8];
                float d = fmaxf(vs[KT + c] - un, -60.0f), sum[2] = {0.0f, 0.0f};
                if constexpr (decltype(masked)::value) d = fminf(d, 100.0f);
                else off += d;
#pragma unroll
                for (uint32_t i = 0; i < 16; i += 4) {
#pragma unroll
                    for (uint32_t e = 0; e < 4; e += 2) {
                        if constexpr (decltype(masked)::value) {  // (as pairs, product and sum came out as one FMA)
                            x[i + e] = __fadd_rn(__fadd_rn(__fmul_rn(x[i + e], cf), off), d);
                            x[i + e + 1] = __fadd_rn(__fadd_rn(__fmul_rn(x[i + e + 1], cf), off), d);
                        } else {
                            fma2(x + i + e, cf, off);
                        }
                    }
#pragma unroll
                    for (uint32_t e = 0; e < 4; e++) {
                        x[i + e] = ex2(x[i + e]);
                        if constexpr (decltype(masked)::value)
                            if ((int)(16 * c + i + e) > left) x[i + e] = 0.0f;
                    }
                    add2(sum, x[i], x[i + 1]);
                    add2(sum, x[i + 2], x[i + 3]);
                    const float4 v4 = *reinterpret_cast<const float4*>(vs + 16 * c + i);
                    mul2(x + i, v4.x, v4.y);
                    mul2(x + i + 2, v4.z, v4.w);
                    if constexpr (decltype(masked)::value) {  // a scale of NaN does not reach rows before it
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++)
                            if ((int)(16 * c + i + e) > left) x[i + e] = 0.0f;
                    }
                    pair16(x[i], x[i + 1], &wh[i / 2], &wl[i / 2]);
                    pair16(x[i + 2], x[i + 3], &wh[i / 2 + 1], &wl[i / 2 + 1]);
                }
                *total = fmaf(sum[0] + sum[1], pow2f(-d), *total);
                tc5::st8(scol + lanes + 16 * c, wh);
                tc5::st8(scol + lanes + 16 * c + 8, wl);
            };
            float o[G::OREG ? HD : 1], alpha = 1.0f;  // OREG: the outputs, and what they take when tile t's are added
#pragma unroll
            for (uint32_t i = 0; i < (G::OREG ? HD : 1); i++) o[i] = 0.0f;
            auto add_o = [&](uint32_t t) {
                wait(&o_done[w], t & 1);
                tc5::fence_after();
#pragma unroll
                for (uint32_t c = 0; c < (G::OREG ? HD / 16 : 0); c++) {
                    float y[16];
                    tc5::ld16(ocol + lanes + 16 * c, y);
                    tc5::wait_ld();
#pragma unroll
                    for (uint32_t i = 0; i < 16; i++) o[16 * c + i] = fmaf(o[16 * c + i], alpha, y[i]);
                }
            };
            // One tile: the scores are read twice, for their maximum and for the
            // weights, so that few registers hold them; the next columns are on
            // their way from TMEM while these are worked on.
            float x[16], y[16];
            auto find_top = [&](auto masked, const float* ks, int left) {
                float top = -INFINITY;
                tc5::ld16(scol + lanes, x);
#pragma unroll 1
                for (uint32_t c = 0; c < 8; c += 2) {
                    tc5::wait_ld();
                    tc5::ld16(scol + lanes + 16 * (c + 1), y);
                    scaled(ks, c, x);
                    top = largest(masked, c, x, top, left);
                    tc5::wait_ld();
                    if (c < 6) tc5::ld16(scol + lanes + 16 * (c + 2), x);
                    scaled(ks, c + 1, y);
                    top = largest(masked, c + 1, y, top, left);
                }
                return top;
            };
            auto all_weights = [&](auto masked, const float* ks, float off, int left) {
                const float* vs = ks + KT;
                float sum = 0.0f;
#pragma unroll 1
                for (uint32_t c = 0; c < 8; c += 2) {
                    tc5::wait_ld();
                    tc5::ld16(scol + lanes + 16 * (c + 1), y);
                    scaled(ks, c, x);
                    weights(masked, vs, c, x, off, left, &sum);
                    tc5::wait_ld();
                    if (c < 6) tc5::ld16(scol + lanes + 16 * (c + 2), x);
                    scaled(ks, c + 1, y);
                    weights(masked, vs, c + 1, y, off, left, &sum);
                }
                l += sum;
            };
            for (uint32_t t = 0; t < tiles; t++) {
                const int left = lim - (int)(t * KT);  // columns 0..left are seen
                wait(&vfull[t % NB], t / NB & 1);
                wait(&s_done[w], t & 1);
                tc5::fence_after();
                const float* ks = sc + t % NB * G::SC;
                const bool full = __all_sync(0xffffffffu, left >= (int)KT - 1);
                float top, u;
                if (full) top = find_top(std::false_type{}, ks, left), u = largest_unit(std::false_type{}, ks + KT, left);
                else top = find_top(std::true_type{}, ks, left), u = largest_unit(std::true_type{}, ks + KT, left);
                __syncwarp();
                if constexpr (G::OREG) {
                    if (t > 0) add_o(t - 1);
                }
                top *= cf;
                u = fmaxf(un, u);
                const bool up = top > mx + kSlack || u > un;
                if (top > mx + kSlack) {
                    top = ceilf(top);
                    alpha = ex2(mx - top);
                    l *= alpha;
                    mx = top;
                } else {
                    alpha = 1.0f;
                }
                alpha *= pow2f(fmaxf(un - u, -127.0f));
                un = u;
                if (!G::OREG && t > 0 && __any_sync(0xffffffffu, up)) {  // outputs so far to the new maximum and unit
                    wait(&o_done[w], (t - 1) & 1);
                    tc5::fence_after();
#pragma unroll 1
                    for (uint32_t c = 0; c < HD / 16; c++) {
                        tc5::ld16(ocol + lanes + 16 * c, y);
                        tc5::wait_ld();
#pragma unroll
                        for (uint32_t i = 0; i < 16; i++) y[i] *= alpha;
                        tc5::st16(ocol + lanes + 16 * c, reinterpret_cast<const uint32_t*>(y));
                    }
                }
                const float off = mx == -INFINITY ? 0.0f : -mx;
                // a product with cf is off by less than a step of 2^-4 up to here
                const bool small = __all_sync(0xffffffffu, fabsf(off) <= 1048576.0f);
                tc5::ld16(scol + lanes, x);
                if (full && small) all_weights(std::false_type{}, ks, off, left);
                else all_weights(std::true_type{}, ks, off, left);
                tc5::wait_st();
                tc5::fence_before();
                bar_sync(1 + w);
                if (issuer) {
                    issue_o(t);
                    // The next scores go where this tile's weights lie, and products with
                    // different accumulators are not bound to run in the order of their issue.
                    if (t + 1 < tiles) {
                        wait(&o_done[w], t & 1);
                        issue_s(t + 1);
                    }
                }
            }
            if constexpr (G::OREG) {  // their sums back where the last tile's were
                add_o(tiles - 1);
#pragma unroll
                for (uint32_t c = 0; c < HD / 8; c++) tc5::st8(ocol + lanes + 8 * c, reinterpret_cast<const uint32_t*>(o + (G::OREG ? 8 * c : 0)));
                tc5::wait_st();
            } else {
                wait(&o_done[w], (tiles - 1) & 1);
                tc5::fence_after();
            }
            // what a row's outputs are divided by goes through shared memory: the
            // registers of this loop stay its own (rows that see nothing: sums of 0)
            const float vunit = pow2f(un);
            if constexpr (SPLIT) row_cf[row] = vunit, row_m[row] = mx, row_l[row] = l;
            else row_cf[row] = lim >= 0 ? vunit * __frcp_rn(l) : 0.0f;
        }
    }
    __syncwarp();
    if constexpr (SPLIT) {
        // Outputs to shared memory, which every product is done with: float4 q of
        // row r at r * HD / 4 + (q ^ r % 8), elements as below.
        tc5::fence_before();
        __syncthreads();
        tc5::fence_after();
        float4* rows = reinterpret_cast<float4*>(smem);
        if (warp < 4 * users) {
            const uint32_t row = warp * 32 + lane, oc = tmem + G::O_COL + warp / 4 * HD + ((warp % 4 * 32) << 16);
            const float unit = row_cf[row];
#pragma unroll 1
            for (uint32_t c = 0; c < HD / 32; c++) {
                float y[4][8];
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) tc5::ld8(oc + e * (HD / 4) + 8 * c, y[e]);
                tc5::wait_ld();
#pragma unroll
                for (uint32_t q = 0; q < 8; q++)
                    rows[row * (HD / 4) + ((8 * c + q) ^ (row & 7))] = make_float4(y[0][q] * unit, y[1][q] * unit, y[2][q] * unit, y[3][q] * unit);
            }
        }
        cg::cluster_group cl = cg::this_cluster();
        cluster_sync();
        for (uint32_t i = part * 256 + tid; i < live * (HD / 4); i += kKv8ChunkSplits * 256) {
            const uint32_t row = i / (HD / 4), q = i % (HD / 4);
            float mm = -INFINITY, ll = 0.0f, mr[kKv8ChunkSplits];
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (uint32_t r = 0; r < kKv8ChunkSplits; r++) {
                mr[r] = *cl.map_shared_rank(&row_m[row], r);
                mm = fmaxf(mm, mr[r]);
            }
#pragma unroll
            for (uint32_t r = 0; r < kKv8ChunkSplits; r++) {
                const float f = mr[r] == mm ? 1.0f : ex2(mr[r] - mm);  // (both may be -inf)
                ll = fmaf(*cl.map_shared_rank(&row_l[row], r), f, ll);
                const float4 x = *cl.map_shared_rank(&rows[row * (HD / 4) + (q ^ (row & 7))], r);
                acc.x = fmaf(x.x, f, acc.x), acc.y = fmaf(x.y, f, acc.y);
                acc.z = fmaf(x.z, f, acc.z), acc.w = fmaf(x.w, f, acc.w);
            }
            const float inv = (uint64_t)pos0 + (f0 + row) / group < a.kv.max_ctx ? __frcp_rn(ll) : 0.0f;
            store4<DT>(const_cast<void*>(a.out.p), row_out[row] + 4 * q, a.out_vec,
                       make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv));
        }
        __syncwarp();
        cluster_sync();  // no CTA leaves while others read its rows
    } else if (warp < 4 * users) {
        // Rows out, 32 columns at a time through the warp's share of q's space:
        // a float4 q of row r lies at r * 8 + (q ^ r % 8). Column e * HD / 4 + i
        // of O' is element 4 i + e. (Every product that reads q is done: the
        // tile's last outputs are.)
        const uint32_t w = warp / 4, row0 = warp * 32;
        const float unit = row_cf[row0 + lane];
        float4* stage = reinterpret_cast<float4*>(smem + G::Q_AT + w * G::Q_BYTES + warp % 4 * 4096);
        const uint32_t oc = tmem + G::O_COL + w * HD + ((warp % 4 * 32) << 16);
        bar_sync(1 + w);
#pragma unroll 1
        for (uint32_t c = 0; c < HD / 32; c++) {
            float y[4][8];
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) tc5::ld8(oc + e * (HD / 4) + 8 * c, y[e]);
            tc5::wait_ld();
#pragma unroll
            for (uint32_t q = 0; q < 8; q++)
                stage[lane * 8 + (q ^ (lane & 7))] = make_float4(y[0][q] * unit, y[1][q] * unit, y[2][q] * unit, y[3][q] * unit);
            __syncwarp();
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                const uint32_t r = 4 * i + lane / 8, q = lane % 8;
                if (row0 + r < live)
                    store4<DT>(const_cast<void*>(a.out.p), row_out[row0 + r] + 32 * c + 4 * q, a.out_vec, stage[r * 8 + (q ^ (r & 7))]);
            }
            __syncwarp();
        }
    }
    tc5::fence_before();
    __syncthreads();
    if (warp == 0) {
        tc5::fence_after();
        tc5::dealloc(tmem, 512);
    }
}

template <int HD, int DT>
cudaError_t attend_dt(const Kv8AttendArgs& a, cudaStream_t st) {
    if (a.rows.row_start) {
        using G = ChunkGeom<HD, DT>;
        const uint64_t tiles = (uint64_t)a.rows.n_rows * a.group / G::ROWS + a.rows.n_slots;
        k_kv8_chunk<HD, DT, false><<<(uint32_t)(tiles * a.kv.nkv), G::THREADS, G::BYTES, st>>>(a);
        cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess || !kv8_chunk_shared(1, a.kv.max_ctx - 1, a.kv.nkv)) return e;
        // Which rows are shared is known on the device only (and must not depend
        // on the batch): the CTAs set aside for them leave where there are none.
        Kv8AttendArgs b = a;
        b.slot_clusters = (uint32_t)std::min<uint64_t>(kKv8ChunkClusters / a.kv.nkv, ((uint64_t)a.rows.n_rows * a.group + G::ROWS - 1) / G::ROWS) * a.kv.nkv;
        uint64_t clusters = (uint64_t)b.slot_clusters * a.rows.n_slots;
        if (tiles * a.kv.nkv < clusters) clusters = tiles * a.kv.nkv, b.slot_clusters = 0;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((uint32_t)clusters * kKv8ChunkSplits);
        cfg.blockDim = dim3(G::THREADS);
        cfg.dynamicSmemBytes = G::BYTES;
        cfg.stream = st;
        cudaLaunchAttribute attr = {};
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = kKv8ChunkSplits;
        attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, k_kv8_chunk<HD, DT, true>, b);
    }
    const bool wide = kv8_single_cols(a.group) == 16;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.kv.nkv * a.chunks, (a.max_splits + a.cluster - 1) / a.cluster * a.cluster, a.rows.n_slots);
    cfg.blockDim = dim3(wide ? DecGeom<HD, DT, 2>::THREADS : DecGeom<HD, DT, 1>::THREADS);
    cfg.dynamicSmemBytes = wide ? DecGeom<HD, DT, 2>::RING : DecGeom<HD, DT, 1>::RING;
    cfg.stream = st;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1;
    attr.val.clusterDim.y = a.cluster;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return wide ? cudaLaunchKernelEx(&cfg, k_kv8_single<HD, DT, 2>, a) : cudaLaunchKernelEx(&cfg, k_kv8_single<HD, DT, 1>, a);
}

template <int HD, int DT>
cudaError_t set_limits() {
    cudaError_t e = cudaFuncSetAttribute(k_kv8_single<HD, DT, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecGeom<HD, DT, 1>::RING);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(k_kv8_single<HD, DT, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, DecGeom<HD, DT, 2>::RING);
    for (auto* chunk : {k_kv8_chunk<HD, DT, false>, k_kv8_chunk<HD, DT, true>}) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(chunk, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkGeom<HD, DT>::BYTES);
        // what setmaxnreg deals out has to be there
        cudaFuncAttributes at{};
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, chunk);
        if (e == cudaSuccess && ChunkGeom<HD, DT>::OREG && at.numRegs * 3 < 2 * kChunkRegsRow + kChunkRegsCode)
            e = cudaErrorInvalidConfiguration;
    }
    return e;
}

}  // namespace

// Per device, before the first launch there.
cudaError_t kv8_attend_set_smem_limits() {
    cudaError_t e = set_limits<64, HS_F32>();
    if (e == cudaSuccess) e = set_limits<64, HS_F16>();
    if (e == cudaSuccess) e = set_limits<64, HS_BF16>();
    if (e == cudaSuccess) e = set_limits<128, HS_F32>();
    if (e == cudaSuccess) e = set_limits<128, HS_F16>();
    if (e == cudaSuccess) e = set_limits<128, HS_BF16>();
    return e;
}

cudaError_t launch_kv8_attend(uint32_t hd, const Kv8AttendArgs& a, cudaStream_t st) {
    if (!a.rows.n_rows) return cudaSuccess;
    if (hd == 64)
        return a.q.dtype == HS_F32 ? attend_dt<64, HS_F32>(a, st)
               : a.q.dtype == HS_F16 ? attend_dt<64, HS_F16>(a, st) : attend_dt<64, HS_BF16>(a, st);
    return a.q.dtype == HS_F32 ? attend_dt<128, HS_F32>(a, st)
           : a.q.dtype == HS_F16 ? attend_dt<128, HS_F16>(a, st) : attend_dt<128, HS_BF16>(a, st);
}

}  // namespace hs
