// Attention over the 8-bit KV cache.
//
// Codes are integers of at most 127, which f16 holds exactly, so both
// products run on the tensor cores with the codes as one operand and no loss:
// the scales are taken outside, on the scores (K) and on the weights (V). The
// other operand is an f16 pair hi + lo (22 bits) for f32 rows, one f16 for
// 16-bit rows, after scaling by powers of two that keep it in f16's range:
//   q:       its largest element to [2^13, 2^14)
//   weights: w = exp(S - m) s_v 2^(10 - e), 2^e at or above the largest s_v so
//            far, so that weights down to 2^-34 of the largest still count
// Scores, statistics and sums are f32.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
    // f32 rows keep q and the weights as pairs; f16 ones the weights (one f16
    // would double their result's own rounding); q of 16 bits is exact in one
    static constexpr bool QPAIR = DT == HS_F32, WPAIR = DT != HS_BF16;
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
                uint32_t w0, w1, x0 = 0, x1 = 0;
                pair16(w[0], w[1], &w0, &x0);
                pair16(w[2], w[3], &w1, &x1);
                w0 = transpose8x8(w0), w1 = transpose8x8(w1);
                if constexpr (G::WPAIR) x0 = transpose8x8(x0), x1 = transpose8x8(x1);
#pragma unroll
                for (uint32_t i = 0; i < KS; i++) {
                    if constexpr (G::WPAIR) mma16816(o[nt][i], va[b][i], x0, x1);
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
        store1<DT>(const_cast<void*>(a.out.p), at, acc.x * inv);
        store1<DT>(const_cast<void*>(a.out.p), at + 1, acc.y * inv);
        store1<DT>(const_cast<void*>(a.out.p), at + 2, acc.z * inv);
        store1<DT>(const_cast<void*>(a.out.p), at + 3, acc.w * inv);
    };
    if (splits == 1) {
        __syncthreads();
        for (uint32_t i = tid; i < cols * (HD / 4); i += THREADS) {
            const uint32_t col = i / (HD / 4), d = i % (HD / 4) * 4;
            store(col, d, *reinterpret_cast<const float4*>(&sm_o[0][col][d]), cta_l[col]);
        }
        return;
    }

    // a cluster's splits: CTA `rank` joins its share of the outputs
    cg::cluster_group cl = cg::this_cluster();
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
    // no CTA leaves while others read its record
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n barrier.cluster.wait.aligned;" ::: "memory");
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
//   warps 8-11      codes from the cache to f16 tiles in shared memory: K as
//                   it lies, V transposed
//
//   S = Q K^T    A = Q (shared), B = K (shared), 128 x 128
//   O' = W V     A = W (TMEM),   B = V^T (shared), 128 x head_dim
//
// While one row tile's threads are at their softmax the other's products run.
// O' is summed over one tile of positions only and then added in registers:
// sums over thousands of positions stay f32 with rounding to nearest, and a
// rise of the maximum costs no pass over TMEM.
template <int HD, int DT>
struct ChunkGeom {
    static constexpr bool QPAIR = DT == HS_F32, WPAIR = DT != HS_BF16;
    static constexpr uint32_t KT = 128, ROWS = 256, THREADS = 384;
    static constexpr uint32_t SLAB = 128 * 128;            // 128 rows of 64 f16
    static constexpr uint32_t Q_BYTES = HD / 64 * SLAB;    // one row tile, hi or lo
    static constexpr uint32_t K_BYTES = HD / 64 * SLAB, V_BYTES = 2 * HD * 128;
    static constexpr uint32_t NB = HD == 128 && QPAIR ? 1 : 2;  // K and V buffers
    static constexpr uint32_t Q_AT = 0, K_AT = Q_AT + 2 * (QPAIR ? 2 : 1) * Q_BYTES, V_AT = K_AT + NB * K_BYTES;
    static constexpr uint32_t SC_AT = V_AT + NB * V_BYTES;  // scales: K [NB][128], V [NB][128]
    static constexpr uint32_t BYTES = SC_AT + NB * 2 * KT * 4 + 1024;
    static constexpr uint32_t S_COL = 0, O_COL = 256;       // TMEM columns: S of both tiles, O' of both
    static constexpr bool HOLD = HD == 64;                  // scores stay in registers between maximum and weights
};

constexpr uint32_t kChunkLimit = 1u << 22;
// Registers a thread of the row tiles' warps and of the code warps; the
// launch's 168 a thread cover two of the first and one of the second.
constexpr int kChunkRegsRow = 200, kChunkRegsCode = 104;

__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void bar_sync(uint32_t id) { asm volatile("bar.sync %0, 128;" ::"r"(id) : "memory"); }

template <int HD, int DT>
__global__ void __launch_bounds__(384, 1) k_kv8_chunk(const Kv8AttendArgs a) {
    using G = ChunkGeom<HD, DT>;
    constexpr uint32_t KT = G::KT, NB = G::NB;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ uint64_t kfull[NB], kempty[NB], vfull[NB], vempty[NB], s_done[2], o_done[2];
    __shared__ uint32_t tmem_slot;
    __shared__ float vtop[4], vratio[NB], vunit;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t group = a.group;

    // the tile: slot, its rows' first pair, its last position. Tiles of slot i
    // start at row_start[i] * group / 256 + i, room for all that it can have.
    const uint32_t bt = gridDim.x / a.kv.nkv - 1 - blockIdx.x / a.kv.nkv, kvh = blockIdx.x % a.kv.nkv;  // long ones first
    uint32_t lo = 0, hi = a.rows.n_slots;
    while (lo < hi) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((uint64_t)__ldg(a.rows.row_start + mid) * group / G::ROWS + mid <= bt)
            lo = mid + 1;
        else
            hi = mid;
    }
    if (lo == 0) return;
    const uint32_t slot = lo - 1, r0 = __ldg(a.rows.row_start + slot);
    const uint32_t r1 = min(__ldg(a.rows.row_start + slot + 1), a.rows.n_rows), m = r1 > r0 ? r1 - r0 : 0;
    const uint64_t f0 = (bt - ((uint64_t)r0 * group / G::ROWS + slot)) * G::ROWS, pairs = (uint64_t)m * group;
    if (f0 >= pairs) return;
    const uint32_t pos0 = __ldg(a.rows.pos + slot);
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
    const uint32_t end = (uint32_t)min(plast + 1, (uint64_t)a.kv.max_ctx);  // positions seen: [0, end)
    const uint32_t tiles = (end + KT - 1) / KT;
    const uint32_t users = live > 128 ? 2 : 1;  // row tiles at work

    if (tid == 0) {
        for (uint32_t i = 0; i < NB; i++) {
            mbar_init(&kfull[i], 128);
            mbar_init(&vfull[i], 128);
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
    tc5::fence_before();
    __syncthreads();
    tc5::fence_after();
    const uint32_t tmem = tmem_slot;
    float* sc = reinterpret_cast<float*>(smem + G::SC_AT);  // [NB][K 128 | V 128]
    // A wait that runs out marks the call and no longer waits: every thread
    // still passes every barrier, and the CTA ends.
    bool dead = false;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (!dead && !mbar_wait_bounded(bar, parity, kChunkLimit)) {
            dead = true;
            atomicOr(a.rows.err, ERR_TIMEOUT);
        }
    };

    if (warp >= 8) {
        // ---------------------------------------------------- codes to f16
        tc5::setmaxnreg_dec<kChunkRegsCode>();
        const uint32_t th = tid - 256;
        const uint8_t* base = reinterpret_cast<const uint8_t*>(a.kv.base[slot]);
        const uint8_t* kp = base + a.kv.code_off(0, kvh, 0);
        const uint8_t* vp = base + a.kv.code_off(1, kvh, 0);
        const float* ksp = reinterpret_cast<const float*>(base + a.kv.scale_off(0, kvh, 0));
        const float* vsp = reinterpret_cast<const float*>(base + a.kv.scale_off(1, kvh, 0));
        const uint64_t ps = a.kv.pos_stride;
        // K: a thread's 16 codes of a row, eight passes over the rows
        constexpr uint32_t CPR = HD / 16, RPP = 128 / CPR, KP = KT / RPP;
        const uint32_t kc = th % CPR, kr = th / CPR;
        // V: eight positions (one 16-byte piece of a transposed row) by HD / 8 of d
        constexpr uint32_t DW = HD / 32;  // words of a V row that a thread takes
        const uint32_t vg = (th / 64) * 8 + th % 8, vd = ((th % 64) / 8) * (HD / 8);
        uint4 kw[KP];
        uint32_t vw[8][DW];
        float ks, vs;
        auto load_k = [&](uint32_t t) {
#pragma unroll
            for (uint32_t i = 0; i < KP; i++)
                kw[i] = __ldg(reinterpret_cast<const uint4*>(kp + min(t * KT + kr + i * RPP, end - 1) * ps + 16 * kc));
            ks = __ldg(ksp + (min(t * KT + th, end - 1) >> a.kv.block_shift) * a.kv.sblk_stride);
        };
        auto load_v = [&](uint32_t t) {
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) {
                const uint8_t* p = vp + min(t * KT + 8 * vg + i, end - 1) * ps + vd;
                if constexpr (HD == 64) {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
                    vw[i][0] = w.x, vw[i][1] = w.y;
                } else {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
                    vw[i][0] = w.x, vw[i][1] = w.y, vw[i][2] = w.z, vw[i][3] = w.w;
                }
            }
            vs = t * KT + th < end ? __ldg(vsp + (min(t * KT + th, end - 1) >> a.kv.block_shift) * a.kv.sblk_stride) : 0.0f;
        };
        float vmax = 0.0f, vfit = 0.0f;
        load_k(0);
        load_v(0);
        for (uint32_t t = 0; t < tiles; t++) {
            const uint32_t b = t % NB, use = t / NB;
            if (use > 0) wait(&kempty[b], (use - 1) & 1);
            uint8_t* kt = smem + G::K_AT + b * G::K_BYTES;
#pragma unroll
            for (uint32_t i = 0; i < KP; i++) {
                const uint32_t r = kr + i * RPP;
                const uint4 w = kw[i];
                // codes 0, 2, 1, 3 of every four, as q's elements lie
                const uint4 x = make_uint4(even_bytes(w.x), odd_bytes(w.x), even_bytes(w.y), odd_bytes(w.y));
                const uint4 y = make_uint4(even_bytes(w.z), odd_bytes(w.z), even_bytes(w.w), odd_bytes(w.w));
                const uint32_t c = 2 * kc, flip = kc / 4 & 1;  // the slabs' lanes write different banks
                uint8_t* row = kt + c / 8 * G::SLAB + r * 128;
                uint8_t *px = row + ((c % 8) ^ (r & 7)) * 16, *py = row + ((c % 8 + 1) ^ (r & 7)) * 16;
                *reinterpret_cast<uint4*>(flip ? py : px) = flip ? y : x;
                *reinterpret_cast<uint4*>(flip ? px : py) = flip ? x : y;
            }
            fence_proxy_async_smem();
            mbar_arrive(&kfull[b]);
            const float ks_now = ks;
            if (t + 1 < tiles) load_k(t + 1);

            // V's scales under a power of two at or above the largest so far
            float top = vs;
#pragma unroll
            for (uint32_t d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (use > 0) wait(&vempty[b], (use - 1) & 1);
            if (lane == 0) vtop[warp - 8] = top;
            bar_sync(3);
            top = fmaxf(fmaxf(vtop[0], vtop[1]), fmaxf(vtop[2], vtop[3]));
            float ratio = 1.0f;
            if (top > vmax) {
                const uint32_t e = min((__float_as_uint(top) >> 23) + 1, 254u);
                const float fit = __uint_as_float(min(264u - e, 254u) << 23);
                ratio = vfit > 0.0f ? fit / vfit : 1.0f;
                vfit = fit;
                vmax = __uint_as_float(e << 23);
            }
            // both tiles' scales go with V: they are read until the weights are written
            sc[b * 2 * KT + th] = ks_now;
            sc[b * 2 * KT + KT + th] = vs * vfit;
            if (th == 0) {
                vratio[b] = ratio;
                if (t + 1 == tiles) vunit = vfit > 0.0f ? 1.0f / vfit : 0.0f;
            }
            uint8_t* vt = smem + G::V_AT + b * G::V_BYTES + (vg / 8) * (HD * 128);
#pragma unroll
            for (uint32_t i = 0; i < DW; i++) {
                uint32_t f[4][4];  // d, d + 1, d + 2, d + 3 by position pairs
#pragma unroll
                for (uint32_t p = 0; p < 4; p++) {
                    const uint32_t w0 = vw[2 * p][i], w1 = vw[2 * p + 1][i];
                    const uint32_t x = __byte_perm(w0, w1, 0x5410), y = __byte_perm(w0, w1, 0x7632);
                    f[0][p] = even_bytes(x), f[1][p] = odd_bytes(x), f[2][p] = even_bytes(y), f[3][p] = odd_bytes(y);
                }
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) {
                    const uint32_t d = vd + 4 * i + e;
                    *reinterpret_cast<uint4*>(vt + d * 128 + ((vg % 8) ^ (d & 7)) * 16) = make_uint4(f[e][0], f[e][1], f[e][2], f[e][3]);
                }
            }
            fence_proxy_async_smem();
            mbar_arrive(&vfull[b]);
            if (t + 1 < tiles) load_v(t + 1);
            bar_sync(3);  // vtop is free
        }
    } else {
        // ---------------------------------------------------- one row tile
        tc5::setmaxnreg_inc<kChunkRegsRow>();
        const uint32_t w = warp / 4, th = tid % 128, row = w * 128 + th;
        if (w < users) {
            const bool on = row < live;
            const uint64_t f = f0 + row;
            const uint32_t j = (uint32_t)(f / group), h = kvh * group + (uint32_t)(f - (uint64_t)j * group);
            const uint64_t p = (uint64_t)pos0 + j;
            const int lim = on && p < a.kv.max_ctx ? (int)p : -1;  // the last position this row sees
            uint8_t* qt = smem + G::Q_AT + w * G::Q_BYTES;
            float cf;
            {
                // q to f16 rows of 64, elements 0, 2, 1, 3 of every four as K's codes lie
                const uint64_t at = (r0 + (uint64_t)j) * a.q.row + (uint64_t)h * a.q.head;
                float top = 0.0f;
                if (on)
                    for (uint32_t d = 0; d < HD; d++) top = fmaxf(top, fabsf(load1<DT>(a.q.p, at + d)));
                float inv;
                const float fit = fit_f16(top, &inv);
                cf = (a.scale * kLog2e) * inv;
#pragma unroll 4
                for (uint32_t c = 0; c < HD / 8; c++) {
                    float x[8];
                    uint32_t hi4[4], lo4[4];
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) x[e] = on ? load1<DT>(a.q.p, at + 8 * c + e) * fit : 0.0f;
#pragma unroll
                    for (uint32_t e = 0; e < 2; e++) {
                        pair16(x[4 * e], x[4 * e + 2], &hi4[2 * e], &lo4[2 * e]);
                        pair16(x[4 * e + 1], x[4 * e + 3], &hi4[2 * e + 1], &lo4[2 * e + 1]);
                    }
                    uint8_t* to = qt + c / 8 * G::SLAB + th * 128 + ((c % 8) ^ (th & 7)) * 16;
                    *reinterpret_cast<uint4*>(to) = make_uint4(hi4[0], hi4[1], hi4[2], hi4[3]);
                    if constexpr (G::QPAIR) *reinterpret_cast<uint4*>(to + 2 * G::Q_BYTES) = make_uint4(lo4[0], lo4[1], lo4[2], lo4[3]);
                }
            }
            fence_proxy_async_smem();
            bar_sync(1 + w);

            const uint32_t scol = tmem + G::S_COL + w * KT, ocol = tmem + G::O_COL + w * HD;
            const uint32_t lanes = (warp % 4 * 32) << 16;
            auto issue_s = [&](uint32_t t) {
                const uint32_t b = t % NB;
                wait(&kfull[b], t / NB & 1);
                tc5::fence_after();
                const uint32_t kb = smem_u32(smem + G::K_AT + b * G::K_BYTES), qb = smem_u32(qt);
#pragma unroll
                for (uint32_t k = 0; k < HD / 16; k++) {
                    const uint64_t kd = tc5::sw128_desc(kb + k / 4 * G::SLAB) + 2 * (k % 4);
                    const uint64_t qd = tc5::sw128_desc(qb + k / 4 * G::SLAB) + 2 * (k % 4);
                    if constexpr (G::QPAIR) {
                        const uint64_t ld = tc5::sw128_desc(qb + 2 * G::Q_BYTES + k / 4 * G::SLAB) + 2 * (k % 4);
                        tc5::mma_ss(scol, ld, kd, tc5::idesc_f16(128, KT), k > 0);
                        tc5::mma_ss(scol, qd, kd, tc5::idesc_f16(128, KT), true);
                    } else {
                        tc5::mma_ss(scol, qd, kd, tc5::idesc_f16(128, KT), k > 0);
                    }
                }
                tc5::commit(&s_done[w]);
                tc5::commit(&kempty[b]);
            };
            auto issue_o = [&](uint32_t t) {
                const uint32_t b = t % NB;
                wait(&vfull[b], t / NB & 1);
                tc5::fence_after();
                const uint32_t vb = smem_u32(smem + G::V_AT + b * G::V_BYTES);
#pragma unroll
                for (uint32_t k = 0; k < KT / 16; k++) {
                    const uint64_t vd = tc5::sw128_desc(vb + k / 4 * (HD * 128)) + 2 * (k % 4);
                    const uint32_t wc = scol + k / 2 * 32 + k % 2 * 8;
                    if constexpr (G::WPAIR) {
                        tc5::mma_ts(ocol, wc + 16, vd, tc5::idesc_f16(128, HD), k > 0);
                        tc5::mma_ts(ocol, wc, vd, tc5::idesc_f16(128, HD), true);
                    } else {
                        tc5::mma_ts(ocol, wc, vd, tc5::idesc_f16(128, HD), k > 0);
                    }
                }
                tc5::commit(&o_done[w]);
                tc5::commit(&vempty[b]);
            };
            if (th == 0) issue_s(0);

            float o[HD], mx = -INFINITY, l = 0.0f, alpha = 1.0f;
#pragma unroll
            for (uint32_t i = 0; i < HD; i++) o[i] = 0.0f;
            auto add_o = [&](uint32_t t) {  // the outputs of tile t, once they are there
                wait(&o_done[w], t & 1);
                tc5::fence_after();
#pragma unroll
                for (uint32_t c = 0; c < HD / 32; c++) {
                    float x[32];
                    tc5::ld32(ocol + lanes + 32 * c, x);
                    tc5::wait_ld();
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) o[32 * c + i] = fmaf(o[32 * c + i], alpha, x[i]);
                }
            };
            for (uint32_t t = 0; t < tiles; t++) {
                const uint32_t b = t % NB;
                const float* ks = sc + b * 2 * KT;
                const int left = lim - (int)(t * KT);  // columns 0..left are seen
                const bool full = __all_sync(0xffffffffu, left >= (int)KT - 1);
                wait(&vfull[b], t / NB & 1);
                wait(&s_done[w], t & 1);
                tc5::fence_after();
                float s[G::HOLD ? KT : 32], top = -INFINITY;
                auto scores = [&](uint32_t c, float* x) {  // columns 32 c.. under K's scales, unseen ones -inf
                    tc5::ld32(scol + lanes + 32 * c, x);
                    tc5::wait_ld();
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 4) {
                        const float4 k4 = *reinterpret_cast<const float4*>(ks + 32 * c + i);
                        x[i] *= k4.x, x[i + 1] *= k4.y, x[i + 2] *= k4.z, x[i + 3] *= k4.w;
                    }
                    if (!full) {
#pragma unroll
                        for (uint32_t i = 0; i < 32; i++)
                            if ((int)(32 * c + i) > left) x[i] = -INFINITY;
                    }
                };
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) {
                    float* x = s + (G::HOLD ? 32 * c : 0);
                    scores(c, x);
#pragma unroll
                    for (uint32_t i = 0; i < 32; i++) top = fmaxf(top, x[i]);
                }
                if (t > 0) add_o(t - 1);
                alpha = 1.0f;
                if ((top - mx) * cf > kSlack) {
                    alpha = ex2((mx - top) * cf);
                    mx = top;
                    l *= alpha;
                }
                const float off = mx == -INFINITY ? 0.0f : -mx * cf;
                alpha *= vratio[b];
                const float* vs = ks + KT;
                float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t c = 0; c < 4; c++) {
                    float* x = s + (G::HOLD ? 32 * c : 0);
                    if constexpr (!G::HOLD) scores(c, x);
                    uint32_t wh[16], wl[16];
#pragma unroll
                    for (uint32_t i = 0; i < 32; i += 4) {
                        const float4 v4 = *reinterpret_cast<const float4*>(vs + 32 * c + i);
                        const float v[4] = {v4.x, v4.y, v4.z, v4.w};
                        float y[4];
#pragma unroll
                        for (uint32_t e = 0; e < 4; e++) {
                            const bool out = !full && (int)(32 * c + i + e) > left;
                            const float pr = out ? 0.0f : ex2(fmaf(x[i + e], cf, off));
                            l4[e] += pr;
                            y[e] = out ? 0.0f : pr * v[e];  // a scale of NaN does not reach rows before it
                        }
                        pair16(y[0], y[1], &wh[i / 2], &wl[i / 2]);
                        pair16(y[2], y[3], &wh[i / 2 + 1], &wl[i / 2 + 1]);
                    }
                    tc5::st16(scol + lanes + 32 * c, wh);
                    if constexpr (G::WPAIR) tc5::st16(scol + lanes + 32 * c + 16, wl);
                }
                l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                tc5::wait_st();
                tc5::fence_before();
                bar_sync(1 + w);
                if (th == 0) {
                    tc5::fence_after();
                    issue_o(t);
                    if (t + 1 < tiles) issue_s(t + 1);
                }
                __syncwarp();
            }
            add_o(tiles - 1);
            if (on) {
                const float unit = lim >= 0 ? vunit * __frcp_rn(l) : 0.0f;
                const uint64_t at = (r0 + (uint64_t)j) * a.out.row + (uint64_t)h * a.out.head;
#pragma unroll
                for (uint32_t i = 0; i < HD; i++) store1<DT>(const_cast<void*>(a.out.p), at + i, lim >= 0 ? o[i] * unit : 0.0f);
            }
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
        k_kv8_chunk<HD, DT><<<(uint32_t)(tiles * a.kv.nkv), G::THREADS, G::BYTES, st>>>(a);
        return cudaGetLastError();
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
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(k_kv8_chunk<HD, DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, ChunkGeom<HD, DT>::BYTES);
    // the chunk kernel deals the registers of its launch out anew: all of them must be there
    cudaFuncAttributes at{};
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&at, k_kv8_chunk<HD, DT>);
    if (e == cudaSuccess && at.numRegs * 3 < kChunkRegsRow * 2 + kChunkRegsCode) e = cudaErrorInvalidConfiguration;
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
