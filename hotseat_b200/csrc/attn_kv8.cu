// Attention over the 8-bit KV cache.
//
// Codes are integers of at most 127, which f16 holds exactly, so both
// products run on the tensor cores with the codes as one operand and no loss:
// the scales are taken outside, on the scores (K) and on the weights (V). The
// other operand is an f16 pair hi + lo (22 bits) for f32 rows, one f16 for
// 16-bit rows, after scaling by powers of two that keep it in f16's range:
//   q:       its largest element to [2^13, 2^14)
//   weights: w = exp(S - m) s_v 2^(14 - e), 2^e at or above the largest s_v so
//            far, so that weights down to 2^-38 of the largest still count
// Scores, statistics and sums are f32.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.h"
#include "device.cuh"
#include "kernels.h"
#include "kv8.h"

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

// One warp per (row, query head): the positions in turn, with the running
// maximum and sum of the softmax.
template <int HD, int DT>
__global__ void __launch_bounds__(128) k_kv8_attend_simple(const Kv8AttendArgs a) {
    constexpr uint32_t N = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint64_t r = item / a.nh;
    const uint32_t h = (uint32_t)(item - r * a.nh), kvh = h / (a.nh / a.kv.nkv);
    if (r >= a.rows.n_rows || (a.rows.row_start && r >= a.rows.row_start[a.rows.n_slots])) return;
    float q[N], o[N], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < N; i++) {
        q[i] = load1<DT>(a.q.p, r * a.q.row + h * a.q.head + lane * N + i) * a.scale;
        o[i] = 0.0f;
    }
    uint32_t slot, pos;
    if (kv8_place(a.rows, a.kv.max_ctx, (uint32_t)r, &slot, &pos)) {
        const uint8_t* base = reinterpret_cast<const uint8_t*>(a.kv.base[slot]);
        for (uint32_t p = 0; p <= pos; p++) {
            const int8_t* kc = reinterpret_cast<const int8_t*>(base + a.kv.code_off(0, kvh, p)) + lane * N;
            const int8_t* vc = reinterpret_cast<const int8_t*>(base + a.kv.code_off(1, kvh, p)) + lane * N;
            const float ks = *reinterpret_cast<const float*>(base + a.kv.scale_off(0, kvh, p >> a.kv.block_shift));
            const float vs = *reinterpret_cast<const float*>(base + a.kv.scale_off(1, kvh, p >> a.kv.block_shift));
            float s = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < N; i++) s = fmaf(q[i], (float)kc[i], s);
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            s *= ks;
            const float mn = fmaxf(m, s), c = expf(m - mn), w = expf(s - mn);
            l = l * c + w;
            m = mn;
#pragma unroll
            for (uint32_t i = 0; i < N; i++) o[i] = fmaf(w * vs, (float)vc[i], o[i] * c);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < N; i++)
        store1<DT>(const_cast<void*>(a.out.p), r * a.out.row + h * a.out.head + lane * N + i, l > 0.0f || isnan(l) ? o[i] / l : 0.0f);
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
constexpr uint32_t kDecWarps = 4;

// A single row per slot: one CTA takes a split of the positions of one
// (slot, KV head), its warps blocks of BP positions in turn. A warp computes
// S^T = K q^T (16 positions by 8 query heads an instruction; the codes are
// the operand of 16 rows, so a group of up to 8 heads wastes none of it) and
// O^T += V^T w^T, with K's and V's codes loaded straight into the operand
// layout: a lane's 16 bytes of a K row are its share of four k-steps (a dot
// product does not mind which), its bytes of four V rows its share of the
// m-tiles. No code passes through shared memory.
template <int HD, int DT, int NT>
struct DecGeom {
    static constexpr uint32_t BP = HD == 64 ? 32 : 16;  // positions of a block: 4 KB of codes either way
    static constexpr uint32_t MB = BP / 16;
    static constexpr uint32_t KS = HD / 16;             // k-steps of the scores, m-tiles of the output
    static constexpr bool PAIR = DT == HS_F32;
    static constexpr uint32_t NC = 8 * NT;
};

template <int HD>
struct DecBlock {  // codes and scales of BP positions as one lane holds them
    static constexpr uint32_t MB = HD == 64 ? 2 : 1;
    uint4 k[MB][2][HD / 64];   // K rows g and g + 8 of each 16: 16 bytes a 64-byte part
    uint32_t v[MB][4][HD / 32];  // V rows 2t, 2t+1, 2t+8, 2t+9: HD / 8 bytes
    float ks[MB][2], vs[MB][2];
};

template <int HD, int DT, int NT>
__global__ void __launch_bounds__(kDecWarps * 32) k_kv8_single(const Kv8AttendArgs a) {
    using G = DecGeom<HD, DT, NT>;
    constexpr uint32_t BP = G::BP, MB = G::MB, KS = G::KS, NC = G::NC;
    constexpr bool PAIR = G::PAIR;
    __shared__ float sm_o[kDecWarps][NC][HD + 4];
    __shared__ float sm_m[kDecWarps][NC], sm_l[kDecWarps][NC];
    __shared__ uint32_t sm_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t group = a.nh / a.kv.nkv, chunks = (group + NC - 1) / NC;
    const uint32_t item = blockIdx.x;
    const uint32_t slot = item / (a.kv.nkv * chunks), rest = item - slot * a.kv.nkv * chunks;
    const uint32_t kvh = rest / chunks, chunk = rest - kvh * chunks;
    const uint32_t h0 = kvh * group + chunk * NC, cols = min(NC, group - chunk * NC);
    const uint32_t split = blockIdx.y;
    const uint32_t pos = __ldg(a.rows.pos + slot);
    const uint8_t* base = reinterpret_cast<const uint8_t*>(__ldg(reinterpret_cast<const unsigned long long*>(a.kv.base + slot)));
    if (pos >= a.kv.max_ctx) {
        if (split == 0) {
            if (pos != kPosNone && tid == 0) atomicOr(a.rows.err, ERR_POS);
            for (uint32_t i = tid; i < cols * HD; i += kDecWarps * 32)
                store1<DT>(const_cast<void*>(a.out.p), slot * a.out.row + (h0 + i / HD) * a.out.head + i % HD, 0.0f);
        }
        return;
    }
    const uint32_t n = pos + 1, len = kv8_split_len(n, HD, a.max_splits), splits = (n + len - 1) / len;
    if (split >= splits) return;
    const uint32_t from = split * len, to = min(n, from + len);

    const uint8_t* kp = base + a.kv.code_off(0, kvh, 0);
    const uint8_t* vp = base + a.kv.code_off(1, kvh, 0);
    const float* ksp = reinterpret_cast<const float*>(base + a.kv.scale_off(0, kvh, 0));
    const float* vsp = reinterpret_cast<const float*>(base + a.kv.scale_off(1, kvh, 0));
    const uint64_t ps = a.kv.pos_stride;

    // Positions past the split are read as its last one and get no weight.
    DecBlock<HD> buf;
    auto load = [&](uint32_t p0) {
#pragma unroll
        for (uint32_t b = 0; b < MB; b++) {
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) {
                const uint32_t p = min(p0 + 16 * b + 8 * r + g, to - 1);
#pragma unroll
                for (uint32_t c = 0; c < HD / 64; c++)
                    buf.k[b][r][c] = __ldg(reinterpret_cast<const uint4*>(kp + p * ps + 64 * c + 16 * t));
                buf.ks[b][r] = __ldg(ksp + (p >> a.kv.block_shift) * a.kv.sblk_stride);
                buf.vs[b][r] = __ldg(vsp + (p >> a.kv.block_shift) * a.kv.sblk_stride);
            }
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                const uint32_t p = min(p0 + 16 * b + 2 * t + (r & 1) + 8 * (r >> 1), to - 1);
                const uint8_t* q = vp + p * ps + (HD / 8) * g;
                if constexpr (HD == 64) {
                    const uint2 w = __ldg(reinterpret_cast<const uint2*>(q));
                    buf.v[b][r][0] = w.x, buf.v[b][r][1] = w.y;
                } else {
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(q));
                    buf.v[b][r][0] = w.x, buf.v[b][r][1] = w.y, buf.v[b][r][2] = w.z, buf.v[b][r][3] = w.w;
                }
            }
        }
    };
    uint32_t p0 = from + warp * BP;
    if (p0 < to) load(p0);

    // q as the second operand: column g of n-tile nt is head h0 + 8 nt + g
    uint32_t qh[NT][KS][2], ql[PAIR ? NT : 1][PAIR ? KS : 1][2];
    float cf[NT][2];  // columns 2t, 2t + 1: softmax scale x log2(e) x what q was scaled by
#pragma unroll
    for (uint32_t nt = 0; nt < NT; nt++) {
        float x[HD / 4], top = 0.0f;
        const uint32_t col = 8 * nt + g;
#pragma unroll
        for (uint32_t i = 0; i < HD / 4; i++) {
            x[i] = col < cols ? load1<DT>(a.q.p, slot * a.q.row + (uint64_t)(h0 + col) * a.q.head + (i / 16) * 64 + 16 * t + i % 16) : 0.0f;
            top = fmaxf(top, fabsf(x[i]));
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        float inv;
        const float fit = fit_f16(top, &inv);
        const float back = (a.scale * kLog2e) * inv;
        cf[nt][0] = __shfl_sync(0xffffffffu, back, 8 * t);
        cf[nt][1] = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (uint32_t j = 0; j < KS; j++) {
            const float* e = x + 4 * j;
            if constexpr (PAIR) {
                pair16(e[0] * fit, e[2] * fit, &qh[nt][j][0], &ql[nt][j][0]);
                pair16(e[1] * fit, e[3] * fit, &qh[nt][j][1], &ql[nt][j][1]);
            } else {
                const __half2 u = __floats2half2_rn(e[0] * fit, e[2] * fit), v = __floats2half2_rn(e[1] * fit, e[3] * fit);
                qh[nt][j][0] = *reinterpret_cast<const uint32_t*>(&u);
                qh[nt][j][1] = *reinterpret_cast<const uint32_t*>(&v);
            }
        }
    }

    float o[NT][KS][4] = {}, m[NT][2], l[NT][2] = {}, vmax = 0.0f, vfit = 0.0f;
#pragma unroll
    for (uint32_t nt = 0; nt < NT; nt++) m[nt][0] = m[nt][1] = -INFINITY;

    for (; p0 < to; p0 += kDecWarps * BP) {
        // scores: rows g and g + 8 of each 16 positions, columns 2t and 2t + 1
        float s[NT][MB][4] = {};
#pragma unroll
        for (uint32_t b = 0; b < MB; b++)
#pragma unroll
            for (uint32_t j = 0; j < KS; j++) {
                const uint4 w0 = buf.k[b][0][j / 4], w1 = buf.k[b][1][j / 4];
                const uint32_t u = j % 4 == 0 ? w0.x : j % 4 == 1 ? w0.y : j % 4 == 2 ? w0.z : w0.w;
                const uint32_t v = j % 4 == 0 ? w1.x : j % 4 == 1 ? w1.y : j % 4 == 2 ? w1.z : w1.w;
                const uint32_t f[4] = {even_bytes(u), even_bytes(v), odd_bytes(u), odd_bytes(v)};
#pragma unroll
                for (uint32_t nt = 0; nt < NT; nt++) {
                    if constexpr (PAIR) mma16816(s[nt][b], f, ql[nt][j][0], ql[nt][j][1]);
                    mma16816(s[nt][b], f, qh[nt][j][0], qh[nt][j][1]);
                }
            }
        float vs[MB][2], top[NT][2];
        bool grew = false, vgrew = false;
#pragma unroll
        for (uint32_t nt = 0; nt < NT; nt++) top[nt][0] = m[nt][0], top[nt][1] = m[nt][1];
#pragma unroll
        for (uint32_t b = 0; b < MB; b++)
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) {
                const bool in = p0 + 16 * b + 8 * r + g < to;
                vs[b][r] = in ? buf.vs[b][r] : 0.0f;
                vgrew |= vs[b][r] > vmax;
#pragma unroll
                for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
                    for (uint32_t c = 0; c < 2; c++) {
                        float& x = s[nt][b][2 * r + c];
                        x = in ? x * (buf.ks[b][r] * cf[nt][c]) : -INFINITY;
                        top[nt][c] = fmaxf(top[nt][c], x);
                    }
            }
        uint32_t va[MB][KS][4];  // V^T: (row 2i or 2i + 1 of the lane's bytes) by position pairs
#pragma unroll
        for (uint32_t b = 0; b < MB; b++)
#pragma unroll
            for (uint32_t i = 0; i < KS / 2; i++)
#pragma unroll
                for (uint32_t h = 0; h < 2; h++) {
                    const uint32_t w0 = buf.v[b][2 * h][i], w1 = buf.v[b][2 * h + 1][i];
                    const uint32_t lo = __byte_perm(w0, w1, 0x5410), hi = __byte_perm(w0, w1, 0x7632);
                    va[b][2 * i][2 * h] = even_bytes(lo), va[b][2 * i][2 * h + 1] = odd_bytes(lo);
                    va[b][2 * i + 1][2 * h] = even_bytes(hi), va[b][2 * i + 1][2 * h + 1] = odd_bytes(hi);
                }
        if (p0 + kDecWarps * BP < to) load(p0 + kDecWarps * BP);

#pragma unroll
        for (uint32_t nt = 0; nt < NT; nt++) grew |= top[nt][0] > m[nt][0] || top[nt][1] > m[nt][1];
        if (__any_sync(0xffffffffu, grew || vgrew)) {
            // new maxima for the warp (over the 8 row groups), older sums scaled to them
            float vnew = vmax;
#pragma unroll
            for (uint32_t b = 0; b < MB; b++) vnew = fmaxf(vnew, fmaxf(vs[b][0], vs[b][1]));
#pragma unroll
            for (uint32_t d = 4; d < 32; d <<= 1) vnew = fmaxf(vnew, __shfl_xor_sync(0xffffffffu, vnew, d));
            float vback = 1.0f;
            if (vnew > vmax) {  // the power of two above vnew, unless it is held already
                const uint32_t e = min((__float_as_uint(vnew) >> 23) + 1, 254u);
                const float fit = __uint_as_float(min(268u - e, 254u) << 23);  // largest weight 2^14
                vback = vfit > 0.0f ? fit / vfit : 1.0f;
                vfit = fit;
                vmax = __uint_as_float(e << 23);
            }
#pragma unroll
            for (uint32_t nt = 0; nt < NT; nt++)
#pragma unroll
                for (uint32_t c = 0; c < 2; c++) {
                    float x = top[nt][c];
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
                uint32_t h0, h1, l0 = 0, l1 = 0;
                pair16(w[0], w[1], &h0, &l0);
                pair16(w[2], w[3], &h1, &l1);
                h0 = transpose8x8(h0), h1 = transpose8x8(h1);
                if constexpr (PAIR) l0 = transpose8x8(l0), l1 = transpose8x8(l1);
#pragma unroll
                for (uint32_t i = 0; i < KS; i++) {
                    if constexpr (PAIR) mma16816(o[nt][i], va[b][i], l0, l1);
                    mma16816(o[nt][i], va[b][i], h0, h1);
                }
            }
    }

    // the warps' records, then the CTA's
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
#pragma unroll
            for (uint32_t i = 0; i < KS; i++) {
                sm_o[warp][col][(HD / 8) * g + 2 * i] = o[nt][i][c] * vinv;
                sm_o[warp][col][(HD / 8) * g + 2 * i + 1] = o[nt][i][2 + c] * vinv;
            }
        }
    __syncthreads();
    constexpr uint32_t TH = kDecWarps * 32;
    float* rec = a.part + (((uint64_t)item * a.max_splits + split) * NC) * (HD + 2);
    for (uint32_t i = tid; i < cols * HD; i += TH) {
        const uint32_t col = i / HD, d = i % HD;
        float mm = -INFINITY, ll = 0.0f, acc = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < kDecWarps; w++) mm = fmaxf(mm, sm_m[w][col]);
#pragma unroll
        for (uint32_t w = 0; w < kDecWarps; w++) {
            if (from + w * BP >= to) break;  // warps without a block
            const float f = ex2(sm_m[w][col] - mm);
            ll = fmaf(sm_l[w][col], f, ll);
            acc = fmaf(sm_o[w][col][d], f, acc);
        }
        if (splits == 1) {
            store1<DT>(const_cast<void*>(a.out.p), slot * a.out.row + (uint64_t)(h0 + col) * a.out.head + d, acc / ll);
        } else {
            rec[i] = acc;
            if (d == 0) rec[NC * HD + col] = mm, rec[NC * HD + NC + col] = ll;
        }
    }
    if (splits == 1) return;
    // the last CTA of this (slot, KV head, chunk) joins the splits in order
    __threadfence();
    __syncthreads();
    if (tid == 0) sm_last = atomicAdd(a.counters + item, 1u);
    __syncthreads();
    if (sm_last != splits - 1) return;
    __threadfence();
    if (tid == 0) a.counters[item] = 0;
    const float* r0 = a.part + ((uint64_t)item * a.max_splits * NC) * (HD + 2);
    const uint64_t rs = (uint64_t)NC * (HD + 2);
    for (uint32_t i = tid; i < cols * HD; i += TH) {
        const uint32_t col = i / HD, d = i % HD;
        float mm = -INFINITY, ll = 0.0f, acc = 0.0f;
        for (uint32_t w = 0; w < splits; w++) mm = fmaxf(mm, __ldcg(r0 + w * rs + NC * HD + col));
#pragma unroll 8
        for (uint32_t w = 0; w < splits; w++) {
            const float f = ex2(__ldcg(r0 + w * rs + NC * HD + col) - mm);
            ll = fmaf(__ldcg(r0 + w * rs + NC * HD + NC + col), f, ll);
            acc = fmaf(__ldcg(r0 + w * rs + i), f, acc);
        }
        store1<DT>(const_cast<void*>(a.out.p), slot * a.out.row + (uint64_t)(h0 + col) * a.out.head + d, acc / ll);
    }
}

template <int HD, int DT>
cudaError_t attend_dt(const Kv8AttendArgs& a, cudaStream_t st) {
    if (a.rows.row_start) {
        const uint64_t items = (uint64_t)a.rows.n_rows * a.nh;
        k_kv8_attend_simple<HD, DT><<<(uint32_t)((items + 3) / 4), 128, 0, st>>>(a);
        return cudaGetLastError();
    }
    const uint32_t nc = kv8_single_cols(a.nh / a.kv.nkv);
    const dim3 grid(a.rows.n_slots * a.kv.nkv * ((a.nh / a.kv.nkv + nc - 1) / nc), a.max_splits);
    if (nc == 8) k_kv8_single<HD, DT, 1><<<grid, kDecWarps * 32, 0, st>>>(a);
    else k_kv8_single<HD, DT, 2><<<grid, kDecWarps * 32, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_kv8_attend(uint32_t hd, const Kv8AttendArgs& a, cudaStream_t st) {
    if (!a.rows.n_rows) return cudaSuccess;
    if (hd == 64)
        return a.q.dtype == HS_F32 ? attend_dt<64, HS_F32>(a, st)
               : a.q.dtype == HS_F16 ? attend_dt<64, HS_F16>(a, st) : attend_dt<64, HS_BF16>(a, st);
    return a.q.dtype == HS_F32 ? attend_dt<128, HS_F32>(a, st)
           : a.q.dtype == HS_F16 ? attend_dt<128, HS_F16>(a, st) : attend_dt<128, HS_BF16>(a, st);
}

}  // namespace hs
