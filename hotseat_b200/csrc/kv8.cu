// The 8-bit KV cache: rows quantised as they are written, and read back.
//
// Both kernels move bytes once: a row of one head is taken by a team of
// head_dim / 8 lanes, eight elements a lane (16 bytes of f16/bf16 or 32 of
// f32 against 8 bytes of codes), so every access is a whole sector.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "common.h"
#include "device.cuh"
#include "kernels.h"
#include "kv8.h"

namespace hs {
namespace {

constexpr uint32_t kThreads = 256;

// Eight consecutive elements of a row as floats (exact) and back (one
// rounding). VEC: 16-byte accesses, which base and strides must allow.
template <int DT, bool VEC>
__device__ __forceinline__ void load8(const void* base, uint64_t e, float* x) {
    if constexpr (DT == HS_F32) {
        const float* p = static_cast<const float*>(base) + e;
        if constexpr (VEC) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) x[i] = __ldg(p + i);
        }
    } else {
        const uint16_t* p = static_cast<const uint16_t*>(base) + e;
        uint32_t w[4];
        if constexpr (VEC) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = (uint32_t)__ldg(p + 2 * i) | (uint32_t)__ldg(p + 2 * i + 1) << 16;
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DT == HS_F16) {
                const float2 f = __half22float2(*reinterpret_cast<__half2*>(&w[i]));
                x[2 * i] = f.x, x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}
template <int DT, bool VEC>
__device__ __forceinline__ void store8(void* base, uint64_t e, const float* x) {
    if constexpr (DT == HS_F32) {
        float* p = static_cast<float*>(base) + e;
        if constexpr (VEC) {
            reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = x[i];
        }
    } else {
        uint16_t* p = static_cast<uint16_t*>(base) + e;
        uint16_t h[8];
#pragma unroll
        for (int i = 0; i < 8; i++)
            h[i] = DT == HS_F16 ? __half_as_ushort(__float2half_rn(x[i])) : __bfloat16_as_ushort(__float2bfloat16_rn(x[i]));
        if constexpr (VEC) {
            *reinterpret_cast<uint4*>(p) = make_uint4(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16,
                                                      h[4] | (uint32_t)h[5] << 16, h[6] | (uint32_t)h[7] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) p[i] = h[i];
        }
    }
}

// max|x|, with NaN kept: infinities and NaN both end as a scale of NaN.
__device__ __forceinline__ float amax8(const float* x) {
    float m = 0.0f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        m = fmaxf(m, fabsf(x[i]));
        bad |= !(fabsf(x[i]) <= 3.402823466e38f);
    }
    return bad ? INFINITY : m;
}

// The scale that rows of largest magnitude m ask for: m times 1/127, both
// rounded to f32 (m / s is then at most 127 (1 + 2^-22), which rounds to 127).
__device__ __forceinline__ float scale_for(float m) {
    if (!(m <= 3.402823466e38f)) return __int_as_float(0x7fc00000);
    const float s = __fmul_rn(m, 1.0f / 127.0f);
    return s < 1.17549435e-38f ? 0.0f : s;
}

// The doublings k >= 0 that take the scale `held` to `need` or above (both
// normal and positive): from the exponents, one more if the mantissa falls short.
__device__ __forceinline__ int doublings(float held, float need) {
    const uint32_t h = __float_as_uint(held), n = __float_as_uint(need);
    const int k = (int)(n >> 23) - (int)(h >> 23) + ((n & 0x7fffffu) > (h & 0x7fffffu) ? 1 : 0);
    return k > 0 ? k : 0;
}

// Eight codes of x under scale s (not 0 or NaN): the integer nearest to x / s,
// ties to even. x times the rounded reciprocal is off by at most 127 x 2^-23
// of a step, so only a product that near to a half needs a second look: there
// the remainder x - c s is exact in one FMA, and says which side x / s is on.
__device__ __forceinline__ uint2 codes8(const float* x, float s, float inv) {
    int c[8];
    float near = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = __fmul_rn(x[i], inv), r = rintf(y);
        near = fmaxf(near, fabsf(__fsub_rn(y, r)));
        c[i] = (int)r;
    }
    if (near > 0.4999f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r2 = 2.0f * __fmaf_rn(-(float)c[i], s, x[i]);
            if (r2 > s || (r2 == s && (c[i] & 1))) c[i]++;
            else if (r2 < -s || (r2 == -s && (c[i] & 1))) c[i]--;
        }
    }
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; i++) {
        c[i] = max(-127, min(127, c[i]));
        w[i >> 2] |= (uint32_t)(c[i] & 0xff) << (8 * (i & 3));
    }
    return make_uint2(w[0], w[1]);
}

// Sets the page bits of `len` bytes at `off`, after they are visible (a
// harvest may run concurrently).
__device__ __forceinline__ void mark_pages(const Kv8View& kv, uint32_t slot, uint64_t off, uint32_t len) {
    uint64_t* dirty = kv.dirty[slot];
    for (uint64_t pg = off >> kv.page_shift; pg <= (off + len - 1) >> kv.page_shift; pg++)
        atomicOr(reinterpret_cast<unsigned long long*>(&dirty[pg >> 6]), 1ull << (pg & 63));
}
__device__ __forceinline__ bool tracked(const Kv8View& kv, uint32_t slot) {
    return *reinterpret_cast<const volatile uint32_t*>(kv.tracking[slot]) != 0;
}

// Append, a scale for every position: a team per (row, head, K or V).
template <int HD, int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_append_rows(const Kv8View kv, const Kv8Rows rows, const Kv8Mat k,
                                                          const Kv8Mat v) {
    constexpr uint32_t TL = HD / 8, TEAMS = kThreads / TL;
    const uint32_t tl = threadIdx.x % TL;
    const uint64_t item = (uint64_t)blockIdx.x * TEAMS + threadIdx.x / TL;
    const uint64_t r64 = item / (2 * kv.nkv);
    const uint32_t which = (uint32_t)(item - r64 * 2 * kv.nkv), is_v = which >= kv.nkv ? 1 : 0;
    const uint32_t head = which - is_v * kv.nkv;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    uint32_t slot = 0, pos = 0;
    const bool live = r64 < rows.n_rows && kv8_place(rows, kv.max_ctx, (uint32_t)r64, &slot, &pos);
    const Kv8Mat& m = is_v ? v : k;
    if (live) load8<DT, VEC>(m.p, r64 * m.row + head * m.head + 8 * tl, x);
    float top = amax8(x);
#pragma unroll
    for (uint32_t o = TL / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!live) return;
    const float s = scale_for(top);
    uint2 c = make_uint2(0, 0);
    if (s > 0.0f) c = codes8(x, s, __fdiv_rn(1.0f, s));
    uint8_t* base = reinterpret_cast<uint8_t*>(kv.base[slot]);
    const uint64_t at = kv.code_off(is_v, head, pos), sat = kv.scale_off(is_v, head, pos);
    *reinterpret_cast<uint2*>(base + at + 8 * tl) = c;
    if (tl == 0) *reinterpret_cast<float*>(base + sat) = s;
    if (tracked(kv, slot)) {
        __threadfence();
        __syncwarp(__activemask());
        if (tl == 0) {
            mark_pages(kv, slot, at, HD);
            mark_pages(kv, slot, sat, 4);
        }
    }
}

// Append, a scale for every B positions: WPU warps take one unit = (slot,
// block, head, K or V) and hold its new rows in registers between the maximum
// and the codes, RL rows a lane; the unit's older rows are rescaled where the
// scale doubles. Units of slot i start at unit row_start[i] / B + 2 i, which
// leaves room for every block that its rows can touch.
template <int HD, int DT, bool VEC, int B>
__global__ void __launch_bounds__(kThreads) k_append_blocks(const Kv8View kv, const Kv8Rows rows, const Kv8Mat k,
                                                            const Kv8Mat v) {
    constexpr uint32_t TL = HD / 8, RPW = 32 / TL;
    constexpr uint32_t WPU = B / (4 * RPW) > 8 ? 8 : B / (4 * RPW), RL = B / (WPU * RPW), UPC = 8 / WPU;
    __shared__ float tops[8];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tl = lane % TL;
    const uint32_t j0 = (warp % WPU) * RPW + lane / TL;  // this lane's rows of the block: j0 + i * WPU * RPW
    const uint64_t unit = (uint64_t)blockIdx.x * UPC + warp / WPU;
    const uint64_t u64 = unit / (2 * kv.nkv);
    const uint32_t which = (uint32_t)(unit - u64 * 2 * kv.nkv), is_v = which >= kv.nkv ? 1 : 0;
    const uint32_t head = which - is_v * kv.nkv;

    // the unit's slot, its rows [r0, r0 + m) and its block
    uint32_t slot = 0, r0 = 0, m = 0, p0 = kPosNone, blk = 0;
    bool live;
    if (!rows.row_start) {
        slot = r0 = (uint32_t)u64;
        live = u64 < rows.n_rows;
        m = 1;
        if (live) p0 = __ldg(rows.pos + slot);
        blk = p0 / B;
    } else {
        uint32_t lo = 0, hi = rows.n_slots;  // the last slot whose first unit is <= u64
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (__ldg(rows.row_start + mid) / B + 2ull * mid <= u64)
                lo = mid + 1;
            else
                hi = mid;
        }
        live = lo > 0;
        if (live) {
            slot = lo - 1;
            r0 = __ldg(rows.row_start + slot);
            const uint32_t end = min(__ldg(rows.row_start + slot + 1), rows.n_rows);
            m = end > r0 ? end - r0 : 0;
            p0 = __ldg(rows.pos + slot);
            blk = p0 / B + (uint32_t)(u64 - (r0 / B + 2ull * slot));
        }
    }
    live = live && m > 0 && p0 != kPosNone;
    const uint64_t b0 = (uint64_t)blk * B, end = (uint64_t)p0 + m;  // the rows' positions: [p0, end)
    live = live && b0 < end;
    if (live && end > kv.max_ctx && tl == 0 && j0 == 0) atomicOr(rows.err, ERR_POS);
    live = live && b0 < kv.max_ctx;

    float x[RL][8];
    float top = 0.0f;
    const Kv8Mat& mat = is_v ? v : k;
#pragma unroll
    for (uint32_t i = 0; i < RL; i++) {
        const uint64_t p = b0 + j0 + i * WPU * RPW;
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
        if (live && p >= p0 && p < end && p < kv.max_ctx)
            load8<DT, VEC>(mat.p, (r0 + (p - p0)) * mat.row + head * mat.head + 8 * tl, x[i]);
        top = fmaxf(top, amax8(x[i]));
    }
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (WPU > 1) {
        if (lane == 0) tops[warp] = top;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < WPU; w++) top = fmaxf(top, tops[warp / WPU * WPU + w]);
    }
    uint8_t* base = live ? reinterpret_cast<uint8_t*>(kv.base[slot]) : nullptr;
    const uint64_t sat = kv.scale_off(is_v, head, blk);
    float s = scale_for(top), held = 0.0f;
    int k2 = 0;
    if (live && b0 < p0) held = *reinterpret_cast<const float*>(base + sat);
    if (WPU > 1) __syncthreads();  // every warp holds the old scale before one writes the new one
    if (!live) return;
    if (isnan(held)) {
        s = held;
    } else if (held > 0.0f && !isnan(s)) {
        if (s > 0.0f) k2 = doublings(held, s);
        s = __fmul_rn(__fmul_rn(held, pow2i(k2 / 2)), pow2i(k2 - k2 / 2));  // 2^k2 itself may pass f32
    }
    const float inv = s > 0.0f ? __fdiv_rn(1.0f, s) : 0.0f;
    const bool track = tracked(kv, slot);
#pragma unroll
    for (uint32_t i = 0; i < RL; i++) {
        const uint64_t p = b0 + j0 + i * WPU * RPW;
        if (p >= end || p >= kv.max_ctx || (p < p0 && k2 == 0)) continue;
        const uint64_t at = kv.code_off(is_v, head, (uint32_t)p);
        uint2* to = reinterpret_cast<uint2*>(base + at + 8 * tl);
        uint2 c = make_uint2(0, 0);
        if (p >= p0) {
            if (s > 0.0f) c = codes8(x[i], s, inv);
        } else {
            const uint2 old = *to;
            const float half = pow2i(-min(k2, 16));
            uint32_t w[2] = {old.x, old.y}, n[2] = {0, 0};
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int o = (int)(int8_t)(w[e >> 2] >> (8 * (e & 3)));
                n[e >> 2] |= (uint32_t)((int)rintf(__fmul_rn((float)o, half)) & 0xff) << (8 * (e & 3));
            }
            c = make_uint2(n[0], n[1]);
        }
        *to = c;
        if (track) {
            __threadfence();
            if (tl == 0) mark_pages(kv, slot, at, HD);
        }
    }
    if (j0 == 0 && tl == 0) {
        *reinterpret_cast<float*>(base + sat) = s;
        if (track) {
            __threadfence();
            mark_pages(kv, slot, sat, 4);
        }
    }
}

// Read back: a team per (row, head, K or V).
template <int HD, int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_read_rows(const Kv8View kv, const Kv8Rows rows, const Kv8Mat k,
                                                        const Kv8Mat v) {
    constexpr uint32_t TL = HD / 8, TEAMS = kThreads / TL;
    const uint32_t tl = threadIdx.x % TL;
    const uint64_t item = (uint64_t)blockIdx.x * TEAMS + threadIdx.x / TL;
    const uint64_t r64 = item / (2 * kv.nkv);
    const uint32_t which = (uint32_t)(item - r64 * 2 * kv.nkv), is_v = which >= kv.nkv ? 1 : 0;
    const uint32_t head = which - is_v * kv.nkv;
    uint32_t slot = 0, pos = 0;
    if (r64 >= rows.n_rows || !kv8_place(rows, kv.max_ctx, (uint32_t)r64, &slot, &pos)) return;
    const Kv8Mat& m = is_v ? v : k;
    if (!m.p) return;
    const uint8_t* base = reinterpret_cast<const uint8_t*>(kv.base[slot]);
    const uint2 c = *reinterpret_cast<const uint2*>(base + kv.code_off(is_v, head, pos) + 8 * tl);
    const float s = *reinterpret_cast<const float*>(base + kv.scale_off(is_v, head, pos >> kv.block_shift));
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __fmul_rn((float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3))), s);
    store8<DT, VEC>(const_cast<void*>(m.p), r64 * m.row + head * m.head + 8 * tl, x);
}

bool vec_ok(const Kv8Mat& m) {
    const uint64_t b = dtype_bytes(m.dtype);
    return reinterpret_cast<uintptr_t>(m.p) % 16 == 0 && m.row * b % 16 == 0 && m.head * b % 16 == 0;
}

// f(dtype constant, vector constant)
template <typename F>
void by_type(uint32_t dtype, bool vec, F f) {
    auto go = [&](auto v) {
        if (dtype == HS_F32) f(std::integral_constant<int, HS_F32>{}, v);
        else if (dtype == HS_F16) f(std::integral_constant<int, HS_F16>{}, v);
        else f(std::integral_constant<int, HS_BF16>{}, v);
    };
    if (vec) go(std::true_type{});
    else go(std::false_type{});
}

template <int HD>
void append_hd(const Kv8View& kv, const Kv8Rows& rows, const Kv8Mat& k, const Kv8Mat& v, cudaStream_t st) {
    by_type(k.dtype, vec_ok(k) && vec_ok(v), [&](auto dt, auto vec) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool VEC = decltype(vec)::value;
        if (kv.block_shift == 0) {
            const uint64_t items = (uint64_t)rows.n_rows * 2 * kv.nkv, per = kThreads / (HD / 8);
            k_append_rows<HD, DT, VEC><<<(uint32_t)((items + per - 1) / per), kThreads, 0, st>>>(kv, rows, k, v);
            return;
        }
        const uint32_t B = 1u << kv.block_shift;
        const uint64_t units =
            (rows.row_start ? (uint64_t)rows.n_rows / B + 2ull * rows.n_slots : (uint64_t)rows.n_rows) * 2 * kv.nkv;
        auto go = [&](auto b) {
            constexpr int BB = decltype(b)::value;
            constexpr uint32_t RPW = 32 / (HD / 8), WPU = BB / (4 * RPW) > 8 ? 8 : BB / (4 * RPW), UPC = 8 / WPU;
            k_append_blocks<HD, DT, VEC, BB><<<(uint32_t)((units + UPC - 1) / UPC), kThreads, 0, st>>>(kv, rows, k, v);
        };
        if (B == 16) go(std::integral_constant<int, 16>{});
        else if (B == 32) go(std::integral_constant<int, 32>{});
        else if (B == 64) go(std::integral_constant<int, 64>{});
        else go(std::integral_constant<int, 128>{});
    });
}

}  // namespace

cudaError_t launch_kv8_append(uint32_t hd, const Kv8View& kv, const Kv8Rows& rows, const Kv8Mat& k, const Kv8Mat& v,
                              cudaStream_t st) {
    if (!rows.n_rows) return cudaSuccess;
    if (hd == 64) append_hd<64>(kv, rows, k, v, st);
    else append_hd<128>(kv, rows, k, v, st);
    return cudaGetLastError();
}

cudaError_t launch_kv8_read(uint32_t hd, const Kv8View& kv, const Kv8Rows& rows, const Kv8Mat& k, const Kv8Mat& v,
                            cudaStream_t st) {
    if (!rows.n_rows) return cudaSuccess;
    const bool vec = (!k.p || vec_ok(k)) && (!v.p || vec_ok(v));
    by_type(k.dtype, vec, [&](auto dt, auto ve) {
        constexpr int DT = decltype(dt)::value;
        constexpr bool VEC = decltype(ve)::value;
        const uint64_t items = (uint64_t)rows.n_rows * 2 * kv.nkv, per = kThreads / (hd / 8);
        const uint32_t grid = (uint32_t)((items + per - 1) / per);
        if (hd == 64) k_read_rows<64, DT, VEC><<<grid, kThreads, 0, st>>>(kv, rows, k, v);
        else k_read_rows<128, DT, VEC><<<grid, kThreads, 0, st>>>(kv, rows, k, v);
    });
    return cudaGetLastError();
}

}  // namespace hs
