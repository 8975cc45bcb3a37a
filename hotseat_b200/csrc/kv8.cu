// The 8-bit KV cache: rows quantised as they are written, and read back.
//
// The kernels move bytes once: a row of one head is taken by head_dim / 8 lanes,
// eight elements a lane (16 bytes of f16/bf16 or 32 of f32 against 8 bytes of
// codes), so that accesses are whole sectors.
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

// max|x| as bits, whose order is that of the numbers, with infinities and then
// NaN above them.
__device__ __forceinline__ uint32_t amax8(const float* x) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; i++) m = max(m, __float_as_uint(x[i]) & 0x7fffffffu);
    return m;
}

// The scale that rows of largest magnitude m (bits) ask for: m times 1/127, both
// rounded to f32 (m / s is then at most 127 (1 + 2^-22), which rounds to 127).
__device__ __forceinline__ float scale_for(uint32_t m) {
    if (m >= 0x7f800000u) return __int_as_float(0x7fc00000);
    const float s = __fmul_rn(__uint_as_float(m), 1.0f / 127.0f);
    return s < 1.17549435e-38f ? 0.0f : s;
}
// 1 / s to within 2^-23 of itself (s is normal, and so is 1 / s).
__device__ __forceinline__ float reciprocal(float s) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(s));
    return y;
}

// The doublings k >= 0 that take the scale `held` to `need` or above (both
// normal and positive): from the exponents, one more if the mantissa falls short.
__device__ __forceinline__ int doublings(float held, float need) {
    const uint32_t h = __float_as_uint(held), n = __float_as_uint(need);
    const int k = (int)(n >> 23) - (int)(h >> 23) + ((n & 0x7fffffu) > (h & 0x7fffffu) ? 1 : 0);
    return k > 0 ? k : 0;
}

// Eight codes of x under scale s (not 0 or NaN): the integer nearest to x / s,
// ties to even. x times the reciprocal is off by at most 127 x 2^-22 of a step,
// so only a product that near to a half needs a second look: there
// the remainder x - c s is exact in one FMA, and says which side x / s is on.
// Adding 1.5 x 2^23 rounds to an integer, ties to even, and leaves it in the low
// bits: no conversion instruction, a quarter as fast, is needed.
__device__ __forceinline__ uint2 codes8(const float* x, float s, float inv) {
    constexpr float kMagic = 12582912.0f;
    uint32_t c[8];
    float near = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const float y = __fmul_rn(x[i], inv), m = __fadd_rn(y, kMagic);
        near = fmaxf(near, fabsf(__fsub_rn(y, __fsub_rn(m, kMagic))));
        c[i] = __float_as_uint(m);
    }
    if (near > 0.4999f) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float r2 = 2.0f * __fmaf_rn(-__fsub_rn(__uint_as_float(c[i]), kMagic), s, x[i]);
            if (r2 > s || (r2 == s && (c[i] & 1))) c[i]++;
            else if (r2 < -s || (r2 == -s && (c[i] & 1))) c[i]--;
        }
    }
    return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}

// The values of eight codes under scale s: a byte with its sign bit flipped,
// under the exponent of 2^23, is 2^23 + 128 + code, exactly.
__device__ __forceinline__ void values8(uint2 c, float s, float* x) {
    const uint32_t w[2] = {c.x ^ 0x80808080u, c.y ^ 0x80808080u};
#pragma unroll
    for (int e = 0; e < 8; e++)
        x[e] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(w[e >> 2], 0x4b000000u, 0x7440 | (e & 3))), 8388736.0f), s);
}

// Sets the page bits of `len` bytes at `off`. A harvest and an arm may run
// concurrently, so a warp that stored rows first fences, then reads whether the
// region is tracked (an arm that this read misses comes after the stores, and so
// do the copies behind it), then meets its other lanes, then marks.
__device__ __forceinline__ void mark_pages(const Kv8View& kv, uint32_t slot, uint64_t off, uint32_t len) {
    uint64_t* dirty = kv.dirty[slot];
    for (uint64_t pg = off >> kv.page_shift; pg <= (off + len - 1) >> kv.page_shift; pg++)
        atomicOr(reinterpret_cast<unsigned long long*>(&dirty[pg >> 6]), 1ull << (pg & 63));
}
__device__ __forceinline__ bool tracked(const Kv8View& kv, uint32_t slot) {
    return *reinterpret_cast<const volatile uint32_t*>(kv.tracking[slot]) != 0;
}

// What one lane takes of a row: piece c of the row's 2 x nkv x HD / 8 pieces of
// eight elements, K's heads first.
template <int HD>
struct Piece {
    uint32_t v, head, e;  // 1 for V, the head, the first element
    __device__ __forceinline__ Piece(uint32_t c, uint32_t nkv) {
        const uint32_t h = c / (HD / 8);
        v = h >= nkv ? 1 : 0;
        head = h - v * nkv;
        e = c % (HD / 8) * 8;
    }
};

// How many of n ascending values f(0), f(1), ... are at most `limit`: the lanes
// of a (converged) warp look at 32 at once, one trip to memory for up to 128,
// where a search by halves takes one a step.
template <typename F>
__device__ __forceinline__ uint32_t count_upto(uint32_t n, uint64_t limit, F f) {
    const uint32_t lane = threadIdx.x & 31;
    if (n > 512) {
        uint32_t lo = 0, hi = n;
        while (lo < hi) {
            const uint32_t mid = (lo + hi) >> 1;
            if (f(mid) <= limit) lo = mid + 1;
            else hi = mid;
        }
        return lo;
    }
    uint32_t count = 0;
#pragma unroll 4
    for (uint32_t i = 0; i < n; i += 32) count += __popc(__ballot_sync(0xffffffffu, i + lane < n && f(i + lane) <= limit));
    return count;
}

// The rows that one warp walks: where row r lies, and how many from it on lie
// behind one another in the same slot.
struct Walk {
    uint8_t* base = nullptr;
    uint32_t slot = 0, first = 0, end = 0, p0 = 0;
    // False: no place for row r (behind the last sequence, no position, past max_ctx).
    __device__ __forceinline__ bool to(const Kv8View& kv, const Kv8Rows& rows, uint32_t r, uint32_t last, uint32_t* pos,
                                       uint32_t* n) {
        if (r < first || r >= end) {
            if (rows.row_start) {
                slot = count_upto(rows.n_slots, r, [&](uint32_t i) { return __ldg(rows.row_start + i + 1); });
                first = slot < rows.n_slots ? __ldg(rows.row_start + slot) : r;
                end = slot < rows.n_slots ? __ldg(rows.row_start + slot + 1) : last;
                if (first > r) first = r, end = r + 1, slot = rows.n_slots;
            } else {
                slot = first = r;
                end = r + 1;
            }
            p0 = slot < rows.n_slots ? __ldg(rows.pos + slot) : kPosNone;
            base = slot < rows.n_slots ? reinterpret_cast<uint8_t*>(kv.base[slot]) : nullptr;
        }
        *n = min(end, last) - r;
        if (p0 == kPosNone) return false;
        const uint64_t p = (uint64_t)p0 + (r - first);
        if (p >= kv.max_ctx) {
            atomicOr(rows.err, ERR_POS);
            return false;
        }
        *n = (uint32_t)min((uint64_t)*n, kv.max_ctx - p);
        *pos = (uint32_t)p;
        return true;
    }
};

// Append, a scale for every position: a warp takes `per` rows in turn, HD / 8
// lanes a head. The row's slot is searched once a row, the same for all lanes.
// Bound by the latency of a row's chain (slot, loads, maximum, codes, the fence
// behind the stores): 64 rows of 2 heads of 64, f32: 3.4 us, of which a launch is
// 2 and the fence 0.6.
template <int HD, int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_append_rows(const Kv8View kv, const Kv8Rows rows, const Kv8Mat k,
                                                          const Kv8Mat v, uint32_t per) {
    constexpr uint32_t TL = HD / 8;
    const uint32_t lane = threadIdx.x & 31, pieces = 2 * kv.nkv * TL;
    const uint32_t first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * per, last = min(first + per, rows.n_rows);
    constexpr uint32_t N = 4;
    Walk walk;
    uint32_t n, pos;
    for (uint32_t r0 = first; r0 < last; r0 += n) {
        if (!walk.to(kv, rows, r0, last, &pos, &n)) continue;
        n = min(n, N);
        for (uint32_t c0 = 0; c0 < pieces; c0 += 32) {
            const uint32_t c = c0 + lane;
            const bool in = c < pieces;
            const Piece<HD> p(in ? c : 0, kv.nkv);
            const Kv8Mat& m = p.v ? v : k;
            float x[N][8];
            uint32_t top[N];
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
#pragma unroll
                for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
                if (in && i < n) load8<DT, VEC>(m.p, (r0 + i) * m.row + p.head * m.head + p.e, x[i]);
            }
#pragma unroll
            for (uint32_t i = 0; i < N; i++) {
                top[i] = amax8(x[i]);
#pragma unroll
                for (uint32_t o = TL / 2; o > 0; o >>= 1) top[i] = max(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
            }
            uint8_t* code = walk.base + kv.code_off(p.v, p.head, pos) + p.e;
            uint8_t* scale = walk.base + kv.scale_off(p.v, p.head, pos);
#pragma unroll
            for (uint32_t i = 0; i < N; i++, code += kv.pos_stride, scale += 4 * kv.sblk_stride)
                if (in && i < n) {
                    const float s = scale_for(top[i]);
                    *reinterpret_cast<uint2*>(code) = s > 0.0f ? codes8(x[i], s, reciprocal(s)) : make_uint2(0, 0);
                    if (p.e == 0) *reinterpret_cast<float*>(scale) = s;
                }
        }
        __threadfence();
        __syncwarp();
        if (tracked(kv, walk.slot)) {
            for (uint32_t h = lane; h < 2 * kv.nkv * n; h += 32) {
                const uint32_t i = h / (2 * kv.nkv), w = h / kv.nkv & 1, head = h % kv.nkv;
                mark_pages(kv, walk.slot, kv.code_off(w, head, pos + i), HD);
                mark_pages(kv, walk.slot, kv.scale_off(w, head, pos + i), 4);
            }
        }
    }
}

// Append, a scale for every B positions: WPU warps take one unit = (slot,
// block, head, K or V) and hold its new rows in registers between the maximum
// and the codes, RL rows a lane; the unit's older rows are rescaled where the
// scale doubles. Units of slot i start at unit row_start[i] / B + 2 i, which
// leaves room for every block that its rows can touch. Bound by the latency of
// loading, reducing, storing and waiting for the stores in turn, a unit a warp
// with nothing of the next on its way: 16 x 2,048 rows of 2 heads of 128, bf16,
// blocks of 32: 30 us (1.7 TB/s moved), five of them the stores' end.
template <int HD, int DT, bool VEC, int B>
__global__ void __launch_bounds__(kThreads) k_append_blocks(const Kv8View kv, const Kv8Rows rows, const Kv8Mat k,
                                                            const Kv8Mat v) {
    constexpr uint32_t TL = HD / 8, RPW = 32 / TL;
    constexpr uint32_t WPU = B / (4 * RPW) > 8 ? 8 : B / (4 * RPW), RL = B / (WPU * RPW), UPC = 8 / WPU;
    __shared__ uint32_t tops[8];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tl = lane % TL;
    const uint32_t j0 = (warp % WPU) * RPW + lane / TL;  // this lane's rows of the block: j0 + i * WPU * RPW
    const uint32_t unit = blockIdx.x * UPC + warp / WPU, blk_no = unit / (2 * kv.nkv);  // the check on rows keeps units in 32 bits
    const uint32_t which = unit - blk_no * 2 * kv.nkv, is_v = which >= kv.nkv ? 1 : 0;
    const uint32_t head = which - is_v * kv.nkv;

    // the unit's slot, its rows [r0, r0 + m) and its block
    uint32_t slot = 0, r0 = 0, m = 0, p0 = kPosNone, blk = 0;
    bool live;
    if (!rows.row_start) {
        slot = r0 = (uint32_t)blk_no;
        live = blk_no < rows.n_rows;
        m = 1;
        if (live) p0 = __ldg(rows.pos + slot);
        blk = p0 / B;
    } else {
        // the last slot whose first unit is <= blk_no
        const uint32_t upto = count_upto(rows.n_slots, blk_no, [&](uint32_t i) { return __ldg(rows.row_start + i) / B + 2ull * i; });
        live = upto > 0;
        if (live) {
            slot = upto - 1;
            r0 = __ldg(rows.row_start + slot);
            const uint32_t end = min(__ldg(rows.row_start + slot + 1), rows.n_rows);
            m = end > r0 ? end - r0 : 0;
            p0 = __ldg(rows.pos + slot);
            blk = p0 / B + (uint32_t)(blk_no - (r0 / B + 2ull * slot));
        }
    }
    live = live && m > 0 && p0 != kPosNone;
    const uint64_t b0 = (uint64_t)blk * B, end = (uint64_t)p0 + m;  // the rows' positions: [p0, end)
    live = live && b0 < end;
    if (live && end > kv.max_ctx && tl == 0 && j0 == 0) atomicOr(rows.err, ERR_POS);
    live = live && b0 < kv.max_ctx;

    float x[RL][8];
    uint32_t top = 0;
    const Kv8Mat& mat = is_v ? v : k;
#pragma unroll
    for (uint32_t i = 0; i < RL; i++) {
        const uint64_t p = b0 + j0 + i * WPU * RPW;
#pragma unroll
        for (int e = 0; e < 8; e++) x[i][e] = 0.0f;
        if (live && p >= p0 && p < end && p < kv.max_ctx)
            load8<DT, VEC>(mat.p, (r0 + (p - p0)) * mat.row + head * mat.head + 8 * tl, x[i]);
        top = max(top, amax8(x[i]));
    }
#pragma unroll
    for (uint32_t o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (WPU > 1) {
        if (lane == 0) tops[warp] = top;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < WPU; w++) top = max(top, tops[warp / WPU * WPU + w]);
    }
    uint8_t* base = live ? reinterpret_cast<uint8_t*>(kv.base[slot]) : nullptr;
    const uint64_t sat = kv.scale_off(is_v, head, blk);
    float s = scale_for(top), held = 0.0f;
    int k2 = 0;
    if (live && b0 < p0) held = *reinterpret_cast<const float*>(base + sat);
    // every thread of the unit holds the old scale before one writes the new one
    if (WPU > 1) __syncthreads();
    else __syncwarp();
    if (!live) return;  // the whole unit
    if (isnan(held)) {
        s = held;
    } else if (held > 0.0f && !isnan(s)) {
        if (s > 0.0f) k2 = doublings(held, s);
        s = __fmul_rn(__fmul_rn(held, pow2i(k2 / 2)), pow2i(k2 - k2 / 2));  // 2^k2 itself may pass f32
    }
    const float inv = s > 0.0f ? reciprocal(s) : 0.0f;
    // new rows, and older ones where the scale grew
    auto stored = [&](uint64_t p) { return p < end && p < kv.max_ctx && (p >= p0 || k2 > 0); };
#pragma unroll
    for (uint32_t i = 0; i < RL; i++) {
        const uint64_t p = b0 + j0 + i * WPU * RPW;
        if (!stored(p)) continue;
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
    }
    if (j0 == 0 && tl == 0) *reinterpret_cast<float*>(base + sat) = s;
    __threadfence();
    __syncwarp();
    if (tl != 0 || !tracked(kv, slot)) return;
#pragma unroll 1
    for (uint32_t i = 0; i < RL; i++) {
        const uint64_t p = b0 + j0 + i * WPU * RPW;
        if (stored(p)) mark_pages(kv, slot, kv.code_off(is_v, head, (uint32_t)p), HD);
    }
    if (j0 == 0) mark_pages(kv, slot, sat, 4);
}

// Read back: as k_append_rows, four rows' pieces in flight at once; bound by
// memory and the start: 32,768 rows of 2 heads of 128 to f16: 14 us (3.6 TB/s).
template <int HD, int DT, bool VEC>
__global__ void __launch_bounds__(kThreads) k_read_rows(const Kv8View kv, const Kv8Rows rows, const Kv8Mat k,
                                                        const Kv8Mat v, uint32_t per) {
    constexpr uint32_t TL = HD / 8, AT_ONCE = 4;
    const uint32_t lane = threadIdx.x & 31, pieces = 2 * kv.nkv * TL;
    const uint32_t first = (blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5)) * per, last = min(first + per, rows.n_rows);
    Walk walk;
    uint32_t n, pos;
    for (uint32_t r0 = first; r0 < last; r0 += n) {
        if (!walk.to(kv, rows, r0, last, &pos, &n)) continue;
        n = min(n, AT_ONCE);
        for (uint32_t c = lane; c < pieces; c += 32) {
            const Piece<HD> p(c, kv.nkv);
            const Kv8Mat& m = p.v ? v : k;
            if (!m.p) continue;
            uint2 code[AT_ONCE];
            float s[AT_ONCE];
            const uint8_t* from = walk.base + kv.code_off(p.v, p.head, pos) + p.e;
#pragma unroll
            for (uint32_t i = 0; i < AT_ONCE; i++, from += kv.pos_stride)
                if (i < n) {
                    code[i] = __ldg(reinterpret_cast<const uint2*>(from));
                    s[i] = __ldg(reinterpret_cast<const float*>(walk.base + kv.scale_off(p.v, p.head, (pos + i) >> kv.block_shift)));
                }
#pragma unroll
            for (uint32_t i = 0; i < AT_ONCE; i++)
                if (i < n) {
                    float x[8];
                    values8(code[i], s[i], x);
                    store8<DT, VEC>(const_cast<void*>(m.p), (r0 + i) * m.row + p.head * m.head + p.e, x);
                }
        }
    }
}

// Rows a warp takes: one while that leaves SMs idle, eight from 16 warps an SM on.
uint32_t rows_per_warp(uint32_t n_rows) { return n_rows >= 148 * 16 * 8 ? 8 : n_rows >= 148 * 16 * 4 ? 4 : 1; }

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
            const uint32_t per = rows_per_warp(rows.n_rows), cta = per * (kThreads / 32);
            k_append_rows<HD, DT, VEC><<<(rows.n_rows + cta - 1) / cta, kThreads, 0, st>>>(kv, rows, k, v, per);
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
        const uint32_t per = rows_per_warp(rows.n_rows), cta = per * (kThreads / 32), grid = (rows.n_rows + cta - 1) / cta;
        if (hd == 64) k_read_rows<64, DT, VEC><<<grid, kThreads, 0, st>>>(kv, rows, k, v, per);
        else k_read_rows<128, DT, VEC><<<grid, kThreads, 0, st>>>(kv, rows, k, v, per);
    });
    return cudaGetLastError();
}

}  // namespace hs
