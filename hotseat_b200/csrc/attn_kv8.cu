// Attention over the 8-bit KV cache.
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

}  // namespace

cudaError_t launch_kv8_attend(uint32_t hd, const Kv8AttendArgs& a, cudaStream_t st) {
    if (!a.rows.n_rows) return cudaSuccess;
    const uint64_t items = (uint64_t)a.rows.n_rows * a.nh;
    const uint32_t grid = (uint32_t)((items + 3) / 4);
    auto go = [&](auto h) {
        constexpr int HD = decltype(h)::value;
        if (a.q.dtype == HS_F32) k_kv8_attend_simple<HD, HS_F32><<<grid, 128, 0, st>>>(a);
        else if (a.q.dtype == HS_F16) k_kv8_attend_simple<HD, HS_F16><<<grid, 128, 0, st>>>(a);
        else k_kv8_attend_simple<HD, HS_BF16><<<grid, 128, 0, st>>>(a);
    };
    if (hd == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    return cudaGetLastError();
}

}  // namespace hs
