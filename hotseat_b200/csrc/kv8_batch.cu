// The batched path over 8-bit regions: the QKV product's rows to rotated f32
// rows before the cache, and attention's f32 rows to the f16 pairs that the
// output projection reads.
#include "attn_body.cuh"
#include "common.h"
#include "device.cuh"
#include "kernels.h"
#include "kv8.h"

namespace hs {
namespace {

// A warp per (slot, head of q, k or v): split-K partials in split order, then
// the bias, then RoPE on q and k (model.rs:365-373), as the f32 regions' append
// forms them. Slots' positions go to `pos` (none: inactive or past max_ctx).
template <int HD>
__global__ void __launch_bounds__(256) k_qkv_rows(const SplitAttnArgs a, uint32_t slots, float* q, float* k, float* v,
                                                  uint32_t* pos_out, uint32_t* row_start) {
    constexpr uint32_t HALF = HD / 2;
    const uint32_t lane = threadIdx.x & 31, heads = a.nh + 2 * a.nkv;
    const uint32_t item = blockIdx.x * 8 + (threadIdx.x >> 5), slot = item / heads, h = item - slot * heads;
    if (slot >= slots) return;
    DevCtl* ctl = a.ctl + slot;
    const uint32_t pos = ctl->pos;
    const bool active = ctl->active != 0, in = active && pos < a.max_ctx;
    if (h == 0 && lane == 0) {
        if (active && !in) atomicOr(&ctl->err, ERR_POS);
        pos_out[slot] = in ? pos : kPosNone;
        if (slot == 0) row_start[0] = 0, row_start[1] = slots;
    }
    if (!in) return;
    const float* src = a.qkv + (size_t)slot * a.qkv_rows;
    auto row = [&](uint32_t r) {
        float4 p = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (uint32_t s = 0; s < a.n_part; s++) p = attn::f4add(p, __ldcg(reinterpret_cast<const float4*>(src + s * a.part_stride + r)));
        if (a.bias) p = attn::f4add(p, *reinterpret_cast<const float4*>(a.bias + r));
        return p;
    };
    if (h >= a.nh + a.nkv) {
        if (lane < HD / 4)
            reinterpret_cast<float4*>(v + ((size_t)slot * a.nkv + h - a.nh - a.nkv) * HD)[lane] = row(h * HD + 4 * lane);
        return;
    }
    if (lane >= HALF / 4) return;
    float4 x0 = row(h * HD + 4 * lane), x1 = row(h * HD + HALF + 4 * lane);
    const float4 c = *reinterpret_cast<const float4*>(a.rope_cos + (size_t)pos * HALF + 4 * lane);
    const float4 sn = *reinterpret_cast<const float4*>(a.rope_sin + (size_t)pos * HALF + 4 * lane);
    auto rot = [](float& u, float& w, float cc, float ss) {
        const float u0 = u, w0 = w;
        u = __fsub_rn(__fmul_rn(u0, cc), __fmul_rn(w0, ss));
        w = __fadd_rn(__fmul_rn(u0, ss), __fmul_rn(w0, cc));
    };
    rot(x0.x, x1.x, c.x, sn.x);
    rot(x0.y, x1.y, c.y, sn.y);
    rot(x0.z, x1.z, c.z, sn.z);
    rot(x0.w, x1.w, c.w, sn.w);
    float* to = h < a.nh ? q + ((size_t)slot * a.nh + h) * HD : k + ((size_t)slot * a.nkv + h - a.nh) * HD;
    reinterpret_cast<float4*>(to)[lane] = x0;
    reinterpret_cast<float4*>(to + HALF)[lane] = x1;
}

__global__ void __launch_bounds__(256) k_to_pairs(const float* x, uint64_t n4, uint16_t* hi, uint16_t* lo) {
    const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n4) return;
    const float4 v = reinterpret_cast<const float4*>(x)[i];
    const float f[4] = {v.x, v.y, v.z, v.w};
    uint16_t h[4], l[4];
#pragma unroll
    for (int e = 0; e < 4; e++) {
        h[e] = f2h_rn(f[e]);
        l[e] = f2h_rn(__fsub_rn(f[e], h2f(h[e])));
    }
    reinterpret_cast<uint2*>(hi)[i] = make_uint2(h[0] | (uint32_t)h[1] << 16, h[2] | (uint32_t)h[3] << 16);
    reinterpret_cast<uint2*>(lo)[i] = make_uint2(l[0] | (uint32_t)l[1] << 16, l[2] | (uint32_t)l[3] << 16);
}

}  // namespace

cudaError_t launch_kv8_qkv_rows(uint32_t hd, const SplitAttnArgs& a, uint32_t slots, float* q, float* k, float* v,
                                uint32_t* pos, uint32_t* row_start, cudaStream_t st) {
    const uint32_t grid = (slots * (a.nh + 2 * a.nkv) + 7) / 8;
    if (hd == 64) k_qkv_rows<64><<<grid, 256, 0, st>>>(a, slots, q, k, v, pos, row_start);
    else k_qkv_rows<128><<<grid, 256, 0, st>>>(a, slots, q, k, v, pos, row_start);
    return cudaGetLastError();
}

cudaError_t launch_kv8_to_pairs(const float* x, uint64_t n, uint16_t* hi, uint16_t* lo, cudaStream_t st) {
    k_to_pairs<<<(uint32_t)((n / 4 + 255) / 256), 256, 0, st>>>(x, n / 4, hi, lo);
    return cudaGetLastError();
}

}  // namespace hs
