// Scores of logit rows: log probabilities of given tokens, entropy, rank and
// the top alternatives.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <string>

#include "common.h"
#include "device.cuh"
#include "kernels.h"
#include "kv_region.h"

namespace hs {
namespace {

template <int DT>
__device__ __forceinline__ float logit(const void* p, uint64_t e) {
    if constexpr (DT == HS_F32) return static_cast<const float*>(p)[e];
    else if constexpr (DT == HS_F16) return __half2float(static_cast<const __half*>(p)[e]);
    else return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[e]);
}

// A key that is larger for a token that comes earlier in the order (logit
// descending, NaN first, -0 equal to 0; id ascending).
__device__ __forceinline__ uint64_t order_key(float x, uint32_t id) {
    uint32_t b = __float_as_uint(__fadd_rn(x, 0.0f));
    b = (b & 0x80000000u) ? ~b : b | 0x80000000u;
    if (isnan(x)) b = 0xffffffffu;
    return ((uint64_t)b << 32) | (0xffffffffu - id);
}

constexpr uint32_t kThreads = 512;

template <int DT>
__global__ void __launch_bounds__(kThreads) k_logprobs_simple(const LogprobArgs a) {
    __shared__ float fa[16];
    __shared__ double da[16], db[16];
    __shared__ uint32_t ua[16];
    __shared__ uint64_t ka[16];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint64_t r = blockIdx.x;
    const uint8_t* row = static_cast<const uint8_t*>(a.logits) + r * a.row_stride * (DT == HS_F32 ? 4 : 2);
    const uint32_t id = a.ids ? a.ids[r] : 0xffffffffu;
    const float xt = id < a.vocab ? logit<DT>(row, id) : __int_as_float(0x7fffffff);
    const uint64_t kt = order_key(xt, id);
    float m = -INFINITY;
    for (uint32_t i = tid; i < a.vocab; i += kThreads) m = fmaxf(m, logit<DT>(row, i));
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) fa[warp] = m;
    __syncthreads();
    for (int w = 0; w < 16; w++) m = fmaxf(m, fa[w]);
    __syncthreads();
    double l = 0.0, t = 0.0;
    uint32_t before = 0;
    for (uint32_t i = tid; i < a.vocab; i += kThreads) {
        const float x = logit<DT>(row, i), d = x - m, e = expf(d);
        l += e;
        if (e != 0.0f) t += (double)e * d;
        before += order_key(x, i) > kt;
    }
    for (int o = 16; o > 0; o >>= 1) {
        l += __shfl_xor_sync(0xffffffffu, l, o);
        t += __shfl_xor_sync(0xffffffffu, t, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    if (lane == 0) da[warp] = l, db[warp] = t, ua[warp] = before;
    __syncthreads();
    l = t = 0.0;
    before = 0;
    for (int w = 0; w < 16; w++) l += da[w], t += db[w], before += ua[w];
    const float lz = (float)log(l);
    if (tid == 0) {
        if (a.logp) a.logp[r] = (xt - m) - lz;
        if (a.entropy) a.entropy[r] = (float)(log(l) - t / l);
        if (a.rank) a.rank[r] = id < a.vocab ? before : 0xffffffffu;
    }
    uint64_t last = ~0ull;
    for (uint32_t j = 0; j < a.top; j++) {
        uint64_t best = 0;
        for (uint32_t i = tid; i < a.vocab; i += kThreads) {
            const uint64_t k = order_key(logit<DT>(row, i), i);
            if ((j == 0 || k < last) && k > best) best = k;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const uint64_t k = __shfl_xor_sync(0xffffffffu, best, o);
            best = k > best ? k : best;
        }
        if (lane == 0) ka[warp] = best;
        __syncthreads();
        for (int w = 0; w < 16; w++) best = ka[w] > best ? ka[w] : best;
        __syncthreads();
        last = best;
        if (tid == 0) {
            const uint32_t i = 0xffffffffu - (uint32_t)best;
            if (a.top_ids) a.top_ids[r * a.top + j] = i;
            if (a.top_logp) a.top_logp[r * a.top + j] = (logit<DT>(row, i) - m) - lz;
        }
    }
}

}  // namespace

cudaError_t launch_logprobs(const LogprobArgs& a, cudaStream_t st) {
    if (!a.rows) return cudaSuccess;
    if (a.dtype == HS_F32) k_logprobs_simple<HS_F32><<<a.rows, kThreads, 0, st>>>(a);
    else if (a.dtype == HS_F16) k_logprobs_simple<HS_F16><<<a.rows, kThreads, 0, st>>>(a);
    else k_logprobs_simple<HS_BF16><<<a.rows, kThreads, 0, st>>>(a);
    return cudaGetLastError();
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
