// The 8-bit KV cache: int8 codes with one f32 scale for each block of
// `block` positions, each KV head, K and V apart (value = code * scale).
//
// Bytes of a region, layer after layer:
//     K codes | V codes | K scales | V scales
// each plane padded to 256 bytes. Code rows are head_dim bytes, [pos][head]
// or [head][pos] by the region's layout; scales are [block][head] or
// [head][block] accordingly.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.h"

namespace hs {

constexpr uint32_t kPosNone = 0xffffffffu;  // HS_POS_NONE

struct Kv8Geo {
    uint64_t plane = 0, splane = 0, layers = 0;  // bytes of a code plane, of a scale plane
    __host__ __device__ uint64_t layer_bytes() const { return 2 * (plane + splane); }
    uint64_t bytes() const { return layers * layer_bytes(); }
};
inline Kv8Geo kv8_geo(const hs_kv_spec& s, uint32_t block) {
    auto pad = [](uint64_t v) { return (v + 255) / 256 * 256; };
    Kv8Geo g;
    g.layers = s.n_layers;
    g.plane = pad((uint64_t)s.max_ctx * s.n_kv_heads * s.head_dim);
    g.splane = pad(((uint64_t)s.max_ctx + block - 1) / block * s.n_kv_heads * 4);
    return g;
}
// A shape that the 8-bit kernels take: HS_OK or an error.
int kv8_check_shape(const hs_kv_spec& s, uint32_t block);

// One layer of n regions as the kernels see it.
struct Kv8View {
    float* const* base = nullptr;             // per slot (device table)
    uint64_t* const* dirty = nullptr;
    const uint32_t* const* tracking = nullptr;
    uint64_t layer_off = 0, plane = 0, splane = 0;
    uint64_t pos_stride = 0, head_stride = 0;    // codes, bytes
    uint64_t sblk_stride = 0, shead_stride = 0;  // scales, elements
    uint32_t nkv = 0, max_ctx = 0, block_shift = 0, page_shift = 0;

    __device__ uint64_t code_off(uint32_t v, uint32_t head, uint32_t pos) const {
        return layer_off + (v ? plane : 0) + (uint64_t)pos * pos_stride + (uint64_t)head * head_stride;
    }
    __device__ uint64_t scale_off(uint32_t v, uint32_t head, uint32_t blk) const {
        return layer_off + 2 * plane + (v ? splane : 0) +
               ((uint64_t)blk * sblk_stride + (uint64_t)head * shead_stride) * 4;
    }
};
inline Kv8View kv8_view(const hs_kv_spec& s, uint32_t block, uint32_t layer) {
    const Kv8Geo g = kv8_geo(s, block);
    Kv8View v;
    v.layer_off = layer * g.layer_bytes();
    v.plane = g.plane;
    v.splane = g.splane;
    const uint64_t hd = s.head_dim, nb = (s.max_ctx + block - 1) / block;
    v.pos_stride = s.layout == HS_LAYOUT_TOKEN_MAJOR ? s.n_kv_heads * hd : hd;
    v.head_stride = s.layout == HS_LAYOUT_TOKEN_MAJOR ? hd : (uint64_t)s.max_ctx * hd;
    v.sblk_stride = s.layout == HS_LAYOUT_TOKEN_MAJOR ? s.n_kv_heads : 1;
    v.shead_stride = s.layout == HS_LAYOUT_TOKEN_MAJOR ? 1 : nb;
    v.nkv = s.n_kv_heads;
    v.max_ctx = s.max_ctx;
    v.block_shift = (uint32_t)__builtin_ctz(block);
    return v;
}

// Rows of a ragged batch: slot i's are row_start[i] .. row_start[i + 1] - 1
// (row_start null: row i alone), at positions pos[i], pos[i] + 1, ...
struct Kv8Rows {
    uint32_t n_rows = 0, n_slots = 0;
    const uint32_t* row_start = nullptr;
    const uint32_t* pos = nullptr;
    uint32_t* err = nullptr;  // ERR_POS is set here for rows past max_ctx
};

// Element types of rows (HS_F32, HS_F16, HS_BF16) with their strides in
// elements; a row's head_dim elements are consecutive.
struct Kv8Mat {
    const void* p = nullptr;
    uint64_t row = 0, head = 0;
    uint32_t dtype = 0;
};
inline uint32_t dtype_bytes(uint32_t dtype) { return dtype == HS_F32 ? 4 : 2; }

cudaError_t launch_kv8_append(uint32_t hd, const Kv8View& kv, const Kv8Rows& rows, const Kv8Mat& k, const Kv8Mat& v,
                              cudaStream_t st);
cudaError_t launch_kv8_read(uint32_t hd, const Kv8View& kv, const Kv8Rows& rows, const Kv8Mat& k, const Kv8Mat& v,
                            cudaStream_t st);

// A single row's positions are split between CTAs by its own length and the
// region's shape alone, so that its bits do not depend on the batch: in
// eight (a cluster), but splits of at least 32 KB and at most 128 KB of codes
// and no more than kv8_max_splits. Short splits finish a lone row sooner (2,048
// positions, 14/2 heads of 64: 6.2 us in eight, 7.6 in four), long ones keep a
// large batch's CTAs from spending their time on starting and joining (64
// sequences of 8,192: 46 us with 128 KB, 58 with 64 KB).
constexpr uint32_t kv8_max_splits(uint32_t nkv) {
    return nkv <= 2 ? 148 : 296 / nkv < 16 ? 16 : 296 / nkv;
}
__host__ __device__ constexpr uint32_t kv8_min_split(uint32_t hd) { return 16384 / hd; }
__host__ __device__ inline uint32_t kv8_split_len(uint32_t n, uint32_t hd, uint32_t max_splits) {
    const uint32_t least = kv8_min_split(hd), most = 4 * least;
    uint32_t len = (n / 8 + 63) / 64 * 64;
    len = len < least ? least : len > most ? most : len;
    if (n <= len * max_splits) return len;
    return ((n + max_splits - 1) / max_splits + 63) / 64 * 64;
}
// Query heads of one KV head that a CTA takes together.
constexpr uint32_t kv8_single_cols(uint32_t group) { return group <= 8 ? 8 : 16; }

// Chunks of rows: whether a cluster shares the positions of each tile of 256
// (row, head) pairs, by the slot's own rows (`tiles` of them, from position
// pos0 on) and the region's shape alone: where a slot's tiles are few, and for
// 512 positions a CTA at least. 16 rows a slot, 12/2 heads of 128, bf16, over
// 5,000 positions: 33 us shared, 169 by one CTA for each KV head; 16 such slots
// 93 and 166; 64 slots, which fill the GPU by themselves and pay for the CTAs'
// starts and joins, 290 and 171 (at 9,000: 428 and 294). One slot over 9,000: 48
// and 293, over 32,768: 139 and 1,035. The rule is for the slot alone; a large
// batch of such rows pays for it.
constexpr uint32_t kKv8ChunkSplits = 8, kKv8ChunkClusters = 8;  // CTAs of a cluster, clusters of a slot
__host__ __device__ constexpr bool kv8_chunk_shared(uint64_t tiles, uint32_t pos0, uint32_t nkv) {
    return tiles * nkv <= kKv8ChunkClusters && pos0 >= 512 * kKv8ChunkSplits;
}

// Floats of a cluster's record: outputs, and for each of 8 shares its columns' maxima and sums.
__host__ __device__ constexpr uint32_t kv8_record(uint32_t hd, uint32_t cols) { return cols * (hd + 16); }

struct Kv8AttendArgs {
    Kv8View kv;
    Kv8Rows rows;
    Kv8Mat q, out;
    uint32_t group = 0, chunks = 0;  // query heads of a KV head, and CTAs of kv8_single_cols for these
    float scale = 1.0f;
    uint32_t slot_clusters = 0;  // split chunks: clusters set aside for each slot; 0: for each tile that the rows can need
    bool q_vec = false, out_vec = false;  // four elements of a row at once: base and strides allow it
    // single rows: CTAs of `cluster` splits join in shared memory; where a
    // region's rows can need more of them, their records [slot][KV head][head
    // chunk][max_clusters][kv8_record] and, for each (slot, KV head, chunk),
    // eight counters that are zero between calls
    uint32_t max_splits = 0, cluster = 1, max_clusters = 0;
    float* part = nullptr;
    uint32_t* counters = nullptr;
};
cudaError_t kv8_attend_set_smem_limits();
cudaError_t launch_kv8_attend(uint32_t hd, const Kv8AttendArgs& a, cudaStream_t st);

// The splits and workspace of single rows for n slots: what Kv8AttendArgs needs.
struct Kv8Plan {
    uint32_t group = 0, chunks = 0, max_splits = 0, cluster = 1, max_clusters = 0;
    uint64_t part_floats = 0, counters = 0;  // 0: none needed
};
inline Kv8Plan kv8_plan(const hs_kv_spec& s, uint32_t nh, uint32_t n) {
    Kv8Plan p;
    p.group = nh / s.n_kv_heads;
    const uint32_t nc = kv8_single_cols(p.group), least = kv8_min_split(s.head_dim);
    p.chunks = (p.group + nc - 1) / nc;
    const uint64_t items = (uint64_t)n * s.n_kv_heads * p.chunks;
    const uint32_t splits = (s.max_ctx + least - 1) / least;
    p.max_splits = splits < kv8_max_splits(s.n_kv_heads) ? splits : kv8_max_splits(s.n_kv_heads);
    while (p.cluster < 8 && p.cluster < p.max_splits) p.cluster *= 2;
    p.max_clusters = (p.max_splits + p.cluster - 1) / p.cluster;
    if (p.max_clusters > 1) {
        p.part_floats = items * p.max_clusters * kv8_record(s.head_dim, nc);
        p.counters = items * 8;
    }
    return p;
}
inline void kv8_use_plan(Kv8AttendArgs* a, const Kv8Plan& p) {
    a->group = p.group;
    a->chunks = p.chunks;
    a->max_splits = p.max_splits;
    a->cluster = p.cluster;
    a->max_clusters = p.max_clusters;
}

// The batched path (kv8_batch.cu): slots' q, k, v rows [slot][head][head_dim]
// and positions from the QKV product, and rows to f16 pairs.
struct SplitAttnArgs;
cudaError_t launch_kv8_qkv_rows(uint32_t hd, const SplitAttnArgs& a, uint32_t slots, float* q, float* k, float* v,
                                uint32_t* pos, uint32_t* row_start, cudaStream_t st);
cudaError_t launch_kv8_to_pairs(const float* x, uint64_t n, uint16_t* hi, uint16_t* lo, cudaStream_t st);

}  // namespace hs
