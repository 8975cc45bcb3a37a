// Host side of the 8-bit KV cache: its shapes and live ranges, sets of
// regions, and the calls that append to them, read them and attend over them.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <vector>

#include "common.h"
#include "kernels.h"
#include "kv8.h"
#include "kv_region.h"

namespace hs {

int kv8_check_shape(const hs_kv_spec& s, uint32_t block) {
    if (s.layout > 1) return fail(HS_E_ARG, "unknown KV layout");
    if (!s.n_layers || !s.n_kv_heads || !s.max_ctx) return fail(HS_E_ARG, "empty KV shape");
    if (s.head_dim != 64 && s.head_dim != 128) return fail(HS_E_UNSUPPORTED, "head_dim must be 64 or 128");
    if (block != 1 && block != 16 && block != 32 && block != 64 && block != 128)
        return fail(HS_E_UNSUPPORTED, "the scale block must be 1, 16, 32, 64 or 128 positions");
    // offsets are 64 bits wide; the region itself must be addressable (a layer of
    // the largest shape has 2^51 bytes, so the sum of layers could pass 64 bits)
    if (s.n_kv_heads > 4096 || s.max_ctx > (1u << 30) || s.n_layers > (1ull << 48) / kv8_geo(s, block).layer_bytes())
        return fail(HS_E_UNSUPPORTED, "KV shape too large");
    return HS_OK;
}

}  // namespace hs

using namespace hs;

struct hs_kv8_set {
    hs_kv_spec spec{};
    int device = 0;
    uint32_t block = 0, page_shift = 0, n = 0, nh = 0;
    void** tab = nullptr;       // device: n region bases, n bitmaps, n tracking flags
    float* part = nullptr;      // records and counters of single-row attention (Kv8AttendArgs)
    uint32_t* counters = nullptr;
    Kv8Plan plan;
    uint32_t* err = nullptr;    // device error word (ERR_POS)
    uint32_t* err_h = nullptr;  // pinned
    ~hs_kv8_set() {
        DeviceGuard g(device);
        cudaFree(tab);
        cudaFree(part);
        cudaFree(counters);
        cudaFree(err);
        cudaFreeHost(err_h);
    }
};

namespace {

// The arguments that the calls on a set share.
int check_call(const hs_kv8_set* s, uint32_t layer, uint32_t n_rows, const uint32_t* row_start, const uint32_t* pos,
               uint32_t dtype) {
    if (!s) return fail(HS_E_ARG, "null set");
    if (layer >= s->spec.n_layers) return fail(HS_E_ARG, "layer past the regions' layers");
    if (dtype > HS_BF16) return fail(HS_E_ARG, "unknown element type");
    if (!pos) return fail(HS_E_ARG, "null positions");
    if (!row_start && n_rows != s->n) return fail(HS_E_ARG, "without row_start there is one row for each slot");
    // grids and the blocks' numbers (n_rows + 2 n_slots at most, for each head of K and V) in 31 bits
    if (((uint64_t)n_rows + 2ull * s->n) * 2 * std::max(s->spec.n_kv_heads, s->nh) > 0x7fffffffull)
        return fail(HS_E_UNSUPPORTED, "too many rows in one call");
    return HS_OK;
}

int check_matrix(const void* p, uint32_t dtype, uint32_t n_rows, const char* what) {
    if (!p && n_rows) return fail(HS_E_ARG, std::string("null ") + what);
    if (reinterpret_cast<uintptr_t>(p) % dtype_bytes(dtype))
        return fail(HS_E_ARG, std::string(what) + " is not aligned to its element type");
    return HS_OK;
}

// A written matrix also holds each element in a place of its own.
int check_output(const void* p, uint32_t dtype, uint64_t n_rows, uint64_t heads, uint64_t hd, uint64_t row,
                 uint64_t head, const char* what) {
    int rc = check_matrix(p, dtype, (uint32_t)n_rows, what);
    if (rc || !n_rows) return rc;
    const bool heads_in = (heads == 1 || head >= hd) && (n_rows == 1 || row >= (heads - 1) * head + hd);
    const bool rows_in = (n_rows == 1 || row >= hd) && (heads == 1 || head >= (n_rows - 1) * row + hd);
    return heads_in || rows_in ? HS_OK : fail(HS_E_ARG, std::string(what) + ": rows or heads overlap");
}

Kv8View view_of(const hs_kv8_set* s, uint32_t layer) {
    Kv8View v = kv8_view(s->spec, s->block, layer);
    v.base = reinterpret_cast<float* const*>(s->tab);
    v.dirty = reinterpret_cast<uint64_t* const*>(s->tab + s->n);
    v.tracking = reinterpret_cast<const uint32_t* const*>(s->tab + 2 * s->n);
    v.page_shift = s->page_shift;
    return v;
}

Kv8Rows rows_of(const hs_kv8_set* s, uint32_t n_rows, const uint32_t* row_start, const uint32_t* pos) {
    Kv8Rows r;
    r.n_rows = n_rows;
    r.n_slots = s->n;
    r.row_start = row_start;
    r.pos = pos;
    r.err = s->err;
    return r;
}

// Whether four consecutive elements of a row can be taken at once.
bool fours(const Kv8Mat& m) {
    const uint64_t b = 4 * dtype_bytes(m.dtype);
    return reinterpret_cast<uintptr_t>(m.p) % b == 0 && m.row % 4 == 0 && m.head % 4 == 0;
}

int launched(cudaError_t e, const char* what) {
    return e == cudaSuccess ? HS_OK : fail(HS_E_CUDA, std::string(what) + " launch: " + cudaGetErrorString(e));
}

}  // namespace

extern "C" {

uint64_t hs_kv8_live_ranges_between(const hs_kv_spec* s, uint32_t block, uint32_t from, uint32_t to, uint64_t* out,
                                    uint64_t cap) {
    if (!s || !block || (block & (block - 1)) || to <= from) return 0;
    const Kv8Geo g = kv8_geo(*s, block);
    const uint64_t b0 = from / block, b1 = ((uint64_t)to + block - 1) / block, p0 = b0 * block;
    const uint64_t nb = ((uint64_t)s->max_ctx + block - 1) / block;
    uint64_t count = 0;
    // a plane's units [a, b): `w` bytes for each unit and head, n units a head
    auto plane = [&](uint64_t off, uint64_t a, uint64_t b, uint64_t w, uint64_t n) {
        const bool tok = s->layout == HS_LAYOUT_TOKEN_MAJOR;
        for (uint64_t h = 0; h < (tok ? 1 : s->n_kv_heads); h++) {
            const uint64_t unit = tok ? s->n_kv_heads * w : w;
            if (out && count < cap) {
                out[2 * count] = off + (h * n + a) * unit;
                out[2 * count + 1] = (b - a) * unit;
            }
            count++;
        }
    };
    for (uint64_t l = 0; l < s->n_layers; l++) {
        const uint64_t at = l * g.layer_bytes();
        plane(at, p0, to, s->head_dim, s->max_ctx);
        plane(at + g.plane, p0, to, s->head_dim, s->max_ctx);
        plane(at + 2 * g.plane, b0, b1, 4, nb);
        plane(at + 2 * g.plane + g.splane, b0, b1, 4, nb);
    }
    return count;
}

int hs_kv8_set_new(hs_kv* const* kvs, uint32_t n, uint32_t n_heads, hs_kv8_set** out) {
    if (!kvs || !out) return fail(HS_E_ARG, "null argument");
    *out = nullptr;
    if (n == 0 || n > 4096) return fail(HS_E_ARG, "a set holds 1..4096 regions");
    std::vector<const hs_kv*> seen;
    for (uint32_t i = 0; i < n; i++) {
        const hs_kv* k = kvs[i];
        if (!k) return fail(HS_E_ARG, "null KV region");
        if (!k->block8) return fail(HS_E_ARG, "an f32 KV region in an 8-bit set");
        if (k->ipc_view) return fail(HS_E_ARG, "the region belongs to another process");
        if (std::memcmp(&k->spec, &kvs[0]->spec, sizeof k->spec) != 0 || k->block8 != kvs[0]->block8 ||
            k->page_shift != kvs[0]->page_shift || k->device != kvs[0]->device)
            return fail(HS_E_ARG, "the regions of a set must share shape, block, page size and device");
        seen.push_back(k);
    }
    std::sort(seen.begin(), seen.end());
    if (std::adjacent_find(seen.begin(), seen.end()) != seen.end())
        return fail(HS_E_ARG, "a KV region appears twice in one set");
    const uint32_t nkv = kvs[0]->spec.n_kv_heads;
    if (n_heads % nkv || n_heads / nkv > 256)
        return fail(HS_E_ARG, "n_heads must be a multiple of the KV heads, at most 256 for each");
    auto s = std::make_unique<hs_kv8_set>();
    s->spec = kvs[0]->spec;
    s->device = kvs[0]->device;
    s->block = kvs[0]->block8;
    s->page_shift = kvs[0]->page_shift;
    s->n = n;
    s->nh = n_heads;
    DeviceGuard g(s->device);
    HS_CUDA_TRY(g.err);
    std::vector<void*> tab(3 * (size_t)n);
    for (uint32_t i = 0; i < n; i++) {
        tab[i] = kvs[i]->base;
        tab[n + i] = kvs[i]->dirty;
        tab[2 * n + i] = kvs[i]->tracking;
    }
    if (cudaMalloc(&s->tab, tab.size() * sizeof(void*)) != cudaSuccess || cudaMalloc(&s->err, 4) != cudaSuccess ||
        cudaMallocHost(&s->err_h, 4) != cudaSuccess) {
        cudaGetLastError();
        return fail(HS_E_NOMEM, "8-bit set: out of memory");
    }
    HS_CUDA_TRY(cudaMemcpy(s->tab, tab.data(), tab.size() * sizeof(void*), cudaMemcpyHostToDevice));
    HS_CUDA_TRY(cudaMemset(s->err, 0, 4));
    if (n_heads) {
        HS_CUDA_TRY(kv8_attend_set_smem_limits());
        s->plan = kv8_plan(s->spec, n_heads, n);
        if (s->plan.counters) {
            if (cudaMalloc(&s->part, s->plan.part_floats * 4) != cudaSuccess ||
                cudaMalloc(&s->counters, s->plan.counters * 4) != cudaSuccess) {
                cudaGetLastError();
                return fail(HS_E_NOMEM, "8-bit set: out of memory");
            }
            HS_CUDA_TRY(cudaMemset(s->counters, 0, s->plan.counters * 4));
        }
    }
    HS_CUDA_TRY(cudaStreamSynchronize(nullptr));
    *out = s.release();
    return HS_OK;
}

void hs_kv8_set_free(hs_kv8_set* s) { delete s; }

int hs_kv8_set_check(hs_kv8_set* s, void* stream) {
    if (!s) return fail(HS_E_ARG, "null set");
    DeviceGuard g(s->device);
    HS_CUDA_TRY(g.err);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    HS_CUDA_TRY(cudaMemcpyAsync(s->err_h, s->err, 4, cudaMemcpyDeviceToHost, st));
    HS_CUDA_TRY(cudaMemsetAsync(s->err, 0, 4, st));
    HS_CUDA_TRY(cudaStreamSynchronize(st));
    if (*s->err_h & ERR_TIMEOUT) return fail(HS_E_CUDA, "attention reported a bounded-wait timeout");
    if (*s->err_h & ERR_POS) return fail(HS_E_ARG, "position past max_ctx");
    return HS_OK;
}

int hs_kv8_append(hs_kv8_set* s, uint32_t layer, uint32_t n_rows, const uint32_t* row_start, const uint32_t* pos,
                  const void* k, const void* v, uint32_t dtype, uint64_t row_stride, uint64_t head_stride,
                  void* stream) {
    int rc = check_call(s, layer, n_rows, row_start, pos, dtype);
    if (rc) return rc;
    const uint64_t hd = s->spec.head_dim;
    if ((rc = check_matrix(k, dtype, n_rows, "k")) || (rc = check_matrix(v, dtype, n_rows, "v"))) return rc;
    if (!n_rows) return HS_OK;
    DeviceGuard g(s->device);
    HS_CUDA_TRY(g.err);
    const Kv8Mat mk{k, row_stride, head_stride, dtype}, mv{v, row_stride, head_stride, dtype};
    return launched(launch_kv8_append((uint32_t)hd, view_of(s, layer), rows_of(s, n_rows, row_start, pos), mk, mv,
                                      static_cast<cudaStream_t>(stream)),
                    "append");
}

int hs_kv8_read(hs_kv8_set* s, uint32_t layer, uint32_t n_rows, const uint32_t* row_start, const uint32_t* pos,
                void* k, void* v, uint32_t dtype, uint64_t row_stride, uint64_t head_stride, void* stream) {
    int rc = check_call(s, layer, n_rows, row_start, pos, dtype);
    if (rc) return rc;
    const uint64_t hd = s->spec.head_dim, nkv = s->spec.n_kv_heads;
    if ((k && (rc = check_output(k, dtype, n_rows, nkv, hd, row_stride, head_stride, "k"))) ||
        (v && (rc = check_output(v, dtype, n_rows, nkv, hd, row_stride, head_stride, "v"))))
        return rc;
    if (!n_rows || (!k && !v)) return HS_OK;
    DeviceGuard g(s->device);
    HS_CUDA_TRY(g.err);
    const Kv8Mat mk{k, row_stride, head_stride, dtype}, mv{v, row_stride, head_stride, dtype};
    return launched(launch_kv8_read((uint32_t)hd, view_of(s, layer), rows_of(s, n_rows, row_start, pos), mk, mv,
                                    static_cast<cudaStream_t>(stream)),
                    "read");
}

int hs_kv8_attend(hs_kv8_set* s, uint32_t layer, uint32_t n_rows, const uint32_t* row_start, const uint32_t* pos,
                  const void* q, uint64_t q_row_stride, uint64_t q_head_stride, void* out, uint64_t out_row_stride,
                  uint64_t out_head_stride, uint32_t dtype, float scale, void* stream) {
    int rc = check_call(s, layer, n_rows, row_start, pos, dtype);
    if (rc) return rc;
    if (!s->nh) return fail(HS_E_ARG, "the set was made without query heads");
    if (!(scale > 0.0f) || std::isinf(scale)) return fail(HS_E_ARG, "scale must be positive and finite");
    const uint64_t hd = s->spec.head_dim;
    if ((rc = check_matrix(q, dtype, n_rows, "q")) ||
        (rc = check_output(out, dtype, n_rows, s->nh, hd, out_row_stride, out_head_stride, "out")))
        return rc;
    if (!n_rows) return HS_OK;
    DeviceGuard g(s->device);
    HS_CUDA_TRY(g.err);
    Kv8AttendArgs a;
    a.kv = view_of(s, layer);
    a.rows = rows_of(s, n_rows, row_start, pos);
    a.q = Kv8Mat{q, q_row_stride, q_head_stride, dtype};
    a.out = Kv8Mat{out, out_row_stride, out_head_stride, dtype};
    kv8_use_plan(&a, s->plan);
    a.scale = scale;
    a.q_vec = fours(a.q);
    a.out_vec = fours(a.out);
    a.part = s->part;
    a.counters = s->counters;
    return launched(launch_kv8_attend((uint32_t)hd, a, static_cast<cudaStream_t>(stream)), "attention");
}

}  // extern "C"
