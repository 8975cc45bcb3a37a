// A KV region on one GPU: the object behind hs_kv.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "common.h"
#include "kernels.h"

struct hs_kv {
    hs_kv_spec spec{};
    int device = 0;
    uint64_t bytes = 0, n_pages = 0, n_words = 0;
    uint32_t page_size = 0, page_shift = 0;
    float* base = nullptr;
    uint64_t* dirty = nullptr;
    uint64_t* harvest_buf = nullptr;
    uint32_t* tracking = nullptr;
    uint64_t fingerprint = 0;
    cudaStream_t st = nullptr;
    int n_sm = 148;
    // byte-run transfers: packed staging (grown on demand), the run table
    // (pinned upload buffer and device copy) and the event after its last use
    uint8_t* stage = nullptr;
    uint64_t stage_cap = 0;
    hs::XferRun *tab_h = nullptr, *tab_dev = nullptr;
    uint64_t tab_cap = 0;
    cudaEvent_t tab_ev = nullptr;
    // 0: f32 rows in the reference's layout; else int8 codes with a scale per
    // `block8` positions and KV head (kv8.h)
    uint32_t block8 = 0;
    bool ipc_view = false;  // `base` maps another process's region (hs_kv_open_ipc)
    ~hs_kv() {
        cudaSetDevice(device);
        if (tab_ev) cudaEventSynchronize(tab_ev);
        if (st) cudaStreamDestroy(st);
        if (tab_ev) cudaEventDestroy(tab_ev);
        cudaFreeHost(tab_h);
        cudaFree(tab_dev);
        cudaFree(stage);
        if (ipc_view)
            cudaIpcCloseMemHandle(base);
        else
            cudaFree(base);
        cudaFree(dirty);
        cudaFree(harvest_buf);
        cudaFree(tracking);
    }
};


namespace hs {

// Restores the calling thread's current device on leaving the scope.
struct DeviceGuard {
    int prev = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&prev);
        if (err == cudaSuccess && prev != device)
            err = cudaSetDevice(device);
        else
            prev = -1;
    }
    ~DeviceGuard() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

// Allocates a region (block8 0: f32; else 8-bit, kv8.h), or with `handle`
// maps another process's region of that shape.
int kv_create(int device, const hs_kv_spec& spec, uint32_t block8, uint32_t page_size, uint64_t fingerprint,
              const void* handle, hs_kv** out);

}  // namespace hs
