// ops.h -- what the operators over device memory (page plan, K/V row store,
// paged attention, beam selection, cache reordering) share on the host side.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/tie_b200.h"
#include "common.cuh"

namespace tie {

// Sequences (or requests) one call takes: each CTA keeps a prefix sum over
// them in shared memory.
constexpr int kOpsMaxSeqs = 4096;
// Physical pages of a pool: slots (page * 16 + row) are int32.
constexpr int kOpsMaxPages = 1 << 27;
constexpr int kHeadDim = 64;

// Records `e` for tie_last_device_error (model.cu).
void note_device_error(cudaError_t e, const char* what, const char* file, int line);

// Kernels launched by the operators on the calling thread.
extern thread_local uint64_t op_launches;

#define TIE_OP_CU(expr)                                                    \
    do {                                                                   \
        cudaError_t e_ = (expr);                                           \
        if (e_ != cudaSuccess) {                                           \
            ::tie::note_device_error(e_, #expr, __FILE__, __LINE__);       \
            cudaGetLastError();                                            \
            return MODEL_ERR_DEVICE;                                       \
        }                                                                  \
    } while (0)

inline bool aligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }
inline bool aligned16(const void* p) { return aligned(p, 16); }

// For the length of a call, makes the device that holds `p` the current one
// (the caller's pointers need not be on it). status() is MODEL_ERR_ARG for
// memory the device cannot own (pageable or pinned host memory) and
// MODEL_ERR_DEVICE without a device.
class OnDeviceOf {
public:
    explicit OnDeviceOf(const void* p) {
        cudaPointerAttributes a;
        cudaError_t e = cudaPointerGetAttributes(&a, p);
        if (e != cudaSuccess) {
            note_device_error(e, "cudaPointerGetAttributes", __FILE__, __LINE__);
            cudaGetLastError();
            rc_ = MODEL_ERR_DEVICE;
            return;
        }
        if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged) { rc_ = MODEL_ERR_ARG; return; }
        int cur = 0;
        if (cudaGetDevice(&cur) != cudaSuccess) { cudaGetLastError(); rc_ = MODEL_ERR_DEVICE; return; }
        device_ = a.device;
        if (a.type == cudaMemoryTypeManaged) device_ = cur;
        if (device_ != cur) {
            if (cudaSetDevice(device_) != cudaSuccess) { cudaGetLastError(); rc_ = MODEL_ERR_DEVICE; return; }
            back_ = cur;
        }
    }
    ~OnDeviceOf() {
        if (back_ >= 0) cudaSetDevice(back_);
    }
    OnDeviceOf(const OnDeviceOf&) = delete;
    OnDeviceOf& operator=(const OnDeviceOf&) = delete;
    model_status status() const { return rc_; }
    int device() const { return device_; }

private:
    model_status rc_ = MODEL_OK;
    int device_ = 0, back_ = -1;
};

// SMs of a device (asked once per device).
int sm_count(int device);

// Rows of `pages` pages fit the addressing of these operators.
inline bool pool_shape_ok(int format, int n_pages, int n_kv_head) {
    return (format == TIE_KV_F32 || format == TIE_KV_BF16) && n_pages > 0 && n_pages <= kOpsMaxPages &&
           n_kv_head > 0 && n_kv_head <= 1024;
}

}  // namespace tie
