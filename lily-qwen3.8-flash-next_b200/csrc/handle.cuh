// The handle behind include/lily_sampler.h and what every entry point's host side does with it:
// error texts, the current device, the fault latch, tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cmath>
#include <string>
#include <vector>

#include "../../include/lily_sampler.h"

namespace lily_host {

constexpr int RING = 8;

struct StageLayout {
    size_t params, steps, slots, hist_len, total;
};

inline StageLayout stage_layout(uint32_t max_rows) {
    StageLayout l;
    size_t off = 0;
    l.params = off;
    off += sizeof(lily_sampling_params_t) * max_rows;
    l.steps = off;
    off += sizeof(uint32_t) * max_rows;
    l.slots = off;
    off += sizeof(uint32_t) * max_rows;
    l.hist_len = off;
    off += sizeof(uint32_t) * max_rows;
    l.total = (off + 255) & ~size_t(255);
    return l;
}

}  // namespace lily_host

struct lily_sampler {
    int device = 0;
    uint32_t vocab = 0, max_rows = 0, max_history = 0, max_list = 0, flags = 0;
    std::string last_error;
    int32_t fault = 0;
    uint64_t wait_ns = 1000000000ull;     // bound of the waits inside the kernels
    uint32_t lost_arrival = 0;            // test hook: what SplitArgs::lost of the next row-kernel launch is
    uint32_t lost_stage = 0xFFFFFFFFu;    // test hook: a weight copy the next head launch leaves out
    int sm_count = 0;
    int max_smem = 0;
    uint2 *part = nullptr;
    uint32_t *part_n = nullptr;
    uint32_t *tickets = nullptr;
    uint32_t *status_word = nullptr;
    char *arena = nullptr;  // the device workspaces below are places in it, the staging ring's host side lies behind h_status
    uint32_t *counts_scratch = nullptr;
    uint32_t *counts_table = nullptr;
    uint32_t *seen_table = nullptr;
    uint32_t seen_words = 0;
    lily_host::StageLayout layout{};
    char *h_stage[lily_host::RING] = {};
    char *d_stage[lily_host::RING] = {};
    cudaEvent_t ev[lily_host::RING] = {};
    int ring_pos = 0;
    uint32_t *h_status = nullptr;
    long long *phase_clocks = nullptr;
    // The parameters a sharded call staged last: a decode step stages the same
    // rows for its candidate call and its merge call, and usually again next step.
    uint64_t slot_serial[lily_host::RING] = {};
    int shard_slot = -1;
    uint64_t shard_serial = 0;
    std::vector<char> shard_bytes;
    float *lm_logits = nullptr;  // LILY_FLAG_LMHEAD: F32 [64, lm_ld]
    uint64_t lm_ld = 0;
    // The LM head's workspaces: the hidden states' images (for lm_tokens padded tokens) and
    // the flags of sums handed on. lm_more: those of calls of more tokens than max_rows or of
    // more than CHUNK_K columns, made by the first of them.
    char *lm_prepared = nullptr, *lm_more = nullptr;
    uint32_t *lm_flags = nullptr;
    uint32_t lm_tokens = 0;
};

namespace lily_host {

inline int32_t fail(lily_sampler *h, int32_t code, const char *msg) {
    if (h) {
        h->last_error = msg;
    }
    return code;
}

inline int32_t cuda_fail(lily_sampler *h, cudaError_t e, const char *what) {
    if (h) {
        h->last_error = std::string(what) + ": " + cudaGetErrorString(e);
    }
    return LILY_ERR_CUDA;
}

#define CU(h, call)                              \
    do {                                         \
        cudaError_t e_ = (call);                 \
        if (e_ != cudaSuccess) {                 \
            return cuda_fail((h), e_, #call);    \
        }                                        \
    } while (0)

struct DeviceGuard {
    int prev = -1;
    bool ok = true, moved = false;
    explicit DeviceGuard(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) {
            prev = -1;
        }
        if (prev != dev) {
            moved = true;
            ok = cudaSetDevice(dev) == cudaSuccess;
        }
    }
    ~DeviceGuard() {
        if (moved && prev >= 0) {
            cudaSetDevice(prev);
        }
    }
};

inline bool params_ok(const lily_sampling_params_t &p) {
    return std::isfinite(p.temperature) && p.temperature >= 0.0f && std::isfinite(p.top_p) &&
           p.top_p > 0.0f && p.top_p <= 1.0f && std::isfinite(p.min_p) && p.min_p >= 0.0f &&
           p.min_p <= 1.0f && std::isfinite(p.repetition_penalty) &&
           p.repetition_penalty > 0.0f && std::isfinite(p.presence_penalty) &&
           std::isfinite(p.frequency_penalty);
}

inline int32_t check_handle(lily_sampler *h) {
    if (h == nullptr) {
        return LILY_ERR_ARG;
    }
    if (h->fault != 0) {
        return fail(h, LILY_ERR_FAULT, "a fault is latched on this sampler");
    }
    return LILY_OK;
}

// cuTensorMapEncodeTiled through the runtime's entry-point query: the library
// does not link against the driver.
typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *,
                                  CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                  CUtensorMapFloatOOBfill);

inline EncodeTiledFn tensor_map_encoder() {
    static EncodeTiledFn fn = nullptr;
    if (fn == nullptr) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &res) == cudaSuccess &&
            res == cudaDriverEntryPointSuccess) {
            fn = reinterpret_cast<EncodeTiledFn>(p);
        }
    }
    return fn;
}

// Every kernel that the norm, the product and the adjusted logits can come to, loaded on the current device (once;
// norm.cu, linear.cu, adjust.cu).
cudaError_t norm_ready();
cudaError_t linear_ready();
cudaError_t adjust_ready();

// f() if the current device has not been through it before; `seen`: a bit for each.
template <typename F>
cudaError_t once_per_device(std::atomic<uint64_t> &seen, F f) {
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    const uint64_t bit = 1ull << (device & 63);
    if (e == cudaSuccess && !(seen.load(std::memory_order_acquire) & bit)) {
        e = f();
        seen.fetch_or(e == cudaSuccess ? bit : 0u, std::memory_order_release);
    }
    return e;
}

// Loads a kernel; `smem`: its limit of dynamic shared memory, if that has to be raised.
template <typename Kernel>
cudaError_t load_kernel(Kernel kernel, uint32_t smem = 0) {
    cudaFuncAttributes fa;
    const cudaError_t e = cudaFuncGetAttributes(&fa, kernel);  // (this loads it)
    return e != cudaSuccess || smem == 0u ? e : cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
}

}  // namespace lily_host
