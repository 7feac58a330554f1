// What the entry points of include/homura_cuda_layers.h share: their checks of a description, and how an operand of
// three dimensions is walked.
#pragma once

#include <atomic>
#include <string>

#include "../../include/homura_cuda_layers.h"

#include "common.cuh"
#include "elem.cuh"
#include "map.cuh"

namespace hmc {

enum class Use { kInput, kOutput };

// `d` has exactly these sizes and the dtype; an output's elements are distinct; every element's byte offset fits 63 bits.
inline hmc_status check_layer(const hmc_tensor_desc *d, const char *what, int dtype, int ndim, const int64_t *sizes, Use use) {
    hmc_status s = check_desc(d, what);
    if (s != HMC_OK) return s;
    if (d->dtype != dtype) return fail(HMC_INVALID, std::string(what) + " has the wrong dtype");
    if (d->ndim != ndim) return fail(HMC_INVALID, std::string(what) + " needs " + std::to_string(ndim) + " dimensions");
    bool empty = false;
    for (int k = 0; k < ndim; ++k) {
        if (d->sizes[k] != sizes[k]) return fail(HMC_INVALID, std::string(what) + " has the wrong sizes");
        empty = empty || d->sizes[k] == 0;
    }
    if (empty) return HMC_OK;
    int64_t reach = d->offset;
    for (int k = 0; k < ndim; ++k) {
        int64_t step = 0;
        if (__builtin_mul_overflow(d->sizes[k] - 1, d->strides[k], &step) || __builtin_add_overflow(reach, step, &reach)) {
            return fail(HMC_INVALID, std::string(what) + " reaches beyond 63 bits");
        }
        if (use == Use::kOutput && d->sizes[k] > 1 && d->strides[k] == 0) {
            return fail(HMC_INVALID, std::string("the elements of ") + what + " are not distinct");
        }
    }
    if (reach > INT64_MAX / 16) return fail(HMC_INVALID, std::string(what) + " reaches beyond 63 bits");
    if (d->data == nullptr) return fail(HMC_INVALID, "null data pointer");
    return HMC_OK;
}

// The number of elements of three sizes, or an error when it needs more than 62 bits.
inline hmc_status count_layer(const int64_t *sizes, int ndim, int64_t *count) {
    int64_t n = 1;
    for (int k = 0; k < ndim; ++k) {
        if (sizes[k] == 0) {
            *count = 0;
            return HMC_OK;
        }
    }
    for (int k = 0; k < ndim; ++k) {
        if (__builtin_mul_overflow(n, sizes[k], &n) || n > (INT64_MAX >> 1)) return fail(HMC_INVALID, "the number of elements overflows 62 bits");
    }
    *count = n;
    return HMC_OK;
}

inline char *layer_base(const hmc_tensor_desc *d) {
    return d == nullptr ? nullptr : static_cast<char *>(d->data) + d->offset * element_size(d->dtype);
}

// Whether vectors of `bytes` bytes along the last dimension (of stride 1) are aligned at every position of the others.
inline bool layer_vectors(const hmc_tensor_desc *d, int bytes) {
    if (d == nullptr) return true;
    const int es = element_size(d->dtype);
    const int last = d->ndim - 1;
    if (d->sizes[last] * es % bytes != 0 || (d->strides[last] != 1 && d->sizes[last] != 1)) return false;
    if (reinterpret_cast<uintptr_t>(layer_base(d)) % bytes != 0) return false;
    for (int k = 0; k < last; ++k) {
        if (d->sizes[k] > 1 && d->strides[k] * es % bytes != 0) return false;
    }
    return true;
}

// Lets a kernel use `bytes` of dynamic shared memory, once a device; `known` belongs to the kernel. (Static and dynamic
// parts together need no asking up to 48 KB; no kernel here has 32 KB of the former. Threads that come at the same time repeat
// the call.)
struct SharedKnown {
    static constexpr int kDevices = 64;
    std::atomic<bool> allowed[kDevices] = {};
};
template <class Kernel> inline hmc_status allow_shared(hmc_context_t ctx, Kernel kernel, SharedKnown &known, int bytes, const char *what) {
    if (bytes <= 16384) return HMC_OK;
    const bool kept = ctx->device < SharedKnown::kDevices;
    if (kept && known.allowed[ctx->device].load(std::memory_order_relaxed)) return HMC_OK;
    HMC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what);
    if (kept) known.allowed[ctx->device].store(true, std::memory_order_relaxed);
    return HMC_OK;
}

}  // namespace hmc
