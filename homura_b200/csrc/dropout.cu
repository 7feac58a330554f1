// Dropout from the counter-based generator (include/homura_cuda_layers.h): the mask of element i is a word of a Philox
// block named by i alone, so it is recomputed where the gradient needs it and never stored.
//
// A thread takes two Philox blocks, eight neighbouring elements, with one vector access per operand. Ten rounds of two
// wide multiplications per four elements are about 15 integer operations an element beside 4 (bf16, no residual) to 12
// bytes of traffic.
#include <cmath>

#include "layers.cuh"
#include "math.cuh"
#include "philox.cuh"

namespace hmc {
namespace {

constexpr int kDropThreads = 256;
constexpr int kPer = 8;  // elements a thread takes: two Philox blocks

template <class C> struct DropRule {
    uint64_t seed, offset;
    uint32_t threshold;  // a word below it drops its element
    bool all;            // every element is dropped (p rounds to 1)
    C scale;
};

template <class T, bool RES>
__device__ __forceinline__ typename Comp<T>::C drop(uint32_t word, T x, T residual, const DropRule<typename Comp<T>::C> &rule) {
    using C = typename Comp<T>::C;
    const bool keep = word >= rule.threshold && !rule.all;
    // (selected, not multiplied by 0: a dropped NaN or infinity leaves nothing)
    if constexpr (RES) {
        const C r = up(residual);
        return keep ? m_fma(up(x), rule.scale, r) : r;
    } else {
        return keep ? up(x) * rule.scale : C(0);
    }
}

template <class T, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_flat_kernel(T *out, const T *src, const T *residual, int64_t n, bool vectors,
                                                                    const DropRule<typename Comp<T>::C> rule) {
    using C = typename Comp<T>::C;
    const int64_t pieces = (n + kPer - 1) / kPer;
    for (int64_t piece = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; piece < pieces;
         piece += static_cast<int64_t>(gridDim.x) * kDropThreads) {
        const int64_t i0 = piece * kPer;
        const bool whole = vectors && i0 + kPer <= n;
        Pack<T, kPer> x, r, y;
        if (whole) {
            vector_load<T, kPer>(x, src + i0, false);
            if constexpr (RES) vector_load<T, kPer>(r, residual + i0, false);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) {
                if (i0 + j < n) {
                    x.v[j] = src[i0 + j];
                    if constexpr (RES) r.v[j] = residual[i0 + j];
                }
            }
        }
        C v[kPer];
#pragma unroll
        for (int b = 0; b < kPer / 4; ++b) {
            const Words4 w = philox_block(rule.offset + static_cast<uint64_t>(piece) * (kPer / 4) + b, rule.seed);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[4 * b + j] = drop<T, RES>(w.w[j], x.v[4 * b + j], r.v[4 * b + j], rule);
        }
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int j = 0; j < kPer; j += 2) down2(y.v[j], y.v[j + 1], v[j], v[j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j) y.v[j] = down<T>(v[j]);
        }
        if (whole) {
            vector_store<T, kPer>(out + i0, y, false);
        } else {
#pragma unroll
            for (int j = 0; j < kPer; ++j)
                if (i0 + j < n) out[i0 + j] = y.v[j];
        }
    }
}

// Any strides: a thread takes one Philox block, four neighbours in row-major order.
struct StridedArgs {
    char *base[3];  // out, src, residual
    int32_t ndim;
    int64_t n;
    int64_t sizes[HMC_MAX_DIMS];
    int64_t strides[3][HMC_MAX_DIMS];
};

template <class T, bool RES>
__global__ void __launch_bounds__(kDropThreads) dropout_strided_kernel(const __grid_constant__ StridedArgs a,
                                                                       const DropRule<typename Comp<T>::C> rule) {
    T *out = reinterpret_cast<T *>(a.base[0]);
    const T *src = reinterpret_cast<const T *>(a.base[1]);
    const T *residual = reinterpret_cast<const T *>(a.base[2]);
    const int64_t blocks = (a.n + 3) / 4;
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; b < blocks;
         b += static_cast<int64_t>(gridDim.x) * kDropThreads) {
        const Words4 w = philox_block(rule.offset + static_cast<uint64_t>(b), rule.seed);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            int64_t rest = 4 * b + j;
            if (rest >= a.n) break;
            int64_t oo = 0, so = 0, ro = 0;
            for (int d = a.ndim - 1; d >= 0; --d) {
                const int64_t q = rest / a.sizes[d];
                const int64_t i = rest - q * a.sizes[d];
                oo += i * a.strides[0][d];
                so += i * a.strides[1][d];
                if constexpr (RES) ro += i * a.strides[2][d];
                rest = q;
            }
            out[oo] = down<T>(drop<T, RES>(w.w[j], src[so], RES ? residual[ro] : T{}, rule));
        }
    }
}

}  // namespace
}  // namespace hmc

using namespace hmc;

HMC_API hmc_status hmc_dropout(hmc_context_t ctx, const hmc_tensor_desc *out, const hmc_tensor_desc *src,
                               const hmc_tensor_desc *residual, double p, uint64_t seed, uint64_t offset) {
    return guarded([&]() -> hmc_status {
        hmc_status s = check_desc(src, "the input");
        if (s != HMC_OK) return s;
        if (!dtype_is_float(src->dtype)) return fail(HMC_INVALID, "dropout needs floating point tensors");
        if (!(p >= 0.0 && p <= 1.0)) return fail(HMC_INVALID, "dropout needs a probability between 0 and 1");
        s = check_layer(src, "the input", src->dtype, src->ndim, src->sizes, Use::kInput);
        if (s == HMC_OK) s = check_layer(out, "the output", src->dtype, src->ndim, src->sizes, Use::kOutput);
        if (s == HMC_OK && residual != nullptr) s = check_layer(residual, "the residual", src->dtype, src->ndim, src->sizes, Use::kInput);
        int64_t n = 0;
        if (s == HMC_OK) s = count_layer(src->sizes, src->ndim, &n);
        if (s != HMC_OK) return s;
        HMC_ENTER(ctx);
        if (n == 0) return HMC_OK;
        const double threshold = std::nearbyint(p * 4294967296.0);
        const bool all = threshold >= 4294967296.0;
        const int dims = src->ndim;
        auto flat = [&](const hmc_tensor_desc *d) {
            return d == nullptr || dims == 0 || (dims == 1 && (d->strides[0] == 1 || d->sizes[0] == 1));
        };
        const bool is_flat = flat(out) && flat(src) && flat(residual);
        auto aligned = [&](const hmc_tensor_desc *d) { return reinterpret_cast<uintptr_t>(layer_base(d)) % 16 == 0; };
        const bool vectors = aligned(out) && aligned(src) && (residual == nullptr || aligned(residual));
        const int64_t pieces = ceil_div(n, is_flat ? kPer : 4);
        const int64_t blocks = ceil_div(pieces, kDropThreads);
        const unsigned grid = static_cast<unsigned>(blocks < (int64_t{1} << 30) ? blocks : (int64_t{1} << 30));
        return dispatch_float(src->dtype, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            using C = typename Comp<T>::C;
            const DropRule<C> rule{seed, offset, all ? 0u : static_cast<uint32_t>(threshold), all, all ? C(0) : static_cast<C>(1.0 / (1.0 - p))};
            if (is_flat) {
                T *o = reinterpret_cast<T *>(layer_base(out));
                const T *x = reinterpret_cast<const T *>(layer_base(src)), *r = reinterpret_cast<const T *>(layer_base(residual));
                if (r != nullptr) dropout_flat_kernel<T, true><<<grid, kDropThreads, 0, ctx->stream>>>(o, x, r, n, vectors, rule);
                else dropout_flat_kernel<T, false><<<grid, kDropThreads, 0, ctx->stream>>>(o, x, r, n, vectors, rule);
            } else {
                StridedArgs a{};
                const hmc_tensor_desc *d[3] = {out, src, residual};
                a.ndim = dims;
                a.n = n;
                for (int k = 0; k < 3; ++k) {
                    a.base[k] = layer_base(d[k]);
                    for (int j = 0; j < dims; ++j) {
                        a.sizes[j] = src->sizes[j];
                        a.strides[k][j] = d[k] != nullptr ? d[k]->strides[j] : 0;
                    }
                }
                if (residual != nullptr) dropout_strided_kernel<T, true><<<grid, kDropThreads, 0, ctx->stream>>>(a, rule);
                else dropout_strided_kernel<T, false><<<grid, kDropThreads, 0, ctx->stream>>>(a, rule);
            }
            return launch_status("dropout kernel launch");
        });
    });
}
