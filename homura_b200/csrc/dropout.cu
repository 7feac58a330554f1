// Dropout from the counter-based generator (include/homura_cuda_layers.h): the mask of element i is a word of a Philox
// block named by i alone, so it is recomputed where the gradient needs it and never stored.
//
// A thread takes two Philox blocks, eight neighbouring elements, at a time. Ten rounds of two wide multiplications and two
// three-way exclusive ors per four elements are ten integer operations an element beside 4 (bf16, no residual) to 12 bytes
// of traffic: arithmetic and memory bind alike.
#include <cmath>

#include "layers.cuh"
#include "math.cuh"
#include "philox.cuh"

namespace hmc {
namespace {

constexpr int kDropThreads = 256;
constexpr int kPer = 8;     // neighbouring elements a thread takes at a time: two Philox blocks
template <class C> struct DropRule {
    PhiloxKeys keys;
    uint64_t offset;
    uint32_t above;  // a word above it keeps its element
    C scale;
};

// RNG: false where nothing is dropped.
template <class T, bool RES, bool RNG>
__device__ __forceinline__ typename Comp<T>::C drop(uint32_t word, T x, T residual, const DropRule<typename Comp<T>::C> &rule) {
    using C = typename Comp<T>::C;
    const bool keep = !RNG || word > rule.above;
    // (selected, not multiplied by 0: a dropped NaN or infinity leaves nothing)
    if constexpr (RES) {
        const C r = up(residual);
        return keep ? m_fma(up(x), rule.scale, r) : r;
    } else {
        return keep ? up(x) * rule.scale : C(0);
    }
}

// Eight neighbours from their two Philox blocks, the first of which is offset + 2 * piece. SAME: the upper half of all block
// numbers is the one the keys were made for; then a block's first product is its neighbour's and a sum.
template <class T, bool RES, bool RNG, bool SAME>
__device__ __forceinline__ Pack<T, kPer> drop_piece(int64_t piece, const Pack<T, kPer> &x, const Pack<T, kPer> &r,
                                                    const DropRule<typename Comp<T>::C> &rule) {
    using C = typename Comp<T>::C;
    C v[kPer];
    const uint64_t block = rule.offset + static_cast<uint64_t>(piece) * (kPer / 4);
    const uint64_t product = static_cast<uint64_t>(kPhiloxM0) * static_cast<uint32_t>(block);
#pragma unroll
    for (int b = 0; b < kPer / 4; ++b) {
        Words4 w{};
        if constexpr (RNG) w = SAME ? philox_block_same_high(product + static_cast<uint64_t>(b) * kPhiloxM0, rule.keys) : philox_block(block + b, rule.keys);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * b + j] = drop<T, RES, RNG>(w.w[j], x.v[4 * b + j], r.v[4 * b + j], rule);
    }
    Pack<T, kPer> y;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < kPer; j += 2) down2(y.v[j], y.v[j + 1], v[j], v[j + 1]);
    } else {
#pragma unroll
        for (int j = 0; j < kPer; ++j) y.v[j] = down<T>(v[j]);
    }
    return y;
}

// What is left of a piece element by element: the last one, or all where an operand does not start on 16 bytes or the block
// numbers pass a multiple of 2^32.
template <class T, bool RES, bool RNG>
__device__ __forceinline__ void drop_ragged(T *out, const T *src, const T *residual, int64_t n, int64_t piece, const DropRule<typename Comp<T>::C> &rule) {
    Pack<T, kPer> x, r;
    const int64_t i0 = piece * kPer;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        if (i0 + j < n) {
            x.v[j] = src[i0 + j];
            if constexpr (RES) r.v[j] = residual[i0 + j];
        }
    }
    const Pack<T, kPer> y = drop_piece<T, RES, RNG, false>(piece, x, r, rule);
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (i0 + j < n) out[i0 + j] = y.v[j];
}
template <class T, bool RES, bool RNG>
__global__ void __launch_bounds__(kDropThreads) dropout_ragged_kernel(T *out, const T *src, const T *residual, int64_t n,
                                                                      const __grid_constant__ DropRule<typename Comp<T>::C> rule) {
    const int64_t pieces = (n + kPer - 1) / kPer;
    for (int64_t piece = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; piece < pieces;
         piece += static_cast<int64_t>(gridDim.x) * kDropThreads) {
        drop_ragged<T, RES, RNG>(out, src, residual, n, piece, rule);
    }
}

// Contiguous operands on 16-byte boundaries, block numbers that agree in their upper half: a resident grid walks the pieces, and a thread's next pieces come through a
// ring in shared memory that its own asynchronous copies fill while it works out the present one's words: the rounds of the
// generator and the memory's latency overlap without a register spent on data in flight.
template <class T, bool RES> struct DropRing {
    static constexpr int kWords = kPer * static_cast<int>(sizeof(T)) / 16;          // copies an operand and piece
    static constexpr int kPiece = (RES ? 2 : 1) * kWords * kDropThreads * 16;       // bytes a block and piece
    static constexpr int kStages = kPiece <= 8192 ? 4 : (kPiece <= 16384 ? 3 : 2);  // the one being worked on among them
    static constexpr int kBytes = kStages * kPiece;                                 // (64 KB at most: F64 with a residual)
};

template <class T, bool RES, bool RNG>
__global__ void __launch_bounds__(kDropThreads, sizeof(T) == 8 ? 2 : 4) dropout_flat_kernel(T *out, const T *src, const T *residual, int64_t n,
                                                                                          const __grid_constant__ DropRule<typename Comp<T>::C> rule) {
    using G = DropRing<T, RES>;
    extern __shared__ __align__(16) unsigned char ring[];
    const int64_t pieces = (n + kPer - 1) / kPer, whole = n / kPer, stride = static_cast<int64_t>(gridDim.x) * kDropThreads;
    unsigned char *mine = ring + threadIdx.x * 16;  // this thread's copies, kDropThreads * 16 bytes apart
    const auto fetch = [&](int64_t piece, int stage) {
        if (piece < whole) {
#pragma unroll
            for (int w = 0; w < G::kWords; ++w) {
                async_copy_16(mine + stage * G::kPiece + w * (kDropThreads * 16), reinterpret_cast<const char *>(src + piece * kPer) + 16 * w);
                if constexpr (RES) {
                    async_copy_16(mine + stage * G::kPiece + (G::kWords + w) * (kDropThreads * 16),
                                  reinterpret_cast<const char *>(residual + piece * kPer) + 16 * w);
                }
            }
        }
        async_copy_commit();
    };
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x;
#pragma unroll
    for (int k = 0; k + 1 < G::kStages; ++k) fetch(first + k * stride, k);
    int stage = 0;
    for (int64_t piece = first; piece < pieces; piece += stride) {
        fetch(piece + (G::kStages - 1) * stride, stage == 0 ? G::kStages - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(G::kStages - 1) : "memory");
        if (piece < whole) {
            Pack<T, kPer> x, r;
#pragma unroll
            for (int w = 0; w < G::kWords; ++w) {
                memcpy(reinterpret_cast<char *>(&x) + 16 * w, mine + stage * G::kPiece + w * (kDropThreads * 16), 16);
                if constexpr (RES) memcpy(reinterpret_cast<char *>(&r) + 16 * w, mine + stage * G::kPiece + (G::kWords + w) * (kDropThreads * 16), 16);
            }
            vector_store<T, kPer>(out + piece * kPer, drop_piece<T, RES, RNG, true>(piece, x, r, rule), false);
        } else {
            drop_ragged<T, RES, RNG>(out, src, residual, n, piece, rule);
        }
        stage = stage + 1 == G::kStages ? 0 : stage + 1;
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

template <class T, bool RES, bool RNG>
__global__ void __launch_bounds__(kDropThreads) dropout_strided_kernel(const __grid_constant__ StridedArgs a,
                                                                       const __grid_constant__ DropRule<typename Comp<T>::C> rule) {
    T *out = reinterpret_cast<T *>(a.base[0]);
    const T *src = reinterpret_cast<const T *>(a.base[1]);
    const T *residual = reinterpret_cast<const T *>(a.base[2]);
    const int64_t blocks = (a.n + 3) / 4;
    for (int64_t b = static_cast<int64_t>(blockIdx.x) * kDropThreads + threadIdx.x; b < blocks;
         b += static_cast<int64_t>(gridDim.x) * kDropThreads) {
        const Words4 w = philox_block(rule.offset + static_cast<uint64_t>(b), rule.keys);
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
            out[oo] = down<T>(drop<T, RES, RNG>(w.w[j], src[so], RES ? residual[ro] : T{}, rule));
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
        const double threshold = std::nearbyint(p * 4294967296.0);  // words below it drop their element
        const bool none = threshold < 1.0, all = threshold >= 4294967296.0;
        const int dims = src->ndim;
        auto flat = [&](const hmc_tensor_desc *d) {
            return d == nullptr || dims == 0 || (dims == 1 && (d->strides[0] == 1 || d->sizes[0] == 1));
        };
        const bool is_flat = flat(out) && flat(src) && flat(residual);
        auto aligned = [&](const hmc_tensor_desc *d) { return reinterpret_cast<uintptr_t>(layer_base(d)) % 16 == 0; };
        const bool vectors = aligned(out) && aligned(src) && (residual == nullptr || aligned(residual));
        const uint64_t last_block = offset + (static_cast<uint64_t>(n) - 1) / 4;
        const bool same_high = last_block >> 32 == offset >> 32;
        const int64_t pieces = ceil_div(n, is_flat ? kPer : 4);
        const int64_t blocks = ceil_div(pieces, kDropThreads);
        const unsigned grid = static_cast<unsigned>(blocks < (int64_t{1} << 30) ? blocks : (int64_t{1} << 30));
        return dispatch_float(src->dtype, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            using C = typename Comp<T>::C;
            const DropRule<C> rule{philox_keys(seed, static_cast<uint32_t>(offset >> 32)), offset, none ? 0u : (all ? 0xFFFFFFFFu : static_cast<uint32_t>(threshold) - 1u),
                                   all ? C(0) : static_cast<C>(1.0 / (1.0 - p))};
            const auto launch = [&](auto with_residual, auto with_words) -> hmc_status {
                constexpr bool RES = decltype(with_residual)::value, RNG = decltype(with_words)::value;
                if (is_flat) {
                    T *o = reinterpret_cast<T *>(layer_base(out));
                    const T *x = reinterpret_cast<const T *>(layer_base(src)), *r = reinterpret_cast<const T *>(layer_base(residual));
                    if (vectors && same_high) {
                        using G = DropRing<T, RES>;
                        static SharedKnown known;
                        const hmc_status allowed = allow_shared(ctx, dropout_flat_kernel<T, RES, RNG>, known, G::kBytes, "shared memory size of the dropout kernel");
                        if (allowed != HMC_OK) return allowed;
                        const int64_t resident = static_cast<int64_t>(ctx->sm_count) * (sizeof(T) == 8 ? 2 : 4);
                        const unsigned flat_grid = static_cast<unsigned>(blocks < resident ? blocks : resident);
                        dropout_flat_kernel<T, RES, RNG><<<flat_grid, kDropThreads, G::kBytes, ctx->stream>>>(o, x, r, n, rule);
                    } else {
                        dropout_ragged_kernel<T, RES, RNG><<<grid, kDropThreads, 0, ctx->stream>>>(o, x, r, n, rule);
                    }
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
                    dropout_strided_kernel<T, RES, RNG><<<grid, kDropThreads, 0, ctx->stream>>>(a, rule);
                }
                return launch_status("dropout kernel launch");
            };
            using Yes = std::true_type;
            using No = std::false_type;
            if (residual != nullptr) return none ? launch(Yes{}, No{}) : launch(Yes{}, Yes{});
            return none ? launch(No{}, No{}) : launch(No{}, Yes{});
        });
    });
}
