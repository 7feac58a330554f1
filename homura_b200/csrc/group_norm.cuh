// Shared by the forward and the backward kernels of group norm with an activation, channels last
// (include/homura_cuda_layers.h): the activations, the affine parameters, and how a tile of channels lies over the groups.
//
// The tensors are [samples, positions, channels] with unit channel stride, so a row of channels is contiguous and a group is
// a strip of cg = channels / groups columns. A block of 256 threads covers a tile of channels, V neighbouring ones a
// thread (16 bytes where the layout allows), with tx threads along the channels and ty rows at a time. A tile is as many
// whole groups as fit, so that narrow groups share coalesced rows, or a segment of one group that is wider than a tile.
#pragma once

#include "layers.cuh"
#include "math.cuh"

namespace hmc {
namespace gnorm {

constexpr int kBlock = 256;
constexpr int kWarps = kBlock / 32;
constexpr int kBlocksWanted = 148 * 4;  // a constant, not the device's count: the order of folding is the same everywhere

// ---- activations ----

// 1 / (1 + exp(-z)): for f32 by the special function unit, relative error at most (2 |z| + 9) 2^-24.
__device__ __forceinline__ float logistic(float z) { return fast_sigmoid(z); }
__device__ __forceinline__ double logistic(double z) { return 1.0 / (1.0 + exp(-z)); }

// The normal distribution's function, 0.5 erfc(-z / sqrt(2)). For f32 from erfc(x) = t exp(-x^2 + P(t)), t = 1 / (1 + x / 2),
// x >= 0, the Chebyshev fit of Press, Teukolsky, Vetterling and Flannery (Numerical Recipes, "erfcc"): about twenty operations
// without a branch, half of erff's. The fit is good to 1.2e-7 of its value everywhere; the roundings of the exponential's
// argument, which grows as z^2 / 2, add up to 3 z^2 2^-24 for z < 0 (seen: 3e-7 down to z = -1, 9e-7 to -3, 4e-6 to -6, 1e-5 to
// -13, where z times it is 1e-37), which an absolute error of a unit of z never shows. With erfcf and expf in the place of this and
// of density's exponential, the gradients of f32 [16384, 1, 4096] with gelu take 240 us instead of 195 and are off by 1.1e-7
// of their size instead of 1.2e-7: what is left is the f32 arithmetic around them.
__device__ __forceinline__ float normal_cdf(float z) {
    const float x = fabsf(z) * 0.70710678118654752440f;
    float t;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(__fmaf_rn(0.5f, x, 1.0f)));
    float p = 0.17087277f;
    p = __fmaf_rn(p, t, -0.82215223f);
    p = __fmaf_rn(p, t, 1.48851587f);
    p = __fmaf_rn(p, t, -1.13520398f);
    p = __fmaf_rn(p, t, 0.27886807f);
    p = __fmaf_rn(p, t, -0.18628806f);
    p = __fmaf_rn(p, t, 0.09678418f);
    p = __fmaf_rn(p, t, 0.37409196f);
    p = __fmaf_rn(p, t, 1.00002368f);
    p = __fmaf_rn(p, t, -1.26551223f);
    const float half = 0.5f * t * fast_exp(__fmaf_rn(-x, x, p));
    return z > 0.0f ? 1.0f - half : half;  // (a NaN comes through: t, p and half are NaN)
}
__device__ __forceinline__ double normal_cdf(double z) { return 0.5 * erfc(z * -0.70710678118654752440); }
__device__ __forceinline__ float density(float z) { return 0.39894228040143267794f * fast_exp(-0.5f * z * z); }
__device__ __forceinline__ double density(double z) { return 0.39894228040143267794 * exp(-0.5 * z * z); }

template <class C> __device__ __forceinline__ C gelu_inner(C z, C &slope) {
    // 2 u with gelu_tanh(z) = z * sigmoid(2 u), u = sqrt(2 / pi) (z + 0.044715 z^3); slope = 2 du/dz
    const C k = static_cast<C>(1.59576912160573071176), c = static_cast<C>(0.044715);
    const C q = c * z * z;
    slope = k * m_fma(C(3), q, C(1));
    return k * z * (C(1) + q);
}

// z between -64 and 64, a NaN passed on.
__device__ __forceinline__ float within_64(float z) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(-64.0f));
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(z) : "f"(64.0f));
    return z;
}
__device__ __forceinline__ double within_64(double z) { return z > 64.0 ? 64.0 : (z < -64.0 ? -64.0 : z); }

// xhat * w + b: in two roundings before relu, whose derivative goes by the sign alone, so that the sign is that of the
// plain formula; fused otherwise. Every forward and backward kernel takes the same steps from x on, (x - mean) * rstd first,
// so that all find the same z: moments and parameters are not folded into one product and sum, which leaves
// mean * rstd * 2^-24 of noise (0.4 for a group of 30000s, whose z is its bias).
template <int ACT, class C> __device__ __forceinline__ C scaled(C xhat, C w, C b) {
    if constexpr (ACT == HMC_UNARY_RELU) return xhat * w + b;
    else return m_fma(xhat, w, b);
}
template <int ACT, class C> __device__ __forceinline__ C activate(C z) {
    if constexpr (ACT == HMC_UNARY_RELU) return (z != z || z > C(0)) ? z : C(0);
    else if constexpr (ACT == HMC_UNARY_SILU) return z * logistic(z);
    else if constexpr (ACT == HMC_UNARY_GELU) return z * normal_cdf(z);
    else if constexpr (ACT == HMC_UNARY_GELU_TANH) {
        C slope;
        return z * logistic(gelu_inner(z, slope));
    } else return z;
}
// d * act'(z)
template <int ACT, class C> __device__ __forceinline__ C through(C d, C z) {
    if constexpr (ACT == HMC_UNARY_RELU) return z > C(0) ? d : (z != z ? z : C(0));
    else if constexpr (ACT == HMC_UNARY_SILU) {
        const C s = logistic(z);
        return d * (s * m_fma(z, C(1) - s, C(1)));
    } else if constexpr (ACT == HMC_UNARY_GELU) {
        return d * m_fma(z, density(z), normal_cdf(z));
    } else if constexpr (ACT == HMC_UNARY_GELU_TANH) {
        // (beyond 64 s is 0 or 1 to the last bit, but the inner slope and its product with z overflow in the end: held there)
        C slope;
        const C held = within_64(z), s = logistic(gelu_inner(held, slope));
        return d * (s * m_fma(held * (C(1) - s), slope, C(1)));
    } else return d;
}

// 1 / sqrt(v): f32 to two units in the last place.
__device__ __forceinline__ float inverse_root(float v) { return rsqrtf(v); }
__device__ __forceinline__ double inverse_root(double v) { return 1.0 / sqrt(v); }

// sum / count from share = 1 / count rounded: the product with share is off by up to an ulp and a half where count is no
// power of two, and one step of Newton's method on it gives every quotient that the type holds, so that the mean of a constant
// group is its value. What is no finite number keeps the product.
template <class C> __device__ __forceinline__ C quotient(C sum, C count, C share) {
    const C q = sum * share, rest = m_fma(-q, count, sum);
    return rest == rest ? m_fma(rest, share, q) : q;
}

// ---- operands ----

// weight and bias, or null; of T or of f32.
struct Affine {
    const char *weight, *bias;
    int64_t weight_stride, bias_stride;
    int32_t is_f32;
};
template <class T> __device__ __forceinline__ typename Comp<T>::C parameter(const char *p, int64_t at, int is_f32) {
    using C = typename Comp<T>::C;
    if (is_f32) return static_cast<C>(reinterpret_cast<const float *>(p)[at]);
    return up(reinterpret_cast<const T *>(p)[at]);
}

struct Rows {
    int64_t n, s;  // strides of samples and positions, in elements
};

template <class C> struct alignas(2 * sizeof(C)) Two {
    C a, b;
};

template <int BYTES> __device__ __forceinline__ void copy_async(void *shared_dst, const void *src) {
    if constexpr (BYTES == 16) async_copy_16(shared_dst, src);
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared_dst))), "l"(src), "n"(BYTES) : "memory");
}

// ---- tiles ----

struct Tiling {
    int64_t channels, groups, cg;   // cg channels a group
    int32_t v;                      // channels a thread
    int32_t tile;                   // channels a tile
    int32_t tx, ty;                 // threads along channels, rows at a time
    int32_t groups_per_tile;        // 1 when a group has several segments
    int32_t segments;               // segments a group
    int64_t tiles;
};

inline Tiling make_tiling(int64_t channels, int64_t groups, int vector, bool vectors) {
    Tiling t{};
    t.channels = channels;
    t.groups = groups;
    t.cg = channels / groups;
    const auto gcd = [](int64_t a, int64_t b) {
        while (b != 0) {
            const int64_t r = a % b;
            a = b;
            b = r;
        }
        return a;
    };
    for (int v = vectors ? vector : 1;; v = 1) {
        const int64_t widest = static_cast<int64_t>(kBlock) * v;
        const int64_t unit = v / gcd(t.cg, v);  // groups after which the channel is a multiple of v again
        t.v = v;
        if (unit * t.cg <= widest) {
            int64_t per = widest / t.cg / unit * unit;
            if (per > groups) per = groups;  // (then the tile is the whole row, a multiple of v)
            t.groups_per_tile = static_cast<int32_t>(per);
            t.segments = 1;
            t.tile = static_cast<int32_t>(per * t.cg);
            t.tiles = ceil_div(groups, per);
            break;
        }
        if (unit == 1) {
            t.groups_per_tile = 1;
            t.segments = static_cast<int32_t>(ceil_div(t.cg, widest));
            t.tile = static_cast<int32_t>(widest);
            t.tiles = groups * t.segments;
            break;
        }
    }
    t.tx = static_cast<int32_t>(ceil_div(t.tile, t.v));
    t.ty = kBlock / t.tx;
    return t;
}

// One tile: its first channel and group, its width, and what part of each of its groups it holds.
struct Tile {
    int64_t channel, group;
    int width, groups;     // channels and (parts of) groups in it
    int part;              // channels of a group in it
    int segment;
};
__device__ __forceinline__ Tile tile_at(const Tiling &t, int64_t index) {
    Tile r;
    if (t.segments == 1) {
        r.group = index * t.groups_per_tile;
        r.groups = static_cast<int>(t.groups - r.group < t.groups_per_tile ? t.groups - r.group : t.groups_per_tile);
        r.channel = r.group * t.cg;
        r.part = static_cast<int>(t.cg);
        r.width = r.groups * r.part;
        r.segment = 0;
    } else {
        r.group = index / t.segments;
        r.segment = static_cast<int>(index - r.group * t.segments);
        r.groups = 1;
        r.channel = r.group * t.cg + static_cast<int64_t>(r.segment) * t.tile;
        const int64_t rest = t.cg - static_cast<int64_t>(r.segment) * t.tile;
        r.part = r.width = static_cast<int>(rest < t.tile ? rest : t.tile);
    }
    return r;
}

// Sums of the block's columns by group: `columns` holds ty rows of tile.width values, done(group, sum) is called once for
// each group of the tile, by one thread, always adding in the same order. A thread a group where a group has few
// values, otherwise a warp.
template <class S, class F> __device__ __forceinline__ void by_group(const S *columns, const Tile &tile, int ty, F &&done) {
    const int values = tile.part * ty;
    if (values <= 64) {
        for (int q = threadIdx.x; q < tile.groups; q += kBlock) {
            S sum = S(0);
            for (int y = 0; y < ty; ++y)
                for (int c = 0; c < tile.part; ++c) sum += columns[y * tile.width + q * tile.part + c];
            done(q, sum);
        }
    } else {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        for (int q = warp; q < tile.groups; q += kWarps) {
            S sum = S(0);
            for (int y = 0; y < ty; ++y)
                for (int c = lane; c < tile.part; c += 32) sum += columns[y * tile.width + q * tile.part + c];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
            if (lane == 0) done(q, sum);
        }
    }
}

// ---- checks of the entry points ----

struct Problem {
    int64_t samples, positions, channels, groups;
    int dtype, stat_dtype;
};
inline hmc_status check_problem(const hmc_tensor_desc *src, int32_t groups, Problem *out) {
    hmc_status s = check_desc(src, "the input");
    if (s != HMC_OK) return s;
    if (!dtype_is_float(src->dtype)) return fail(HMC_INVALID, "group norm needs floating point tensors");
    s = check_layer(src, "the input", src->dtype, 3, src->sizes, Use::kInput);
    if (s != HMC_OK) return s;
    if (groups <= 0 || src->sizes[2] % groups != 0) return fail(HMC_INVALID, "the channels do not divide into the groups");
    int64_t n = 0;
    s = count_layer(src->sizes, 3, &n);
    if (s != HMC_OK) return s;
    // (workspaces hold at most some tens of bytes an element: their sizes stay within 63 bits)
    if (n > (int64_t{1} << 56)) return fail(HMC_INVALID, "the tensor has too many elements");
    const int64_t stats[2] = {src->sizes[0], groups};
    s = count_layer(stats, 2, &n);
    if (s != HMC_OK) return s;
    *out = Problem{src->sizes[0], src->sizes[1], src->sizes[2], groups, src->dtype, src->dtype == HMC_F64 ? HMC_F64 : HMC_F32};
    return HMC_OK;
}
inline hmc_status check_channels_last(const hmc_tensor_desc *d, const char *what) {
    if (d->sizes[2] > 1 && d->strides[2] != 1) return fail(HMC_INVALID, std::string(what) + " is not channels last: its channels are not neighbours");
    return HMC_OK;
}
inline hmc_status check_affine(const hmc_tensor_desc *weight, const hmc_tensor_desc *bias, const Problem &p, Affine *out) {
    *out = Affine{};
    if ((weight == nullptr) != (bias == nullptr)) return fail(HMC_INVALID, "group norm takes both weight and bias or neither");
    if (weight == nullptr) return HMC_OK;
    hmc_status s = check_desc(weight, "the weight");
    if (s != HMC_OK) return s;
    if (weight->dtype != p.dtype && weight->dtype != HMC_F32) return fail(HMC_INVALID, "the weight has neither the input's dtype nor F32");
    s = check_layer(weight, "the weight", weight->dtype, 1, &p.channels, Use::kInput);
    if (s == HMC_OK) s = check_layer(bias, "the bias", weight->dtype, 1, &p.channels, Use::kInput);
    if (s != HMC_OK) return s;
    *out = Affine{layer_base(weight), layer_base(bias), weight->strides[0], bias->strides[0], weight->dtype == HMC_F32 ? 1 : 0};
    return HMC_OK;
}
inline hmc_status check_stats(const hmc_tensor_desc *mean, const hmc_tensor_desc *rstd, const Problem &p, Use use) {
    if ((mean == nullptr) != (rstd == nullptr)) return fail(HMC_INVALID, "group norm takes both mean and rstd or neither");
    if (mean == nullptr) return HMC_OK;
    const int64_t sizes[2] = {p.samples, p.groups};
    hmc_status s = check_layer(mean, "the mean", p.stat_dtype, 2, sizes, use);
    if (s == HMC_OK) s = check_layer(rstd, "the rstd", p.stat_dtype, 2, sizes, use);
    return s;
}
inline hmc_status check_activation(int32_t activation) {
    switch (activation) {
        case HMC_ACTIVATION_NONE: case HMC_UNARY_RELU: case HMC_UNARY_SILU: case HMC_UNARY_GELU: case HMC_UNARY_GELU_TANH: return HMC_OK;
        default: return fail(HMC_INVALID, "group norm's activation is none, relu, silu, gelu or gelu_tanh");
    }
}
inline hmc_status check_workspace(int64_t need, const void *workspace, int64_t bytes) {
    if (need == 0) return HMC_OK;
    if (workspace == nullptr || bytes < need) {
        return fail(HMC_INVALID, "the workspace has " + std::to_string(workspace == nullptr ? 0 : bytes) + " bytes, group norm needs " + std::to_string(need));
    }
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0) return fail(HMC_INVALID, "the workspace is not 16-byte aligned");
    return HMC_OK;
}
template <class F> inline hmc_status dispatch_activation(int32_t activation, F &&f) {
    switch (activation) {
        case HMC_UNARY_RELU: return f(std::integral_constant<int, HMC_UNARY_RELU>{});
        case HMC_UNARY_SILU: return f(std::integral_constant<int, HMC_UNARY_SILU>{});
        case HMC_UNARY_GELU: return f(std::integral_constant<int, HMC_UNARY_GELU>{});
        case HMC_UNARY_GELU_TANH: return f(std::integral_constant<int, HMC_UNARY_GELU_TANH>{});
        default: return f(std::integral_constant<int, HMC_ACTIVATION_NONE>{});
    }
}
// How regular the operands are: vectors of 16 bytes, words of 4, or neither.
enum class Align { kAny, kWord, kLine };
template <class... D> inline Align alignment(int dtype, const D *...d) {
    if ((layer_vectors(d, 16) && ...)) return Align::kLine;
    return element_size(dtype) >= 4 || (layer_vectors(d, 4) && ...) ? Align::kWord : Align::kAny;
}
constexpr int narrow_vector(int es) { return es == 2 ? 2 : 1; }  // elements of a word
template <class T> constexpr int kVector = 16 / static_cast<int>(sizeof(T));

inline unsigned grid_for(int64_t blocks) { return static_cast<unsigned>(blocks < (int64_t{1} << 30) ? blocks : (int64_t{1} << 30)); }

// Work over rows: every (sample, tile) is cut into `chunks` runs of `run` positions, multiples of `step` rows.
struct Cut {
    int64_t run, chunks, units;
};
inline Cut cut_rows(const Problem &p, const Tiling &t, int64_t step) {
    const int64_t strips = p.samples * t.tiles;
    int64_t want = ceil_div(kBlocksWanted, strips);
    const int64_t most = ceil_div(p.positions, step);
    if (want > most) want = most;
    Cut c;
    c.run = ceil_div(ceil_div(p.positions, want), step) * step;
    c.chunks = ceil_div(p.positions, c.run);
    c.units = strips * c.chunks;
    return c;
}

}  // namespace gnorm
}  // namespace hmc
