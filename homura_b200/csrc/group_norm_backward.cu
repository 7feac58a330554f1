// Group norm with an activation, channels last, the gradients (include/homura_cuda_layers.h); tiles as in group_norm.cuh.
//
// Three steps: sums over each run of rows of dz and dz * xhat (by channel for weight and bias, by group, weighted, for
// the input), a small kernel that folds the runs in order, and an elementwise pass. A thread adds at most 64 rows of a
// run in the computation type. Channel sums are kept in f64 across the runs a block takes, and folded over the blocks in f64.
#include <algorithm>

#include "group_norm_resident.cuh"

namespace hmc {
namespace gnorm {
namespace {

// Rows that a thread adds in the computation type before the sums go on in f64: within a run where it has up to kNarrow channels,
// by shorter runs where the f64 sums of more would not find registers beside them (f16 [700, 300, 515] in 1 group: 1015 us with
// runs of 300 rows, 1124 with runs of 64).
constexpr int kLongest = 64, kNarrow = 2;

struct GradArgs {
    char *dsrc, *dweight, *dbias;  // dweight, dbias: or null
    const char *src, *dout, *mean, *rstd;
    Rows wdsrc, wsrc, wdout;
    int64_t mean_n, mean_g, rstd_n, rstd_g, dweight_stride, dbias_stride;
    int32_t dparam_f32;
    Tiling t;
    Cut cut;              // of the sums
    int64_t columns;      // blocks that share a tile of channels
    Cut apply;
    int64_t positions, samples;
    Affine affine;
    void *pieces;         // Two<C> [samples][groups][chunks * segments]
    void *means;          // Two<C> [samples][groups]: the means of p and of p * xhat
    void *by_channel;     // [columns][2][channels], f64 (C after the one-pass kernel); null when neither dweight nor dbias is wanted
};

// One element: xhat and dz, with the forward pass's steps up to z.
template <int ACT, class C>
__device__ __forceinline__ void element(C x, C dy, C mean, C rstd, C w, C b, C &xhat, C &dz) {
    xhat = (x - mean) * rstd;
    dz = through<ACT>(dy, scaled<ACT>(xhat, w, b));
}

template <class T, int V> struct Coefficients {
    typename Comp<T>::C mean[V], rstd[V], w[V], b[V];
    __device__ __forceinline__ void load(const GradArgs &a, int64_t sample, const Tile &tile, int at) {
        using C = typename Comp<T>::C;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int64_t group = tile.group + (at + i) / tile.part;
            mean[i] = reinterpret_cast<const C *>(a.mean)[sample * a.mean_n + group * a.mean_g];
            rstd[i] = reinterpret_cast<const C *>(a.rstd)[sample * a.rstd_n + group * a.rstd_g];
        }
    }
    __device__ __forceinline__ void load_affine(const GradArgs &a, int64_t channel) {
        using C = typename Comp<T>::C;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = a.affine.weight != nullptr ? parameter<T>(a.affine.weight, (channel + i) * a.affine.weight_stride, a.affine.is_f32) : C(1);
            b[i] = a.affine.weight != nullptr ? parameter<T>(a.affine.bias, (channel + i) * a.affine.bias_stride, a.affine.is_f32) : C(0);
        }
    }
};

// Block b of tile t takes the (sample, chunk) pairs b, b + columns, ... in order.
template <class T, int V, int ACT>
__global__ void __launch_bounds__(kBlock, 2) sums_kernel(const __grid_constant__ GradArgs a) {
    using C = typename Comp<T>::C;
    __shared__ union {
        C by_row[2][kBlock * V];
        double by_column[kBlock * V];
    } shared;
    __shared__ C first[kBlock * V];
    const int tx = threadIdx.x % a.t.tx, ty = threadIdx.x / a.t.tx;
    const int64_t index = blockIdx.x / a.columns, column = blockIdx.x - index * a.columns;
    const Tile tile = tile_at(a.t, index);
    const bool live = tx * V < tile.width && ty < a.t.ty;
    const int64_t channel = tile.channel + tx * V;
    Coefficients<T, V> k;
    if (live) k.load_affine(a, channel);
    double dw[V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = 0.0;
    const int64_t pairs = a.samples * a.cut.chunks;
    const int64_t pieces = a.cut.chunks * a.t.segments;
    for (int64_t pair = column; pair < pairs; pair += a.columns) {
        const int64_t sample = pair / a.cut.chunks, chunk = pair - sample * a.cut.chunks;
        const int64_t begin = chunk * a.cut.run;
        const int64_t end = begin + a.cut.run < a.positions ? begin + a.cut.run : a.positions;
        C s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = C(0);
        if (live) {
            k.load(a, sample, tile, tx * V);
            const T *src = reinterpret_cast<const T *>(a.src) + sample * a.wsrc.n + channel;
            const T *dout = reinterpret_cast<const T *>(a.dout) + sample * a.wdout.n + channel;
            const auto add = [&](int64_t from, int64_t to) {
#pragma unroll 4
                for (int64_t row = from; row < to; row += a.t.ty) {
                    const Pack<T, V> x = *reinterpret_cast<const Pack<T, V> *>(src + row * a.wsrc.s);
                    const Pack<T, V> d = *reinterpret_cast<const Pack<T, V> *>(dout + row * a.wdout.s);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        C xhat, dz;
                        element<ACT>(up(x.v[i]), up(d.v[i]), k.mean[i], k.rstd[i], k.w[i], k.b[i], xhat, dz);
                        s1[i] += dz;
                        s2[i] = m_fma(dz, xhat, s2[i]);
                    }
                }
            };
            if constexpr (V > kNarrow) {
                add(begin + ty, end);
            } else {
                const int64_t longest = static_cast<int64_t>(a.t.ty) * kLongest;
                double t1[V], t2[V];
#pragma unroll
                for (int i = 0; i < V; ++i) t1[i] = t2[i] = 0.0;
                for (int64_t from = begin; from < end; from += longest) {
                    add(from + ty, from + longest < end ? from + longest : end);
                    if (end - begin <= longest) break;
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        t1[i] += static_cast<double>(s1[i]);
                        t2[i] += static_cast<double>(s2[i]);
                        s1[i] = s2[i] = C(0);
                    }
                }
                if (end - begin > longest) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        s1[i] = static_cast<C>(t1[i]);
                        s2[i] = static_cast<C>(t2[i]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < V; ++i) {
                db[i] += static_cast<double>(s1[i]);
                dw[i] += static_cast<double>(s2[i]);
                shared.by_row[0][ty * tile.width + tx * V + i] = s1[i] * k.w[i];
                shared.by_row[1][ty * tile.width + tx * V + i] = s2[i] * k.w[i];
            }
        }
        __syncthreads();
        Two<C> *to = reinterpret_cast<Two<C> *>(pieces == 1 ? a.means : a.pieces) + (sample * a.t.groups + tile.group) * pieces + chunk * a.t.segments + tile.segment;
        const C scale = pieces == 1 ? C(1) / (static_cast<C>(a.positions) * static_cast<C>(a.t.cg)) : C(1);
        by_group(shared.by_row[0], tile, a.t.ty, [&](int q, C s) { first[q] = s; });
        __syncthreads();
        by_group(shared.by_row[1], tile, a.t.ty, [&](int q, C s) { to[q * pieces] = Two<C>{first[q] * scale, s * scale}; });
        __syncthreads();
    }
    if (a.by_channel == nullptr) return;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        if (live) {
#pragma unroll
            for (int i = 0; i < V; ++i) shared.by_column[ty * tile.width + tx * V + i] = which == 0 ? dw[i] : db[i];
        }
        __syncthreads();
        for (int c = threadIdx.x; c < tile.width; c += kBlock) {
            double sum = 0.0;
            for (int y = 0; y < a.t.ty; ++y) sum += shared.by_column[y * tile.width + c];
            reinterpret_cast<double *>(a.by_channel)[(column * 2 + which) * a.t.channels + tile.channel + c] = sum;
        }
        __syncthreads();
    }
}

// A warp folds the pieces of a group: every lane its own in order, then the lanes in a fixed tree.
template <class C> __global__ void __launch_bounds__(kBlock) fold_groups_kernel(const __grid_constant__ GradArgs a, int64_t total) {
    const int lane = threadIdx.x & 31;
    const int64_t pieces = a.cut.chunks * a.t.segments;
    const double count = static_cast<double>(a.positions) * static_cast<double>(a.t.cg);
    for (int64_t g = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); g < total; g += static_cast<int64_t>(gridDim.x) * kWarps) {
        const Two<C> *p = reinterpret_cast<const Two<C> *>(a.pieces) + g * pieces;
        double s = 0.0, t = 0.0;
        for (int64_t k = lane; k < pieces; k += 32) {
            s += static_cast<double>(p[k].a);
            t += static_cast<double>(p[k].b);
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) {
            s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
            t += __shfl_xor_sync(0xFFFFFFFFu, t, d);
        }
        if (lane == 0) reinterpret_cast<Two<C> *>(a.means)[g] = Two<C>{static_cast<C>(s / count), static_cast<C>(t / count)};
    }
}

// dweight and dbias: 32 channels a block, eight warps along the blocks that hold partial sums.
template <class T, class P> __global__ void __launch_bounds__(kBlock) fold_channels_kernel(const __grid_constant__ GradArgs a) {
    __shared__ double part[kWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int which = static_cast<int>(blockIdx.x & 1);
    char *to = which == 0 ? a.dweight : a.dbias;
    if (to == nullptr) return;
    const int64_t stride = which == 0 ? a.dweight_stride : a.dbias_stride;
    for (int64_t block = blockIdx.x >> 1; block * 32 < a.t.channels; block += gridDim.x >> 1) {
        const int64_t channel = block * 32 + lane;
        double sum = 0.0;
        if (channel < a.t.channels) {
            for (int64_t k = warp; k < a.columns; k += kWarps) sum += static_cast<double>(reinterpret_cast<const P *>(a.by_channel)[(k * 2 + which) * a.t.channels + channel]);
        }
        part[warp][lane] = sum;
        __syncthreads();
        if (warp == 0 && channel < a.t.channels) {
            for (int w = 1; w < kWarps; ++w) sum += part[w][lane];
            if (a.dparam_f32) reinterpret_cast<float *>(to)[channel * stride] = static_cast<float>(sum);
            else reinterpret_cast<T *>(to)[channel * stride] = from_f64<T>(sum);
        }
        __syncthreads();
    }
}

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kBlock) grad_kernel(const __grid_constant__ GradArgs a) {
    using C = typename Comp<T>::C;
    const int tx = threadIdx.x % a.t.tx, ty = threadIdx.x / a.t.tx;
    for (int64_t unit = blockIdx.x; unit < a.apply.units; unit += gridDim.x) {
        const int64_t strip = unit / a.apply.chunks, chunk = unit - strip * a.apply.chunks;
        const int64_t sample = strip / a.t.tiles;
        const Tile tile = tile_at(a.t, strip - sample * a.t.tiles);
        if (tx * V >= tile.width || ty >= a.t.ty) continue;
        const int64_t channel = tile.channel + tx * V;
        Coefficients<T, V> k;
        k.load(a, sample, tile, tx * V);
        k.load_affine(a, channel);
        C m1[V], m2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const Two<C> m = reinterpret_cast<const Two<C> *>(a.means)[sample * a.t.groups + tile.group + (tx * V + i) / tile.part];
            m1[i] = m.a;
            m2[i] = m.b;
        }
        const int64_t begin = chunk * a.apply.run;
        const int64_t end = begin + a.apply.run < a.positions ? begin + a.apply.run : a.positions;
        const T *src = reinterpret_cast<const T *>(a.src) + sample * a.wsrc.n + channel;
        const T *dout = reinterpret_cast<const T *>(a.dout) + sample * a.wdout.n + channel;
        T *dsrc = reinterpret_cast<T *>(a.dsrc) + sample * a.wdsrc.n + channel;
#pragma unroll 2
        for (int64_t row = begin + ty; row < end; row += a.t.ty) {
            const Pack<T, V> x = *reinterpret_cast<const Pack<T, V> *>(src + row * a.wsrc.s);
            const Pack<T, V> d = *reinterpret_cast<const Pack<T, V> *>(dout + row * a.wdout.s);
            Pack<T, V> y;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                C xhat, dz;
                element<ACT>(up(x.v[i]), up(d.v[i]), k.mean[i], k.rstd[i], k.w[i], k.b[i], xhat, dz);
                y.v[i] = down<T>(k.rstd[i] * (dz * k.w[i] - m1[i] - xhat * m2[i]));
            }
            *reinterpret_cast<Pack<T, V> *>(dsrc + row * a.wdsrc.s) = y;
        }
    }
}

struct Plan {
    Tiling t;
    Cut sums, apply;
    int64_t columns;
    int64_t pieces_bytes, means_bytes, bytes;
};
Plan make_plan(const Problem &p, Align align) {
    Plan r{};
    const int es = element_size(p.dtype);
    r.t = make_tiling(p.channels, p.groups, align == Align::kLine ? 16 / es : narrow_vector(es), align != Align::kAny);
    // (a tiling by lines that does not come out is one by single values; by words it may)
    if (align == Align::kLine && r.t.v == 1) r.t = make_tiling(p.channels, p.groups, narrow_vector(es), true);
    r.sums = cut_rows(p, r.t, static_cast<int64_t>(r.t.ty) * 4);
    // however many strips there are, a thread adds no more than kLongest rows in the computation type
    const int64_t most = static_cast<int64_t>(r.t.ty) * kLongest;
    if (r.t.v > kNarrow && r.sums.run > most) {
        r.sums.run = most;
        r.sums.chunks = ceil_div(p.positions, most);
        r.sums.units = p.samples * r.t.tiles * r.sums.chunks;
    }
    r.apply = cut_rows(p, r.t, r.t.ty);
    const int64_t pairs = p.samples * r.sums.chunks;
    r.columns = ceil_div(kBlocksWanted, r.t.tiles);
    if (r.columns > pairs) r.columns = pairs;
    const int64_t pieces = r.sums.chunks * r.t.segments, wide = element_size(p.stat_dtype);
    r.pieces_bytes = pieces == 1 ? 0 : ceil_div(p.samples * p.groups * pieces * 2 * wide, 16) * 16;
    r.means_bytes = ceil_div(p.samples * p.groups * 2 * wide, 16) * 16;
    r.bytes = r.pieces_bytes + r.means_bytes + r.columns * 2 * p.channels * 8;
    return r;
}

// The one-pass kernel: at most 64 samples a team (what f32 sums of dz are kept over), fewer where that leaves SMs idle.
struct RowRuns {
    Teams t;
    int64_t run, row_blocks, partials, bytes;
};
RowRuns make_runs(const Problem &p, Align align) {
    RowRuns r{};
    r.t = make_teams(p, align, true);
    if (r.t.v == 0) return r;
    const int64_t rounds = ceil_div(p.samples, r.t.samples_at_once);
    int64_t run = ceil_div(rounds * r.t.tiles, 148 * 8);
    run = run < 8 ? 8 : (run > 64 ? 64 : run);
    if (ceil_div(rounds, run) > 65535 || r.t.tiles > (int64_t{1} << 30)) {  // beyond a grid's second dimension
        r.t.v = 0;
        return r;
    }
    r.run = run;
    r.row_blocks = ceil_div(rounds, run);
    r.partials = r.row_blocks * r.t.samples_at_once * p.positions;
    r.bytes = ceil_div(r.partials * 2 * p.channels * element_size(p.stat_dtype), 16) * 16;
    return r;
}

// Clusters that share a tile of the resident kernel.
int64_t resident_columns(const Problem &p, const Resident &r) {
    int64_t wanted = ceil_div(kBlocksWanted, r.t.tiles * r.cluster);
    const int64_t least = ceil_div(p.samples, 64);  // samples whose sums one block keeps in the computation type
    if (wanted < least) wanted = least;
    if (wanted >= p.samples) return p.samples;
    return ceil_div(p.samples, ceil_div(p.samples, wanted));  // the same number of samples for all but the last
}

}  // namespace

int64_t backward_workspace(const Problem &p) {
    const int es = element_size(p.dtype), vector = 16 / es;
    const auto need = [&](Align align) -> int64_t {
        const RowRuns r = make_runs(p, align);
        if (r.t.v > 0) return r.bytes;
        const Resident resident = find_resident(p, align, 2);
        if (resident.t.v > 0) {
            return ceil_div(resident_columns(p, resident) * resident.cluster * 2 * p.channels * element_size(p.stat_dtype), 16) * 16;
        }
        return make_plan(p, align).bytes;
    };
    int64_t most = es >= 4 ? 0 : need(Align::kAny);
    if (p.channels * es % 4 == 0) most = std::max(most, need(Align::kWord));
    if (p.channels % vector == 0) most = std::max(most, need(Align::kLine));
    return most;
}
int64_t forward_workspace(const Problem &p);

}  // namespace gnorm
}  // namespace hmc

using namespace hmc;
using namespace hmc::gnorm;

HMC_API hmc_status hmc_group_norm_workspace(const hmc_tensor_desc *src, int32_t groups, int32_t backward, int64_t *bytes) {
    return guarded([&]() -> hmc_status {
        if (bytes == nullptr) return fail(HMC_INVALID, "null workspace size");
        *bytes = 0;
        hmc_tensor_desc shape{};
        if (src != nullptr) {  // the size depends on sizes and dtype only: no memory is needed to ask for it
            shape = *src;
            static char nothing[16];
            shape.data = nothing;
        }
        Problem p{};
        hmc_status s = check_problem(src != nullptr ? &shape : nullptr, groups, &p);
        if (s != HMC_OK) return s;
        if (p.samples == 0 || p.positions == 0 || p.channels == 0) return HMC_OK;
        *bytes = backward ? backward_workspace(p) : forward_workspace(p);
        return HMC_OK;
    });
}

HMC_API hmc_status hmc_group_norm_backward(hmc_context_t ctx, const hmc_tensor_desc *dsrc, const hmc_tensor_desc *dweight,
                                           const hmc_tensor_desc *dbias, const hmc_tensor_desc *src, const hmc_tensor_desc *dout,
                                           const hmc_tensor_desc *mean, const hmc_tensor_desc *rstd, const hmc_tensor_desc *weight,
                                           const hmc_tensor_desc *bias, int32_t groups, int32_t activation, void *workspace,
                                           int64_t workspace_bytes) {
    return guarded([&]() -> hmc_status {
        Problem p{};
        Affine affine{};
        hmc_status s = check_problem(src, groups, &p);
        if (s == HMC_OK) s = check_channels_last(src, "the input");
        if (s == HMC_OK) s = check_layer(dout, "the output's gradient", p.dtype, 3, src->sizes, Use::kInput);
        if (s == HMC_OK) s = check_channels_last(dout, "the output's gradient");
        if (s == HMC_OK) s = check_layer(dsrc, "the input's gradient", p.dtype, 3, src->sizes, Use::kOutput);
        if (s == HMC_OK) s = check_channels_last(dsrc, "the input's gradient");
        if (s == HMC_OK) s = check_affine(weight, bias, p, &affine);
        if (s == HMC_OK && (mean == nullptr || rstd == nullptr)) s = fail(HMC_INVALID, "the gradients of group norm need mean and rstd");
        if (s == HMC_OK) s = check_stats(mean, rstd, p, Use::kInput);
        if (s == HMC_OK) s = check_activation(activation);
        int param = -1;
        for (const hmc_tensor_desc *d : {dweight, dbias}) {
            if (s != HMC_OK || d == nullptr) continue;
            if (param < 0) param = weight != nullptr ? weight->dtype : d->dtype;
            if (weight == nullptr && param != p.dtype && param != HMC_F32) s = fail(HMC_INVALID, "the weight's gradient has neither the input's dtype nor F32");
            if (s == HMC_OK) s = check_layer(d, d == dweight ? "the weight's gradient" : "the bias's gradient", param, 1, &p.channels, Use::kOutput);
        }
        if (s != HMC_OK) return s;
        const bool empty = p.samples == 0 || p.positions == 0 || p.channels == 0;
        if (!empty) s = check_workspace(backward_workspace(p), workspace, workspace_bytes);
        if (s != HMC_OK) return s;
        HMC_ENTER(ctx);
        const bool sums_wanted = dweight != nullptr || dbias != nullptr;
        if (p.channels == 0 || (empty && !sums_wanted)) return HMC_OK;
        GradArgs a{};
        a.dsrc = layer_base(dsrc);
        a.dweight = layer_base(dweight);
        a.dbias = layer_base(dbias);
        a.dweight_stride = dweight != nullptr ? dweight->strides[0] : 0;
        a.dbias_stride = dbias != nullptr ? dbias->strides[0] : 0;
        a.dparam_f32 = param == HMC_F32 ? 1 : 0;
        a.samples = p.samples;
        a.positions = p.positions;
        const int64_t channel_blocks = 2 * ceil_div(p.channels, 32);
        if (empty) {  // sums over nothing
            a.t.channels = p.channels;
            return dispatch_float(p.dtype, [&](auto tag) -> hmc_status {
                fold_channels_kernel<decltype(tag), double><<<grid_for(channel_blocks), kBlock, 0, ctx->stream>>>(a);
                return launch_status("group norm channel kernel launch");
            });
        }
        const Align align = alignment(p.dtype, src, dout, dsrc);
        const RowRuns rows = make_runs(p, align);
        const Resident resident = rows.t.v > 0 ? Resident{} : find_resident(p, align, 2);
        const Plan plan = rows.t.v > 0 || resident.t.v > 0 ? Plan{} : make_plan(p, align);
        a.src = layer_base(src);
        a.dout = layer_base(dout);
        a.mean = layer_base(mean);
        a.rstd = layer_base(rstd);
        a.wdsrc = Rows{dsrc->strides[0], dsrc->strides[1]};
        a.wsrc = Rows{src->strides[0], src->strides[1]};
        a.wdout = Rows{dout->strides[0], dout->strides[1]};
        a.mean_n = mean->strides[0];
        a.mean_g = mean->strides[1];
        a.rstd_n = rstd->strides[0];
        a.rstd_g = rstd->strides[1];
        const auto fold_by_channel = [&](int64_t partials, auto tag) -> hmc_status {
            a.t.channels = p.channels;
            a.columns = partials;
            a.by_channel = workspace;
            using T = decltype(tag);
            fold_channels_kernel<T, typename Comp<T>::C><<<grid_for(channel_blocks), kBlock, 0, ctx->stream>>>(a);
            return launch_status("group norm channel kernel launch");
        };
        if (rows.t.v > 0) {
            RowsBackwardArgs b{};
            b.dsrc = a.dsrc;
            b.src = a.src;
            b.dout = a.dout;
            b.mean = a.mean;
            b.rstd = a.rstd;
            b.wdsrc = a.wdsrc;
            b.wsrc = a.wsrc;
            b.wdout = a.wdout;
            b.mean_n = a.mean_n;
            b.mean_g = a.mean_g;
            b.rstd_n = a.rstd_n;
            b.rstd_g = a.rstd_g;
            b.t = rows.t;
            b.samples = p.samples;
            b.groups = p.groups;
            b.cg = p.channels / p.groups;
            b.channels = p.channels;
            b.positions = p.positions;
            b.run = rows.run;
            b.affine = affine;
            b.by_channel = sums_wanted ? workspace : nullptr;
            s = launch_rows_backward(ctx, p.dtype, activation, b, rows.row_blocks);
            if (s != HMC_OK || !sums_wanted) return s;
            return dispatch_float(p.dtype, [&](auto tag) -> hmc_status { return fold_by_channel(rows.partials, tag); });
        }
        if (resident.t.v > 0) {
            ResidentBackwardArgs b{};
            b.dsrc = a.dsrc;
            b.src = a.src;
            b.dout = a.dout;
            b.mean = a.mean;
            b.rstd = a.rstd;
            b.wdsrc = a.wdsrc;
            b.wsrc = a.wsrc;
            b.wdout = a.wdout;
            b.mean_n = a.mean_n;
            b.mean_g = a.mean_g;
            b.rstd_n = a.rstd_n;
            b.rstd_g = a.rstd_g;
            b.r = resident;
            b.samples = p.samples;
            b.positions = p.positions;
            b.columns = resident_columns(p, resident);
            b.affine = affine;
            b.by_channel = sums_wanted ? workspace : nullptr;
            s = launch_resident_backward(ctx, p.dtype, activation, b);
            if (s != HMC_OK || !sums_wanted) return s;
            return dispatch_float(p.dtype, [&](auto tag) -> hmc_status { return fold_by_channel(b.columns * resident.cluster, tag); });
        }
        a.t = plan.t;
        a.cut = plan.sums;
        a.columns = plan.columns;
        a.apply = plan.apply;
        a.affine = affine;
        a.pieces = workspace;
        a.means = static_cast<char *>(workspace) + plan.pieces_bytes;
        a.by_channel = sums_wanted ? static_cast<char *>(a.means) + plan.means_bytes : nullptr;
        return dispatch_float(p.dtype, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            using C = typename Comp<T>::C;
            const auto run = [&](auto width) -> hmc_status {
                constexpr int V = decltype(width)::value;
                return dispatch_activation(activation, [&](auto act) -> hmc_status {
                    constexpr int ACT = decltype(act)::value;
                    sums_kernel<T, V, ACT><<<static_cast<unsigned>(plan.columns * plan.t.tiles), kBlock, 0, ctx->stream>>>(a);
                    hmc_status l = launch_status("group norm sums kernel launch");
                    if (l == HMC_OK && plan.sums.chunks * plan.t.segments > 1) {
                        const int64_t total = p.samples * p.groups;
                        fold_groups_kernel<C><<<grid_for(ceil_div(total, kWarps)), kBlock, 0, ctx->stream>>>(a, total);
                        l = launch_status("group norm fold kernel launch");
                    }
                    if (l == HMC_OK && sums_wanted) {
                        fold_channels_kernel<T, double><<<grid_for(channel_blocks), kBlock, 0, ctx->stream>>>(a);
                        l = launch_status("group norm channel kernel launch");
                    }
                    if (l != HMC_OK) return l;
                    grad_kernel<T, V, ACT><<<grid_for(plan.apply.units), kBlock, 0, ctx->stream>>>(a);
                    return launch_status("group norm gradient kernel launch");
                });
            };
            if (plan.t.v == kVector<T>) return run(std::integral_constant<int, kVector<T>>{});
            if constexpr (sizeof(T) == 2) {
                if (plan.t.v == 2) return run(std::integral_constant<int, 2>{});
            }
            return run(std::integral_constant<int, 1>{});
        });
    });
}
