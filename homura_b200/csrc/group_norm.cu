// Group norm with an activation, channels last, forward (include/homura_cuda_layers.h); tiles as in group_norm.cuh.
//
// Three steps: every block takes the moments of its run of rows (held in registers: the mean first, then the squares of
// the deviations from it, run by run merged pairwise), a small kernel merges the pieces of each group, and an elementwise
// pass normalises. Where one block holds a whole group the middle step falls away.
#include <algorithm>

#include "group_norm_resident.cuh"

namespace hmc {
namespace gnorm {
namespace {

constexpr int kRows = 8;  // rows a thread holds at a time

struct StatArgs {
    const char *src;
    Rows wsrc;
    Tiling t;
    Cut cut;
    int64_t positions;
    void *pieces;   // Two<double> [samples][groups][chunks * segments]: mean and sum of squared deviations
    void *stats;    // Two<C> [samples][groups]: mean and rstd, written here when there is one piece
    char *mean, *rstd;  // or null
    int64_t mean_n, mean_g, rstd_n, rstd_g;
    double eps;
};

// Pairwise merge of (count, mean, sum of squared deviations), Chan, Golub and LeVeque.
struct Moments {
    double count, mean, m2;
};
__device__ __forceinline__ Moments merge(const Moments &x, const Moments &y) {
    if (y.count == 0.0) return x;
    if (x.count == 0.0) return y;
    const double n = x.count + y.count, d = y.mean - x.mean, share = y.count / n;
    return Moments{n, x.mean + d * share, x.m2 + y.m2 + d * d * (x.count * share)};
}
template <class C> __device__ __forceinline__ void finish(const StatArgs &a, int64_t sample, int64_t group, const Moments &m) {
    const C mean = static_cast<C>(m.mean);
    const C rstd = static_cast<C>(1.0 / sqrt(m.m2 / m.count + a.eps));
    reinterpret_cast<Two<C> *>(a.stats)[sample * a.t.groups + group] = Two<C>{mean, rstd};
    if (a.mean != nullptr) {
        reinterpret_cast<C *>(a.mean)[sample * a.mean_n + group * a.mean_g] = mean;
        reinterpret_cast<C *>(a.rstd)[sample * a.rstd_n + group * a.rstd_g] = rstd;
    }
}

template <class T, int V>
__global__ void __launch_bounds__(kBlock, 3) moments_kernel(const __grid_constant__ StatArgs a) {
    using C = typename Comp<T>::C;
    __shared__ C columns[kBlock * V];
    __shared__ C centre[kBlock * V];
    __shared__ Two<double> running[kBlock * V];
    const int tx = threadIdx.x % a.t.tx, ty = threadIdx.x / a.t.tx;
    for (int64_t unit = blockIdx.x; unit < a.cut.units; unit += gridDim.x) {
        const int64_t strip = unit / a.cut.chunks, chunk = unit - strip * a.cut.chunks;
        const int64_t sample = strip / a.t.tiles;
        const Tile tile = tile_at(a.t, strip - sample * a.t.tiles);
        const bool live = tx * V < tile.width && ty < a.t.ty;
        const int64_t first = chunk * a.cut.run;
        const int64_t end = first + a.cut.run < a.positions ? first + a.cut.run : a.positions;
        const T *src = reinterpret_cast<const T *>(a.src) + sample * a.wsrc.n + tile.channel + tx * V;
        int group[V];  // of each of this thread's channels, within the tile
#pragma unroll
        for (int i = 0; i < V; ++i) group[i] = (tx * V + i) / tile.part;
        const int64_t step = static_cast<int64_t>(a.t.ty) * kRows;
        double before = 0.0;  // values merged into `running` so far
        for (int64_t row = first; row < end; row += step) {
            Pack<T, V> x[kRows];
            const T *p = src + (row + ty) * a.wsrc.s;
            const int rows = static_cast<int>(end - row < step ? end - row : step);
            C sum[V];
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = C(0);
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                if (live && r * a.t.ty + ty < rows) x[r] = *reinterpret_cast<const Pack<T, V> *>(p + r * a.t.ty * a.wsrc.s);
            }
#pragma unroll
            for (int r = 0; r < kRows; ++r) {
                if (live && r * a.t.ty + ty < rows) {
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += up(x[r].v[i]);
                }
            }
            if (live) {
#pragma unroll
                for (int i = 0; i < V; ++i) columns[ty * tile.width + tx * V + i] = sum[i];
            }
            __syncthreads();
            const double count = static_cast<double>(rows) * tile.part;
            by_group(columns, tile, a.t.ty, [&](int q, C s) { centre[q] = s / static_cast<C>(count); });
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) sum[i] = C(0);
            if (live) {
                C c[V];
#pragma unroll
                for (int i = 0; i < V; ++i) c[i] = centre[group[i]];
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    if (r * a.t.ty + ty < rows) {
#pragma unroll
                        for (int i = 0; i < V; ++i) {
                            const C d = up(x[r].v[i]) - c[i];
                            sum[i] = m_fma(d, d, sum[i]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < V; ++i) columns[ty * tile.width + tx * V + i] = sum[i];
            }
            __syncthreads();
            by_group(columns, tile, a.t.ty, [&](int q, C s) {
                Moments m{count, static_cast<double>(centre[q]), static_cast<double>(s)};
                if (before > 0.0) m = merge(Moments{before, running[q].a, running[q].b}, m);
                running[q] = Two<double>{m.mean, m.m2};
            });
            before += count;
            __syncthreads();
        }
        const int64_t pieces = a.cut.chunks * a.t.segments;
        for (int q = threadIdx.x; q < tile.groups; q += kBlock) {
            if (pieces == 1) {
                finish<C>(a, sample, tile.group + q, Moments{before, running[q].a, running[q].b});
            } else {
                reinterpret_cast<Two<double> *>(a.pieces)[(sample * a.t.groups + tile.group + q) * pieces + chunk * a.t.segments + tile.segment] = running[q];
            }
        }
        __syncthreads();
    }
}

// A warp merges the pieces of a group: every lane its own in order, then the lanes in a fixed tree.
template <class C> __global__ void __launch_bounds__(kBlock) merge_kernel(const __grid_constant__ StatArgs a, int64_t total) {
    const int lane = threadIdx.x & 31;
    const int64_t pieces = a.cut.chunks * a.t.segments;
    for (int64_t g = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); g < total; g += static_cast<int64_t>(gridDim.x) * kWarps) {
        const Two<double> *p = reinterpret_cast<const Two<double> *>(a.pieces) + g * pieces;
        Moments m{0.0, 0.0, 0.0};
        for (int64_t k = lane; k < pieces; k += 32) {
            const int64_t chunk = k / a.t.segments, segment = k - chunk * a.t.segments;
            const int64_t row = chunk * a.cut.run, rows = a.positions - row < a.cut.run ? a.positions - row : a.cut.run;
            const int64_t from = a.t.segments == 1 ? 0 : segment * a.t.tile;
            const int64_t width = a.t.segments == 1 ? a.t.cg : (a.t.cg - from < a.t.tile ? a.t.cg - from : a.t.tile);
            m = merge(m, Moments{static_cast<double>(rows) * static_cast<double>(width), p[k].a, p[k].b});
        }
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const Moments other{__shfl_down_sync(0xFFFFFFFFu, m.count, d), __shfl_down_sync(0xFFFFFFFFu, m.mean, d), __shfl_down_sync(0xFFFFFFFFu, m.m2, d)};
            m = merge(m, other);
        }
        if (lane == 0) finish<C>(a, g / a.t.groups, g % a.t.groups, m);
    }
}

struct ApplyArgs {
    char *out;
    const char *src;
    Rows wout, wsrc;
    Tiling t;
    Cut cut;
    int64_t positions;
    Affine affine;
    const void *stats;
};

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kBlock) apply_kernel(const __grid_constant__ ApplyArgs a) {
    using C = typename Comp<T>::C;
    const int tx = threadIdx.x % a.t.tx, ty = threadIdx.x / a.t.tx;
    for (int64_t unit = blockIdx.x; unit < a.cut.units; unit += gridDim.x) {
        const int64_t strip = unit / a.cut.chunks, chunk = unit - strip * a.cut.chunks;
        const int64_t sample = strip / a.t.tiles;
        const Tile tile = tile_at(a.t, strip - sample * a.t.tiles);
        if (tx * V >= tile.width || ty >= a.t.ty) continue;
        const int64_t channel = tile.channel + tx * V;
        C mean[V], rstd[V], w[V], b[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const Two<C> st = reinterpret_cast<const Two<C> *>(a.stats)[sample * a.t.groups + tile.group + (tx * V + i) / tile.part];
            mean[i] = st.a;
            rstd[i] = st.b;
            w[i] = a.affine.weight != nullptr ? parameter<T>(a.affine.weight, (channel + i) * a.affine.weight_stride, a.affine.is_f32) : C(1);
            b[i] = a.affine.weight != nullptr ? parameter<T>(a.affine.bias, (channel + i) * a.affine.bias_stride, a.affine.is_f32) : C(0);
        }
        const int64_t first = chunk * a.cut.run;
        const int64_t end = first + a.cut.run < a.positions ? first + a.cut.run : a.positions;
        const T *src = reinterpret_cast<const T *>(a.src) + sample * a.wsrc.n + channel;
        T *out = reinterpret_cast<T *>(a.out) + sample * a.wout.n + channel;
#pragma unroll 4
        for (int64_t row = first + ty; row < end; row += a.t.ty) {
            const Pack<T, V> x = *reinterpret_cast<const Pack<T, V> *>(src + row * a.wsrc.s);
            Pack<T, V> y;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                y.v[i] = down<T>(activate<ACT>(scaled<ACT>((up(x.v[i]) - mean[i]) * rstd[i], w[i], b[i])));
            }
            *reinterpret_cast<Pack<T, V> *>(out + row * a.wout.s) = y;
        }
    }
}

struct Plan {
    Tiling t;
    Cut moments, apply;
    int64_t pieces_bytes, bytes;
};
Plan make_plan(const Problem &p, Align align) {
    Plan r{};
    const int es = element_size(p.dtype);
    r.t = make_tiling(p.channels, p.groups, align == Align::kLine ? 16 / es : narrow_vector(es), align != Align::kAny);
    // (a tiling by lines that does not come out is one by single values; by words it may)
    if (align == Align::kLine && r.t.v == 1) r.t = make_tiling(p.channels, p.groups, narrow_vector(es), true);
    r.moments = cut_rows(p, r.t, static_cast<int64_t>(r.t.ty) * kRows);
    r.apply = cut_rows(p, r.t, r.t.ty);
    const int64_t pieces = r.moments.chunks * r.t.segments;
    r.pieces_bytes = pieces == 1 ? 0 : p.samples * p.groups * pieces * static_cast<int64_t>(sizeof(Two<double>));
    r.bytes = r.pieces_bytes + p.samples * p.groups * 2 * element_size(p.stat_dtype);
    return r;
}

}  // namespace

// What the forward pass needs whatever the alignment of its operands.
int64_t forward_workspace(const Problem &p) {
    const int es = element_size(p.dtype), vector = 16 / es;
    const auto need = [&](Align align) -> int64_t {
        if (make_teams(p, align, false).v > 0 || find_resident(p, align, 1).t.v > 0) return 0;
        return make_plan(p, align).bytes;
    };
    int64_t most = es >= 4 ? 0 : need(Align::kAny);
    if (p.channels * es % 4 == 0) most = std::max(most, need(Align::kWord));
    if (p.channels % vector == 0) most = std::max(most, need(Align::kLine));
    return most;
}

}  // namespace gnorm
}  // namespace hmc

using namespace hmc;
using namespace hmc::gnorm;

HMC_API hmc_status hmc_group_norm(hmc_context_t ctx, const hmc_tensor_desc *out, const hmc_tensor_desc *src,
                                  const hmc_tensor_desc *weight, const hmc_tensor_desc *bias, const hmc_tensor_desc *mean,
                                  const hmc_tensor_desc *rstd, int32_t groups, double eps, int32_t activation, void *workspace,
                                  int64_t workspace_bytes) {
    return guarded([&]() -> hmc_status {
        Problem p{};
        Affine affine{};
        hmc_status s = check_problem(src, groups, &p);
        if (s == HMC_OK) s = check_channels_last(src, "the input");
        if (s == HMC_OK) s = check_layer(out, "the output", p.dtype, 3, src->sizes, Use::kOutput);
        if (s == HMC_OK) s = check_channels_last(out, "the output");
        if (s == HMC_OK) s = check_affine(weight, bias, p, &affine);
        if (s == HMC_OK) s = check_stats(mean, rstd, p, Use::kOutput);
        if (s == HMC_OK) s = check_activation(activation);
        if (s == HMC_OK && !(eps >= 0.0)) s = fail(HMC_INVALID, "group norm needs an eps of at least 0");
        if (s != HMC_OK) return s;
        if (p.samples == 0 || p.positions == 0 || p.channels == 0) {
            if (p.samples > 0 && mean != nullptr) return fail(HMC_INVALID, "the moments of empty groups are not defined");
            HMC_ENTER(ctx);
            return HMC_OK;
        }
        s = check_workspace(forward_workspace(p), workspace, workspace_bytes);
        if (s != HMC_OK) return s;
        HMC_ENTER(ctx);
        const Align align = alignment(p.dtype, src, out);
        const Teams teams = make_teams(p, align, false);
        if (teams.v > 0) {
            RowsForwardArgs r{};
            r.out = layer_base(out);
            r.src = layer_base(src);
            r.wout = Rows{out->strides[0], out->strides[1]};
            r.wsrc = Rows{src->strides[0], src->strides[1]};
            r.t = teams;
            r.samples = p.samples;
            r.groups = p.groups;
            r.cg = p.channels / p.groups;
            r.affine = affine;
            r.mean = layer_base(mean);
            r.rstd = layer_base(rstd);
            if (mean != nullptr) {
                r.mean_n = mean->strides[0];
                r.mean_g = mean->strides[1];
                r.rstd_n = rstd->strides[0];
                r.rstd_g = rstd->strides[1];
            }
            r.eps = eps;
            return launch_rows_forward(ctx, p.dtype, activation, r);
        }
        const Resident resident = find_resident(p, align, 1);
        if (resident.t.v > 0) {
            ResidentForwardArgs r{};
            r.out = layer_base(out);
            r.src = layer_base(src);
            r.wout = Rows{out->strides[0], out->strides[1]};
            r.wsrc = Rows{src->strides[0], src->strides[1]};
            r.r = resident;
            r.samples = p.samples;
            r.positions = p.positions;
            r.affine = affine;
            r.mean = layer_base(mean);
            r.rstd = layer_base(rstd);
            if (mean != nullptr) {
                r.mean_n = mean->strides[0];
                r.mean_g = mean->strides[1];
                r.rstd_n = rstd->strides[0];
                r.rstd_g = rstd->strides[1];
            }
            r.eps = eps;
            return launch_resident_forward(ctx, p.dtype, activation, r);
        }
        const Plan plan = make_plan(p, align);
        StatArgs st{};
        st.src = layer_base(src);
        st.wsrc = Rows{src->strides[0], src->strides[1]};
        st.t = plan.t;
        st.cut = plan.moments;
        st.positions = p.positions;
        st.pieces = workspace;
        st.stats = static_cast<char *>(workspace) + plan.pieces_bytes;
        st.mean = layer_base(mean);
        st.rstd = layer_base(rstd);
        if (mean != nullptr) {
            st.mean_n = mean->strides[0];
            st.mean_g = mean->strides[1];
            st.rstd_n = rstd->strides[0];
            st.rstd_g = rstd->strides[1];
        }
        st.eps = eps;
        ApplyArgs ap{};
        ap.out = layer_base(out);
        ap.src = st.src;
        ap.wout = Rows{out->strides[0], out->strides[1]};
        ap.wsrc = st.wsrc;
        ap.t = plan.t;
        ap.cut = plan.apply;
        ap.positions = p.positions;
        ap.affine = affine;
        ap.stats = st.stats;
        return dispatch_float(p.dtype, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            using C = typename Comp<T>::C;
            const auto run = [&](auto width) -> hmc_status {
                constexpr int V = decltype(width)::value;
                moments_kernel<T, V><<<grid_for(st.cut.units), kBlock, 0, ctx->stream>>>(st);
                hmc_status l = launch_status("group norm moments kernel launch");
                if (l != HMC_OK) return l;
                if (st.cut.chunks * st.t.segments > 1) {
                    const int64_t total = p.samples * p.groups;
                    merge_kernel<C><<<grid_for(ceil_div(total, kWarps)), kBlock, 0, ctx->stream>>>(st, total);
                    l = launch_status("group norm merge kernel launch");
                    if (l != HMC_OK) return l;
                }
                return dispatch_activation(activation, [&](auto act) -> hmc_status {
                    apply_kernel<T, V, decltype(act)::value><<<grid_for(ap.cut.units), kBlock, 0, ctx->stream>>>(ap);
                    return launch_status("group norm kernel launch");
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
