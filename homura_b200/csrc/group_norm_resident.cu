// Group norm with an activation in one pass over a cluster's shared memory, forward; the split is group_norm_resident.cuh's.
#include "group_norm_resident.cuh"

namespace hmc {
namespace gnorm {
namespace {

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kBlock, 2) resident_kernel(const __grid_constant__ ResidentForwardArgs a) {
    using C = typename Comp<T>::C;
    constexpr int kBytes = V * static_cast<int>(sizeof(T));
    extern __shared__ __align__(16) unsigned char memory[];
    const Memory m = carve<C, V>(memory, a.r, 1);
    const Tiling &t = a.r.t;
    const int tx = threadIdx.x % t.tx, ty = threadIdx.x / t.tx;
    const int rank = a.r.cluster == 1 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
    Pack<T, V> *mine = reinterpret_cast<Pack<T, V> *>(m.data) + threadIdx.x;  // this thread's vectors, kBlock apart
    if (a.r.cluster > 1) cg::this_cluster().sync();  // every block runs before anyone writes to its shared memory
    const int64_t units = a.samples * t.tiles;
    const int64_t first = rank * a.r.run;
    const int rows = static_cast<int>(a.positions - first < a.r.run ? (a.positions > first ? a.positions - first : 0) : a.r.run);
    int generation = 0;
    for (int64_t unit = blockIdx.x / a.r.cluster; unit < units; unit += gridDim.x / a.r.cluster) {
        const int64_t sample = unit / t.tiles;
        const Tile tile = tile_at(t, unit - sample * t.tiles);
        const bool live = tx * V < tile.width && ty < t.ty;
        const int64_t channel = tile.channel + tx * V;
        const int have = live && rows > ty ? (rows - ty + t.ty - 1) / t.ty : 0;  // rows of this thread: ty, ty + t.ty, ...
        {
            const T *p = reinterpret_cast<const T *>(a.src) + sample * a.wsrc.n + (first + ty) * a.wsrc.s + channel;
            const int64_t step = t.ty * a.wsrc.s;
#pragma unroll 4
            for (int k = 0; k < have; ++k, p += step) copy_async<kBytes>(mine + k * kBlock, p);
            async_copy_commit();
        }
        const Columns<V> column(tile, tx, ty, t.ty);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // The mean of this thread's rows of each channel, and the squares of their deviations from it: nothing large
        // cancels, whatever stands in the other rows.
        C mean[V];
        {
            C sum[V];
#pragma unroll
            for (int i = 0; i < V; ++i) mean[i] = sum[i] = C(0);
            double total[V];
            const bool many = have > 64;
            if (many) {
#pragma unroll
                for (int i = 0; i < V; ++i) total[i] = 0.0;
            }
            for (int k0 = 0; k0 < have; k0 += 64) {
                const int k1 = k0 + 64 < have ? k0 + 64 : have;
#pragma unroll 4
                for (int k = k0; k < k1; ++k) {
                    const Pack<T, V> x = mine[k * kBlock];
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += up(x.v[i]);
                }
                if (many) {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        total[i] += static_cast<double>(sum[i]);
                        sum[i] = C(0);
                    }
                }
            }
            if (have > 0) {
                const C rows_here = static_cast<C>(have), share = C(1) / rows_here;
#pragma unroll
                for (int i = 0; i < V; ++i) mean[i] = many ? static_cast<C>(total[i] / have) : quotient(sum[i], rows_here, share);
            }
            if (many) {
#pragma unroll
                for (int i = 0; i < V; ++i) total[i] = 0.0;
            }
            for (int k0 = 0; k0 < have; k0 += 64) {
                const int k1 = k0 + 64 < have ? k0 + 64 : have;
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] = C(0);
#pragma unroll 4
                for (int k = k0; k < k1; ++k) {
                    const Pack<T, V> x = mine[k * kBlock];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const C d = up(x.v[i]) - mean[i];
                        sum[i] = m_fma(d, d, sum[i]);
                    }
                }
                if (many) {
#pragma unroll
                    for (int i = 0; i < V; ++i) total[i] += static_cast<double>(sum[i]);
                }
            }
            if (live) {
#pragma unroll
                for (int i = 0; i < V; ++i) reinterpret_cast<Two<C> *>(m.columns)[column.at[i]] = Two<C>{mean[i], many ? static_cast<C>(total[i]) : sum[i]};
            }
        }
        __syncthreads();
        // Sums of the values and of their squares in f64, from the threads' means and deviations.
        const int per_row = tile.part;
        fold_columns<C>(m.columns, tile, t.ty,
                        [&](const Two<C> &v, int e) {
                            const int y = e / per_row;
                            const double n = static_cast<double>(rows > y ? (rows - y + t.ty - 1) / t.ty : 0), mu = static_cast<double>(v.a);
                            return Two<double>{n * mu, static_cast<double>(v.b) + n * mu * mu};
                        },
                        [&](int q, Two<double> s) { leave(m, a.r, generation, rank, q, s); });
        meet(a.r);
        const double count = static_cast<double>(a.positions) * tile.part;
        for (int q = threadIdx.x; q < tile.groups; q += kBlock) {
            const Two<double> s = gather(m, a.r, generation, q);
            const double mu = s.a / count, var = s.b / count - mu * mu, rstd = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + a.eps);
            m.folded[q] = Two<double>{mu, rstd};
            if (rank == 0 && a.mean != nullptr) {
                reinterpret_cast<C *>(a.mean)[sample * a.mean_n + (tile.group + q) * a.mean_g] = static_cast<C>(mu);
                reinterpret_cast<C *>(a.rstd)[sample * a.rstd_n + (tile.group + q) * a.rstd_g] = static_cast<C>(rstd);
            }
        }
        generation ^= 1;
        __syncthreads();
        if (live) {
            C rstd[V], w[V], b[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const Two<double> st = m.folded[column.group[i]];
                mean[i] = static_cast<C>(st.a);
                rstd[i] = static_cast<C>(st.b);
            }
            parameters<T, V>(w, a.affine.weight, channel, a.affine.weight_stride, a.affine.is_f32, C(1));
            parameters<T, V>(b, a.affine.bias, channel, a.affine.bias_stride, a.affine.is_f32, C(0));
            T *out = reinterpret_cast<T *>(a.out) + sample * a.wout.n + (first + ty) * a.wout.s + channel;
            const int64_t step = t.ty * a.wout.s;
#pragma unroll 2
            for (int k = 0; k < have; ++k, out += step) {
                const Pack<T, V> x = mine[k * kBlock];
                C y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = activate<ACT>(scaled<ACT>((up(x.v[i]) - mean[i]) * rstd[i], w[i], b[i]));
                *reinterpret_cast<Pack<T, V> *>(out) = pack_of<T, V>(y);
            }
        }
        // (every thread has read m.columns and m.folded, and begun on the next sample's, only behind a barrier in between)
    }
}

}  // namespace

hmc_status launch_resident_forward(hmc_context_t ctx, int dtype, int32_t activation, const ResidentForwardArgs &a) {
    return dispatch_float(dtype, [&](auto tag) -> hmc_status {
        using T = decltype(tag);
        if constexpr (std::is_same_v<T, double>) return fail(HMC_INTERNAL_ERROR, "F64 moments are merged from pieces");  // (make_resident)
        else return dispatch_activation(activation, [&](auto act) -> hmc_status {
            const int64_t units = a.samples * a.r.t.tiles;
            const int64_t most = (int64_t{1} << 30) / a.r.cluster;
            if (a.r.t.v == kVector<T>) {
                static SharedKnown known;
                return launch_resident(ctx, resident_kernel<T, kVector<T>, decltype(act)::value>, known, units < most ? units : most, a.r, a, "group norm kernel launch");
            }
            static SharedKnown known;
            return launch_resident(ctx, resident_kernel<T, narrow_vector(sizeof(T)), decltype(act)::value>, known, units < most ? units : most, a.r, a, "group norm kernel launch");
        });
    });
}

}  // namespace gnorm
}  // namespace hmc
