// Group norm with an activation in one pass over a cluster's shared memory, the gradients; the split is
// group_norm_resident.cuh's. A cluster takes the samples of one tile one after another and keeps its channels' sums for
// dweight and dbias in registers, over at most 64 samples.
#include "group_norm_resident.cuh"

namespace hmc {
namespace gnorm {
namespace {

template <class T, int V, int ACT>
__global__ void __launch_bounds__(kBlock, 2) resident_backward_kernel(const __grid_constant__ ResidentBackwardArgs a) {
    using C = typename Comp<T>::C;
    constexpr int kBytes = V * static_cast<int>(sizeof(T));
    extern __shared__ __align__(16) unsigned char memory[];
    const Memory m = carve<C, V>(memory, a.r, 2);
    const Tiling &t = a.r.t;
    const int tx = threadIdx.x % t.tx, ty = threadIdx.x / t.tx;
    const int rank = a.r.cluster == 1 ? 0 : static_cast<int>(cg::this_cluster().block_rank());
    Pack<T, V> *xs = reinterpret_cast<Pack<T, V> *>(m.data) + threadIdx.x;  // this thread's vectors, kBlock apart
    Pack<T, V> *ds = reinterpret_cast<Pack<T, V> *>(m.data + a.r.data_bytes) + threadIdx.x;
    if (a.r.cluster > 1) cg::this_cluster().sync();  // every block runs before anyone writes to its shared memory
    const int64_t index = blockIdx.x / a.r.cluster / a.columns, column = blockIdx.x / a.r.cluster - index * a.columns;
    const Tile tile = tile_at(t, index);
    const bool live = tx * V < tile.width && ty < t.ty;
    const int64_t channel = tile.channel + tx * V;
    const int64_t first = rank * a.r.run;
    const int rows = static_cast<int>(a.positions - first < a.r.run ? (a.positions > first ? a.positions - first : 0) : a.r.run);
    const int have = live && rows > ty ? (rows - ty + t.ty - 1) / t.ty : 0;  // rows of this thread: ty, ty + t.ty, ...
    C w[V], b[V];
    if (live) {
        parameters<T, V>(w, a.affine.weight, channel, a.affine.weight_stride, a.affine.is_f32, C(1));
        parameters<T, V>(b, a.affine.bias, channel, a.affine.bias_stride, a.affine.is_f32, C(0));
    }
    C dw[V], db[V];
#pragma unroll
    for (int i = 0; i < V; ++i) dw[i] = db[i] = C(0);
    const Columns<V> column_of(tile, tx, ty, t.ty);
    const double count = static_cast<double>(a.positions) * tile.part;
    int generation = 0;
    for (int64_t sample = column; sample < a.samples; sample += a.columns) {
        {
            const T *px = reinterpret_cast<const T *>(a.src) + sample * a.wsrc.n + (first + ty) * a.wsrc.s + channel;
            const T *pd = reinterpret_cast<const T *>(a.dout) + sample * a.wdout.n + (first + ty) * a.wdout.s + channel;
            const int64_t x_step = t.ty * a.wsrc.s, d_step = t.ty * a.wdout.s;
            for (int k = 0; k < have; ++k, px += x_step, pd += d_step) {
                copy_async<kBytes>(xs + k * kBlock, px);
                copy_async<kBytes>(ds + k * kBlock, pd);
            }
            async_copy_commit();
        }
        C mean[V], rstd[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int64_t group = tile.group + column_of.group[i];
            mean[i] = live ? reinterpret_cast<const C *>(a.mean)[sample * a.mean_n + group * a.mean_g] : C(0);
            rstd[i] = live ? reinterpret_cast<const C *>(a.rstd)[sample * a.rstd_n + group * a.rstd_g] : C(0);
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // (vectors of 8 and 16 bytes: shared memory holds at most 54 and 27 rows of a thread; words up to 108, whose sums go on in
        // f64 every 64 rows)
        constexpr int kRun = 64;
        C s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = C(0);
        const auto add = [&](int k0, int k1) {
#pragma unroll 2
            for (int k = k0; k < k1; ++k) {
                const Pack<T, V> x = xs[k * kBlock], d = ds[k * kBlock];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const C xhat = (up(x.v[i]) - mean[i]) * rstd[i];
                    const C dz = through<ACT>(up(d.v[i]), scaled<ACT>(xhat, w[i], b[i]));
                    s1[i] += dz;
                    s2[i] = m_fma(dz, xhat, s2[i]);
                }
            }
        };
        if constexpr (kResidentShared / (2 * kBlock * kBytes) <= kRun) {
            add(0, have);
        } else {
            double t1[V], t2[V];
            for (int k0 = 0; k0 < have; k0 += kRun) {
                add(k0, k0 + kRun < have ? k0 + kRun : have);
                if (have <= kRun) break;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    t1[i] = static_cast<double>(s1[i]) + (k0 > 0 ? t1[i] : 0.0);
                    t2[i] = static_cast<double>(s2[i]) + (k0 > 0 ? t2[i] : 0.0);
                    s1[i] = s2[i] = C(0);
                }
            }
            if (have > kRun) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s1[i] = static_cast<C>(t1[i]);
                    s2[i] = static_cast<C>(t2[i]);
                }
            }
        }
        if (live) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                db[i] += s1[i];
                dw[i] += s2[i];
                reinterpret_cast<Two<C> *>(m.columns)[column_of.at[i]] = Two<C>{s1[i] * w[i], s2[i] * w[i]};
            }
        }
        __syncthreads();
        fold_columns<C>(m.columns, tile, t.ty, [](const Two<C> &v, int) { return Two<double>{static_cast<double>(v.a), static_cast<double>(v.b)}; },
                        [&](int q, Two<double> s) { leave(m, a.r, generation, rank, q, s); });
        meet(a.r);
        for (int q = threadIdx.x; q < tile.groups; q += kBlock) {
            const Two<double> s = gather(m, a.r, generation, q);
            m.folded[q] = Two<double>{s.a / count, s.b / count};
        }
        generation ^= 1;
        __syncthreads();
        if (live) {
            C m1[V], m2[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const Two<double> s = m.folded[column_of.group[i]];
                m1[i] = static_cast<C>(s.a);
                m2[i] = static_cast<C>(s.b);
            }
            T *dsrc = reinterpret_cast<T *>(a.dsrc) + sample * a.wdsrc.n + (first + ty) * a.wdsrc.s + channel;
            const int64_t step = t.ty * a.wdsrc.s;
#pragma unroll 2
            for (int k = 0; k < have; ++k, dsrc += step) {
                const Pack<T, V> x = xs[k * kBlock], d = ds[k * kBlock];
                C y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const C xhat = (up(x.v[i]) - mean[i]) * rstd[i];
                    const C dz = through<ACT>(up(d.v[i]), scaled<ACT>(xhat, w[i], b[i]));
                    y[i] = rstd[i] * (dz * w[i] - m1[i] - xhat * m2[i]);
                }
                *reinterpret_cast<Pack<T, V> *>(dsrc) = pack_of<T, V>(y);
            }
        }
        // (every thread has read m.columns and m.folded, and begun on the next sample's, only behind a barrier in between)
    }
    if (a.by_channel == nullptr) return;
    __syncthreads();
    if (live) {
#pragma unroll
        for (int i = 0; i < V; ++i) reinterpret_cast<Two<C> *>(m.columns)[column_of.at[i]] = Two<C>{dw[i], db[i]};
    }
    __syncthreads();
    C *to = reinterpret_cast<C *>(a.by_channel) + (column * a.r.cluster + rank) * 2 * t.channels + tile.channel;
    for (int c = threadIdx.x; c < tile.width; c += kBlock) {
        const int q = c / tile.part;
        const Two<C> *from = reinterpret_cast<const Two<C> *>(m.columns) + q * t.ty * tile.part + (c - q * tile.part);
        Two<double> sum{0.0, 0.0};
#pragma unroll 4
        for (int y = 0; y < t.ty; ++y) {
            sum.a += static_cast<double>(from[y * tile.part].a);
            sum.b += static_cast<double>(from[y * tile.part].b);
        }
        to[c] = static_cast<C>(sum.a);
        to[t.channels + c] = static_cast<C>(sum.b);
    }
}

}  // namespace

hmc_status launch_resident_backward(hmc_context_t ctx, int dtype, int32_t activation, const ResidentBackwardArgs &a) {
    return dispatch_float(dtype, [&](auto tag) -> hmc_status {
        using T = decltype(tag);
        return dispatch_activation(activation, [&](auto act) -> hmc_status {
            if (a.r.t.v == kVector<T>) {
                static SharedKnown known;
                return launch_resident(ctx, resident_backward_kernel<T, kVector<T>, decltype(act)::value>, known, a.columns * a.r.t.tiles, a.r, a, "group norm gradient kernel launch");
            }
            static SharedKnown known;
            return launch_resident(ctx, resident_backward_kernel<T, narrow_vector(sizeof(T)), decltype(act)::value>, known, a.columns * a.r.t.tiles, a.r, a, "group norm gradient kernel launch");
        });
    });
}

}  // namespace gnorm
}  // namespace hmc
