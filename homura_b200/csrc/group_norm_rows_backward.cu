// Group norm with an activation, one position a sample and a group in the registers of a team of lanes: the gradients in
// one pass; the split is group_norm_rows.cuh's. A team takes `run` samples one after another and keeps its channels' sums
// for dweight and dbias in registers (f32 for at most 64 samples, then a partial that is folded in f64).
#include "group_norm_rows.cuh"

namespace hmc {
namespace gnorm {
namespace {

template <class T, int V, int K, bool WIDE, int ACT>
__global__ void __launch_bounds__(kBlock, sizeof(T) == 8 ? 1 : 2) rows_backward_kernel(const __grid_constant__ RowsBackwardArgs a) {
    using C = typename Comp<T>::C;
    constexpr bool kFast = sizeof(T) == 2;
    constexpr bool kKeep = K * V <= 8;  // parameters in registers
    constexpr int U = K == 1 ? 2 : 1;
    __shared__ C scratch[2 * U][kWarps];
    const int team = threadIdx.x / a.t.lanes, lane = threadIdx.x - team * a.t.lanes;
    const int beside = team / a.t.groups_per_tile;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * a.t.groups_per_tile + (team - beside * a.t.groups_per_tile);
    const bool team_live = beside < a.t.samples_at_once && group < a.groups;
    const int64_t first_channel = group * a.cg;
    bool have[K];
    C w[kKeep ? K : 1][V], b[kKeep ? K : 1][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int vector = lane + k * a.t.lanes;
        have[k] = team_live && vector < a.t.vectors;
        if constexpr (kKeep) {
            if (have[k]) {
                parameters<T, V>(w[k], a.affine.weight, first_channel + vector * V, a.affine.weight_stride, a.affine.is_f32, C(1));
                parameters<T, V>(b[k], a.affine.bias, first_channel + vector * V, a.affine.bias_stride, a.affine.is_f32, C(0));
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = C(0);
    }
    const C share = C(1) / (static_cast<C>(a.t.vectors) * C(V));
    const int64_t begin = static_cast<int64_t>(blockIdx.y) * a.run * a.t.samples_at_once;
    for (int64_t r = 0; r < a.run && begin + r * a.t.samples_at_once < a.samples; r += U) {
        Pack<T, V> x[U][K], d[U][K];
        C mean[U], rstd[U];
        bool live[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t n = begin + (r + u) * a.t.samples_at_once + beside;
            live[u] = team_live && r + u < a.run && n < a.samples;
            mean[u] = rstd[u] = C(0);
            if (live[u]) {
                mean[u] = reinterpret_cast<const C *>(a.mean)[n * a.mean_n + group * a.mean_g];
                rstd[u] = reinterpret_cast<const C *>(a.rstd)[n * a.rstd_n + group * a.rstd_g];
            }
            const T *src = reinterpret_cast<const T *>(a.src) + n * a.wsrc.n + first_channel;
            const T *dout = reinterpret_cast<const T *>(a.dout) + n * a.wdout.n + first_channel;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int at = (lane + k * a.t.lanes) * V;
                if (live[u] && have[k]) {
                    x[u][k] = *reinterpret_cast<const Pack<T, V> *>(src + at);
                    d[u][k] = *reinterpret_cast<const Pack<T, V> *>(dout + at);
                }
            }
        }
        C sums[2 * U];   // of p and of p * xhat
        C dz[U][K][V];   // kept where registers allow, otherwise taken again
#pragma unroll
        for (int u = 0; u < U; ++u) {
            sums[2 * u] = sums[2 * u + 1] = C(0);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!live[u] || !have[k]) continue;
                if constexpr (!kKeep) {
                    const int64_t channel = first_channel + (lane + k * a.t.lanes) * V;
                    parameters<T, V>(w[0], a.affine.weight, channel, a.affine.weight_stride, a.affine.is_f32, C(1));
                    parameters<T, V>(b[0], a.affine.bias, channel, a.affine.bias_stride, a.affine.is_f32, C(0));
                }
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const C xhat = (up(x[u][k].v[i]) - mean[u]) * rstd[u];
                    const C z = xhat * w[kKeep ? k : 0][i] + b[kKeep ? k : 0][i];
                    const C g = through<ACT, C, kFast>(up(d[u][k].v[i]), z);
                    dw[k][i] = m_fma(g, xhat, dw[k][i]);
                    db[k][i] += g;
                    const C p = g * w[kKeep ? k : 0][i];
                    dz[u][k][i] = p;
                    sums[2 * u] += p;
                    sums[2 * u + 1] = m_fma(p, xhat, sums[2 * u + 1]);
                }
            }
        }
        team_sum<2 * U, WIDE>(sums, a.t.lanes, scratch);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t n = begin + (r + u) * a.t.samples_at_once + beside;
            const C m1 = sums[2 * u] * share, m2 = sums[2 * u + 1] * share;
            T *dsrc = reinterpret_cast<T *>(a.dsrc) + n * a.wdsrc.n + first_channel;
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!live[u] || !have[k]) continue;
                C y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const C xhat = (up(x[u][k].v[i]) - mean[u]) * rstd[u];
                    y[i] = rstd[u] * (dz[u][k][i] - m1 - xhat * m2);
                }
                *reinterpret_cast<Pack<T, V> *>(dsrc + (lane + k * a.t.lanes) * V) = pack_of<T, V>(y);
            }
        }
    }
    if (a.by_channel == nullptr || !team_live) return;
    C *to = reinterpret_cast<C *>(a.by_channel) + (static_cast<int64_t>(blockIdx.y) * a.t.samples_at_once + beside) * 2 * a.channels + first_channel;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!have[k]) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            to[(lane + k * a.t.lanes) * V + i] = dw[k][i];
            to[a.channels + (lane + k * a.t.lanes) * V + i] = db[k][i];
        }
    }
}

}  // namespace

hmc_status launch_rows_backward(hmc_context_t ctx, int dtype, int32_t activation, const RowsBackwardArgs &a, int64_t row_blocks) {
    return dispatch_float(dtype, [&](auto tag) -> hmc_status {
        using T = decltype(tag);
        return dispatch_teams<T, true>(a.t, [&](auto v, auto k, auto wide) -> hmc_status {
            constexpr int V = decltype(v)::value, K = decltype(k)::value;
            constexpr bool WIDE = decltype(wide)::value;
            return dispatch_activation(activation, [&](auto act) -> hmc_status {
                const dim3 grid(static_cast<unsigned>(a.t.tiles), static_cast<unsigned>(row_blocks));
                rows_backward_kernel<T, V, K, WIDE, decltype(act)::value><<<grid, kBlock, 0, ctx->stream>>>(a);
                return launch_status("group norm gradient kernel launch");
            });
        });
    });
}

}  // namespace gnorm
}  // namespace hmc
