// Group norm with an activation where a group of one sample fits the registers of a team of lanes, forward; the split is
// group_norm_rows.cuh's.
#include "group_norm_rows.cuh"

namespace hmc {
namespace gnorm {
namespace {

template <class T, int V, int K, bool WIDE, int ACT>
__global__ void __launch_bounds__(kBlock, sizeof(T) == 8 || (sizeof(T) * V == 2 && K == 16) ? 1 : (sizeof(T) * V == 16 && K * V <= 8 ? 3 : 2)) rows_kernel(const __grid_constant__ RowsForwardArgs a) {
    using C = typename Comp<T>::C;
    constexpr int U = samples_at_a_time(K);
    constexpr bool kKeep = K * V <= 16;  // parameters in registers
    __shared__ C scratch[U][kWarps];
    extern __shared__ __align__(16) unsigned char memory[];
    using Ring = RowRing<T, V, U * K>;
    Ring ring(memory);
    const int team = threadIdx.x / a.t.lanes, lane = threadIdx.x - team * a.t.lanes;
    const int beside = team / a.t.groups_per_tile;  // which of the samples side by side
    const int64_t group = static_cast<int64_t>(blockIdx.x) * a.t.groups_per_tile + (team - beside * a.t.groups_per_tile);
    const bool team_live = beside < a.t.samples_at_once && group < a.groups;
    // this lane's vectors: where they lie within a sample, and their channels
    int64_t in[K], to[K], channel[K];
    bool have[K];
    C w[kKeep ? K : 1][V], b[kKeep ? K : 1][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int vector = lane + k * a.t.lanes;
        have[k] = team_live && vector < a.t.vectors;
        const int position = vector / a.t.row_vectors;
        channel[k] = group * a.cg + static_cast<int64_t>(vector - position * a.t.row_vectors) * V;
        in[k] = position * a.wsrc.s + channel[k];
        to[k] = position * a.wout.s + channel[k];
        if constexpr (kKeep) {
            if (have[k]) {
                parameters<T, V>(w[k], a.affine.weight, channel[k], a.affine.weight_stride, a.affine.is_f32, C(1));
                parameters<T, V>(b[k], a.affine.bias, channel[k], a.affine.bias_stride, a.affine.is_f32, C(0));
            }
        }
    }
    const C count = static_cast<C>(a.t.vectors) * C(V), share = C(1) / count;
    const bool exact = (a.t.vectors & (a.t.vectors - 1)) == 0;  // then share is (V is a power of two)
    const int64_t step = static_cast<int64_t>(a.t.samples_at_once) * U * gridDim.y;
    const int64_t first = static_cast<int64_t>(blockIdx.y) * a.t.samples_at_once * U;
    int64_t n = first + beside;  // of the samples at a time, samples_at_once apart, the first
    const T *src = reinterpret_cast<const T *>(a.src) + n * a.wsrc.n;
    T *out = reinterpret_cast<T *>(a.out) + n * a.wout.n;
    const int64_t src_next = a.t.samples_at_once * a.wsrc.n, out_next = a.t.samples_at_once * a.wout.n;
    const auto load = [&](int64_t from, int stage) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (have[k] && from + u * a.t.samples_at_once < a.samples) ring.fetch(stage, u * K + k, src + u * src_next + in[k]);
            }
        }
        ring.commit();
        src += step * a.wsrc.n;
    };
    // rounds on their way: all stages but the one being worked on, or the next in registers
    constexpr int kAhead = Ring::kUsed ? Ring::kStages - 1 : 1;
#pragma unroll
    for (int s = 0; s < kAhead; ++s) load(n + s * step, s);
    int stage = 0;
    // (the loop runs alike for the whole block: the shuffles and barriers of a team's sums stand in it. Lanes without a
    // vector, or without a sample, add nothing and write nothing.)
    for (int64_t base = first; base < a.samples; base += step, n += step) {
        C x[U][K][V];
        if constexpr (Ring::kUsed) {
            load(n + kAhead * step, stage == 0 ? Ring::kStages - 1 : stage - 1);
            ring.wait();
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const Pack<T, V> v = ring.get(stage, u * K + k);
#pragma unroll
                for (int i = 0; i < V; ++i) x[u][k][i] = have[k] ? up(v.v[i]) : C(0);
            }
        }
        if constexpr (Ring::kUsed) stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
        else load(n + step, 0);
        C mean[U], sq[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] = C(0);
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) mean[u] += x[u][k][i];
            }
        }
        team_sum<U, WIDE>(mean, a.t.lanes, scratch);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            mean[u] = exact ? mean[u] * share : quotient(mean[u], count, share);
            sq[u] = C(0);
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    x[u][k][i] = have[k] ? x[u][k][i] - mean[u] : C(0);
                    sq[u] = m_fma(x[u][k][i], x[u][k][i], sq[u]);
                }
            }
        }
        team_sum<U, WIDE>(sq, a.t.lanes, scratch);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const C rstd = inverse_root(m_fma(sq[u], share, static_cast<C>(a.eps)));
            if (n + u * a.t.samples_at_once >= a.samples) continue;
            if (a.mean != nullptr && lane == 0 && team_live) {
                reinterpret_cast<C *>(a.mean)[(n + u * a.t.samples_at_once) * a.mean_n + group * a.mean_g] = mean[u];
                reinterpret_cast<C *>(a.rstd)[(n + u * a.t.samples_at_once) * a.rstd_n + group * a.rstd_g] = rstd;
            }
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (!have[k]) continue;
                if constexpr (!kKeep) {
                    parameters<T, V>(w[0], a.affine.weight, channel[k], a.affine.weight_stride, a.affine.is_f32, C(1));
                    parameters<T, V>(b[0], a.affine.bias, channel[k], a.affine.bias_stride, a.affine.is_f32, C(0));
                }
                C y[V];
#pragma unroll
                for (int i = 0; i < V; ++i) y[i] = activate<ACT>(scaled<ACT>(x[u][k][i] * rstd, w[kKeep ? k : 0][i], b[kKeep ? k : 0][i]));
                *reinterpret_cast<Pack<T, V> *>(out + u * out_next + to[k]) = pack_of<T, V>(y);
            }
        }
        out += step * a.wout.n;
    }
}

}  // namespace

hmc_status launch_rows_forward(hmc_context_t ctx, int dtype, int32_t activation, const RowsForwardArgs &a) {
    return dispatch_float(dtype, [&](auto tag) -> hmc_status {
        using T = decltype(tag);
        return dispatch_teams<T, false>(a.t, [&](auto v, auto k, auto wide) -> hmc_status {
            constexpr int V = decltype(v)::value, K = decltype(k)::value;
            constexpr bool WIDE = decltype(wide)::value;
            return dispatch_activation(activation, [&](auto act) -> hmc_status {
                // blocks for some rounds each, so that the parameters and the first copies are paid once for many samples; more
                // and shorter ones where two vectors a lane leave three blocks on an SM
                const int64_t rounds = ceil_div(a.samples, static_cast<int64_t>(a.t.samples_at_once) * samples_at_a_time(K));
                const int64_t wanted = ceil_div(148 * (K * V * static_cast<int>(sizeof(T)) <= 32 ? 16 : 4), a.t.tiles);
                const int64_t y = rounds < wanted ? rounds : wanted;
                const dim3 grid(static_cast<unsigned>(a.t.tiles), static_cast<unsigned>(y < 65535 ? y : 65535));
                constexpr int kShared = RowRing<T, V, samples_at_a_time(K) * K>::kBytes;
                static SharedKnown known;
                const auto kernel = rows_kernel<T, V, K, WIDE, decltype(act)::value>;
                const hmc_status s = allow_shared(ctx, kernel, known, kShared, "shared memory size of a group norm kernel");
                if (s != HMC_OK) return s;
                kernel<<<grid, kBlock, kShared, ctx->stream>>>(a);
                return launch_status("group norm kernel launch");
            });
        });
    });
}

}  // namespace gnorm
}  // namespace hmc
