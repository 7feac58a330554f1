// Group norm with an activation where a group of one sample fits the registers of a team of lanes: the gradients in one
// pass; the split is group_norm_rows.cuh's. A team takes `run` samples one after another and keeps its channels' sums
// for dweight and dbias in registers (f32 for at most 64 samples, then a partial that is folded in f64).
#include "group_norm_rows.cuh"

namespace hmc {
namespace gnorm {
namespace {

template <class T, int V, int K, bool WIDE, int ACT>
__global__ void __launch_bounds__(kBlock, sizeof(T) == 8 || K == 16 ? 1 : 2) rows_backward_kernel(const __grid_constant__ RowsBackwardArgs a) {
    using C = typename Comp<T>::C;
    constexpr bool kKeep = K * V <= 8;  // parameters in registers
    __shared__ C scratch[2][kWarps];
    extern __shared__ __align__(16) unsigned char memory[];
    using Ring = RowRing<T, V, 2 * K>;  // src, then dout
    Ring ring(memory);
    const int team = threadIdx.x / a.t.lanes, lane = threadIdx.x - team * a.t.lanes;
    const int beside = team / a.t.groups_per_tile;
    const int64_t group = static_cast<int64_t>(blockIdx.x) * a.t.groups_per_tile + (team - beside * a.t.groups_per_tile);
    const bool team_live = beside < a.t.samples_at_once && group < a.groups;
    const int64_t first_channel = group * a.cg;
    // this lane's vectors: position, first channel within the group
    int position[K], at[K];
    bool have[K];
    C w[kKeep ? K : 1][V], b[kKeep ? K : 1][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int vector = lane + k * a.t.lanes;
        have[k] = team_live && vector < a.t.vectors;
        position[k] = vector / a.t.row_vectors;
        at[k] = (vector - position[k] * a.t.row_vectors) * V;
        if constexpr (kKeep) {
            if (have[k]) {
                parameters<T, V>(w[k], a.affine.weight, first_channel + at[k], a.affine.weight_stride, a.affine.is_f32, C(1));
                parameters<T, V>(b[k], a.affine.bias, first_channel + at[k], a.affine.bias_stride, a.affine.is_f32, C(0));
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = C(0);
    }
    const C share = C(1) / (static_cast<C>(a.t.vectors) * C(V));
    const int64_t first = static_cast<int64_t>(blockIdx.y) * a.run * a.t.samples_at_once;
    int64_t n = first + beside;
    const T *src = reinterpret_cast<const T *>(a.src) + n * a.wsrc.n + first_channel;
    const T *dout = reinterpret_cast<const T *>(a.dout) + n * a.wdout.n + first_channel;
    T *dsrc = reinterpret_cast<T *>(a.dsrc) + n * a.wdsrc.n + first_channel;
    const int64_t src_next = a.t.samples_at_once * a.wsrc.n, dout_next = a.t.samples_at_once * a.wdout.n, dsrc_next = a.t.samples_at_once * a.wdsrc.n;
    const auto load = [&](int64_t sample, int64_t r, int stage) {
        if (r < a.run && sample < a.samples) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                if (have[k]) {
                    ring.fetch(stage, k, src + position[k] * a.wsrc.s + at[k]);
                    ring.fetch(stage, K + k, dout + position[k] * a.wdout.s + at[k]);
                }
            }
        }
        ring.commit();
        src += src_next;
        dout += dout_next;
    };
    // rounds on their way: all stages but the one being worked on, or the next in registers
    constexpr int kAhead = Ring::kUsed ? Ring::kStages - 1 : 1;
#pragma unroll
    for (int s = 0; s < kAhead; ++s) load(n + s * a.t.samples_at_once, s, s);
    C mean_ahead = C(0), rstd_ahead = C(0);
    const auto load_moments = [&](int64_t sample) {
        if (sample < a.samples && team_live) {
            mean_ahead = reinterpret_cast<const C *>(a.mean)[sample * a.mean_n + group * a.mean_g];
            rstd_ahead = reinterpret_cast<const C *>(a.rstd)[sample * a.rstd_n + group * a.rstd_g];
        }
    };
    load_moments(n);
    int stage = 0;
    // (the loop runs alike for the whole block: the shuffles and barriers of a team's sums stand in it)
    for (int64_t r = 0; r < a.run && first + r * a.t.samples_at_once < a.samples; ++r, n += a.t.samples_at_once) {
        const bool live = n < a.samples && team_live;
        const C mean = mean_ahead, rstd = rstd_ahead;
        load_moments(n + a.t.samples_at_once);
        if constexpr (Ring::kUsed) {
            load(n + kAhead * a.t.samples_at_once, r + kAhead, stage == 0 ? Ring::kStages - 1 : stage - 1);
            ring.wait();
        }
        C xhat[K][V], p[K][V], sums[2] = {C(0), C(0)};  // of p and of p * xhat
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if constexpr (!kKeep) {
                if (have[k]) {
                    parameters<T, V>(w[0], a.affine.weight, first_channel + at[k], a.affine.weight_stride, a.affine.is_f32, C(1));
                    parameters<T, V>(b[0], a.affine.bias, first_channel + at[k], a.affine.bias_stride, a.affine.is_f32, C(0));
                }
            }
            if (!live || !have[k]) continue;
            const Pack<T, V> x = ring.get(stage, k), d = ring.get(stage, K + k);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                xhat[k][i] = (up(x.v[i]) - mean) * rstd;
                const C g = through<ACT>(up(d.v[i]), scaled<ACT>(xhat[k][i], w[kKeep ? k : 0][i], b[kKeep ? k : 0][i]));
                dw[k][i] = m_fma(g, xhat[k][i], dw[k][i]);
                db[k][i] += g;
                p[k][i] = g * w[kKeep ? k : 0][i];
                sums[0] += p[k][i];
                sums[1] = m_fma(p[k][i], xhat[k][i], sums[1]);
            }
        }
        if constexpr (Ring::kUsed) stage = stage + 1 == Ring::kStages ? 0 : stage + 1;
        else load(n + a.t.samples_at_once, r + 1, 0);
        team_sum<2, WIDE>(sums, a.t.lanes, scratch);
        const C m1 = sums[0] * share, m2 = sums[1] * share;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            if (!live || !have[k]) continue;
            C y[V];
#pragma unroll
            for (int i = 0; i < V; ++i) y[i] = rstd * (p[k][i] - m1 - xhat[k][i] * m2);
            *reinterpret_cast<Pack<T, V> *>(dsrc + position[k] * a.wdsrc.s + at[k]) = pack_of<T, V>(y);
        }
        dsrc += dsrc_next;
    }
    if (a.by_channel == nullptr || !team_live) return;
    const int64_t partial = (static_cast<int64_t>(blockIdx.y) * a.t.samples_at_once + beside) * a.positions;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (!have[k]) continue;
        C *to = reinterpret_cast<C *>(a.by_channel) + (partial + position[k]) * 2 * a.channels + first_channel + at[k];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            to[i] = dw[k][i];
            to[a.channels + i] = db[k][i];
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
                constexpr int kShared = RowRing<T, V, 2 * K>::kBytes;
                static SharedKnown known;
                const auto kernel = rows_backward_kernel<T, V, K, WIDE, decltype(act)::value>;
                const hmc_status s = allow_shared(ctx, kernel, known, kShared, "shared memory size of a group norm kernel");
                if (s != HMC_OK) return s;
                kernel<<<grid, kBlock, kShared, ctx->stream>>>(a);
                return launch_status("group norm gradient kernel launch");
            });
        });
    });
}

}  // namespace gnorm
}  // namespace hmc
