// The gated linear recurrence h_t = a_t h_{t-1} + u_t (include/homura_cuda_layers.h); the split is recurrence.cuh's.
#include "recurrence.cuh"

namespace hmc {
namespace recur {
namespace {

struct ForwardArgs {
    char *out;
    const char *gate, *x;
    const char *initial;  // null: zeros
    char *last;           // null: not wanted
    Walk wout, wgate, wx, winitial, wlast;
    int64_t time, channels, tiles, items;
    int32_t warps_time;
};

template <class T, int V> constexpr int kResident = sizeof(T) == 8 ? 2 : (V == 2 ? 3 : 4);

template <class T, int V, int R, bool SIG, bool COMP>
__global__ void __launch_bounds__(kThreads, kResident<T, V>) forward_kernel(const __grid_constant__ ForwardArgs a) {
    using C = typename Comp<T>::C;
    __shared__ Exchange<C, V> shared;
    const Place p = place<V>(a.warps_time);
    const bool alone = a.warps_time == 1 && p.cluster == 1;
    const int64_t round = static_cast<int64_t>(R) * a.warps_time * p.cluster;
    const int64_t mine = static_cast<int64_t>(R) * (p.rank * a.warps_time + p.wt);
    if (p.cluster > 1) cg::this_cluster().sync();  // every block runs before anyone writes to its shared memory
    int generation = 0;
    for (int64_t item = blockIdx.x / p.cluster; item < a.items; item += gridDim.x / p.cluster) {
        const int64_t batch = item / a.tiles;
        const int64_t channel = ((item - batch * a.tiles) * (kWarps / a.warps_time) + p.wc) * (32 * V) + p.slot;
        const bool live = channel < a.channels;
        const int64_t rows = live ? a.time : 0;
        const T *gate = reinterpret_cast<const T *>(a.gate) + batch * a.wgate.b + channel * a.wgate.c;
        const T *x = reinterpret_cast<const T *>(a.x) + batch * a.wx.b + channel * a.wx.c;
        T *out = reinterpret_cast<T *>(a.out) + batch * a.wout.b + channel * a.wout.c;
        C carry[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            carry[i] = C(0);
            if (a.initial != nullptr && live)
                carry[i] = reinterpret_cast<const C *>(a.initial)[batch * a.winitial.b + (channel + i) * a.winitial.c];
        }
        // rows of this lane from t0 on that exist, R at most
        auto count = [&](int64_t t0) { return static_cast<int>(rows - t0 < R ? (rows - t0 > 0 ? rows - t0 : 0) : R); };
        for (int64_t base = 0; base < a.time; base += round) {
            const int64_t t0 = base + mine;
            const int n = count(t0);
            Pack<T, V> rg[R], rx[R];
            {
                const T *pg = gate + t0 * a.wgate.t, *px = x + t0 * a.wx.t;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < n) {
                        rg[r] = load_pack<T, V>(pg);
                        rx[r] = load_pack<T, V>(px);
                    }
                    pg += a.wgate.t;
                    px += a.wx.t;
                }
            }
            C ca[R][V], cu[R][V];
#pragma unroll
            for (int r = 0; r < R; ++r) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    ca[r][i] = C(1);
                    cu[r][i] = C(0);
                    if (r < n) {
                        const C m = gate_code<SIG>(rg[r].v[i]);
                        ca[r][i] = kept<SIG>(m);
                        cu[r][i] = COMP ? left<SIG>(m) * up(rx[r].v[i]) : up(rx[r].v[i]);
                    }
                }
            }
            C h[V];
#pragma unroll
            for (int i = 0; i < V; ++i) h[i] = carry[i];
            if (!alone) {
                Step<C> s[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[i].a = ca[0][i];
                    s[i].b = cu[0][i];
#pragma unroll
                    for (int r = 1; r < R; ++r) {
                        s[i].b = m_fma(ca[r][i], s[i].b, cu[r][i]);
                        s[i].a *= ca[r][i];
                    }
                }
                exchange(shared, p, a.warps_time, generation, s, h, carry);
                generation ^= 1;
            }
            T *po = out + t0 * a.wout.t;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r < n) {
#pragma unroll
                    for (int i = 0; i < V; ++i) h[i] = m_fma(ca[r][i], h[i], cu[r][i]);
                    store_pack<T, V>(po, h);
                }
                po += a.wout.t;
            }
            if (n > 0 && t0 + n == a.time && a.last != nullptr) {
#pragma unroll
                for (int i = 0; i < V; ++i) reinterpret_cast<C *>(a.last)[batch * a.wlast.b + (channel + i) * a.wlast.c] = h[i];
            }
            if (alone) {
#pragma unroll
                for (int i = 0; i < V; ++i) carry[i] = h[i];
            }
        }
        if (a.time == 0 && live && p.rank == 0 && p.wt == 0 && a.last != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) reinterpret_cast<C *>(a.last)[batch * a.wlast.b + (channel + i) * a.wlast.c] = carry[i];
        }
    }
}

template <class T, int V, int R>
hmc_status launch_forward(hmc_context_t ctx, ForwardArgs &a, int64_t batch, int32_t flags) {
    const Shape shape = plan_launch(batch, a.time, a.channels, V, R);
    a.tiles = shape.tiles;
    a.items = shape.items;
    a.warps_time = shape.warps_time;
    const char *what = "linear recurrence kernel launch";
    switch (flags & (HMC_RECURRENCE_SIGMOID | HMC_RECURRENCE_COMPLEMENT)) {
        case 0: return launch(ctx, forward_kernel<T, V, R, false, false>, shape, a, what);
        case HMC_RECURRENCE_SIGMOID: return launch(ctx, forward_kernel<T, V, R, true, false>, shape, a, what);
        case HMC_RECURRENCE_COMPLEMENT: return launch(ctx, forward_kernel<T, V, R, false, true>, shape, a, what);
        default: return launch(ctx, forward_kernel<T, V, R, true, true>, shape, a, what);
    }
}

}  // namespace
}  // namespace recur
}  // namespace hmc

using namespace hmc;
using namespace hmc::recur;

HMC_API hmc_status hmc_linear_recurrence(hmc_context_t ctx, const hmc_tensor_desc *out, const hmc_tensor_desc *gate,
                                         const hmc_tensor_desc *x, const hmc_tensor_desc *initial, const hmc_tensor_desc *last,
                                         int32_t flags) {
    return guarded([&]() -> hmc_status {
        int64_t n = 0;
        hmc_status s = check_recurrence(gate, flags, &n);
        const int64_t *sz = gate != nullptr ? gate->sizes : nullptr;
        const int dt = gate != nullptr ? gate->dtype : 0;
        if (s == HMC_OK) s = check_layer(x, "x", dt, 3, sz, Use::kInput);
        if (s == HMC_OK) s = check_layer(out, "the output", dt, 3, sz, Use::kOutput);
        if (s == HMC_OK) s = check_state(initial, "the initial state", gate, Use::kInput);
        if (s == HMC_OK) s = check_state(last, "the last state", gate, Use::kOutput);
        if (s != HMC_OK) return s;
        HMC_ENTER(ctx);
        const int64_t batch = sz[0], time = sz[1], channels = sz[2];
        if (batch == 0 || channels == 0 || (time == 0 && last == nullptr)) return HMC_OK;
        ForwardArgs a{};
        a.out = layer_base(out);
        a.gate = layer_base(gate);
        a.x = layer_base(x);
        a.initial = layer_base(initial);
        a.last = layer_base(last);
        const bool backwards = (flags & HMC_RECURRENCE_REVERSE) != 0;
        a.wout = walk_rows(out, backwards, &a.out);
        a.wgate = walk_rows(gate, backwards, &a.gate);
        a.wx = walk_rows(x, backwards, &a.x);
        a.winitial = walk_state(initial);
        a.wlast = walk_state(last);
        a.time = time;
        a.channels = channels;
        const bool pairs = layer_vectors(out, 4) && layer_vectors(gate, 4) && layer_vectors(x, 4);
        return dispatch_float(dt, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            if constexpr (sizeof(T) == 2) {
                if (pairs) return time == 1 ? launch_forward<T, 2, 1>(ctx, a, batch, flags) : launch_forward<T, 2, 8>(ctx, a, batch, flags);
            }
            return time == 1 ? launch_forward<T, 1, 1>(ctx, a, batch, flags) : launch_forward<T, 1, 8>(ctx, a, batch, flags);
        });
    });
}
