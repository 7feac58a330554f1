// The gradients of the gated linear recurrence (include/homura_cuda_layers.h); the split is recurrence.cuh's. Rows are
// numbered in the order they are processed, against the order of time: g_s = c_s g_{s-1} + dout_s, where c_s is the gate
// of row s - 1 (1 at the first row, so that dlast enters as it is), and the state before row s in time is row s + 1 of
// the forward output (`initial` for the last row).
#include "recurrence.cuh"

namespace hmc {
namespace recur {
namespace {

struct BackwardArgs {
    char *dgate, *dx;
    char *dinitial;                             // null: not wanted
    const char *gate, *x, *out, *dout;          // x: read with COMP only
    const char *initial, *dlast;                // null: zeros
    Walk wdgate, wdx, wdinitial, wgate, wx, wout, wdout, winitial, wdlast;
    int64_t time, channels, tiles, items;
    int32_t warps_time;
};

template <class T, int V> constexpr int kResident = sizeof(T) == 8 ? 1 : (V == 2 ? 2 : 3);

template <class T, int V, int R, bool SIG, bool COMP>
__global__ void __launch_bounds__(kThreads, kResident<T, V>) backward_kernel(const __grid_constant__ BackwardArgs a) {
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
        const T *x = COMP ? reinterpret_cast<const T *>(a.x) + batch * a.wx.b + channel * a.wx.c : nullptr;
        const T *out = reinterpret_cast<const T *>(a.out) + batch * a.wout.b + channel * a.wout.c;
        const T *dout = reinterpret_cast<const T *>(a.dout) + batch * a.wdout.b + channel * a.wdout.c;
        T *dgate = reinterpret_cast<T *>(a.dgate) + batch * a.wdgate.b + channel * a.wdgate.c;
        T *dx = reinterpret_cast<T *>(a.dx) + batch * a.wdx.b + channel * a.wdx.c;
        C carry[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            carry[i] = C(0);
            if (a.dlast != nullptr && live) carry[i] = reinterpret_cast<const C *>(a.dlast)[batch * a.wdlast.b + (channel + i) * a.wdlast.c];
        }
        for (int64_t base = 0; base < a.time; base += round) {
            const int64_t t0 = base + mine;
            // rows of this lane that exist; `last`: the last row in processing order is among them
            const int n = static_cast<int>(rows - t0 < R ? (rows - t0 > 0 ? rows - t0 : 0) : R);
            const bool last = n > 0 && t0 + n == a.time;
            Pack<T, V> rg[R], rd[R], rh[R], rx[COMP ? R : 1], before;
            {
                const T *pg = gate + t0 * a.wgate.t, *pd = dout + t0 * a.wdout.t, *ph = out + (t0 + 1) * a.wout.t;
                const T *px = COMP ? x + t0 * a.wx.t : nullptr;
                if (n > 0 && t0 > 0) before = load_pack<T, V>(pg - a.wgate.t);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < n) {
                        rg[r] = load_pack<T, V>(pg);
                        rd[r] = load_pack<T, V>(pd);
                        if constexpr (COMP) rx[r] = load_pack<T, V>(px);
                        if (r + 1 < n || !last) rh[r] = load_pack<T, V>(ph);
                    }
                    pg += a.wgate.t;
                    pd += a.wdout.t;
                    ph += a.wout.t;
                    if constexpr (COMP) px += a.wx.t;
                }
            }
            // the gates, in the code that gives both a and 1 - a; first: that of the row before this lane's
            C first[V], m[R][V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                first[i] = n > 0 && t0 > 0 ? kept<SIG>(gate_code<SIG>(before.v[i])) : C(1);
#pragma unroll
                for (int r = 0; r < R; ++r) m[r][i] = r < n ? gate_code<SIG>(rg[r].v[i]) : C(1);
            }
            C g[V];
#pragma unroll
            for (int i = 0; i < V; ++i) g[i] = carry[i];
            if (!alone) {
                Step<C> s[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    s[i].a = first[i];
                    s[i].b = n > 0 ? up(rd[0].v[i]) : C(0);
#pragma unroll
                    for (int r = 1; r < R; ++r) {
                        if (r < n) {
                            const C c = kept<SIG>(m[r - 1][i]);
                            s[i].b = m_fma(c, s[i].b, up(rd[r].v[i]));
                            s[i].a *= c;
                        }
                    }
                }
                exchange(shared, p, a.warps_time, generation, s, g, carry);
                generation ^= 1;
            }
            T *pg = dgate + t0 * a.wdgate.t, *px = dx + t0 * a.wdx.t;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                if (r < n) {
                    C da[V], du[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        g[i] = m_fma(r == 0 ? first[i] : kept<SIG>(m[r - 1 < 0 ? 0 : r - 1][i]), g[i], up(rd[r].v[i]));
                        C h;
                        if (r + 1 == n && last) {
                            h = a.initial == nullptr ? C(0)
                                                     : reinterpret_cast<const C *>(a.initial)[batch * a.winitial.b + (channel + i) * a.winitial.c];
                        } else {
                            h = up(rh[r].v[i]);
                        }
                        if constexpr (COMP) h = h - up(rx[r].v[i]);
                        du[i] = COMP ? g[i] * left<SIG>(m[r][i]) : g[i];
                        da[i] = g[i] * h;
                        if constexpr (SIG) da[i] = da[i] * (kept<SIG>(m[r][i]) * left<SIG>(m[r][i]));
                        if (r + 1 == n && last && a.dinitial != nullptr) {
                            reinterpret_cast<C *>(a.dinitial)[batch * a.wdinitial.b + (channel + i) * a.wdinitial.c] = kept<SIG>(m[r][i]) * g[i];
                        }
                    }
                    store_pack<T, V>(pg, da);
                    store_pack<T, V>(px, du);
                }
                pg += a.wdgate.t;
                px += a.wdx.t;
            }
            if (alone) {
#pragma unroll
                for (int i = 0; i < V; ++i) carry[i] = g[i];
            }
        }
        if (a.time == 0 && live && p.rank == 0 && p.wt == 0 && a.dinitial != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) reinterpret_cast<C *>(a.dinitial)[batch * a.wdinitial.b + (channel + i) * a.wdinitial.c] = carry[i];
        }
    }
}

template <class T, int V, int R>
hmc_status launch_backward(hmc_context_t ctx, BackwardArgs &a, int64_t batch, int32_t flags) {
    const Shape shape = plan_launch(batch, a.time, a.channels, V, R);
    a.tiles = shape.tiles;
    a.items = shape.items;
    a.warps_time = shape.warps_time;
    const char *what = "linear recurrence gradient kernel launch";
    switch (flags & (HMC_RECURRENCE_SIGMOID | HMC_RECURRENCE_COMPLEMENT)) {
        case 0: return launch(ctx, backward_kernel<T, V, R, false, false>, shape, a, what);
        case HMC_RECURRENCE_SIGMOID: return launch(ctx, backward_kernel<T, V, R, true, false>, shape, a, what);
        case HMC_RECURRENCE_COMPLEMENT: return launch(ctx, backward_kernel<T, V, R, false, true>, shape, a, what);
        default: return launch(ctx, backward_kernel<T, V, R, true, true>, shape, a, what);
    }
}

}  // namespace
}  // namespace recur
}  // namespace hmc

using namespace hmc;
using namespace hmc::recur;

HMC_API hmc_status hmc_linear_recurrence_backward(hmc_context_t ctx, const hmc_tensor_desc *dgate, const hmc_tensor_desc *dx,
                                                  const hmc_tensor_desc *dinitial, const hmc_tensor_desc *gate,
                                                  const hmc_tensor_desc *x, const hmc_tensor_desc *out,
                                                  const hmc_tensor_desc *initial, const hmc_tensor_desc *dout,
                                                  const hmc_tensor_desc *dlast, int32_t flags) {
    return guarded([&]() -> hmc_status {
        int64_t n = 0;
        hmc_status s = check_recurrence(gate, flags, &n);
        if (s != HMC_OK) return s;
        const int64_t *sz = gate->sizes;
        const int dt = gate->dtype;
        const bool complement = (flags & HMC_RECURRENCE_COMPLEMENT) != 0;
        if (complement || x != nullptr) s = check_layer(x, "x", dt, 3, sz, Use::kInput);
        if (s == HMC_OK) s = check_layer(out, "the forward output", dt, 3, sz, Use::kInput);
        if (s == HMC_OK) s = check_layer(dout, "the output's gradient", dt, 3, sz, Use::kInput);
        if (s == HMC_OK) s = check_layer(dgate, "the gate's gradient", dt, 3, sz, Use::kOutput);
        if (s == HMC_OK) s = check_layer(dx, "the gradient of x", dt, 3, sz, Use::kOutput);
        if (s == HMC_OK) s = check_state(initial, "the initial state", gate, Use::kInput);
        if (s == HMC_OK) s = check_state(dlast, "the last state's gradient", gate, Use::kInput);
        if (s == HMC_OK) s = check_state(dinitial, "the initial state's gradient", gate, Use::kOutput);
        if (s != HMC_OK) return s;
        HMC_ENTER(ctx);
        const int64_t batch = sz[0], time = sz[1], channels = sz[2];
        if (batch == 0 || channels == 0 || (time == 0 && dinitial == nullptr)) return HMC_OK;
        BackwardArgs a{};
        a.dgate = layer_base(dgate);
        a.dx = layer_base(dx);
        a.dinitial = layer_base(dinitial);
        a.gate = layer_base(gate);
        a.x = complement ? layer_base(x) : nullptr;
        a.out = layer_base(out);
        a.dout = layer_base(dout);
        a.initial = layer_base(initial);
        a.dlast = layer_base(dlast);
        const bool backwards = (flags & HMC_RECURRENCE_REVERSE) == 0;
        a.wdgate = walk_rows(dgate, backwards, &a.dgate);
        a.wdx = walk_rows(dx, backwards, &a.dx);
        a.wgate = walk_rows(gate, backwards, &a.gate);
        a.wx = complement ? walk_rows(x, backwards, &a.x) : Walk{0, 0, 0};
        a.wout = walk_rows(out, backwards, &a.out);
        a.wdout = walk_rows(dout, backwards, &a.dout);
        a.wdinitial = walk_state(dinitial);
        a.winitial = walk_state(initial);
        a.wdlast = walk_state(dlast);
        a.time = time;
        a.channels = channels;
        const bool pairs = layer_vectors(dgate, 4) && layer_vectors(dx, 4) && layer_vectors(gate, 4) && layer_vectors(out, 4) &&
                           layer_vectors(dout, 4) && (!complement || layer_vectors(x, 4));
        return dispatch_float(dt, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            if constexpr (sizeof(T) == 2) {
                if (pairs) return time == 1 ? launch_backward<T, 2, 1>(ctx, a, batch, flags) : launch_backward<T, 2, 8>(ctx, a, batch, flags);
            }
            return time == 1 ? launch_backward<T, 1, 1>(ctx, a, batch, flags) : launch_backward<T, 1, 8>(ctx, a, batch, flags);
        });
    });
}
