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
    int64_t time, channels;
    Columns columns;
    int32_t warps_time;
    int32_t wait_limit;
    int *status;
};

constexpr int kStages = 2;
template <class T> constexpr int kPerSm = sizeof(T) == 8 ? 1 : 2;  // blocks on an SM
template <int R, bool COMP> constexpr int kStageRows = (COMP ? 4 : 3) * R + 1;

template <class T, int V, int R, int COPY, bool SIG, bool COMP>
__global__ void __launch_bounds__(kThreads, kPerSm<T>) backward_kernel(const __grid_constant__ BackwardArgs a) {
    using C = typename Comp<T>::C;
    using G = Ring<T, V, COPY>;
    __shared__ Exchange<C, V> shared;
    extern __shared__ __align__(16) unsigned char memory[];
    // a warp's rows of a stage: the gates (that of the row before first), dout, the states, x
    constexpr int kGate = 0, kDout = R + 1, kState = 2 * R + 1, kX = 3 * R + 1, kStage = kStageRows<R, COMP> * G::kRow;
    unsigned char *ring = memory + (threadIdx.x >> 5) * (kStages * kStage);
    const Place p = place<V>(a.warps_time);
    const bool alone = a.warps_time == 1 && p.cluster == 1;
    const int64_t round = static_cast<int64_t>(R) * a.warps_time * p.cluster;
    const int64_t mine = static_cast<int64_t>(R) * (p.rank * a.warps_time + p.wt);
    begin_exchange(shared, p);
    uint32_t rounds = 0;
    for (int64_t item = blockIdx.x / p.cluster; item < a.columns.items; item += gridDim.x / p.cluster) {
        const Column at_column = column_of<V>(a.columns, item, a.warps_time, p.wc, p.lane);
        const int64_t batch = at_column.batch, channel = at_column.channel;
        const bool live = at_column.live;
        // what this lane loads or copies: its own channels, or its part of a row
        const int64_t column = COPY == 16 ? at_column.tile + G::channel() : channel;
        const bool loads = COPY == 16 ? column < a.channels : live;
        const T *gate = reinterpret_cast<const T *>(a.gate) + batch * a.wgate.b + column * a.wgate.c;
        const T *x = COMP ? reinterpret_cast<const T *>(a.x) + batch * a.wx.b + column * a.wx.c : nullptr;
        const T *out = reinterpret_cast<const T *>(a.out) + batch * a.wout.b + column * a.wout.c;
        const T *dout = reinterpret_cast<const T *>(a.dout) + batch * a.wdout.b + column * a.wdout.c;
        T *dgate = reinterpret_cast<T *>(a.dgate) + batch * a.wdgate.b + channel * a.wdgate.c;
        T *dx = reinterpret_cast<T *>(a.dx) + batch * a.wdx.b + channel * a.wdx.c;
        Vec<C, V> carry;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            carry.v[i] = C(0);
            if (a.dlast != nullptr && live) carry.v[i] = reinterpret_cast<const C *>(a.dlast)[batch * a.wdlast.b + (channel + i) * a.wdlast.c];
        }
        // rows of this warp from t0 on that exist, R at most
        const auto count = [&](int64_t t0) { return static_cast<int>(a.time - t0 < R ? (a.time - t0 > 0 ? a.time - t0 : 0) : R); };
        Pack<T, V> direct[COPY > 0 ? 1 : kStageRows<R, COMP>];
        // the next round's rows (one call a round, in order)
        const int64_t gate_round = round * a.wgate.t, dout_round = round * a.wdout.t, out_round = round * a.wout.t, x_round = round * a.wx.t;
        const int64_t ahead = mine + (COPY > 0 ? G::row() : 0);
        const T *pgate = gate + ahead * a.wgate.t, *pdout = dout + ahead * a.wdout.t, *pout = out + (ahead + 1) * a.wout.t;
        const T *px = COMP ? x + ahead * a.wx.t : nullptr;
        const auto fetch = [&](int64_t t0, int stage) {
            const int n = loads ? count(t0) : 0, states = loads ? count(t0 + 1) : 0, before = n > 0 && t0 > 0 ? 1 : 0;
            if constexpr (COPY > 0) {
                unsigned char *to = ring + stage * kStage;
                copy_rows<T, V, COPY, 1>(to, kGate, pgate - a.wgate.t, a.wgate.t, before);
                copy_rows<T, V, COPY, R>(to, kGate + 1, pgate, a.wgate.t, n);
                copy_rows<T, V, COPY, R>(to, kDout, pdout, a.wdout.t, n);
                copy_rows<T, V, COPY, R>(to, kState, pout, a.wout.t, states);
                if constexpr (COMP) copy_rows<T, V, COPY, R>(to, kX, px, a.wx.t, n);
                async_copy_commit();
            } else {
                if (before) direct[kGate] = load_pack<T, V>(pgate - a.wgate.t);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < n) {
                        direct[kGate + 1 + r] = load_pack<T, V>(pgate + r * a.wgate.t);
                        direct[kDout + r] = load_pack<T, V>(pdout + r * a.wdout.t);
                        if (r < states) direct[kState + r] = load_pack<T, V>(pout + r * a.wout.t);
                        if constexpr (COMP) direct[kX + r] = load_pack<T, V>(px + r * a.wx.t);
                    }
                }
            }
            pgate += gate_round;
            pdout += dout_round;
            pout += out_round;
            if constexpr (COMP) px += x_round;
        };
        T *pdgate = dgate + mine * a.wdgate.t, *pdx = dx + mine * a.wdx.t;
        const int64_t dgate_round = round * a.wdgate.t, dx_round = round * a.wdx.t;
        int filled = 0;
        if constexpr (COPY > 0) {
#pragma unroll
            for (int k = 0; k + 1 < kStages; ++k) fetch(mine + k * round, k);
        }
        for (int64_t base = 0; base < a.time; base += round) {
            const int64_t t0 = base + mine;
            const int n = count(t0);
            const bool last = n > 0 && t0 + n == a.time;  // the last row in processing order is among this warp's
            const int stage = filled;
            if constexpr (COPY > 0) {
                // the stage of the round before is free: the copies of kStages - 1 rounds are on their way
                __syncwarp();
                fetch(t0 + (kStages - 1) * round, stage == 0 ? kStages - 1 : stage - 1);
                wait_for_all_but<kStages - 1>();
                __syncwarp();
                filled = stage + 1 == kStages ? 0 : stage + 1;
            } else {
                fetch(t0, 0);
            }
            const unsigned char *from = ring + stage * kStage + p.lane * static_cast<int>(sizeof(T) * V);
            const auto at = [&](int row) -> Pack<T, V> {
                if constexpr (COPY > 0) return load_pack<T, V>(reinterpret_cast<const T *>(from + row * G::kRow));
                else return direct[row];
            };
            // All R rows exist for most warps (`whole`, the same for a warp's lanes): that form has no conditions in it. The
            // barriers of the exchange stand outside. Lanes beyond the last channel compute on whatever there is and write
            // nothing.
            Vec<C, V> first;  // the gate of the row before this warp's
            Gates<C, V> m[R];
            Vec<C, V> product, sum;
            const auto read = [&](auto whole) {
                constexpr bool kWhole = decltype(whole)::value;
                first = n > 0 && t0 > 0 ? gates_of<SIG, T, V>(at(kGate)).a : splat<C, V>(C(1));
                product = first;
                sum = splat<C, V>(C(0));
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (kWhole || r < n) {
                        m[r] = gates_of<SIG, T, V>(at(kGate + 1 + r));
                        const Vec<C, V> c = r == 0 ? first : m[r == 0 ? 0 : r - 1].a;
                        sum = vfma(c, sum, widen<T, V>(at(kDout + r)));
                        if (r > 0) product = vmul(product, c);
                    }
                }
            };
            if (n == R) read(std::true_type{});
            else read(std::false_type{});
            Vec<C, V> g = carry;
            if (!alone) exchange(shared, p, a.warps_time, rounds, base == 0, product, sum, g, carry, a.wait_limit, a.status);
            const auto write = [&](auto whole) {
                constexpr bool kWhole = decltype(whole)::value;  // (and the last row in processing order is not among them)
                T *to_gate = pdgate, *to_x = pdx;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (kWhole || r < n) {
                        g = vfma(r == 0 ? first : m[r == 0 ? 0 : r - 1].a, g, widen<T, V>(at(kDout + r)));
                        Vec<C, V> h = widen<T, V>(at(kState + r));
                        if constexpr (!kWhole) {
                            if (r + 1 == n && last) {
#pragma unroll
                                for (int i = 0; i < V; ++i) {
                                    h.v[i] = a.initial == nullptr || !live ? C(0)
                                                                           : reinterpret_cast<const C *>(a.initial)[batch * a.winitial.b + (channel + i) * a.winitial.c];
                                    if (a.dinitial != nullptr && live) {
                                        reinterpret_cast<C *>(a.dinitial)[batch * a.wdinitial.b + (channel + i) * a.wdinitial.c] = m[r].a.v[i] * g.v[i];
                                    }
                                }
                            }
                        }
                        if constexpr (COMP) h = vfma(widen<T, V>(at(kX + r)), splat<C, V>(C(-1)), h);  // (exact product: h - x)
                        Vec<C, V> da = vmul(g, h);
                        if constexpr (SIG) da = vmul(da, vmul(m[r].a, m[r].rest));
                        if (live) {
                            store_pack<T, V>(to_gate, da);
                            store_pack<T, V>(to_x, COMP ? vmul(g, m[r].rest) : g);
                        }
                    }
                    to_gate += a.wdgate.t;
                    to_x += a.wdx.t;
                }
            };
            if (n == R && !last) write(std::true_type{});
            else write(std::false_type{});
            pdgate += dgate_round;
            pdx += dx_round;
            if (alone) {
                carry = g;
            } else {
                leave_carry(shared, p, a.warps_time, rounds, g);
                ++rounds;
            }
        }
        if (a.time == 0 && live && p.rank == 0 && p.wt == 0 && a.dinitial != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) reinterpret_cast<C *>(a.dinitial)[batch * a.wdinitial.b + (channel + i) * a.wdinitial.c] = carry.v[i];
        }
    }
    end_exchange(shared, p);
}

template <class T, int V, int R, int COPY>
hmc_status launch_backward(hmc_context_t ctx, BackwardArgs &a, int64_t batch, int32_t flags) {
    const bool flat = COPY != 16 && flat_columns(a.channels, V);
    const Shape shape = plan_launch(batch, a.time, a.channels, flat, V, R, kPerSm<T>, &a.columns);
    a.warps_time = shape.warps_time;
    const auto go = [&](auto sigmoid, auto complement) -> hmc_status {
        static SharedKnown known;
        constexpr int kShared = COPY > 0 ? kWarps * kStages * kStageRows<R, decltype(complement)::value> * Ring<T, V, COPY>::kRow : 0;
        return launch(ctx, backward_kernel<T, V, R, COPY, decltype(sigmoid)::value, decltype(complement)::value>, known, kShared, shape, a,
                      "linear recurrence gradient kernel launch");
    };
    return dispatch_flags(flags, go);
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
        a.wait_limit = wait_limit();
        a.status = ctx->status;
        const bool pairs = layer_vectors(dgate, 4) && layer_vectors(dx, 4) && layer_vectors(gate, 4) && layer_vectors(out, 4) &&
                           layer_vectors(dout, 4) && (!complement || layer_vectors(x, 4));
        const bool wide = layer_vectors(gate, 16) && layer_vectors(out, 16) && layer_vectors(dout, 16) &&
                          (!complement || layer_vectors(x, 16)) && layer_vectors(dgate, 4) && layer_vectors(dx, 4);
        return dispatch_float(dt, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            constexpr int kWord = sizeof(T) == 8 ? 8 : 4, V = sizeof(T) == 2 ? 2 : 1;
            if constexpr (sizeof(T) == 2) {
                if (!pairs) return time == 1 ? launch_backward<T, 1, 1, 0>(ctx, a, batch, flags) : launch_backward<T, 1, 8, 0>(ctx, a, batch, flags);
            }
            if (time == 1) return launch_backward<T, V, 1, 0>(ctx, a, batch, flags);
            return wide && !flat_columns(channels, V) ? launch_backward<T, V, 8, 16>(ctx, a, batch, flags) : launch_backward<T, V, 8, kWord>(ctx, a, batch, flags);
        });
    });
}
