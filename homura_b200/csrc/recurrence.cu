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
    int64_t time, channels;
    Columns columns;
    int32_t warps_time;
    int32_t wait_limit;
    int *status;
};

constexpr int kStages = 2;
// Blocks on an SM: four with eight rows a lane; with sixteen, for launches that fill no more, two.
template <class T> constexpr int per_sm(int rows) { return sizeof(T) == 8 || rows > 8 ? 2 : 4; }

template <class T, int V, int R, int COPY, bool SIG, bool COMP>
__global__ void __launch_bounds__(kThreads, per_sm<T>(R)) forward_kernel(const __grid_constant__ ForwardArgs a) {
    using C = typename Comp<T>::C;
    using G = Ring<T, V, COPY>;
    __shared__ Exchange<C, V> shared;
    extern __shared__ __align__(16) unsigned char memory[];
    constexpr int kStage = 2 * R * G::kRow;  // a warp's gates, then its x
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
        const T *x = reinterpret_cast<const T *>(a.x) + batch * a.wx.b + column * a.wx.c;
        T *out = reinterpret_cast<T *>(a.out) + batch * a.wout.b + channel * a.wout.c;
        Vec<C, V> carry;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            carry.v[i] = C(0);
            if (a.initial != nullptr && live)
                carry.v[i] = reinterpret_cast<const C *>(a.initial)[batch * a.winitial.b + (channel + i) * a.winitial.c];
        }
        // rows of this warp from t0 on that exist, R at most
        const auto count = [&](int64_t t0) { return static_cast<int>(a.time - t0 < R ? (a.time - t0 > 0 ? a.time - t0 : 0) : R); };
        Pack<T, V> rg[R], rx[R];
        // the next round's rows (one call a round, in order)
        const int64_t gate_round = round * a.wgate.t, x_round = round * a.wx.t;
        const int ahead = COPY > 0 ? G::row() : 0;
        const T *pg = gate + (mine + ahead) * a.wgate.t, *px = x + (mine + ahead) * a.wx.t;
        const auto fetch = [&](int64_t t0, int stage) {
            const int n = loads ? count(t0) : 0;
            if constexpr (COPY > 0) {
                copy_rows<T, V, COPY, R>(ring + stage * kStage, 0, pg, a.wgate.t, n);
                copy_rows<T, V, COPY, R>(ring + stage * kStage, R, px, a.wx.t, n);
                async_copy_commit();
            } else {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (r < n) {
                        rg[r] = load_pack<T, V>(pg + r * a.wgate.t);
                        rx[r] = load_pack<T, V>(px + r * a.wx.t);
                    }
                }
            }
            pg += gate_round;
            px += x_round;
        };
        T *po = out + mine * a.wout.t;
        const int64_t out_round = round * a.wout.t;
        int stage = 0;
        if constexpr (COPY > 0) {
#pragma unroll
            for (int k = 0; k + 1 < kStages; ++k) fetch(mine + k * round, k);
        }
        for (int64_t base = 0; base < a.time; base += round) {
            const int64_t t0 = base + mine;
            const int n = count(t0);
            if constexpr (COPY > 0) {
                // the stage of the round before is free: the copies of kStages - 1 rounds are on their way
                __syncwarp();
                fetch(t0 + (kStages - 1) * round, stage == 0 ? kStages - 1 : stage - 1);
                wait_for_all_but<kStages - 1>();
                __syncwarp();
                const unsigned char *from = ring + stage * kStage + p.lane * static_cast<int>(sizeof(T) * V);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    rg[r] = load_pack<T, V>(reinterpret_cast<const T *>(from + r * G::kRow));
                    rx[r] = load_pack<T, V>(reinterpret_cast<const T *>(from + (R + r) * G::kRow));
                }
                stage = stage + 1 == kStages ? 0 : stage + 1;
            } else {
                fetch(t0, 0);
            }
            // All R rows exist for most warps (`whole`, the same for a warp's lanes): that form has no conditions in it. The
            // barriers of the exchange stand outside. Lanes beyond the last channel compute on whatever their registers
            // hold and write nothing.
            Vec<C, V> ca[R], cu[R];
            const auto read = [&](auto whole) {
                constexpr bool kWhole = decltype(whole)::value;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (kWhole || r < n) {
                        const Gates<C, V> g = gates_of<SIG, T, V>(rg[r]);
                        ca[r] = g.a;
                        cu[r] = COMP ? vmul(g.rest, widen<T, V>(rx[r])) : widen<T, V>(rx[r]);
                    } else {
                        ca[r] = splat<C, V>(C(1));
                        cu[r] = splat<C, V>(C(0));
                    }
                }
            };
            if (n == R) read(std::true_type{});
            else read(std::false_type{});
            Vec<C, V> h = carry;
            if (!alone) {
                Vec<C, V> product = ca[0], sum = vfma(ca[0], splat<C, V>(C(0)), cu[0]);
#pragma unroll
                for (int r = 1; r < R; ++r) {
                    sum = vfma(ca[r], sum, cu[r]);
                    product = vmul(product, ca[r]);
                }
                exchange(shared, p, a.warps_time, rounds, base == 0, product, sum, h, carry, a.wait_limit, a.status);
            }
            const auto write = [&](auto whole) {
                constexpr bool kWhole = decltype(whole)::value;
                T *to = po;
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (kWhole || r < n) {
                        h = vfma(ca[r], h, cu[r]);
                        if (live) store_pack<T, V>(to, h);
                    }
                    to += a.wout.t;
                }
            };
            if (n == R) write(std::true_type{});
            else write(std::false_type{});
            po += out_round;
            if (alone) {
                carry = h;
            } else {
                leave_carry(shared, p, a.warps_time, rounds, h);
                ++rounds;
            }
            if (a.last != nullptr && live && n > 0 && t0 + n == a.time) {
#pragma unroll
                for (int i = 0; i < V; ++i) reinterpret_cast<C *>(a.last)[batch * a.wlast.b + (channel + i) * a.wlast.c] = h.v[i];
            }
        }
        if (a.time == 0 && live && p.rank == 0 && p.wt == 0 && a.last != nullptr) {
#pragma unroll
            for (int i = 0; i < V; ++i) reinterpret_cast<C *>(a.last)[batch * a.wlast.b + (channel + i) * a.wlast.c] = carry.v[i];
        }
    }
    end_exchange(shared, p);
}

template <class T, int V, int R, int COPY>
hmc_status launch_forward(hmc_context_t ctx, ForwardArgs &a, int64_t batch, int32_t flags) {
    const bool flat = COPY != 16 && flat_columns(a.channels, V);
    const Shape shape = plan_launch(batch, a.time, a.channels, flat, V, R, per_sm<T>(R), &a.columns);
    a.warps_time = shape.warps_time;
    constexpr int kShared = COPY > 0 ? kWarps * kStages * 2 * R * Ring<T, V, COPY>::kRow : 0;
    const auto go = [&](auto sigmoid, auto complement) -> hmc_status {
        static SharedKnown known;
        return launch(ctx, forward_kernel<T, V, R, COPY, decltype(sigmoid)::value, decltype(complement)::value>, known, kShared, shape, a,
                      "linear recurrence kernel launch");
    };
    return dispatch_flags(flags, go);
}

thread_local int polls_of_a_wait = kPollLimit;

}  // namespace

int wait_limit() { return polls_of_a_wait; }

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
        a.wait_limit = wait_limit();
        a.status = ctx->status;
        const bool pairs = layer_vectors(out, 4) && layer_vectors(gate, 4) && layer_vectors(x, 4);
        const bool wide = layer_vectors(gate, 16) && layer_vectors(x, 16) && layer_vectors(out, 4);
        return dispatch_float(dt, [&](auto tag) -> hmc_status {
            using T = decltype(tag);
            constexpr int kWord = sizeof(T) == 8 ? 8 : 4, V = sizeof(T) == 2 ? 2 : 1;
            if constexpr (sizeof(T) == 2) {
                if (!pairs) return time == 1 ? launch_forward<T, 1, 1, 0>(ctx, a, batch, flags) : launch_forward<T, 1, 8, 0>(ctx, a, batch, flags);
            }
            if (time == 1) return launch_forward<T, V, 1, 0>(ctx, a, batch, flags);
            const bool flat = flat_columns(channels, V), lines = wide && !flat;
            if constexpr (sizeof(T) < 8) {
                // Sixteen rows a lane halve the exchanges, two blocks an SM then: where that many blocks take all channels (bf16
                // [8, 2048, 4096]: 117 us with eight rows and four blocks an SM, 88 with sixteen; f32 [1, 65521, 1000]: 214 and 169).
                const int64_t warps = flat ? ceil_div(batch * channels, int64_t{32} * V) : batch * ceil_div(channels, int64_t{32} * V);
                if (warps <= int64_t{148} * 2 * kWarps) {
                    return lines ? launch_forward<T, V, 16, 16>(ctx, a, batch, flags) : launch_forward<T, V, 16, kWord>(ctx, a, batch, flags);
                }
            }
            return lines ? launch_forward<T, V, 8, 16>(ctx, a, batch, flags) : launch_forward<T, V, 8, kWord>(ctx, a, batch, flags);
        });
    });
}

HMC_API void hmc_test_wait_limit(int32_t polls) { polls_of_a_wait = polls >= 0 ? polls : kPollLimit; }
