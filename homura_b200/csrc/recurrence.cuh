// What the forward and the backward kernel of the gated linear recurrence share.
//
// Both are a scan v_s = c_s v_{s-1} + w_s along one axis for every (batch, channel): forward v = h, c = a, w = u in the
// order of time; backward v = g, c = the gate of the step processed before, w = dout, against the order of time (rows
// are addressed in the order they are processed, with negative strides where that runs backwards). The bound is HBM
// traffic: each element of each operand is moved once.
//
// Split. A lane owns V neighbouring channels and, per round, R neighbouring rows that it keeps in registers; a warp is
// 32 * V channels wide, so a row is one coalesced access. Of a block's eight warps WT divide the time axis among them
// and 8 / WT the channels; where batch * channels leave SMs idle, up to eight blocks of a cluster divide the time axis
// further. A round is then R * WT * cluster rows:
//   1. every lane folds its rows to (A, B): v after the rows = A * (v before) + B;
//   2. warps leave (A, B) in shared memory; the blocks of a cluster send their fold to every block of it (asynchronous
//      stores into distributed shared memory that count themselves off on the receiver's mbarrier: a cluster barrier
//      would wait for the results' stores to global memory as well);
//   3. every lane folds what lies before its rows, always in the order of time, onto the round's carry, and walks its rows
//      once more from registers, now from the true value, writing the results.
// No block waits for a block outside its cluster, nothing is read twice, and the order of the folds is fixed by the sizes.
// With WT = 1 and no cluster a lane walks its channels alone and steps 1 and 2 fall away.
#pragma once

#include <cooperative_groups.h>

#include "layers.cuh"
#include "math.cuh"

namespace hmc {
namespace recur {

namespace cg = cooperative_groups;

constexpr int kThreads = 256;
constexpr int kWarps = 8;
constexpr int kMaxCluster = 8;

template <class C> struct alignas(2 * sizeof(C)) Step {
    C a, b;
};

// A step applied to the value before it. A product of gates may have overflowed: a state of zero stays zero all the same, any
// other becomes infinite or no number, never a finite wrong one. (A NaN or infinite gate shows in b, which is folded from zero.)
// The selection lengthens the chain of folds that a lane waits for: f32 [1, 65536, 8], all of it exchanges, 106 us with products held
// at the largest number instead, 112 with it; bf16 [8, 2048, 4096] 86 and 87.
template <class C> __device__ __forceinline__ C fold(Step<C> s, C v) { return v == C(0) ? s.b : m_fma(s.a, v, s.b); }

// Rows and channels of one operand, in elements; t may be negative.
struct Walk {
    int64_t b, t, c;
};

// V values of the computation type. Pairs of f32 go through the packed instructions, two products or sums an issue.
template <class C, int V> struct Vec {
    C v[V];
};
template <class C, int V> __device__ __forceinline__ Vec<C, V> vfma(const Vec<C, V> &a, const Vec<C, V> &b, const Vec<C, V> &c) {
    Vec<C, V> r;
    if constexpr (std::is_same_v<C, float> && V == 2) {
        asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
            "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
            : "=f"(r.v[0]), "=f"(r.v[1])
            : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]), "f"(c.v[0]), "f"(c.v[1]));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = m_fma(a.v[i], b.v[i], c.v[i]);
    }
    return r;
}
template <class C, int V> __device__ __forceinline__ Vec<C, V> vmul(const Vec<C, V> &a, const Vec<C, V> &b) {
    Vec<C, V> r;
    if constexpr (std::is_same_v<C, float> && V == 2) {
        asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmul.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
            : "=f"(r.v[0]), "=f"(r.v[1])
            : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = a.v[i] * b.v[i];
    }
    return r;
}
template <class C, int V> __device__ __forceinline__ Vec<C, V> vadd(const Vec<C, V> &a, const Vec<C, V> &b) {
    Vec<C, V> r;
    if constexpr (std::is_same_v<C, float> && V == 2) {
        asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
            : "=f"(r.v[0]), "=f"(r.v[1])
            : "f"(a.v[0]), "f"(a.v[1]), "f"(b.v[0]), "f"(b.v[1]));
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = a.v[i] + b.v[i];
    }
    return r;
}
template <class C, int V> __device__ __forceinline__ Vec<C, V> splat(C c) {
    Vec<C, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = c;
    return r;
}
template <class T, int V> __device__ __forceinline__ Vec<typename Comp<T>::C, V> widen(const Pack<T, V> &p) {
    Vec<typename Comp<T>::C, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = up(p.v[i]);
    return r;
}

// a and 1 - a of V gates, each with full relative precision however close to 0 or 1 a is.
template <class C, int V> struct Gates {
    Vec<C, V> a, rest;
};
template <bool SIG, class T, int V> __device__ __forceinline__ Gates<typename Comp<T>::C, V> gates_of(Pack<T, V> stored) {
    using C = typename Comp<T>::C;
    Gates<C, V> r;
    if constexpr (!SIG) {
        r.a = widen<T, V>(stored);
#pragma unroll
        for (int i = 0; i < V; ++i) r.rest.v[i] = C(1) - r.a.v[i];
    } else if constexpr (sizeof(T) == 2) {
        // The special function unit's exponential and reciprocal: a and 1 - a to (12 + 2 |g|) 2^-24, for logits of 8 or 11 bits.
        // Where e = exp(-g) passes 2^126 the reciprocal is flushed to 0, so that a logit of -infinity forgets whatever it meets, and
        // e a is 0 or no number: 1 - a, less what its terms may be off by, is below e a everywhere else and stands in for it there.
        const Vec<C, V> g = widen<T, V>(stored), t = vmul(g, splat<C, V>(-1.44269504088896341f));
        Vec<C, V> e;
#pragma unroll
        for (int i = 0; i < V; ++i) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.v[i]) : "f"(t.v[i]));
        const Vec<C, V> all = vadd(e, splat<C, V>(1.0f));
#pragma unroll
        for (int i = 0; i < V; ++i) asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.a.v[i]) : "f"(all.v[i]));
        const Vec<C, V> product = vmul(e, r.a), low = vfma(r.a, splat<C, V>(-1.0f), splat<C, V>(1.0f - 0x1p-21f));
#pragma unroll
        for (int i = 0; i < V; ++i) r.rest.v[i] = fmaxf(product.v[i], low.v[i]);  // (no number only for a NaN logit)
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const C g = up(stored.v[i]);
            const C e = exp(-m_abs(g)), large = C(1) / (C(1) + e), small = e * large;
            r.a.v[i] = g > C(0) ? large : small;
            r.rest.v[i] = g > C(0) ? small : large;
        }
    }
    return r;
}

// V elements at p, the channels `c` elements apart (V > 1 only where c is 1 and the access aligned).
template <class T, int V> __device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
    return *reinterpret_cast<const Pack<T, V> *>(p);
}
template <class T, int V> __device__ __forceinline__ void store_pack(T *p, const Vec<typename Comp<T>::C, V> &v) {
    Pack<T, V> r;
    if constexpr (V % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < V; i += 2) down2(r.v[i], r.v[i + 1], v.v[i], v.v[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = down<T>(v.v[i]);
    }
    *reinterpret_cast<Pack<T, V> *>(p) = r;
}

// A warp's rows come through a ring in shared memory that its own asynchronous copies fill rounds ahead: no register
// holds data in flight. A copy moves COPY bytes: 16 where every row begins on such a boundary, a quarter of the
// instructions of the copies of one lane's word (4 or 8 bytes) that any layout allows. A warp waits for its own copies
// only. Elements of 2 bytes that do not pair up (odd offsets or strides) are too small for an asynchronous copy and are
// loaded to registers instead (COPY = 0), as is a single step.
template <int BYTES> __device__ __forceinline__ void copy_async(void *shared_dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(shared_dst))), "l"(src), "n"(BYTES)
                 : "memory");
}
template <int N> __device__ __forceinline__ void wait_for_all_but() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <class T, int V, int COPY> struct Ring {
    static constexpr int kRow = 32 * V * static_cast<int>(sizeof(T));  // bytes of a warp's row
    static constexpr int kCopies = COPY > 0 ? kRow / COPY : 32;        // copies a row
    static constexpr int kAtOnce = 32 / kCopies;                       // rows the warp copies with one instruction
    static constexpr int kStep = COPY > 0 ? COPY / static_cast<int>(sizeof(T)) : V;  // elements a copy
    // The row and the channel of the warp's rows that this lane copies.
    __device__ __forceinline__ static int row() { return (threadIdx.x & 31) / kCopies; }
    __device__ __forceinline__ static int channel() { return (threadIdx.x & 31) % kCopies * kStep; }
};

// `rows` rows into the ring from row `to` on, of which `there` exist; p: this lane's part of the first.
template <class T, int V, int COPY, int ROWS>
__device__ __forceinline__ void copy_rows(unsigned char *ring, int to, const T *p, int64_t stride, int there) {
    using G = Ring<T, V, COPY>;
    unsigned char *dst = ring + (to + G::row()) * G::kRow + G::channel() * static_cast<int>(sizeof(T));
    const int64_t next = stride * G::kAtOnce;
    static_assert(ROWS % G::kAtOnce == 0 || ROWS == 1, "whole instructions");
#pragma unroll
    for (int r = 0; r < ROWS; r += G::kAtOnce) {
        if (r + G::row() < there) copy_async<COPY>(dst + r * G::kRow, p);
        p += next;
    }
}

// The columns (batch, V channels) of an item. `flat`: lanes take the columns of all batches one after another, so that few
// channels, or a number that no warp divides, leave no lane idle; every lane then has a batch of its own, and copies are of
// its own word. Otherwise a warp's columns lie side by side in one batch.
struct Columns {
    int64_t channels, tiles, items;
    int64_t per_batch, all;  // flat: columns of a batch and of all batches
    int32_t flat;
};
struct Column {
    int64_t batch, channel, tile;  // tile: the warp's first channel (not flat)
    bool live;
};
template <int V> __device__ __forceinline__ Column column_of(const Columns &c, int64_t item, int warps_time, int wc, int lane) {
    Column r;
    if (c.flat) {
        const int64_t column = (item * (kWarps / warps_time) + wc) * 32 + lane;
        r.live = column < c.all;
        r.batch = r.live ? column / c.per_batch : 0;
        r.channel = r.live ? (column - r.batch * c.per_batch) * V : 0;
        r.tile = 0;
    } else {
        r.batch = item / c.tiles;
        r.tile = ((item - r.batch * c.tiles) * (kWarps / warps_time) + wc) * (32 * V);
        r.channel = r.tile + lane * V;
        r.live = r.channel < c.channels;
    }
    return r;
}

// What a launch looks like; see plan_launch.
struct Shape {
    int32_t warps_time;  // WT
    int32_t cluster;
    int64_t tiles;       // channel tiles of 8 / WT * 32 * V channels
    int64_t items;       // batch * tiles
    unsigned grid;
};

// WT and the cluster grow while every block still finds a place at once, `per_sm` on an SM, and the time axis feeds them:
// a second, partly filled wave costs more than the warps it brings (the gradients of bf16 [4, 4096, 2048] at two blocks an SM:
// 101 us with 512 blocks in clusters of four, 94 with 256 in clusters of two). The constant is B200's SM count, not the device's,
// so that the order of folding is the same everywhere.
inline Shape plan_launch(int64_t batch, int64_t time, int64_t channels, bool flat, int v, int rows, int per_sm, Columns *columns) {
    *columns = Columns{channels, 0, 0, channels / v, batch * (channels / v), flat ? 1 : 0};
    if (flat) {
        channels *= batch;
        batch = 1;
    }
    const int64_t places = int64_t{148} * per_sm;
    Shape s{1, 1, 0, 0, 0};
    const int64_t warps = batch * ceil_div(channels, int64_t{32} * v);  // (both counts are below 2^62 / (32 v))
    while (s.warps_time < kWarps && ceil_div(warps, kWarps / (s.warps_time * 2)) <= places && static_cast<int64_t>(s.warps_time) * rows < time) {
        s.warps_time *= 2;
    }
    while (s.warps_time == kWarps && s.cluster < kMaxCluster && warps * s.cluster * 2 <= places &&
           static_cast<int64_t>(s.warps_time) * s.cluster * rows < time) {
        s.cluster *= 2;
    }
    s.tiles = ceil_div(channels, int64_t{32} * v * (kWarps / s.warps_time));
    s.items = batch * s.tiles;
    columns->tiles = s.tiles;
    columns->items = s.items;
    const int64_t most = (int64_t{1} << 30) / s.cluster;
    s.grid = static_cast<unsigned>((s.items < most ? s.items : most) * s.cluster);
    return s;
}

// ---- checks of the entry points ----
inline hmc_status check_recurrence(const hmc_tensor_desc *gate, int32_t flags, int64_t *count) {
    hmc_status s = check_desc(gate, "the gate");
    if (s != HMC_OK) return s;
    if (!dtype_is_float(gate->dtype)) return fail(HMC_INVALID, "a linear recurrence needs floating point tensors");
    if (flags & ~(HMC_RECURRENCE_SIGMOID | HMC_RECURRENCE_COMPLEMENT | HMC_RECURRENCE_REVERSE)) {
        return fail(HMC_INVALID, "unknown flags of a linear recurrence");
    }
    s = check_layer(gate, "the gate", gate->dtype, 3, gate->sizes, Use::kInput);
    if (s != HMC_OK) return s;
    s = count_layer(gate->sizes, 3, count);
    if (s != HMC_OK) return s;
    const int64_t states[2] = {gate->sizes[0], gate->sizes[2]};
    int64_t ignored = 0;
    return count_layer(states, 2, &ignored);
}
inline hmc_status check_state(const hmc_tensor_desc *d, const char *what, const hmc_tensor_desc *gate, Use use) {
    if (d == nullptr) return HMC_OK;
    const int64_t sizes[2] = {gate->sizes[0], gate->sizes[2]};
    return check_layer(d, what, gate->dtype == HMC_F64 ? HMC_F64 : HMC_F32, 2, sizes, use);
}

// [batch, time, channels] in the order the rows are processed: from the last row on where that runs `backwards`.
template <class P> inline Walk walk_rows(const hmc_tensor_desc *d, bool backwards, P *base) {
    if (d == nullptr) return Walk{0, 0, 0};
    Walk w{d->strides[0], d->strides[1], d->strides[2]};
    if (backwards && d->sizes[1] > 0) {
        *base += (d->sizes[1] - 1) * w.t * element_size(d->dtype);
        w.t = -w.t;
    }
    return w;
}
inline Walk walk_state(const hmc_tensor_desc *d) { return d == nullptr ? Walk{0, 0, 0} : Walk{d->strides[0], 0, d->strides[1]}; }

// Whether the columns of all batches are laid out flat: where warps within one batch would leave a fifth of their lanes idle
// (f32 [20, 28896, 47]: 200 us in warps of one batch, 121 flat). Flat columns cannot use the 16-byte copies, which is worth
// as much (bf16 [8, 2048, 4096]: 191 us by words, 108 by lines, with otherwise the same kernel).
inline bool flat_columns(int64_t channels, int v) { return ceil_div(channels, int64_t{32} * v) * 32 * v * 4 > channels * 5; }

template <class F> hmc_status dispatch_flags(int32_t flags, F &&f) {
    using Yes = std::true_type;
    using No = std::false_type;
    switch (flags & (HMC_RECURRENCE_SIGMOID | HMC_RECURRENCE_COMPLEMENT)) {
        case 0: return f(No{}, No{});
        case HMC_RECURRENCE_SIGMOID: return f(Yes{}, No{});
        case HMC_RECURRENCE_COMPLEMENT: return f(No{}, Yes{});
        default: return f(Yes{}, Yes{});
    }
}

template <class Kernel, class Args>
hmc_status launch(hmc_context_t ctx, Kernel kernel, SharedKnown &known, int shared, const Shape &shape, const Args &args,
                  const char *what) {
    const hmc_status s = allow_shared(ctx, kernel, known, shared, what);
    if (s != HMC_OK) return s;
    cudaLaunchConfig_t config{};
    config.dynamicSmemBytes = static_cast<size_t>(shared);
    config.gridDim = dim3(shape.grid);
    config.blockDim = dim3(kThreads);
    config.stream = ctx->stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = static_cast<unsigned>(shape.cluster);
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = shape.cluster > 1 ? 1 : 0;
    cudaError_t err = cudaLaunchKernelEx(&config, kernel, args);
    if (err != cudaSuccess) return cuda_fail(err, what);
    return HMC_OK;
}

// Where a warp stands: its item's batch and first channel, its place along the time axis.
struct Place {
    int lane, wt, wc;      // lane; the warp's place among the warps along time and along channels
    int rank, cluster;     // the block's place in the cluster
    int slot;              // lane's first column in the exchange arrays
};
template <int V> __device__ __forceinline__ Place place(int warps_time) {
    Place p;
    p.lane = threadIdx.x & 31;
    const int warp = threadIdx.x >> 5;
    p.wt = warp & (warps_time - 1);
    p.wc = warp / warps_time;
    cg::cluster_group cluster = cg::this_cluster();
    p.rank = static_cast<int>(cluster.block_rank());
    p.cluster = static_cast<int>(cluster.num_blocks());
    p.slot = p.lane * V;
    return p;
}

// Shared memory of the exchange, two generations: one is written again two rounds later, behind a barrier (or the arrival
// of the next round's folds) that every reader has passed by then.
template <class C, int V> struct alignas(16) Exchange {
    Step<C> warp[2][kWarps][32 * V];
    Step<C> block[2][kMaxCluster][32 * V];
    C carry[2][kWarps][32 * V];   // by the warp's place along channels
    alignas(8) uint64_t arrived[2];
    int gave_up;                  // a thread of the block has given up a wait
};

__device__ __forceinline__ uint32_t shared_address(const void *p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// Before the first round; every thread of the cluster.
template <class C, int V> __device__ __forceinline__ void begin_exchange(Exchange<C, V> &x, const Place &p) {
    if (p.cluster == 1) return;
    if (threadIdx.x == 0) {
        for (int g = 0; g < 2; ++g) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&x.arrived[g])) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        x.gave_up = 0;
    }
    cg::this_cluster().sync();  // every block runs, its barriers stand, before anyone writes to its shared memory
}
template <class C, int V> __device__ __forceinline__ bool has_given_up(const Exchange<C, V> &x) {
    return *static_cast<const volatile int *>(&x.gave_up) != 0;
}
// After the last: no block ends while another may still write to it. A block that has seen every round's sums arrive knows of
// nothing on its way; for one that gave up, what its neighbours had sent by the barrier gets far more time than the microsecond
// that a store between blocks takes (2^14 looks, some 100 us).
template <class C, int V> __device__ __forceinline__ void end_exchange(Exchange<C, V> &x, const Place &p) {
    if (p.cluster == 1) return;
    cg::this_cluster().sync();
    if (!has_given_up(x)) return;
#pragma unroll 1
    for (int look = 0; look < 1 << 14; ++look) {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%0], 0;\n\t}" ::"r"(shared_address(&x.arrived[look & 1]))
                     : "memory");
    }
}

// One lane's V steps to the same place of another block, counted off on that block's mbarrier.
template <class C, int V> __device__ __forceinline__ void send(const Step<C> *mine, uint64_t *arrived, int block, const Pack<Step<C>, V> &value) {
    uint32_t to, at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(shared_address(mine)), "r"(block));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(shared_address(arrived)), "r"(block));
    constexpr int kWords = static_cast<int>(sizeof(Step<C>)) * V / 8;
    uint64_t w[kWords];
    memcpy(w, &value, sizeof w);
    if constexpr (kWords == 1) {
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to), "l"(w[0]), "r"(at) : "memory");
    } else {
        static_assert(kWords == 2, "one or two words");
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%1, %2}, [%3];" ::"r"(to), "l"(w[0]), "l"(w[1]), "r"(at)
                     : "memory");
    }
}

constexpr int kPollLimit = 1 << 22;
// Polls of a wait: kPollLimit, or what the calling thread has set for its tests (hmc_test_wait_limit).
int wait_limit();

// A wait for the sums of a round that gives up after `limit` polls. `status` is the context's word. A block of which a thread has
// given up waits no more and, from the next round on, sends no more and expects no more: a neighbour that misses its sums gives
// up in turn, and nobody touches a barrier or sums of a round that its block has not seen complete. (The barriers of the whole
// cluster at the kernel's begin and end are the hardware's, among blocks that run at the same time.)
template <class C, int V> __device__ __forceinline__ void await(Exchange<C, V> &x, uint32_t generation, uint32_t parity, int limit, int *status) {
    const uint32_t at = shared_address(&x.arrived[generation]);
#pragma unroll 1
    for (int poll = 0; poll < limit; ++poll) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(at), "r"(parity)
            : "memory");
        if (done) return;
        if (has_given_up(x)) return;
    }
    *static_cast<volatile int *>(&x.gave_up) = 1;
    atomicExch(status, 1);
}

// Step 2 and the folds of step 3: (a, b) is what this lane's rows do; v enters as the item's first value and leaves as the
// value before this lane's rows. `round` counts all rounds of the block. Within a block a round's first value is what the last
// warp along time ended the round before with (left by leave_carry); a cluster folds every block's sum onto the carry that each
// lane keeps.
template <class C, int V>
__device__ __forceinline__ void exchange(Exchange<C, V> &x, const Place &p, int warps_time, uint32_t round, bool first_round,
                                         const Vec<C, V> &a, const Vec<C, V> &b, Vec<C, V> &v, Vec<C, V> &carry, int limit, int *status) {
    using Pair = Pack<Step<C>, V>;
    const uint32_t generation = round & 1u;
    Step<C>(&warps)[kWarps][32 * V] = x.warp[generation];
    const auto at = [&](const Step<C> (&row)[32 * V]) { return *reinterpret_cast<const Pair *>(&row[p.slot]); };
    const int first = p.wc * warps_time;
    {
        Pair mine_packed;
#pragma unroll
        for (int i = 0; i < V; ++i) mine_packed.v[i] = Step<C>{a.v[i], b.v[i]};
        *reinterpret_cast<Pair *>(&warps[first + p.wt][p.slot]) = mine_packed;
    }
    __syncthreads();
    if (p.cluster > 1) {
        if (threadIdx.x == 0 && !has_given_up(x)) {
            asm volatile("mbarrier.arrive.expect_tx.release.cta.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(&x.arrived[generation])),
                         "r"(static_cast<uint32_t>(p.cluster * 32 * V * sizeof(Step<C>)))
                         : "memory");
        }
        // (a cluster is used with all eight warps along time only, so a block has one tile of channels; warp w brings the
        // block's fold to block w)
        if (p.wt < p.cluster && !has_given_up(x)) {
            Pair t = at(warps[0]);
#pragma unroll
            for (int w = 1; w < kWarps; ++w) {
                const Pair s = at(warps[w]);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    t.v[i].b = fold(s.v[i], t.v[i].b);
                    t.v[i].a *= s.v[i].a;
                }
            }
            send<C, V>(&x.block[generation][p.rank][p.slot], &x.arrived[generation], p.wt, t);
        }
        await(x, generation, (round >> 1) & 1u, limit, status);
#pragma unroll 4
        for (int k = 0; k < p.cluster; ++k) {
            const Pair s = at(x.block[generation][k]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if (k == p.rank) v.v[i] = carry.v[i];
                carry.v[i] = fold(s.v[i], carry.v[i]);
            }
        }
    } else if (!first_round) {
        const Pack<C, V> c = *reinterpret_cast<const Pack<C, V> *>(&x.carry[generation][p.wc][p.slot]);
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[i] = c.v[i];
    }
#pragma unroll 4
    for (int w = 0; w < p.wt; ++w) {
        const Pair s = at(warps[first + w]);
#pragma unroll
        for (int i = 0; i < V; ++i) v.v[i] = fold(s.v[i], v.v[i]);
    }
}
// The last warp along time leaves its last value for the next round of the block.
template <class C, int V>
__device__ __forceinline__ void leave_carry(Exchange<C, V> &x, const Place &p, int warps_time, uint32_t round, const Vec<C, V> &v) {
    if (p.cluster > 1 || p.wt != warps_time - 1) return;
    Pack<C, V> c;
#pragma unroll
    for (int i = 0; i < V; ++i) c.v[i] = v.v[i];
    *reinterpret_cast<Pack<C, V> *>(&x.carry[(round + 1) & 1u][p.wc][p.slot]) = c;
}

}  // namespace recur
}  // namespace hmc
