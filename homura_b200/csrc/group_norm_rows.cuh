// Group norm where a group of one sample fits the registers of a team of lanes: every token by itself (one position), or
// few positions. One pass: a value is read once and written once (bf16 [32768, 1, 4096] in 32 groups: 1473 us in tiles of rows
// with a block's sums for every sample, 107 to 115 here).
//
// A team is a power of two of lanes within a warp (or, WIDE, the whole block); a lane keeps K vectors of V neighbouring
// channels of its team's group, the same channels for every sample it takes, so parameters (and, backward, the sums for
// dweight and dbias) stay in registers across samples. The next samples' vectors come through a ring in shared
// memory that a lane's own asynchronous copies fill rounds ahead (a lane reads only what it copied: waiting for its copies is
// all the synchronisation). Sums go through shuffles within the team.
#pragma once

#include "group_norm.cuh"

namespace hmc {
namespace gnorm {

// A lane's vectors at most: 32 values forward, 16 backward, where the sums for dweight and dbias stand beside them, in at
// most eight vectors of 16 bytes or sixteen words (es: bytes of an element).
constexpr int most_vectors(int v, int es, bool backward) {
    const int most = (backward ? 16 : 32) / v, narrow = v * es < 16 ? 16 : 8;
    return most < narrow ? most : narrow;
}

struct Teams {
    int32_t lanes;            // lanes a team
    int32_t k;                // vectors a lane
    int32_t vectors;          // vectors of a group: positions * cg / V
    int32_t row_vectors;      // cg / V
    int32_t groups_per_tile;  // groups side by side in a block
    int32_t samples_at_once;  // samples side by side in a block
    int64_t tiles;
    int32_t v;                // 0: the group does not fit
    bool wide;
};

// K as it is compiled (dispatch_vectors).
constexpr int compiled_k(int k, int v, int es, bool backward) {
    const int most = most_vectors(v, es, backward);
    int c = v * es == 16 ? 1 : 4;
    while (c < k) c *= 2;
    return c < most ? c : most;
}
// The widest team that wastes least: lanes * compiled K as small as possible, lanes as many as possible for coalescing.
inline Teams make_teams(const Problem &p, Align align, bool backward) {
    Teams t{};
    const int64_t cg = p.channels / p.groups;
    const int es = element_size(p.dtype), vector = 16 / es, word = narrow_vector(es);
    const int v = align == Align::kLine && cg % vector == 0 ? vector : (align != Align::kAny && cg % word == 0 ? word : 1);
    const int most_k = most_vectors(v, es, backward);
    const int64_t most = static_cast<int64_t>(kBlock) * most_k;
    if (p.positions > most || cg / v > most || p.positions * (cg / v) > most) return t;
    t.v = v;
    t.vectors = static_cast<int32_t>(p.positions * (cg / v));
    t.row_vectors = static_cast<int32_t>(cg / v);
    // Words of several rows are read in small pieces, at some 150 GB/s; a cluster reads them side by side but spends
    // about 4 us a sample on two blocks an SM, which only samples of about 2 KB (all operands) do not repay.
    if (v < vector && p.positions > 1 && p.positions * p.channels * es * (backward ? 3 : 2) > 2048) {
        t.v = 0;
        return t;
    }
    if (t.vectors > 32 * most_k) {
        if (p.positions > 1) {  // the tiled kernels read several rows of wide groups side by side
            t.v = 0;
            return t;
        }
        t.wide = true;
        t.lanes = kBlock;
        t.k = (t.vectors + kBlock - 1) / kBlock;
    } else {
        int best = 0;
        for (int lanes = 32; lanes >= 1; lanes >>= 1) {
            const int k = (t.vectors + lanes - 1) / lanes;
            if (k > most_k) break;
            const int cost = lanes * compiled_k(k, v, es, backward);
            if (best == 0 || cost < best) {
                best = cost;
                t.lanes = lanes;
                t.k = k;
            }
        }
    }
    const int64_t teams = kBlock / t.lanes;
    t.groups_per_tile = static_cast<int32_t>(p.groups < teams ? p.groups : teams);
    t.samples_at_once = static_cast<int32_t>(teams / t.groups_per_tile);
    t.tiles = ceil_div(p.groups, t.groups_per_tile);
    return t;
}
// Samples a lane takes at once.
constexpr int samples_at_a_time(int k) { return k == 1 ? 2 : 1; }

// Sums `s` over the team; every lane gets the same.
template <int U, bool WIDE, class C> __device__ __forceinline__ void team_sum(C (&s)[U], int lanes, C (*scratch)[kWarps]) {
    if constexpr (WIDE) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) s[u] += __shfl_xor_sync(0xFFFFFFFFu, s[u], d);
            if (lane == 0) scratch[u][warp] = s[u];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = scratch[u][0];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) s[u] += scratch[u][w];
        }
        __syncthreads();
    } else {
        for (int d = lanes >> 1; d > 0; d >>= 1) {
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] += __shfl_xor_sync(0xFFFFFFFFu, s[u], d);
        }
    }
}

// V parameters from channel `at` on, or `otherwise` where there are none.
template <class T, int V> __device__ __forceinline__ void parameters(typename Comp<T>::C (&to)[V], const char *p, int64_t at, int64_t stride,
                                                                     int is_f32, typename Comp<T>::C otherwise) {
    using C = typename Comp<T>::C;
    if (p == nullptr) {
#pragma unroll
        for (int i = 0; i < V; ++i) to[i] = otherwise;
        return;
    }
    if constexpr (V > 1) {
        if (stride == 1 && reinterpret_cast<uintptr_t>(p) % 16 == 0) {  // (at is a multiple of V)
            if (is_f32) {
                constexpr int kHalf = V < 4 ? V : 4;
#pragma unroll
                for (int h = 0; h < V; h += kHalf) {
                    const Pack<float, kHalf> w = *reinterpret_cast<const Pack<float, kHalf> *>(reinterpret_cast<const float *>(p) + at + h);
#pragma unroll
                    for (int i = 0; i < kHalf; ++i) to[h + i] = static_cast<C>(w.v[i]);
                }
            } else {
                const Pack<T, V> w = *reinterpret_cast<const Pack<T, V> *>(reinterpret_cast<const T *>(p) + at);
#pragma unroll
                for (int i = 0; i < V; ++i) to[i] = up(w.v[i]);
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) to[i] = parameter<T>(p, (at + i) * stride, is_f32);
}

template <class T, int V> __device__ __forceinline__ Pack<T, V> pack_of(const typename Comp<T>::C (&v)[V]) {
    Pack<T, V> r;
    if constexpr (V % 2 == 0 && sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < V; i += 2) down2(r.v[i], r.v[i + 1], v[i], v[i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = down<T>(v[i]);
    }
    return r;
}

// `WORDS` vectors (of 4, 8 or 16 bytes) a lane and round; single values of 2 bytes, for which there is no asynchronous copy,
// are loaded to registers a round ahead.
template <class T, int V, int WORDS> struct RowRing {
    static constexpr int kSize = static_cast<int>(sizeof(T)) * V;
    static constexpr bool kUsed = kSize >= 4;
    static constexpr int kRound = WORDS * kBlock * kSize;  // bytes a block and round
    static constexpr int kStages = !kUsed ? 1 : (kRound * 4 <= 49152 ? 4 : (kRound * 3 <= 49152 ? 3 : 2));
    static constexpr int kBytes = kUsed ? kStages * kRound : 0;
    Pack<T, V> direct[kUsed ? 1 : WORDS];
    unsigned char *mine;
    __device__ __forceinline__ explicit RowRing(unsigned char *memory) : mine(memory + threadIdx.x * kSize) {}
    __device__ __forceinline__ void fetch(int stage, int word, const T *p) {
        if constexpr (kUsed) copy_async<kSize>(mine + (stage * WORDS + word) * (kBlock * kSize), p);
        else direct[word] = *reinterpret_cast<const Pack<T, V> *>(p);
    }
    // After the copies of a round; then, before the first read of the oldest round in flight.
    __device__ __forceinline__ void commit() const {
        if constexpr (kUsed) async_copy_commit();
    }
    __device__ __forceinline__ void wait() const {
        if constexpr (kUsed) asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    }
    __device__ __forceinline__ Pack<T, V> get(int stage, int word) const {
        if constexpr (kUsed) return *reinterpret_cast<const Pack<T, V> *>(mine + (stage * WORDS + word) * (kBlock * kSize));
        else return direct[word];
    }
};

struct RowsForwardArgs {
    char *out;
    const char *src;
    Rows wout, wsrc;
    Teams t;
    int64_t samples, groups, cg;
    Affine affine;
    char *mean, *rstd;  // or null
    int64_t mean_n, mean_g, rstd_n, rstd_g;
    double eps;
};
struct RowsBackwardArgs {
    char *dsrc;
    const char *src, *dout, *mean, *rstd;
    Rows wdsrc, wsrc, wdout;
    int64_t mean_n, mean_g, rstd_n, rstd_g;
    Teams t;
    int64_t samples, positions, groups, cg, channels;
    int64_t run;        // samples a team takes
    Affine affine;
    void *by_channel;   // C [row blocks * samples_at_once * positions][2][channels], or null
};

// One launch; the group of a sample fits a team (t.v > 0). dispatch.
hmc_status launch_rows_forward(hmc_context_t ctx, int dtype, int32_t activation, const RowsForwardArgs &a);
hmc_status launch_rows_backward(hmc_context_t ctx, int dtype, int32_t activation, const RowsBackwardArgs &a, int64_t row_blocks);

// f(V, K, WIDE) as compile-time constants. K is the next of 1, 2, 4 and 8, of 4, 8 and 16 for words and single values; 2 at
// least, or the most, for a block.
template <class T, bool BACKWARD, int V, class F> inline hmc_status dispatch_vectors(const Teams &t, F &&f) {
    constexpr int kMost = most_vectors(V, sizeof(T), BACKWARD);
    constexpr bool kLines = V * sizeof(T) == 16;
    const auto with = [&](auto k, auto wide) { return f(std::integral_constant<int, V>{}, k, wide); };
    if (t.wide) {
        if constexpr (kLines) {
            if (t.k <= 2) return with(std::integral_constant<int, 2>{}, std::true_type{});
        }
        return with(std::integral_constant<int, kMost>{}, std::true_type{});
    }
    if constexpr (kLines) {
        if (t.k <= 1) return with(std::integral_constant<int, 1>{}, std::false_type{});
        if (t.k <= 2) return with(std::integral_constant<int, 2>{}, std::false_type{});
    }
    if constexpr (kMost > 4) {
        if (t.k <= 4) return with(std::integral_constant<int, 4>{}, std::false_type{});
    }
    if constexpr (kMost > 8) {
        if (t.k <= 8) return with(std::integral_constant<int, 8>{}, std::false_type{});
    }
    return with(std::integral_constant<int, kMost>{}, std::false_type{});
}
template <class T, bool BACKWARD, class F> inline hmc_status dispatch_teams(const Teams &t, F &&f) {
    if (t.v == kVector<T>) return dispatch_vectors<T, BACKWARD, kVector<T>>(t, f);
    if constexpr (sizeof(T) == 2) {
        if (t.v == 2) return dispatch_vectors<T, BACKWARD, 2>(t, f);
    }
    return dispatch_vectors<T, BACKWARD, 1>(t, f);
}

}  // namespace gnorm
}  // namespace hmc
