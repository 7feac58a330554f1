// Group norm where the rows of a tile of groups fit the shared memory of a cluster: one pass, a value is read from HBM once
// and written once.
//
// The positions of one sample are divided among the blocks of a cluster (one to eight). A thread copies its own column of
// 16-byte vectors (of words of 4 bytes where rows or groups are not that regular, 8 for F64) into shared memory
// asynchronously and reads only what it copied. What a thread finds for its
// channels (over at most 64 rows at a time in the computation type) is laid out by group in shared memory, summed by a warp a
// group in f64, and goes to the other blocks through distributed shared memory, where every block folds it in rank order.
// That is one exchange a sample, whatever the direction.
#pragma once

#include <cooperative_groups.h>

#include "group_norm_rows.cuh"

namespace hmc {
namespace gnorm {

namespace cg = cooperative_groups;

constexpr int kResidentCluster = 8;
constexpr int kResidentShared = 216 * 1024;   // dynamic shared memory of a block at most
constexpr int kResidentWanted = 112 * 1024;   // two blocks an SM

struct Resident {
    Tiling t;           // v = 0: does not fit
    int32_t cluster;
    int64_t run;        // positions a block
    int32_t slots;      // rows a thread keeps
    int32_t data_bytes; // of one operand
    int32_t shared;
};

// Against the pieces merged by a second kernel: f16 [16, 4096, 320] in 32 groups 82 us in pieces, 43 here; f32 [487, 384, 58] in 2
// groups (by words) 97 and 28. `operands` tensors are kept. Tiles are made wide enough for whole 128-byte lines where the groups allow, and, where
// there are few positions, as wide as gives a block some tens of KB of work.
inline Resident make_resident(const Problem &p, int vector, int operands) {
    Resident r{};
    if (p.channels % vector != 0 || p.positions < 2 || p.positions > (int64_t{1} << 20)) return r;
    // (forward, squares are summed in f64, which leaves nothing to spare for F64's own moments: their pieces are merged pairwise)
    if (operands == 1 && p.dtype == HMC_F64) return r;
    const int es = element_size(p.dtype);
    const Tiling full = make_tiling(p.channels, p.groups, vector, true);
    if (full.v != vector || full.segments != 1) return r;
    const int64_t cg = full.cg;
    int64_t unit = 1;  // groups after which a channel is a multiple of the vector again
    while (unit * cg % vector != 0) ++unit;
    const auto shape = [&](int64_t per, int cluster) -> Resident {
        Resident s{};
        s.t = full;
        if (per > p.groups) per = p.groups;
        s.t.groups_per_tile = static_cast<int32_t>(per);
        s.t.tile = static_cast<int32_t>(per * cg);
        s.t.tiles = ceil_div(p.groups, per);
        s.t.tx = s.t.tile / vector;
        s.t.ty = kBlock / s.t.tx;
        s.cluster = cluster;
        s.run = ceil_div(p.positions, cluster);
        const int64_t slots = ceil_div(s.run, s.t.ty), data = ceil_div(slots * kBlock * vector * es, 16) * 16;
        const int64_t rest = kBlock * vector * 2 * (es == 8 ? 8 : 4) + 2 * cluster * per * 16 + per * 16 + 64;
        if (data * operands + rest > kResidentShared) {
            s.t.v = 0;
            return s;
        }
        s.slots = static_cast<int32_t>(slots);
        s.data_bytes = static_cast<int32_t>(data);
        s.shared = static_cast<int32_t>(data * operands + rest);
        return s;
    };
    // the widest tile of which one block holds all positions comfortably, if that is at least a line wide
    const int64_t line = ceil_div(ceil_div(128, es), unit * cg) * unit;
    const int64_t widest = full.groups_per_tile;
    int64_t per = 48 * 1024 / operands / es / cg / p.positions / unit * unit;
    if (per > widest) per = widest;
    if (per >= line || per >= p.groups) {
        r = shape(per < 1 ? 1 : per, 1);
        if (r.t.v > 0) {
            // few samples: narrower tiles, down to a line, so that there are blocks enough
            while (p.samples * r.t.tiles < 148 * 2 && r.t.groups_per_tile >= 2 * line) {
                const Resident s = shape(r.t.groups_per_tile / 2 / unit * unit, 1);
                if (s.t.v == 0) break;
                r = s;
            }
        }
    } else {
        for (int64_t width = line < widest ? line : widest;;) {
            for (int cluster = 1; cluster <= kResidentCluster; cluster *= 2) {
                r = shape(width, cluster);
                if (r.t.v > 0 && r.shared <= kResidentWanted) break;
            }
            if (r.t.v > 0 || width <= unit) break;
            width = width / 2 / unit * unit < unit ? unit : width / 2 / unit * unit;  // (then rows of less than a line)
        }
        if (r.t.v == 0) return r;
    }
    // few samples and tiles: more blocks to a cluster, while each keeps some rows
    while (r.t.v > 0 && r.cluster < kResidentCluster && p.samples * r.t.tiles * r.cluster < 148 * 2 && r.run > 4 * r.t.ty) {
        const Resident s = shape(r.t.groups_per_tile, r.cluster * 2);
        if (s.t.v == 0) break;
        r = s;
    }
    return r;
}

inline Resident find_resident(const Problem &p, Align align, int operands) {
    const int es = element_size(p.dtype);
    if (align == Align::kLine) {
        const Resident r = make_resident(p, 16 / es, operands);
        if (r.t.v > 0) return r;
    }
    if (align != Align::kAny) return make_resident(p, narrow_vector(es), operands);
    return Resident{};
}

struct Memory {  // a block's dynamic shared memory
    unsigned char *data;   // [operands][slots][kBlock] vectors (or words)
    void *columns;         // Two<C> [groups of the tile][rows at a time * channels of a group]: what the threads found
    Two<double> *slots;    // [2][cluster][groups of the tile]
    Two<double> *folded;   // [groups of the tile]
};
template <class C, int V> __device__ __forceinline__ Memory carve(unsigned char *memory, const Resident &r, int operands) {
    Memory m;
    m.data = memory;
    m.columns = memory + static_cast<int64_t>(r.data_bytes) * operands;
    m.slots = reinterpret_cast<Two<double> *>(static_cast<unsigned char *>(m.columns) + kBlock * V * sizeof(Two<C>));
    m.folded = m.slots + 2 * r.cluster * r.t.groups_per_tile;
    return m;
}

// A thread's place in the columns for its V channels: of channel i at[i], in group[i] of the tile.
template <int V> struct Columns {
    int at[V], group[V];
    __device__ __forceinline__ Columns(const Tile &tile, int tx, int ty, int rows) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            group[i] = (tx * V + i) / tile.part;
            at[i] = (group[i] * rows + ty) * tile.part + (tx * V + i - group[i] * tile.part);
        }
    }
};
// done(q, sum over group q's columns of value(column)) once for each group of the tile, always adding in the same order: a
// thread a group where a group has few values, otherwise a warp.
template <class C, class F, class G> __device__ __forceinline__ void fold_columns(const void *columns, const Tile &tile, int rows, F &&value, G &&done) {
    const int values = tile.part * rows;
    const Two<C> *c = reinterpret_cast<const Two<C> *>(columns);
    if (values <= 16) {
        for (int q = threadIdx.x; q < tile.groups; q += kBlock) {
            Two<double> sum{0.0, 0.0};
            for (int e = 0; e < values; ++e) {
                const Two<double> v = value(c[q * values + e], e);
                sum.a += v.a;
                sum.b += v.b;
            }
            done(q, sum);
        }
    } else {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        for (int q = warp; q < tile.groups; q += kWarps) {
            Two<double> sum{0.0, 0.0};
#pragma unroll 4
            for (int e = lane; e < values; e += 32) {
                const Two<double> v = value(c[q * values + e], e);
                sum.a += v.a;
                sum.b += v.b;
            }
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) {
                sum.a += __shfl_xor_sync(0xFFFFFFFFu, sum.a, d);
                sum.b += __shfl_xor_sync(0xFFFFFFFFu, sum.b, d);
            }
            if (lane == 0) done(q, sum);
        }
    }
}

// Leaves this block's sums of group q in slot [generation][rank][q] of every block of the cluster.
__device__ __forceinline__ void leave(const Memory &m, const Resident &r, int generation, int rank, int q, Two<double> value) {
    Two<double> *mine = m.slots + (generation * r.cluster + rank) * r.t.groups_per_tile + q;
    if (r.cluster == 1) {
        *mine = value;
        return;
    }
    cg::cluster_group cluster = cg::this_cluster();
    for (int k = 0; k < r.cluster; ++k) *cluster.map_shared_rank(mine, k) = value;
}
__device__ __forceinline__ void meet(const Resident &r) {
    if (r.cluster == 1) __syncthreads();
    else cg::this_cluster().sync();
}
// The sums of all blocks, in rank order.
__device__ __forceinline__ Two<double> gather(const Memory &m, const Resident &r, int generation, int q) {
    Two<double> s{0.0, 0.0};
    for (int k = 0; k < r.cluster; ++k) {
        const Two<double> v = m.slots[(generation * r.cluster + k) * r.t.groups_per_tile + q];
        s.a += v.a;
        s.b += v.b;
    }
    return s;
}

template <class Kernel, class Args>
hmc_status launch_resident(hmc_context_t ctx, Kernel kernel, SharedKnown &known, int64_t clusters, const Resident &r, const Args &args,
                           const char *what) {
    const hmc_status s = allow_shared(ctx, kernel, known, kResidentShared, what);
    if (s != HMC_OK) return s;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(clusters * r.cluster));
    config.blockDim = dim3(kBlock);
    config.dynamicSmemBytes = static_cast<size_t>(r.shared);
    config.stream = ctx->stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = static_cast<unsigned>(r.cluster);
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    config.attrs = attribute;
    config.numAttrs = r.cluster > 1 ? 1 : 0;
    cudaError_t err = cudaLaunchKernelEx(&config, kernel, args);
    if (err != cudaSuccess) return cuda_fail(err, what);
    return HMC_OK;
}

struct ResidentForwardArgs {
    char *out;
    const char *src;
    Rows wout, wsrc;
    Resident r;
    int64_t samples, positions;
    Affine affine;
    char *mean, *rstd;  // or null
    int64_t mean_n, mean_g, rstd_n, rstd_g;
    double eps;
};
struct ResidentBackwardArgs {
    char *dsrc;
    const char *src, *dout, *mean, *rstd;
    Rows wdsrc, wsrc, wdout;
    int64_t mean_n, mean_g, rstd_n, rstd_g;
    Resident r;
    int64_t samples, positions;
    int64_t columns;      // clusters that share a tile
    Affine affine;
    void *by_channel;     // C [columns * cluster][2][channels], or null
};
hmc_status launch_resident_forward(hmc_context_t ctx, int dtype, int32_t activation, const ResidentForwardArgs &a);
hmc_status launch_resident_backward(hmc_context_t ctx, int dtype, int32_t activation, const ResidentBackwardArgs &a);

}  // namespace gnorm
}  // namespace hmc
