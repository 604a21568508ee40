// awa_cache_join.cuh -- several blocks of a cluster share the keys of a tile of
// query rows: how many, and how their parts become the result. For the fp32
// cache kernels.
#pragma once

#include "awa_cache_device.cuh"
#include "awa_rows.cuh"

#include <cooperative_groups.h>

namespace awa
{

// Writes the rows of tile t of key/value head kv. Every block of the cluster has
// in its shared memory, in the same places, its unscaled O, part_o[row][pitch],
// and (m, l), part_ml[row] (written by its THREADS threads, not yet synchronised);
// they are joined in the order of the ranks, each block taking a share.
template <typename T, int THREADS>
__device__ __forceinline__ void join_cluster(const CacheAttnArgs& a, const QueryTile& t, int kv, int d, int rank,
                                             int cluster_size, float* part_o, int pitch, float2* part_ml)
{
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    T* out = static_cast<T*>(a.out);
    cluster.sync();
    for (int i = rank * THREADS + threadIdx.x; i < t.count * (d / 4); i += cluster_size * THREADS)
    {
        const int r = i / (d / 4), f = (i - r * (d / 4)) * 4;
        float top = -INFINITY;
        for (int c = 0; c < cluster_size; c++)
            top = fmaxf(top, cluster.map_shared_rank(part_ml, c)[r].x);
        const float base = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < cluster_size; c++)
        {
            const float2 ml = cluster.map_shared_rank(part_ml, c)[r];
            const float w = fast_exp2(ml.x - base);
            const float4 x = *reinterpret_cast<const float4*>(cluster.map_shared_rank(part_o, c) + r * pitch + f);
            total = fmaf(ml.y, w, total);
            acc.x = fmaf(x.x, w, acc.x);
            acc.y = fmaf(x.y, w, acc.y);
            acc.z = fmaf(x.z, w, acc.z);
            acc.w = fmaf(x.w, w, acc.w);
        }
        const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
        const int m = t.m0 + r;
        T* dst = out + (int64_t)(t.row0 + m / a.group) * a.out_stride + (int64_t)(kv * a.group + m % a.group) * d + f;
        store1(dst, acc.x * inv);
        store1(dst + 1, acc.y * inv);
        store1(dst + 2, acc.z * inv);
        store1(dst + 3, acc.w * inv);
    }
    cluster.sync();  // a block's shared memory stays until every peer has read it
}

// Blocks that share a tile's keys, at most 8 (the portable cluster size), for
// tiles of `tile` of the batch's rows (row and head of a group) and key blocks of
// `keys`. An SM's blocks share its arithmetic units, so what counts is the most
// that one SM gets of them, times the length of each -- plus what a block pays
// for its start and the join, start_blocks blocks of keys.
inline int cluster_of(const CacheAttnArgs& a, int64_t rows, int tile, int keys, double start_blocks)
{
    const int64_t most = (((int64_t)a.batch.table_width << a.mem.page_shift) + keys - 1) / keys;
    const int64_t full = (rows + tile - 1) / tile + a.batch.sequences / 2;
    int cluster = 1;
    double best = 1e30;
    for (int c = 1; c <= 8; c *= 2)
    {
        const double cost =
            (double)((full * a.mem.heads * c + 147) / 148) / c + start_blocks * c / (double)(most > 0 ? most : 1);
        if (cost < best)
        {
            best = cost;
            cluster = c;
        }
    }
    return cluster;
}

}  // namespace awa
