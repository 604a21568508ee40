// awa_cache_attn_f32.cu -- attention of many rows over an fp32 key/value cache
// with head_dim 64 or 128, to fp32 accuracy on the tensor cores.
//
// A float of 24 significant bits is the sum of three bf16 numbers of 8 bits,
// x = h + m + l with |m| <= 2^-8 |x|, |l| <= 2^-16 |x|, exactly (but for bits
// below bf16's smallest number, 2^-133). Of the nine products of two such sums
// six are taken, in fp32 sums:
//   x y = h h' + (h m' + m h') + (m m' + h l' + l h') + <= 2^-23 |x y|,
// and what is left out is within what one fp32 rounding each of x, y and x y
// moves. The tensor cores cut their fp32 sums off instead of rounding them, so
// sums are kept short: the large products of a score (h h') and the small ones
// are summed apart, and P V of a block of keys starts from 0 and is added to
// O 2^(m - m') by an FMA. Softmax as everywhere: one pass, running maximum and
// sum, base 2, fp32.
//
// Six products at the mma.sync rate (1024 FMAs a clock and SM) are 4/3 of the
// 128 FMAs a clock that the FMA units do, with far fewer loads from shared
// memory per FMA. Measured (B200): 512 rows of 20 heads over 1594 keys 141 us, 31
// TFLOP/s of fp32 (236 us with FMAs). The products' own time is 45 us: they keep
// the tensor pipe 0.48 of the time busy; two warps a scheduler do not cover the
// latency of their MMAs, softmax and splitting, and the registers (255) allow no
// more.
#include "awa_cache_join.cuh"
#include "awa_mma.cuh"

#include <cuda_bf16.h>

namespace awa
{
namespace
{

constexpr int kThreads = 128;  // 4 warps of 16 query rows
constexpr int kRows = 64;
constexpr int kKeys = 32;  // a block of keys

// Shared memory of a block: the keys and values of one block as they come, and
// split in three planes each of bf16 rows, 16 bytes apart from a multiple of 128
// so that the 8 rows of an ldmatrix fall on different banks.
template <int D>
struct Shared
{
    static constexpr int kPitch = D + 8;                    // bf16 of a row of a plane
    static constexpr int kPlane = kKeys * kPitch * 2;       // bytes
    static constexpr int kRaw = kKeys * D * 4;              // bytes, of keys or values
    static constexpr int kPlanes = 2 * kRaw;                // offset of the planes: keys h, m, l, values h, m, l
    static constexpr int kQueries = kPlanes + 6 * kPlane;   // offset of the queries' l as the lanes hold it
    static constexpr int kBytes = kQueries + (D / 16) * kThreads * 16;
    static constexpr int kPartPitch = D + 4;                // floats of a row of O, over the planes
    static_assert(kRows * kPartPitch * 4 <= 6 * kPlane, "O of a tile fits over the planes");
    static_assert(kRows * 8 <= 2 * kRaw, "m and l of a tile fit over the copies");
};

// Two floats as three pairs of bf16.
__device__ __forceinline__ void split(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l)
{
    // the largest floats would round to infinity
    asm("cvt.rn.satfinite.bf16x2.f32 %0, %1, %2;" : "=r"(h) : "f"(y), "f"(x));
    x -= __uint_as_float(h << 16);
    y -= __uint_as_float(h & 0xffff0000u);
    m = pack_bf16x2(x, y);
    x -= __uint_as_float(m << 16);
    y -= __uint_as_float(m & 0xffff0000u);
    l = pack_bf16x2(x, y);
}

__device__ __forceinline__ void product(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    mma(c, a[0], a[1], a[2], a[3], b0, b1);
}

// A block (of a cluster of gridDim.x / tiles that share the keys) takes one tile
// of 64 query rows of one key/value head, a warp 16 of them over all the block's
// keys: lane (g, c) = (lane / 4, lane % 4) holds rows g and g + 8 of S and O at
// columns 2 c, 2 c + 1 of every 8. Two blocks an SM work under each other's
// splitting, softmax and barriers.
template <int D>
__global__ void __launch_bounds__(kThreads, 2) cache_attention_f32_kernel(CacheAttnArgs a, int cluster_size)
{
    using S = Shared<D>;
    extern __shared__ float4 shared4[];
    __shared__ QueryTile tile_s;
    const CacheMemory& mem = a.mem;
    char* const shared = reinterpret_cast<char*>(shared4);
    const uint32_t raw = shared_address(shared), planes = raw + S::kPlanes;
    const int rank = blockIdx.x % cluster_size;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (warp == 0)
    {
        const QueryTile t =
            find_tile(mem, a.batch, a.group, kRows, blockIdx.x / cluster_size, rank == 0 ? a.error_flag : nullptr);
        if (lane == 0)
            tile_s = t;
    }
    __syncthreads();
    const QueryTile t = tile_s;
    if (t.b < 0)
        return;  // the whole cluster
    const int kv = blockIdx.y;
    const RowSpan first = row_span(t.past + t.m0 / a.group, t.length, a.sinks, a.window, a.frame_tokens);
    const RowSpan last =
        row_span(t.past + (t.m0 + t.count - 1) / a.group, t.length, a.sinks, a.window, a.frame_tokens);
    const KeyBlocks blocks = key_blocks(first, last, a.sinks, kKeys);
    const auto first_key = [&](int n) { return (n < blocks.prefix ? n : n + blocks.shift) * kKeys; };

    // Page of key `lane` of block n, -1 for what no row of the tile sees: such
    // keys are not read, their page may be gone.
    const auto page_of_lane = [&](int n) {
        if (n >= blocks.count)
            return -1;
        const int key = first_key(n) + lane;
        if (key >= last.hi || (key < first.lo && key >= a.sinks))
            return -1;
        return page_of(mem, a.batch, t.b, key, a.error_flag);
    };
    // A thread copies, and later splits, the same 16-byte pieces of the rows.
    constexpr int kPieces = D / 4, kRowsAtOnce = kThreads / kPieces;
    const int piece = threadIdx.x % kPieces, row0 = threadIdx.x / kPieces;
    const auto fetch = [&](int n, int page_lane) {
        const int key0 = first_key(n);
#pragma unroll
        for (int i = 0; i < kKeys / kRowsAtOnce; i++)
        {
            const int r = row0 + i * kRowsAtOnce;
            const int page = __shfl_sync(0xffffffffu, page_lane, r);
            const int slot = (key0 + r) & ((1 << mem.page_shift) - 1);
            const int64_t at =
                page < 0 ? 0 : page * mem.page_stride + kv * mem.head_stride + ((int64_t)slot * D + piece * 4) * 4;
            copy_async<16>(raw + (r * D + piece * 4) * 4, mem.k + at, page >= 0);
            copy_async<16>(raw + S::kRaw + (r * D + piece * 4) * 4, mem.v + at, page >= 0);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int next_page = page_of_lane(rank);
    if (rank < blocks.count)
        fetch(rank, next_page);
    next_page = page_of_lane(rank + cluster_size);

    const int g = lane >> 2, c = lane & 3;
    uint32_t qp[2][D / 16][4];  // h and m; l would not fit the registers
    uint4* const ql = reinterpret_cast<uint4*>(shared + S::kQueries) + threadIdx.x;
    RowSpan span[2];
    {
        const float* q = static_cast<const float*>(a.q);
        const float* row[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
            const int m = t.m0 + min(warp * 16 + g + 8 * i, t.count - 1);  // rows past the last one repeat it
            span[i] = row_span(t.past + m / a.group, t.length, a.sinks, a.window, a.frame_tokens);
            row[i] = q + (int64_t)(t.row0 + m / a.group) * a.q_stride + (int64_t)(kv * a.group + m % a.group) * D;
        }
#pragma unroll
        for (int s = 0; s < D / 16; s++)
        {
            uint32_t l[4];
#pragma unroll
            for (int i = 0; i < 4; i++)
            {
                const float2 x = __ldg(reinterpret_cast<const float2*>(row[i & 1] + s * 16 + (i >> 1) * 8 + 2 * c));
                split(x.x, x.y, qp[0][s][i], qp[1][s][i], l[i]);
            }
            ql[s * kThreads] = make_uint4(l[0], l[1], l[2], l[3]);
        }
    }
    const float to_log2 = a.scale * 1.44269504088896341f;
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; n++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            o[n][i] = 0.f;

    // this lane's row of the four 8x8 matrices of an ldmatrix: keys as they lie
    // (n, and k in halves), values transposed (k in halves, and n)
    const uint32_t k_at = planes + (((lane & 7) + ((lane >> 4) & 1) * 8) * S::kPitch + ((lane >> 3) & 1) * 8) * 2;
    const uint32_t v_at = planes + 3 * S::kPlane + ((lane & 15) * S::kPitch + (lane >> 4) * 8) * 2;

    for (int n = rank; n < blocks.count; n += cluster_size)
    {
        const int key0 = first_key(n);
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads();  // the planes are free
#pragma unroll
        for (int kind = 0; kind < 2; kind++)
#pragma unroll
            for (int i = 0; i < kKeys / kRowsAtOnce; i++)
            {
                const int r = row0 + i * kRowsAtOnce;
                const float4 x = *reinterpret_cast<const float4*>(shared + kind * S::kRaw + (r * D + piece * 4) * 4);
                uint2 h, m, l;
                split(x.x, x.y, h.x, m.x, l.x);
                split(x.z, x.w, h.y, m.y, l.y);
                char* dst = shared + S::kPlanes + 3 * kind * S::kPlane + (r * S::kPitch + piece * 4) * 2;
                *reinterpret_cast<uint2*>(dst) = h;
                *reinterpret_cast<uint2*>(dst + S::kPlane) = m;
                *reinterpret_cast<uint2*>(dst + 2 * S::kPlane) = l;
            }
        __syncthreads();
        if (n + cluster_size < blocks.count)
            fetch(n + cluster_size, next_page);
        next_page = page_of_lane(n + 2 * cluster_size);

        // S = Q K^T, 4 tiles of 8 keys: products of h and h', and the small ones
        float big[4][4], small[4][4];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                big[j][i] = small[j][i] = 0.f;
#pragma unroll
        for (int s = 0; s < D / 16; s++)
        {
            uint32_t kp[3][2][4];
#pragma unroll
            for (int p = 0; p < 3; p++)
#pragma unroll
                for (int u = 0; u < 2; u++)
                    ldmatrix_x4(k_at + p * S::kPlane + (u * 16 * S::kPitch + s * 16) * 2, kp[p][u]);
            const uint4 l4 = ql[s * kThreads];
            const uint32_t l[4] = {l4.x, l4.y, l4.z, l4.w};
#pragma unroll
            for (int j = 0; j < 4; j++)
                product(small[j], l, kp[0][j / 2][j % 2 * 2], kp[0][j / 2][j % 2 * 2 + 1]);
#pragma unroll
            for (int p = 0; p < 2; p++)  // h l', m m'
#pragma unroll
                for (int j = 0; j < 4; j++)
                    product(small[j], qp[p][s], kp[2 - p][j / 2][j % 2 * 2], kp[2 - p][j / 2][j % 2 * 2 + 1]);
#pragma unroll
            for (int p = 0; p < 2; p++)  // h m', m h'
#pragma unroll
                for (int j = 0; j < 4; j++)
                    product(small[j], qp[p][s], kp[1 - p][j / 2][j % 2 * 2], kp[1 - p][j / 2][j % 2 * 2 + 1]);
#pragma unroll
            for (int j = 0; j < 4; j++)
                product(big[j], qp[0][s], kp[0][j / 2][j % 2 * 2], kp[0][j / 2][j % 2 * 2 + 1]);
        }

        float old[2];
#pragma unroll
        for (int i = 0; i < 2; i++)
        {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                {
                    float& x = big[j][2 * i + e];
                    const int key = key0 + 8 * j + 2 * c + e;
                    const bool seen = key < span[i].hi && (key >= span[i].lo || key < a.sinks);
                    x = seen ? (x + small[j][2 * i + e]) * to_log2 : -INFINITY;
                    top = fmaxf(top, x);
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            top = fmaxf(top, mx[i]);
            const float base = top == -INFINITY ? 0.f : top;  // nothing seen yet: all exponentials 0
            old[i] = fast_exp2(mx[i] - base);
            mx[i] = top;
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                {
                    float& x = big[j][2 * i + e];
                    x = fast_exp2(x - base);
                    part += x;
                }
            sum[i] = sum[i] * old[i] + part;  // of this lane's keys; added up over c at the end
        }
        uint32_t pp[3][2][4];
#pragma unroll
        for (int s = 0; s < 2; s++)
#pragma unroll
            for (int i = 0; i < 4; i++)
            {
                const float* x = big[2 * s + (i >> 1)] + 2 * (i & 1);
                split(x[0], x[1], pp[0][s][i], pp[1][s][i], pp[2][s][i]);
            }

        // O = O 2^(m - m') + P V, 32 features at a time
#pragma unroll
        for (int f = 0; f < D; f += 32)
        {
            float acc[4][4];
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    acc[j][i] = 0.f;
#pragma unroll
            for (int s = 0; s < 2; s++)
            {
                uint32_t vp[3][2][4];
#pragma unroll
                for (int p = 0; p < 3; p++)
#pragma unroll
                    for (int u = 0; u < 2; u++)
                        ldmatrix_x4_trans(v_at + p * S::kPlane + (s * 16 * S::kPitch + f + u * 16) * 2, vp[p][u]);
#pragma unroll
                for (int p = 0; p < 3; p++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        product(acc[j], pp[p][s], vp[2 - p][j / 2][j % 2 * 2], vp[2 - p][j / 2][j % 2 * 2 + 1]);
#pragma unroll
                for (int p = 0; p < 2; p++)
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        product(acc[j], pp[p][s], vp[1 - p][j / 2][j % 2 * 2], vp[1 - p][j / 2][j % 2 * 2 + 1]);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    product(acc[j], pp[0][s], vp[0][j / 2][j % 2 * 2], vp[0][j / 2][j % 2 * 2 + 1]);
            }
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    o[f / 8 + j][i] = fmaf(o[f / 8 + j][i], old[i >> 1], acc[j][i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
    {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
    }
    __syncthreads();
    float* part_o = reinterpret_cast<float*>(shared + S::kPlanes);
    float2* part_ml = reinterpret_cast<float2*>(shared);
#pragma unroll
    for (int i = 0; i < 2; i++)
    {
        const int r = warp * 16 + g + 8 * i;
#pragma unroll
        for (int n = 0; n < D / 8; n++)
            *reinterpret_cast<float2*>(part_o + r * S::kPartPitch + 8 * n + 2 * c) =
                make_float2(o[n][2 * i], o[n][2 * i + 1]);
        if (c == 0)
            part_ml[r] = make_float2(mx[i], sum[i]);
    }
    join_cluster<float, kThreads>(a, t, kv, D, rank, cluster_size, part_o, S::kPartPitch, part_ml);
}

template <int D>
int run(const CacheAttnArgs& a, cudaStream_t stream)
{
    const int64_t rows = (int64_t)a.batch.rows * a.group;
    const int64_t tiles = rows / kRows + a.batch.sequences;
    // 160 tiles of 28 blocks of keys: 158, 174, 141 and 153 us with 1, 2, 4 and 8 blocks a tile
    const int cluster = cluster_of(a, rows, kRows, kKeys, 4.0);
    if (tiles * cluster > 0x7fffffff)
        return (int)cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)a.mem.heads);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = Shared<D>::kBytes;
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&config, cache_attention_f32_kernel<D>, a, cluster);
}

}  // namespace

int launch_cache_attention_f32(const CacheAttnArgs& a, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_attention_f32", stream);
    return a.mem.head_dim == 128 ? run<128>(a, stream) : run<64>(a, stream);
}

int prepare_cache_attention_f32()
{
    cudaError_t err = cudaFuncSetAttribute((const void*)cache_attention_f32_kernel<64>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, Shared<64>::kBytes);
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute((const void*)cache_attention_f32_kernel<128>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, Shared<128>::kBytes);
    return (int)err;
}

}  // namespace awa
