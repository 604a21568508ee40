// awa_cache_attn_simt.cu -- attention over the paged key/value cache in fp32
// arithmetic, for few rows of fp32 caches and for head sizes without a
// tensor-core kernel.
//
// out = softmax(scale q K^T) V in one pass over the keys a tile of query rows
// sees: per block of 64 keys, S = Q K^T in registers, the running maximum m and
// sum l of each row (base 2, scale folded into the exponent), O = O 2^(m - m')
// + P V.
//
// The FMA units bound it: 4 d flops per visible pair at 128 FMAs a clock and SM.
// Both products go through fma.f32x2, two of them per instruction, so that their
// issue leaves room for the loads from shared memory; two blocks on an SM work
// under each other's waits. Measured (B200): 1024 rows of 32 / 8 heads of 96 over
// 4096 keys 1.58 ms, 28.5 TFLOP/s, 0.38 of the FMA rate (bf16 1.53 ms). For single
// rows the loads count, and a block has none in flight while it computes: 64
// streams of 8192 fp32 keys, 32 / 8 heads of 128, 2.98 ms, 1.4 TB/s; one of 32768
// keys 555 us (8 blocks a tile, 64 SMs); one of 701 keys, 20 heads, 66 us.
#include "awa_cache_join.cuh"

#include <cuda_bf16.h>

namespace awa
{
namespace
{

using bf16 = __nv_bfloat16;

constexpr int kThreads = 256;
constexpr int kKeys = 64;
constexpr int kPad = 4;  // floats: rows start 4 banks apart, so 16-byte reads of 8 rows do not collide

__host__ __device__ constexpr int shared_floats(int rows, int d)
{
    return (rows + 2 * kKeys) * (d + kPad) + rows * (kKeys + kPad);
}

using Pair = unsigned long long;  // two floats

__device__ __forceinline__ Pair pair_of(float a, float b)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(a), "f"(b));
    return p;
}

__device__ __forceinline__ float2 floats_of(Pair p)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p));
    return f;
}

__device__ __forceinline__ void fma2(Pair& acc, Pair a, Pair b)
{
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}

__device__ __forceinline__ void mul2(Pair& acc, Pair a)
{
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(acc) : "l"(a));
}

// T: type of the cache, q and out. D: head_dim, 0 if only the cache knows it. A
// block (of a cluster of gridDim.x / tiles that share the keys) takes one tile of
// R * 16 query rows of one key/value head. Thread (ty, tx) of 16 x 16: rows
// ty * R + i, keys tx + 16 j, output features 4 (tx + 16 j).
template <typename T, int R, int D>
__global__ void __launch_bounds__(kThreads, 2) cache_attention_simt_kernel(CacheAttnArgs a, int cluster_size)
{
    constexpr int kRows = 16 * R;
    extern __shared__ float4 shared4[];
    __shared__ QueryTile tile_s;
    const CacheMemory& mem = a.mem;
    const int d = D ? D : mem.head_dim, pitch = d + kPad;
    float* sq = reinterpret_cast<float*>(shared4);
    float* sk = sq + kRows * pitch;
    float* sv = sk + kKeys * pitch;
    float* sp = sv + kKeys * pitch;
    const int rank = blockIdx.x % cluster_size;
    if (threadIdx.x < 32)
    {
        const QueryTile t =
            find_tile(mem, a.batch, a.group, kRows, blockIdx.x / cluster_size, rank == 0 ? a.error_flag : nullptr);
        if (threadIdx.x == 0)
            tile_s = t;
    }
    __syncthreads();
    const QueryTile t = tile_s;
    if (t.b < 0)
        return;  // the whole cluster
    const int kv = blockIdx.y;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int chunks = d / 8;

    const T* q = static_cast<const T*>(a.q);
    for (int i = threadIdx.x; i < kRows * chunks; i += kThreads)
    {
        const int r = i / chunks, f = (i - r * chunks) * 8;
        float v[8] = {};
        if (r < t.count)
        {
            const int m = t.m0 + r;
            load8(q + (int64_t)(t.row0 + m / a.group) * a.q_stride + (int64_t)(kv * a.group + m % a.group) * d + f, v);
        }
        store8(sq + r * pitch + f, v);
    }

    RowSpan span[R];
#pragma unroll
    for (int i = 0; i < R; i++)
    {
        const int m = min(ty * R + i, t.count - 1);
        span[i] = row_span(t.past + (t.m0 + m) / a.group, t.length, a.sinks, a.window, a.frame_tokens);
    }
    const RowSpan first = row_span(t.past + t.m0 / a.group, t.length, a.sinks, a.window, a.frame_tokens);
    const RowSpan last =
        row_span(t.past + (t.m0 + t.count - 1) / a.group, t.length, a.sinks, a.window, a.frame_tokens);
    const KeyBlocks blocks = key_blocks(first, last, a.sinks, kKeys);

    const float to_log2 = a.scale * 1.44269504088896341f;
    float mx[R], sum[R];
    Pair o[R][2][2];
#pragma unroll
    for (int i = 0; i < R; i++)
    {
        mx[i] = -INFINITY;
        sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < 4; j++)
            o[i][j / 2][j % 2] = 0;
    }

    for (int n = rank; n < blocks.count; n += cluster_size)
    {
        const int key0 = (n < blocks.prefix ? n : n + blocks.shift) * kKeys;
        __syncthreads();
        for (int i = threadIdx.x; i < kKeys * chunks; i += kThreads)
        {
            const int r = i / chunks, f = (i - r * chunks) * 8;
            const int key = key0 + r;
            float k8[8] = {}, v8[8] = {};
            // only what some row sees is read: pages outside may be gone
            if (key < last.hi && (key >= first.lo || key < a.sinks))
            {
                const int page = page_of(mem, a.batch, t.b, key, a.error_flag);
                if (page >= 0)
                {
                    const int slot = key & ((1 << mem.page_shift) - 1);
                    const int64_t at = page * mem.page_stride + kv * mem.head_stride;
                    load8(reinterpret_cast<const T*>(mem.k + at) + slot * d + f, k8);
                    load8(reinterpret_cast<const T*>(mem.v + at) + slot * d + f, v8);
                }
            }
            store8(sk + r * pitch + f, k8);
            store8(sv + r * pitch + f, v8);
        }
        __syncthreads();

        // sums over even and over odd features, added at the end
        Pair s2[R][4];
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
                s2[i][j] = 0;
#pragma unroll 4
        for (int f = 0; f < d; f += 4)
        {
            ulonglong2 qv[R], kk[4];
#pragma unroll
            for (int i = 0; i < R; i++)
                qv[i] = *reinterpret_cast<const ulonglong2*>(sq + (ty * R + i) * pitch + f);
#pragma unroll
            for (int j = 0; j < 4; j++)
                kk[j] = *reinterpret_cast<const ulonglong2*>(sk + (tx + 16 * j) * pitch + f);
#pragma unroll
            for (int i = 0; i < R; i++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                {
                    fma2(s2[i][j], qv[i].x, kk[j].x);
                    fma2(s2[i][j], qv[i].y, kk[j].y);
                }
        }
        float s[R][4];
#pragma unroll
        for (int i = 0; i < R; i++)
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                const float2 x = floats_of(s2[i][j]);
                s[i][j] = x.x + x.y;
            }
#pragma unroll
        for (int i = 0; i < R; i++)
        {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                const int key = key0 + tx + 16 * j;
                const bool seen = key < span[i].hi && (key >= span[i].lo || key < a.sinks);
                s[i][j] = seen ? s[i][j] * to_log2 : -INFINITY;
                top = fmaxf(top, s[i][j]);
            }
#pragma unroll
            for (int off = 1; off < 16; off <<= 1)
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
            top = fmaxf(top, mx[i]);
            const float base = top == -INFINITY ? 0.f : top;  // nothing seen yet: all exponentials 0
            const float old = fast_exp2(mx[i] - base);
            mx[i] = top;
            float part = 0.f;
#pragma unroll
            for (int j = 0; j < 4; j++)
            {
                const float p = fast_exp2(s[i][j] - base);
                part += p;
                sp[(ty * R + i) * (kKeys + kPad) + tx + 16 * j] = p;
            }
            sum[i] = sum[i] * old + part;  // of this thread's keys; added up over tx at the end
#pragma unroll
            for (int j = 0; j < 4; j++)
                mul2(o[i][j / 2][j % 2], pair_of(old, old));
        }
        __syncwarp();  // a row's probabilities come from its own half warp
#pragma unroll 2
        for (int key = 0; key < kKeys; key += 4)
        {
            float4 p[R];
#pragma unroll
            for (int i = 0; i < R; i++)
                p[i] = *reinterpret_cast<const float4*>(sp + (ty * R + i) * (kKeys + kPad) + key);
#pragma unroll
            for (int j = 0; j < 2; j++)
            {
                const int f = 4 * (tx + 16 * j);
                if (f >= d)
                    break;
#pragma unroll
                for (int u = 0; u < 4; u++)
                {
                    const ulonglong2 v = *reinterpret_cast<const ulonglong2*>(sv + (key + u) * pitch + f);
#pragma unroll
                    for (int i = 0; i < R; i++)
                    {
                        const float w = u == 0 ? p[i].x : u == 1 ? p[i].y : u == 2 ? p[i].z : p[i].w;
                        fma2(o[i][j][0], pair_of(w, w), v.x);
                        fma2(o[i][j][1], pair_of(w, w), v.y);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; i++)
#pragma unroll
        for (int off = 1; off < 16; off <<= 1)
            sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], off);

    T* out = static_cast<T*>(a.out);
    if (cluster_size == 1)
    {
#pragma unroll
        for (int i = 0; i < R; i++)
        {
            const int r = ty * R + i;
            if (r >= t.count)
                continue;
            const int m = t.m0 + r;
            const float inv = sum[i] > 0.f ? 1.f / sum[i] : sum[i] == 0.f ? 0.f : sum[i];
            T* dst = out + (int64_t)(t.row0 + m / a.group) * a.out_stride + (int64_t)(kv * a.group + m % a.group) * d;
#pragma unroll
            for (int j = 0; j < 2; j++)
                if (4 * (tx + 16 * j) < d)
#pragma unroll
                    for (int c = 0; c < 2; c++)
                    {
                        const float2 x = floats_of(o[i][j][c]);
                        store1(dst + 4 * (tx + 16 * j) + 2 * c, x.x * inv);
                        store1(dst + 4 * (tx + 16 * j) + 2 * c + 1, x.y * inv);
                    }
        }
        return;
    }

    __syncthreads();
    float* part_o = sq;                // [kRows][pitch]
    float2* part_ml = reinterpret_cast<float2*>(sk);
#pragma unroll
    for (int i = 0; i < R; i++)
    {
        const int r = ty * R + i;
#pragma unroll
        for (int j = 0; j < 2; j++)
            if (4 * (tx + 16 * j) < d)
                *reinterpret_cast<ulonglong2*>(part_o + r * pitch + 4 * (tx + 16 * j)) =
                    make_ulonglong2(o[i][j][0], o[i][j][1]);
        if (tx == 0)
            part_ml[r] = make_float2(mx[i], sum[i]);
    }
    join_cluster<T, kThreads>(a, t, kv, d, rank, cluster_size, part_o, pitch, part_ml);
}

template <typename T, int R, int D>
int run(const CacheAttnArgs& a, cudaStream_t stream)
{
    const int64_t rows = (int64_t)a.batch.rows * a.group;
    const int64_t tiles = rows / (16 * R) + a.batch.sequences;
    // a start and a join cost about 4 blocks of keys (64 rows of 128 features, before
    // they went to the tensor cores, 160 tiles of 14: 291, 236, 244 and 313 us with 1,
    // 2, 4 and 8 blocks a tile)
    const int cluster = cluster_of(a, rows, 16 * R, kKeys, 4.0);
    if (tiles * cluster > 0x7fffffff)
        return (int)cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)a.mem.heads);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = shared_floats(16 * R, a.mem.head_dim) * sizeof(float);
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&config, cache_attention_simt_kernel<T, R, D>, a, cluster);
}

template <typename T, int R>
int run(const CacheAttnArgs& a, cudaStream_t stream)
{
    // the other sizes and types with 64 and 128 features have kernels of their own
    if constexpr (sizeof(T) == 4 && R == 1)
    {
        if (a.mem.head_dim == 128)
            return run<T, R, 128>(a, stream);
        if (a.mem.head_dim == 64)
            return run<T, R, 64>(a, stream);
    }
    return run<T, R, 0>(a, stream);
}

template <typename T>
int run(const CacheAttnArgs& a, int max_rows, cudaStream_t stream)
{
    // 64 rows a tile use the FMA units best; up to 16 rows of a head group,
    // a tile of 16 does a quarter of the work
    return (int64_t)max_rows * a.group <= 16 ? run<T, 1>(a, stream) : run<T, 4>(a, stream);
}

}  // namespace

int launch_cache_attention_simt(const CacheAttnArgs& a, int max_rows, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_attention_simt", stream);
    return a.mem.storage == AWA_F32 ? run<float>(a, max_rows, stream) : run<bf16>(a, max_rows, stream);
}

int prepare_cache_attention_simt()
{
    const struct
    {
        const void* kernel;
        int rows;
    } kernels[] = {{(const void*)cache_attention_simt_kernel<float, 1, 0>, 16},
                   {(const void*)cache_attention_simt_kernel<float, 4, 0>, 64},
                   {(const void*)cache_attention_simt_kernel<float, 1, 64>, 16},
                   {(const void*)cache_attention_simt_kernel<float, 1, 128>, 16},
                   {(const void*)cache_attention_simt_kernel<bf16, 1, 0>, 16},
                   {(const void*)cache_attention_simt_kernel<bf16, 4, 0>, 64}};
    for (const auto& k : kernels)
    {
        const cudaError_t err = cudaFuncSetAttribute(k.kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                     shared_floats(k.rows, kMaxHeadDim) * (int)sizeof(float));
        if (err != cudaSuccess)
            return (int)err;
    }
    return 0;
}

}  // namespace awa
