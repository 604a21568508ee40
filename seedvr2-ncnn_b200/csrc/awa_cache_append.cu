// awa_cache_append.cu -- rows of q, k and v into a paged key/value cache with
// the position rotation applied on the way, and back.
//
// Per row and head: (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) for the rotated
// pairs of q and k, one rounding to the storage type (or to 4-bit codes with a
// scale and a minimum per 64 features). Nothing is read or written twice, so
// memory bounds it: bytes = rows * (q + k + v in, q + k + v out).
#include "awa_cache_device.cuh"
#include "awa_rows.cuh"

#include <cuda_bf16.h>

namespace awa
{
namespace
{

using bf16 = __nv_bfloat16;

constexpr int kThreads = 256;
constexpr int kMaxTileRows = 8;

// Page number `index` of all that the sequences of the batch see, counted
// sequence by sequence. Called by one full warp; the same in all lanes.
struct PageSlot
{
    int b;  // -1: none
    int entry;
};

__device__ __forceinline__ PageSlot find_page(const CacheUnpackArgs& a, int index)
{
    const int lane = threadIdx.x & 31;
    const int page = 1 << a.mem.page_shift;
    int before = 0;
    for (int base = 0; base < a.batch.sequences; base += 32)
    {
        const int b = base + lane;
        KeyBlocks pages;
        pages.prefix = pages.shift = pages.count = 0;
        if (b < a.batch.sequences)
        {
            const int rows = batch_rows(a.batch, b);
            const int past = max(0, __ldg(a.batch.past + b));
            const int length = sequence_length(a.mem, a.batch, past, rows, nullptr);
            if (rows > 0)
                pages = key_blocks(row_span(min(past, length), length, a.sinks, a.window, a.frame_tokens),
                                   row_span(min(past, length) + rows - 1, length, a.sinks, a.window, a.frame_tokens),
                                   a.sinks, page);
        }
        int sum = pages.count;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o)
                sum += up;
        }
        const unsigned holds = __ballot_sync(0xffffffffu, index < before + sum);
        if (holds)
        {
            const int src = __ffs(holds) - 1;
            const int i = index - before - __shfl_sync(0xffffffffu, sum - pages.count, src);
            const int prefix = __shfl_sync(0xffffffffu, pages.prefix, src);
            const int shift = __shfl_sync(0xffffffffu, pages.shift, src);
            return {base + src, i < prefix ? i : i + shift};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return {-1, 0};
}

// 8 consecutive elements, in 16-byte pieces where the rows allow it.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void get8(const T* p, float (&v)[8])
{
    if (ALIGNED)
        load8(p, v);
    else
#pragma unroll
        for (int i = 0; i < 8; i++)
            v[i] = load1(p + i);
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void put8(T* p, const float (&v)[8])
{
    if (ALIGNED)
        store8(p, v);
    else
#pragma unroll
        for (int i = 0; i < 8; i++)
            store1(p + i, v[i]);
}

// The largest bf16 value <= x, and the smallest >= x.
__device__ __forceinline__ float bf16_down(float x)
{
    return __bfloat162float(__float2bfloat16_rd(x));
}
__device__ __forceinline__ float bf16_up(float x)
{
    return __bfloat162float(__float2bfloat16_ru(x));
}

// Codes of 64 features held by 8 neighbouring lanes, 8 each. The scale is
// rounded up and the minimum down, so 16 steps always cover the group: no code
// is clipped by the rounding of its own parameters.
__device__ __forceinline__ void quantize8(const float (&v)[8], uint32_t& codes, uint32_t& params)
{
    float lo = v[0], hi = v[0];
#pragma unroll
    for (int i = 1; i < 8; i++)
    {
        lo = fminf(lo, v[i]);
        hi = fmaxf(hi, v[i]);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1)
    {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    const float minimum = bf16_down(lo);
    const float scale = bf16_up(__fdiv_rn(__fsub_rn(hi, minimum), 15.f));
    const float inverse = scale > 0.f ? __fdiv_rn(1.f, scale) : 0.f;
    codes = 0;
#pragma unroll
    for (int i = 0; i < 8; i++)
    {
        const float c = rintf(__fmul_rn(__fsub_rn(v[i], minimum), inverse));
        codes |= (uint32_t)fminf(fmaxf(c, 0.f), 15.f) << (4 * i);
    }
    params = (__float_as_uint(scale) >> 16) | (__float_as_uint(minimum) & 0xffff0000u);
}

__device__ __forceinline__ void dequantize8(uint32_t codes, uint32_t params, float (&v)[8])
{
    const float scale = __uint_as_float(params << 16), minimum = __uint_as_float(params & 0xffff0000u);
#pragma unroll
    for (int i = 0; i < 8; i++)
        v[i] = __fadd_rn(__fmul_rn((float)((codes >> (4 * i)) & 15u), scale), minimum);
}

// A row of the batch: where it goes and how it turns.
struct RowPlace
{
    int64_t slot;    // byte offset of its head 0 in the pages
    int64_t params;  // the same in the params
    int position;    // -1: nothing to do
    int coord[4];
};

// ST: the cache's storage type. Blocks: x = tiles of `tile_rows` rows, y =
// parts of the heads. A thread keeps its 8 features (and so, within a row, its
// rotation factors) and walks over the heads of q, k and v.
template <typename TIn, typename TQ, int ST, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) cache_append_kernel(CacheAppendArgs a, int tile_rows)
{
    __shared__ RowPlace places[kMaxTileRows];
    const CacheMemory& mem = a.mem;
    const int row0 = blockIdx.x * tile_rows;
    if ((int)threadIdx.x < tile_rows)
    {
        RowPlace p;
        p.position = -1;
        const int row = row0 + threadIdx.x;
        const int b = row < a.batch.rows ? sequence_of_row(a.batch, row) : -1;
        if (b >= 0)
        {
            const int position = position_of_row(a.batch, b, row);
            const int page = page_of(mem, a.batch, b, position, a.error_flag);
            bool good = page >= 0;
            if (a.table)
                for (int x = 0; x < a.axes; x++)
                {
                    p.coord[x] = a.coords ? __ldg(a.coords + (int64_t)row * a.axes + x) : position;
                    if (p.coord[x] < 0 || p.coord[x] >= a.max_coord)
                    {
                        cache_error(a.error_flag, AWA_CACHE_BAD_COORD);
                        good = false;
                    }
                }
            if (good)
            {
                const int slot = position & ((1 << mem.page_shift) - 1);
                const int row_bytes = ST == AWA_INT4 ? mem.head_dim / 2 : mem.head_dim * (ST == AWA_F32 ? 4 : 2);
                p.slot = page * mem.page_stride + (int64_t)slot * row_bytes;
                p.params = page * mem.params_page_stride + (int64_t)slot * (mem.head_dim / AWA_CACHE_GROUP) * 4;
                p.position = position;
            }
        }
        places[threadIdx.x] = p;
    }
    __syncthreads();

    const int chunks = mem.head_dim / 8;
    const int lanes = kThreads / chunks;  // heads side by side
    const int chunk = threadIdx.x % chunks, lane = threadIdx.x / chunks;
    const int f = chunk * 8;
    const int total = a.q_heads + 2 * mem.heads;
    const int step = lanes * gridDim.y;
    const TIn* q = reinterpret_cast<const TIn*>(a.q);
    const TIn* k = reinterpret_cast<const TIn*>(a.k);
    const TIn* v = reinterpret_cast<const TIn*>(a.v);
    TQ* q_out = reinterpret_cast<TQ*>(a.q_out);

    for (int r = 0; r < tile_rows; r++)
    {
        const RowPlace& place = places[r];
        if (place.position < 0)
            continue;
        const int64_t row = row0 + r;
        float2 cs[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            cs[i] = make_float2(1.f, 0.f);
            const int pair = f / 2 + i;
            if (a.table && pair < a.axes * a.pairs)
            {
                const int axis = pair / a.pairs;
                cs[i] = __ldg(a.table + (int64_t)place.coord[axis] * a.pairs + (pair - axis * a.pairs));
            }
        }
        const bool turns = a.table && f < 2 * a.axes * a.pairs;
        // uniform trip count: quantize8 shuffles within the warp
        for (int h0 = blockIdx.y * lanes; h0 < total; h0 += step)
        {
            const int h = h0 + lane;
            const bool mine = lane < lanes && h < total;
            float x[8] = {};
            const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + mem.heads;
            if (mine)
            {
                const TIn* src = is_q   ? q + row * a.q_stride + h * mem.head_dim
                                 : is_k ? k + row * a.k_stride + (h - a.q_heads) * mem.head_dim
                                        : v + row * a.v_stride + (h - a.q_heads - mem.heads) * mem.head_dim;
                get8<TIn, ALIGNED>(src + f, x);
                if (turns && (is_q || is_k))
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (f / 2 + i < a.axes * a.pairs)
                            rope_rotate(x[2 * i], x[2 * i + 1], cs[i].x, cs[i].y, x[2 * i], x[2 * i + 1]);
            }
            if (mine && is_q)
                put8<TQ, ALIGNED>(q_out + row * a.q_out_stride + h * mem.head_dim + f, x);
            const int kv = is_k ? h - a.q_heads : h - a.q_heads - mem.heads;
            char* base = is_k ? mem.k : mem.v;
            if (ST == AWA_INT4)
            {
                uint32_t codes, params;
                quantize8(x, codes, params);
                if (mine && !is_q)
                {
                    *reinterpret_cast<uint32_t*>(base + place.slot + kv * mem.head_stride + f / 2) = codes;
                    if (chunk % 8 == 0)
                        *reinterpret_cast<uint32_t*>((is_k ? mem.k_params : mem.v_params) + place.params +
                                                     kv * mem.params_head_stride + f / AWA_CACHE_GROUP * 4) = params;
                }
            }
            else if (mine && !is_q)
            {
                char* dst = base + place.slot + kv * mem.head_stride;
                if (ST == AWA_F32)
                    store8(reinterpret_cast<float*>(dst) + f, x);
                else
                    store8(reinterpret_cast<bf16*>(dst) + f, x);
            }
        }
    }
}

template <typename TOut, int ST, bool ALIGNED>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(CacheReadArgs a, int tile_rows)
{
    __shared__ RowPlace places[kMaxTileRows];
    const CacheMemory& mem = a.mem;
    const int row0 = blockIdx.x * tile_rows;
    if ((int)threadIdx.x < tile_rows)
    {
        RowPlace p;
        p.position = -1;
        const int row = row0 + threadIdx.x;
        const int b = row < a.batch.rows ? sequence_of_row(a.batch, row) : -1;
        if (b >= 0)
        {
            const int position = position_of_row(a.batch, b, row);
            const int page = page_of(mem, a.batch, b, position, a.error_flag);
            if (page >= 0)
            {
                const int slot = position & ((1 << mem.page_shift) - 1);
                const int row_bytes = ST == AWA_INT4 ? mem.head_dim / 2 : mem.head_dim * (ST == AWA_F32 ? 4 : 2);
                p.slot = page * mem.page_stride + (int64_t)slot * row_bytes;
                p.params = page * mem.params_page_stride + (int64_t)slot * (mem.head_dim / AWA_CACHE_GROUP) * 4;
                p.position = position;
            }
        }
        places[threadIdx.x] = p;
    }
    __syncthreads();

    const int chunks = mem.head_dim / 8;
    const int lanes = kThreads / chunks;
    const int f = (threadIdx.x % chunks) * 8, lane = threadIdx.x / chunks;
    if (lane >= lanes)
        return;
    for (int r = 0; r < tile_rows; r++)
    {
        const RowPlace& place = places[r];
        if (place.position < 0)
            continue;
        const int64_t row = row0 + r;
        for (int h = blockIdx.y * lanes + lane; h < 2 * mem.heads; h += lanes * gridDim.y)
        {
            const bool is_k = h < mem.heads;
            const int kv = is_k ? h : h - mem.heads;
            const char* src = (is_k ? mem.k : mem.v) + place.slot + kv * mem.head_stride;
            float x[8];
            if (ST == AWA_INT4)
            {
                const uint32_t params =
                    *reinterpret_cast<const uint32_t*>((is_k ? mem.k_params : mem.v_params) + place.params +
                                                       kv * mem.params_head_stride + f / AWA_CACHE_GROUP * 4);
                dequantize8(*reinterpret_cast<const uint32_t*>(src + f / 2), params, x);
            }
            else if (ST == AWA_F32)
                load8(reinterpret_cast<const float*>(src) + f, x);
            else
                load8(reinterpret_cast<const bf16*>(src) + f, x);
            TOut* dst = reinterpret_cast<TOut*>(is_k ? a.k_out : a.v_out) + row * (is_k ? a.k_stride : a.v_stride) +
                        (int64_t)kv * mem.head_dim + f;
            put8<TOut, ALIGNED>(dst, x);
        }
    }
}

// One 4-bit page that some row of the batch sees -> its keys and values as
// bf16, and its number in the workspace's page table. Blocks: x = the pages of
// all sequences in order, y = heads.
__global__ void __launch_bounds__(kThreads) cache_unpack_kernel(CacheUnpackArgs a)
{
    __shared__ int which_s[2];
    const CacheMemory& mem = a.mem;
    if (threadIdx.x < 32)
    {
        const PageSlot at = find_page(a, blockIdx.x);
        if (threadIdx.x == 0)
        {
            which_s[0] = at.b;
            which_s[1] = at.entry;
        }
    }
    __syncthreads();
    const int b = which_s[0], entry = which_s[1];
    if (b < 0)
        return;
    const int page = __ldg(a.batch.page_table + b * a.batch.table_stride + entry);
    const bool real = (unsigned)page < (unsigned)mem.pages;
    if (threadIdx.x == 0 && blockIdx.y == 0)
    {
        if (!real)
            cache_error(a.error_flag, AWA_CACHE_BAD_PAGE);
        a.table[(int64_t)b * a.batch.table_width + entry] = blockIdx.x;
    }
    const int kv = blockIdx.y, groups = mem.head_dim / AWA_CACHE_GROUP, row_bytes = mem.head_dim / 2;
    const int64_t page_bytes = (int64_t)row_bytes << mem.page_shift;  // of codes
    const int64_t src = page * mem.page_stride + kv * mem.head_stride;
    const int64_t par = page * mem.params_page_stride + kv * mem.params_head_stride;
    const int64_t dst = ((int64_t)blockIdx.x * mem.heads + kv) * page_bytes * 4;
    // 16 codes, of one group, a thread and turn
    for (int i = threadIdx.x; i < 2 * (int)(page_bytes / 8); i += kThreads)
    {
        const bool is_k = i < (int)(page_bytes / 8);
        const int at = (is_k ? i : i - (int)(page_bytes / 8)) * 8;
        uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
        if (real)
        {
            const uint2 codes = __ldg(reinterpret_cast<const uint2*>((is_k ? mem.k : mem.v) + src + at));
            const int row = at / row_bytes, group = (at - row * row_bytes) / (AWA_CACHE_GROUP / 2);
            const uint32_t params = __ldg(
                reinterpret_cast<const uint32_t*>((is_k ? mem.k_params : mem.v_params) + par) + row * groups + group);
            float v[8];
            dequantize8(codes.x, params, v);
            store8(reinterpret_cast<bf16*>(&out[0]), v);
            dequantize8(codes.y, params, v);
            store8(reinterpret_cast<bf16*>(&out[1]), v);
        }
        uint4* to = reinterpret_cast<uint4*>((is_k ? a.k_out : a.v_out) + dst + (int64_t)at * 4);
        to[0] = out[0];
        to[1] = out[1];
    }
}

struct Shape
{
    dim3 grid;
    int tile_rows;
};

// Few rows: a block per row and part of the heads (a step of 8 rows with 60
// heads of 128 features fills 32 blocks). Many rows: a block takes 8 of them
// whole, so the lookup of sequence, page and coordinates is paid once a tile.
Shape shape_of(int rows, int heads, int head_dim)
{
    Shape s;
    s.tile_rows = rows < 148 * 8 ? 1 : kMaxTileRows;
    const int lanes = kThreads / (head_dim / 8);
    const int passes = (heads + lanes - 1) / lanes;
    s.grid = dim3((unsigned)((rows + s.tile_rows - 1) / s.tile_rows), s.tile_rows == 1 ? (unsigned)passes : 1u);
    return s;
}

template <typename TIn, typename TQ, int ST>
void run_append(const CacheAppendArgs& a, cudaStream_t stream)
{
    const Shape s = shape_of(a.batch.rows, a.q_heads + 2 * a.mem.heads, a.mem.head_dim);
    if (a.aligned)
        cache_append_kernel<TIn, TQ, ST, true><<<s.grid, kThreads, 0, stream>>>(a, s.tile_rows);
    else
        cache_append_kernel<TIn, TQ, ST, false><<<s.grid, kThreads, 0, stream>>>(a, s.tile_rows);
}

template <typename TIn, typename TQ>
void run_append(const CacheAppendArgs& a, cudaStream_t stream)
{
    if (a.mem.storage == AWA_INT4)
        run_append<TIn, TQ, AWA_INT4>(a, stream);
    else if (a.mem.storage == AWA_F32)
        run_append<TIn, TQ, AWA_F32>(a, stream);
    else
        run_append<TIn, TQ, AWA_BF16>(a, stream);
}

template <typename TOut, int ST>
void run_read(const CacheReadArgs& a, cudaStream_t stream)
{
    const Shape s = shape_of(a.batch.rows, 2 * a.mem.heads, a.mem.head_dim);
    if (a.aligned)
        cache_read_kernel<TOut, ST, true><<<s.grid, kThreads, 0, stream>>>(a, s.tile_rows);
    else
        cache_read_kernel<TOut, ST, false><<<s.grid, kThreads, 0, stream>>>(a, s.tile_rows);
}

template <typename TOut>
void run_read(const CacheReadArgs& a, cudaStream_t stream)
{
    if (a.mem.storage == AWA_INT4)
        run_read<TOut, AWA_INT4>(a, stream);
    else if (a.mem.storage == AWA_F32)
        run_read<TOut, AWA_F32>(a, stream);
    else
        run_read<TOut, AWA_BF16>(a, stream);
}

}  // namespace

int launch_cache_append(const CacheAppendArgs& a, int in_dtype, int q_out_dtype, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_append", stream);
    if (in_dtype == AWA_F32)
        q_out_dtype == AWA_F32 ? run_append<float, float>(a, stream) : run_append<float, bf16>(a, stream);
    else
        q_out_dtype == AWA_F32 ? run_append<bf16, float>(a, stream) : run_append<bf16, bf16>(a, stream);
    return (int)cudaGetLastError();
}

int launch_cache_read(const CacheReadArgs& a, int out_dtype, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_read", stream);
    out_dtype == AWA_F32 ? run_read<float>(a, stream) : run_read<bf16>(a, stream);
    return (int)cudaGetLastError();
}

int launch_cache_unpack(const CacheUnpackArgs& a, int pages, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_unpack", stream);
    cache_unpack_kernel<<<dim3((unsigned)pages, (unsigned)a.mem.heads), kThreads, 0, stream>>>(a);
    return (int)cudaGetLastError();
}

}  // namespace awa
