// awa_cache_append.cu -- rows of q, k and v into a paged key/value cache with
// the position rotation applied on the way, and back.
//
// Per row and head: (x0, x1) -> (x0 c - x1 s, x1 c + x0 s) for the rotated
// pairs of q and k, one rounding to the storage type (or to 4-bit codes with a
// scale and a minimum per 64 features). Nothing is read or written twice, so
// memory bounds it: bytes = rows * (q + k + v in, q + k + v out). Measured (B200):
// 86074 rows of 20 heads of 128 in bf16, 2.64 GB, 480 us (5.5 TB/s, 0.84 of the
// measured copy rate); 8 rows 3.9 us. Read back, the rows' k and v take 326 us
// (5.4 TB/s), of an fp32 cache 570 us (6.2 TB/s), of a 4-bit one, to fp32, 406 us
// (5.0 TB/s); to append them to it takes 448 us (2.5 TB/s): the minimum, maximum
// and rounding of 64 values a group keep the SMs' issue 0.6 busy.
#include "awa_cache_device.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace awa
{
namespace
{

using bf16 = __nv_bfloat16;

constexpr int kThreads = 256;     // of cache_unpack_kernel
constexpr int kMaxThreads = 512;  // of the others
constexpr int kMaxTileRows = 16;

// Page number `index` of all that the sequences of the batch see, counted
// sequence by sequence, or with `total` how many there are. Called by one full warp; the same in all lanes.
struct PageSlot
{
    int b;  // -1: none
    int entry;
    int lo, hi;  // the rows of the sequence see its positions [0, sinks) and [lo, hi)
    int run;     // the next pages, this one among them, are the sequence's entries behind one another
};

__device__ __forceinline__ PageSlot find_page(const CacheUnpackArgs& a, int index, int* total = nullptr)
{
    const int lane = threadIdx.x & 31;
    const int page = 1 << a.mem.page_shift;
    int before = 0;
    for (int base = 0; base < a.batch.sequences; base += 32)
    {
        const int b = base + lane;
        KeyBlocks pages;
        pages.prefix = pages.shift = pages.count = 0;
        RowSpan first = {0, 0}, last = {0, 0};
        if (b < a.batch.sequences)
        {
            const int rows = batch_rows(a.batch, b);
            const int past = max(0, __ldg(a.batch.past + b));
            const int length = sequence_length(a.mem, a.batch, past, rows, nullptr);
            if (rows > 0)
            {
                first = row_span(min(past, length), length, a.sinks, a.window, a.frame_tokens);
                last = row_span(min(past, length) + rows - 1, length, a.sinks, a.window, a.frame_tokens);
                pages = key_blocks(first, last, a.sinks, page);
            }
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
        if (holds && !total)
        {
            const int src = __ffs(holds) - 1;
            const int i = index - before - __shfl_sync(0xffffffffu, sum - pages.count, src);
            const int count = __shfl_sync(0xffffffffu, pages.count, src);
            const int prefix = __shfl_sync(0xffffffffu, pages.prefix, src);
            const int shift = __shfl_sync(0xffffffffu, pages.shift, src);
            return {base + src, i < prefix ? i : i + shift, __shfl_sync(0xffffffffu, first.lo, src),
                    __shfl_sync(0xffffffffu, last.hi, src), (i < prefix ? prefix : count) - i};
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (total)
        *total = before;
    return {-1, 0, 0, 0, 0};
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

__device__ __forceinline__ void dequantize8(uint32_t codes, float scale, float minimum, float (&v)[8])
{
#pragma unroll
    for (int i = 0; i < 8; i++)
        v[i] = __fadd_rn(__fmul_rn((float)((codes >> (4 * i)) & 15u), scale), minimum);
}

__device__ __forceinline__ void dequantize8(uint32_t codes, uint32_t params, float (&v)[8])
{
    dequantize8(codes, __uint_as_float(params << 16), __uint_as_float(params & 0xffff0000u), v);
}

// 8 consecutive elements as they are loaded: raw 16-byte pieces where the rows
// allow them, so that several heads' loads fit the registers.
template <typename T, bool ALIGNED>
struct Raw8
{
    float v[8];
    __device__ __forceinline__ void load(const T* p)
    {
        get8<T, ALIGNED>(p, v);
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; i++)
            x[i] = v[i];
    }
};

template <>
struct Raw8<bf16, true>
{
    uint4 w;
    __device__ __forceinline__ void load(const bf16* p)
    {
        w = __ldg(reinterpret_cast<const uint4*>(p));
    }
    __device__ __forceinline__ void floats(float (&x)[8]) const
    {
        const uint32_t words[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            x[2 * i] = __uint_as_float(words[i] << 16);
            x[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
        }
    }
};

// (x0, x1) -> (x0 c - x1 s, x1 c + x0 s), every product and sum rounded: the
// products two at a time (x1 (-s) is -(x1 s) exactly), the sums one by one, since
// a sum of pairs behind them was contracted into fused operations.
__device__ __forceinline__ void rotate_x2(float& x0, float& x1, float c, float s)
{
    float a0, a1, b0, b1;
    asm("{\n\t.reg .b64 x, y, cc, ss;\n\t"
        "mov.b64 x, {%4, %5};\n\t"
        "mov.b64 y, {%5, %4};\n\t"
        "mov.b64 cc, {%6, %6};\n\t"
        "mov.b64 ss, {%7, %8};\n\t"
        "mul.rn.f32x2 x, x, cc;\n\t"
        "mul.rn.f32x2 y, y, ss;\n\t"
        "mov.b64 {%0, %1}, x;\n\t"
        "mov.b64 {%2, %3}, y;\n\t}"
        : "=f"(a0), "=f"(a1), "=f"(b0), "=f"(b1)
        : "f"(x0), "f"(x1), "f"(c), "f"(-s), "f"(s));
    x0 = __fadd_rn(a0, b0);
    x1 = __fadd_rn(a1, b1);
}

// A row of the batch: where it goes and how it turns.
struct RowPlace
{
    int64_t slot;    // byte offset of its head 0 in the pages
    int64_t params;  // the same in the params
    int position;    // -1: nothing to do
    int coord[4];
};

// The places of the block's rows; a block barrier ends it. coords, table: of
// the rotation, NULL without one.
template <int ST>
__device__ __forceinline__ void find_places(const CacheMemory& mem, const CacheBatch& batch, int row0, int rows,
                                            const int* coords, bool rotates, int axes, int max_coord, int* flag,
                                            RowPlace* places)
{
    if ((int)threadIdx.x < rows)
    {
        RowPlace& p = places[threadIdx.x];
        p.position = -1;
        const int row = row0 + threadIdx.x;
        const int b = row < batch.rows ? sequence_of_row(batch, row) : -1;
        if (b >= 0)
        {
            const int position = position_of_row(batch, b, row);
            const int page = page_of(mem, batch, b, position, flag);
            bool good = page >= 0;
            for (int x = 0; rotates && x < axes; x++)
            {
                const int c = coords ? __ldg(coords + (int64_t)row * axes + x) : position;
                p.coord[x] = c;
                if (c < 0 || c >= max_coord)
                {
                    cache_error(flag, AWA_CACHE_BAD_COORD);
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
    }
    __syncthreads();
}

// ST: the cache's storage type. A block takes tile_rows rows: `lanes` heads side
// by side, head_dim / 8 threads each. A thread keeps its 8 features, and so,
// within a row, its rotation factors, and takes every lanes-th head of q, k and v.
template <typename TIn, typename TQ, int ST, bool ALIGNED>
__global__ void __launch_bounds__(kMaxThreads, 2) cache_append_kernel(CacheAppendArgs a, int tile_rows, int lanes)
{
    __shared__ RowPlace places[kMaxTileRows];
    const CacheMemory& mem = a.mem;
    const int row0 = blockIdx.x * tile_rows;
    find_places<ST>(mem, a.batch, row0, tile_rows, a.coords, a.table != nullptr, a.axes, a.max_coord, a.error_flag,
                    places);

    const int chunks = mem.head_dim / 8;
    const int lane = threadIdx.x / chunks, chunk = threadIdx.x - lane * chunks;
    const int f = chunk * 8;
    const int pairs = a.table ? a.axes * a.pairs : 0;
    const int turned = min(4, max(0, pairs - f / 2));  // of this thread's pairs
    const bool exists = lane < lanes;                  // the last warp may be longer than the heads
    const TIn* q = reinterpret_cast<const TIn*>(a.q) + f;
    const TIn* k = reinterpret_cast<const TIn*>(a.k) + f;
    const TIn* v = reinterpret_cast<const TIn*>(a.v) + f;

    const auto turn = [&](float(&x)[8], const float2(&cs)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (i < turned)
                rotate_x2(x[2 * i], x[2 * i + 1], cs[i].x, cs[i].y);
    };
    const auto keep = [&](char* pages, char* params, const RowPlace& place, int h, bool mine, const float(&x)[8]) {
        char* dst = pages + place.slot + h * mem.head_stride;
        if (ST == AWA_INT4)
        {
            uint32_t codes, par;
            quantize8(x, codes, par);  // all lanes: the groups' threads meet
            if (mine)
            {
                *reinterpret_cast<uint32_t*>(dst + f / 2) = codes;
                if (chunk % 8 == 0)
                    *reinterpret_cast<uint32_t*>(params + place.params + h * mem.params_head_stride +
                                                 f / AWA_CACHE_GROUP * 4) = par;
            }
        }
        else if (mine)
        {
            if (ST == AWA_F32)
                store8(reinterpret_cast<float*>(dst) + f, x);
            else
                store8(reinterpret_cast<bf16*>(dst) + f, x);
        }
    };

    for (int r = 0; r < tile_rows; r++)
    {
        const RowPlace& place = places[r];
        if (place.position < 0)
            continue;
        const int64_t row = row0 + r;
        const TIn* qr = q + row * a.q_stride;
        const TIn* kr = k + row * a.k_stride;
        const TIn* vr = v + row * a.v_stride;
        TQ* out = reinterpret_cast<TQ*>(a.q_out) + row * a.q_out_stride + f;
        // the loads of the first head of each kind ahead of the first use
        Raw8<TIn, ALIGNED> q8 = {}, k8 = {}, v8 = {};
        if (lane < a.q_heads && exists)
            q8.load(qr + lane * mem.head_dim);
        if (lane < mem.heads && exists)
        {
            k8.load(kr + lane * mem.head_dim);
            v8.load(vr + lane * mem.head_dim);
        }
        float2 cs[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            cs[i] = make_float2(1.f, 0.f);
            if (i < turned)
            {
                const int pair = f / 2 + i;
                const int axis = pair < a.pairs ? 0 : pair / a.pairs;
                cs[i] = __ldg(a.table + (int64_t)place.coord[axis] * a.pairs + (pair - axis * a.pairs));
            }
        }
        float x[8];
        for (int h = lane; h < a.q_heads && exists; h += lanes)
        {
            q8.floats(x);
            if (h + lanes < a.q_heads)
                q8.load(qr + (h + lanes) * mem.head_dim);
            turn(x, cs);
            put8<TQ, ALIGNED>(out + h * mem.head_dim, x);
        }
        for (int h0 = 0; h0 < mem.heads; h0 += lanes)  // the same count in all threads
        {
            const int h = h0 + lane;
            const bool mine = h < mem.heads && exists, more = h + lanes < mem.heads && exists;
            float y[8];
            k8.floats(x);
            v8.floats(y);
            if (more)
            {
                k8.load(kr + (h + lanes) * mem.head_dim);
                v8.load(vr + (h + lanes) * mem.head_dim);
            }
            turn(x, cs);
            keep(mem.k, mem.k_params, place, h, mine, x);
            keep(mem.v, mem.v_params, place, h, mine, y);
        }
    }
}

template <typename TOut, int ST, bool ALIGNED>
__global__ void __launch_bounds__(kMaxThreads, 2) cache_read_kernel(CacheReadArgs a, int tile_rows, int lanes)
{
    __shared__ RowPlace places[kMaxTileRows];
    const CacheMemory& mem = a.mem;
    const int row0 = blockIdx.x * tile_rows;
    find_places<ST>(mem, a.batch, row0, tile_rows, nullptr, false, 0, 0, a.error_flag, places);

    const int chunks = mem.head_dim / 8;
    const int lane = threadIdx.x / chunks, f = (threadIdx.x - lane * chunks) * 8;
    if (lane >= lanes)
        return;
    for (int r = 0; r < tile_rows; r++)
    {
        const RowPlace& place = places[r];
        if (place.position < 0)
            continue;
        const int64_t row = row0 + r;
        TOut* k = reinterpret_cast<TOut*>(a.k_out) + row * a.k_stride + f;
        TOut* v = reinterpret_cast<TOut*>(a.v_out) + row * a.v_stride + f;
        for (int h = lane; h < mem.heads; h += lanes)
        {
            const int64_t at = place.slot + h * mem.head_stride;
            float x[8], y[8];
            if (ST == AWA_INT4)
            {
                const int64_t par = place.params + h * mem.params_head_stride + f / AWA_CACHE_GROUP * 4;
                const uint32_t kc = *reinterpret_cast<const uint32_t*>(mem.k + at + f / 2);
                const uint32_t vc = *reinterpret_cast<const uint32_t*>(mem.v + at + f / 2);
                const uint32_t kp = *reinterpret_cast<const uint32_t*>(mem.k_params + par);
                const uint32_t vp = *reinterpret_cast<const uint32_t*>(mem.v_params + par);
                dequantize8(kc, kp, x);
                dequantize8(vc, vp, y);
            }
            else if (ST == AWA_F32)
            {
                load8(reinterpret_cast<const float*>(mem.k + at) + f, x);
                load8(reinterpret_cast<const float*>(mem.v + at) + f, y);
            }
            else
            {
                load8(reinterpret_cast<const bf16*>(mem.k + at) + f, x);
                load8(reinterpret_cast<const bf16*>(mem.v + at) + f, y);
            }
            put8<TOut, ALIGNED>(k + h * mem.head_dim, x);
            put8<TOut, ALIGNED>(v + h * mem.head_dim, y);
        }
    }
}

// 8 floats as fp16.
__device__ __forceinline__ uint4 half8(const float (&v)[8])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
    {
        const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The largest magnitudes that the minimum and scale of a group allow, of what
// some row sees, per head and 64 features: kRangeParts parts, x of the grid, for
// cache_unpack_kernel to join (no zeros to begin with, no atomics). Warps share
// the pages, lanes the slots of a page; y = heads.
constexpr int kRangeParts = 32;

template <int GROUPS>
__global__ void __launch_bounds__(kThreads) cache_range_kernel(CacheUnpackArgs a)
{
    constexpr int kWarps = kThreads / 32;
    __shared__ unsigned most_s[kWarps][2 * GROUPS];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const CacheMemory& mem = a.mem;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, page_tokens = 1 << mem.page_shift;
    const int64_t head = blockIdx.y * mem.params_head_stride;
    float most[2 * GROUPS] = {};  // k, v of each group
    int total = a.most_seen;
    if (total > kRangeParts * kWarps)
        find_page(a, 0, &total);
    const int share = (total + kRangeParts * kWarps - 1) / (kRangeParts * kWarps);
    int i = ((int)blockIdx.x * kWarps + warp) * share;
    for (const int end = min(total, i + share); i < end;)
    {
        const PageSlot at = find_page(a, i);
        if (at.b < 0)
            break;
        const int run = min(min(at.run, end - i), 32);
        const int page_lane =
            lane < run ? __ldg(a.batch.page_table + at.b * a.batch.table_stride + at.entry + lane) : -1;
#pragma unroll 2
        for (int n = 0; n < run; n++)
        {
            const int page = __shfl_sync(0xffffffffu, page_lane, n);
            if ((unsigned)page >= (unsigned)mem.pages)
                continue;  // reported where it is unpacked
            for (int slot = lane; slot < page_tokens; slot += 32)
            {
                const int key = ((at.entry + n) << mem.page_shift) + slot;
                if (!(key < at.hi && (key >= at.lo || key < a.sinks)))
                    continue;
                const int64_t from = page * mem.params_page_stride + head + (int64_t)slot * GROUPS * 4;
#pragma unroll
                for (int g = 0; g < 2 * GROUPS; g++)
                {
                    const uint32_t params = __ldg(
                        reinterpret_cast<const uint32_t*>((g & 1 ? mem.v_params : mem.k_params) + from) + (g >> 1));
                    const float scale = __uint_as_float(params << 16), low = __uint_as_float(params & 0xffff0000u);
                    most[g] = fmaxf(most[g], fmaxf(fabsf(low), fabsf(fmaf(15.f, scale, low))));
                }
            }
        }
        i += run;
    }
    // floats that are not negative are ordered as their bits are
#pragma unroll
    for (int g = 0; g < 2 * GROUPS; g++)
    {
        const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(most[g]));
        if (lane == 0)
            most_s[warp][g] = bits;
    }
    __syncthreads();
    if (threadIdx.x < 2 * GROUPS)
    {
        unsigned bits = 0;
        for (int w = 0; w < kWarps; w++)
            bits = max(bits, most_s[w][threadIdx.x]);
        a.range_parts[((int64_t)blockIdx.y * kRangeParts + blockIdx.x) * 2 * GROUPS + threadIdx.x] = bits;
    }
}

// Ends when cache_range_kernel, beside which the unpacking starts, has ended.
__device__ __forceinline__ void wait_for_ranges()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// One part of what cache_range_kernel found. Not __ldg: written while this
// kernel may have been there already.
__device__ __forceinline__ unsigned range_part(const CacheUnpackArgs& a, int kv, int part, int i)
{
    const int each = 2 * (a.mem.head_dim / AWA_CACHE_GROUP);
    return __ldcg(a.range_parts + ((int64_t)kv * kRangeParts + part) * each + i);
}

// 8 features of q a thread; the head_dim / 8 lanes of one head and row, which
// stand side by side, share its power of two, the 8 lanes of a group of features
// look for that of its keys.
__device__ __forceinline__ void unpack_queries(const CacheUnpackArgs& a, int64_t first, int64_t step)
{
    const int d = a.mem.head_dim, shift = d == 64 ? 6 : 7, heads = a.q_row >> shift, lanes = d / 8;
    const int per_kv = heads / a.mem.heads;
    const int64_t chunks = a.q_row / 8, all = chunks * a.batch.rows;
    const int lane = threadIdx.x & 31;
    for (int64_t i = first; i - lane < all; i += step)
    {
        const bool mine = i < all;
        const int64_t row = mine ? i / chunks : 0;
        const int f = mine ? (int)(i - row * chunks) * 8 : 0;  // of the row
        float v[8] = {};
        if (mine)
            load8(static_cast<const bf16*>(a.q) + row * a.q_stride + f, v);
        float most = 0.f;
#pragma unroll
        for (int j = 0; j < 8; j++)
            most = fmaxf(most, fabsf(v[j]));
        const int head = f >> shift, group = (f & (d - 1)) / AWA_CACHE_GROUP;
        unsigned range = 0;
#pragma unroll
        for (int part = 0; part < kRangeParts; part += 8)
            range = max(range, range_part(a, head / per_kv, part + (lane & 7), 2 * group));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1)
            range = max(range, __shfl_xor_sync(0xffffffffu, range, o));
        const int down = half_shift(range);
        int top = most > 0.f ? (int)(__float_as_uint(most) >> 23) - 127 - down : -1024;
        for (int o = 1; o < lanes; o <<= 1)
            top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        const int up = top == -1024 ? 0 : 14 - top;
        // in two factors: one may be outside the floats' range
        const int n0 = max(-126, min(127, up - down)), n1 = max(-126, min(127, up - down - n0));
        const float by0 = power_of_two(n0), by1 = power_of_two(n1);
#pragma unroll
        for (int j = 0; j < 8; j++)
            v[j] = v[j] * by0 * by1;
        if (!mine)
            continue;
        reinterpret_cast<uint4*>(a.q_out)[i] = half8(v);
        // never 0 or infinite, which would make NaN of a masked or an empty score; so
        // far out, scores are next to 0 or beyond the floats
        if ((f & (d - 1)) == 0)
            a.score_scale[row * heads + head] =
                fminf(fmaxf(ldexpf(a.scale * 1.4426950408889634f, -up), 0x1p-126f), 0x1p127f);
    }
}

// The ranges of head blockIdx.y, by one warp, as the powers of two of its keys
// and values or, for the attention, into a.ranges.
__device__ __forceinline__ void join_ranges(const CacheUnpackArgs& a, float* up)
{
    static_assert(kRangeParts == 32, "a lane takes a part");
    const int lane = threadIdx.x & 31, each = 2 * (a.mem.head_dim / AWA_CACHE_GROUP);
    const unsigned* from = a.range_parts + ((int64_t)blockIdx.y * kRangeParts + lane) * each;
    unsigned bits[4] = {};
    if (each == 4)
    {
        const uint4 x = __ldcg(reinterpret_cast<const uint4*>(from));
        bits[0] = x.x, bits[1] = x.y, bits[2] = x.z, bits[3] = x.w;
    }
    else
    {
        const uint2 x = __ldcg(reinterpret_cast<const uint2*>(from));
        bits[0] = x.x, bits[1] = x.y;
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
        bits[i] = __reduce_max_sync(0xffffffffu, bits[i]);
    const unsigned mine = lane == 0 ? bits[0] : lane == 1 ? bits[1] : lane == 2 ? bits[2] : bits[3];
    if (lane >= each)
        return;
    if (up)
        up[lane] = power_of_two(half_shift(mine));
    else
        a.ranges[blockIdx.y * each + lane] = mine;
}

// The 4-bit pages that some row of the batch sees -> their keys and values as fp16
// (rounded by 2^-12, where bf16's 2^-9 of every key would show in the scores),
// and their numbers in the workspace's page table, if it has one. Blocks: x < page_blocks
// share the pages of all sequences in order, y = heads; the blocks x behind them
// take the q rows.
__global__ void __launch_bounds__(kThreads, 8) cache_unpack_kernel(CacheUnpackArgs a, int page_blocks)
{
    __shared__ float up_s[4];  // powers of two: keys and values of each group
    __shared__ PageSlot first_s;
    __shared__ int index_s[2];
    const CacheMemory& mem = a.mem;
    if ((int)blockIdx.x >= page_blocks)
    {
        wait_for_ranges();
        if ((int)blockIdx.x == page_blocks && threadIdx.x < 32)
            join_ranges(a, nullptr);
        unpack_queries(a, ((int64_t)(blockIdx.x - page_blocks) * gridDim.y + blockIdx.y) * kThreads + threadIdx.x,
                       (int64_t)(gridDim.x - page_blocks) * gridDim.y * kThreads);
        return;
    }
    const int warp = threadIdx.x >> 5;
    if (warp == 0)
    {
        int total = a.most_seen;
        if (total > page_blocks)
            find_page(a, 0, &total);
        const int share = (total + page_blocks - 1) / page_blocks, first = (int)blockIdx.x * share;
        const PageSlot at = first < total ? find_page(a, first) : PageSlot{-1, 0, 0, 0, 0};
        if (threadIdx.x == 0)
        {
            first_s = at;
            index_s[0] = first;
            index_s[1] = min(total, first + share);
        }
    }
    else if (warp == 1)  // beside it
    {
        wait_for_ranges();  // every block: the grid must not end ahead of that kernel
        join_ranges(a, up_s);
    }
    __syncthreads();
    int index = index_s[0];
    const int end = index_s[1];
    PageSlot at = first_s;
    const int kv = blockIdx.y, groups = mem.head_dim / AWA_CACHE_GROUP, row_bytes = mem.head_dim / 2;
    const int64_t page_bytes = (int64_t)row_bytes << mem.page_shift;  // of codes
    const int pieces = (int)(page_bytes / 8);                         // of the keys, then as many of the values
    while (at.b >= 0)
    {
        const int run = min(at.run, end - index);
        const int* entries = a.batch.page_table + at.b * a.batch.table_stride + at.entry;
        for (int n = 0; n < run; n++, index++)
        {
            const int page = __ldg(entries + n);
            const bool real = (unsigned)page < (unsigned)mem.pages;
            if (threadIdx.x == 0 && kv == 0)
            {
                if (!real)
                    cache_error(a.error_flag, AWA_CACHE_BAD_PAGE);
                if (a.table)
                    a.table[(int64_t)at.b * a.batch.table_width + at.entry + n] = index;
            }
            if (!a.table && !real)
                continue;  // the attention finds it missing
            const int64_t src = page * mem.page_stride + kv * mem.head_stride;
            const int64_t par = page * mem.params_page_stride + kv * mem.params_head_stride;
            // a page that several sequences see is written by each, with the same bytes
            const int64_t dst = ((int64_t)(a.table ? index : page) * mem.heads + kv) * page_bytes * 4;
            // 16 codes, of one group, a thread and turn
            for (int i = threadIdx.x; i < 2 * pieces; i += kThreads)
            {
                const bool is_k = i < pieces;
                const int from = (is_k ? i : i - pieces) * 8;
                uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
                if (real)
                {
                    const uint2 codes = __ldg(reinterpret_cast<const uint2*>((is_k ? mem.k : mem.v) + src + from));
                    const int row = from / row_bytes, group = (from - row * row_bytes) / (AWA_CACHE_GROUP / 2);
                    const uint32_t params =
                        __ldg(reinterpret_cast<const uint32_t*>((is_k ? mem.k_params : mem.v_params) + par) +
                              row * groups + group);
                    // scaled ahead of the products: the same roundings
                    const float by = up_s[2 * group + (is_k ? 0 : 1)];
                    const float scale = __uint_as_float(params << 16) * by;
                    const float minimum = __uint_as_float(params & 0xffff0000u) * by;
                    float v[8];
                    dequantize8(codes.x, scale, minimum, v);
                    out[0] = half8(v);
                    dequantize8(codes.y, scale, minimum, v);
                    out[1] = half8(v);
                }
                uint4* to = reinterpret_cast<uint4*>((is_k ? a.k_out : a.v_out) + dst + (int64_t)from * 4);
                to[0] = out[0];
                to[1] = out[1];
            }
        }
        if (index >= end)
            break;
        at = find_page(a, index);  // by each warp: none waits for another
    }
}

struct Shape
{
    int blocks, threads, tile_rows, lanes;
};

// Heads side by side: the multiple of the cache's heads that leaves the fewest
// threads idle over q, k and v, at more than 128 threads, if the heads allow it, and
// at most 512. Few rows: a block each.
// More: a block takes several, so that the lookup of sequence, page and
// coordinates, which its threads wait for, is paid once a tile: 4, and 16 where
// that still leaves every SM some blocks (86074 rows: 478 us with 4, 455 with
// 16; 1790 fp32 rows: 12.4 and 24.6).
Shape shape_of(int rows, int q_heads, int heads, int head_dim)
{
    Shape s;
    const int chunks = head_dim / 8, most = kMaxThreads / chunks, least = 128 / chunks + 1;
    s.lanes = most;
    double best = 0;
    for (int lanes = heads < most ? heads : most; lanes <= most; lanes += heads)
    {
        const int passes = (q_heads + lanes - 1) / lanes + 2 * ((heads + lanes - 1) / lanes);
        const double used = (double)(q_heads + 2 * heads) / ((double)passes * lanes);
        if ((lanes >= least || lanes + heads > most) && used >= best)
        {
            best = used;
            s.lanes = lanes;
        }
    }
    s.threads = (s.lanes * chunks + 31) / 32 * 32;
    s.tile_rows = rows < 148 * 8 ? 1 : rows < 148 * 64 ? 4 : kMaxTileRows;
    s.blocks = (rows + s.tile_rows - 1) / s.tile_rows;
    return s;
}

template <typename TIn, typename TQ, int ST>
void run_append(const CacheAppendArgs& a, cudaStream_t stream)
{
    const Shape s = shape_of(a.batch.rows, a.q_heads, a.mem.heads, a.mem.head_dim);
    if (a.aligned)
        cache_append_kernel<TIn, TQ, ST, true><<<s.blocks, s.threads, 0, stream>>>(a, s.tile_rows, s.lanes);
    else
        cache_append_kernel<TIn, TQ, ST, false><<<s.blocks, s.threads, 0, stream>>>(a, s.tile_rows, s.lanes);
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
    const Shape s = shape_of(a.batch.rows, 0, a.mem.heads, a.mem.head_dim);
    if (a.aligned)
        cache_read_kernel<TOut, ST, true><<<s.blocks, s.threads, 0, stream>>>(a, s.tile_rows, s.lanes);
    else
        cache_read_kernel<TOut, ST, false><<<s.blocks, s.threads, 0, stream>>>(a, s.tile_rows, s.lanes);
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

size_t cache_unpack_range_bytes(const CacheMemory& mem, int heads)
{
    return (size_t)heads * kRangeParts * 2 * (mem.head_dim / AWA_CACHE_GROUP) * sizeof(unsigned);
}

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

int launch_cache_unpack(const CacheUnpackArgs& a, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_unpack", stream);
    const dim3 grid(kRangeParts, (unsigned)a.mem.heads);
    if (a.mem.head_dim == AWA_CACHE_GROUP)
        cache_range_kernel<1><<<grid, kThreads, 0, stream>>>(a);
    else
        cache_range_kernel<2><<<grid, kThreads, 0, stream>>>(a);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess)
        return (int)err;
    // 4 pieces of q a thread
    const int64_t pieces = (int64_t)a.batch.rows * (a.q_row / 8), at_once = (int64_t)4 * kThreads * a.mem.heads;
    const int64_t q_blocks = (pieces + at_once - 1) / at_once;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    config.stream = stream;
    // Blocks for the pages: several times what runs at once, so that the last ones
    // even the SMs out (64 x 30000 keys, 8 heads: 1.86 ms, with a quarter of them 2.26)
    const int blocks = 148 * 32 / a.mem.heads + 1, page_blocks = a.most_seen < blocks ? a.most_seen : blocks;
    config.gridDim = dim3((unsigned)(page_blocks + q_blocks), (unsigned)a.mem.heads);
    config.blockDim = dim3(kThreads);
    return (int)cudaLaunchKernelEx(&config, cache_unpack_kernel, a, page_blocks);
}

}  // namespace awa
