// awa_cache_device.cuh -- which sequence a row belongs to, where a position is
// stored and what a row sees: shared by the key/value cache kernels.
#pragma once

#include "awa_cache_internal.h"
#include "awa_device.cuh"

namespace awa
{

__device__ __forceinline__ void cache_error(int* flag, int code)
{
    if (flag)
        atomicCAS(flag, 0, code);
}

// n for the 2^n that brings numbers up to the one with these bits below 2^15,
// for use as fp16 operands: -114 to 126, so that 2^n and 2^-n are normal floats.
__device__ __forceinline__ int half_shift(unsigned bits)
{
    return 14 - max((int)(bits >> 23) - 127, -112);
}

__device__ __forceinline__ float power_of_two(int n)  // -126 to 127
{
    return __int_as_float((n + 127) << 23);
}

// Sequence whose rows contain `row` (largest b with row_starts[b] <= row), or
// -1 if it belongs to nobody. Empty sequences share their start with the next.
__device__ __forceinline__ int sequence_of_row(const CacheBatch& batch, int row)
{
    if (row < __ldg(batch.row_starts) || row >= __ldg(batch.row_starts + batch.sequences))
        return -1;
    int lo = 0, hi = batch.sequences;  // row_starts[lo] <= row < row_starts[hi]
    while (hi - lo > 1)
    {
        const int mid = (lo + hi) >> 1;
        if (__ldg(batch.row_starts + mid) <= row)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Position in sequence b of a row of it. A past that is out of range gives one
// that no page table reaches.
__device__ __forceinline__ int position_of_row(const CacheBatch& batch, int b, int row)
{
    const int64_t p = (int64_t)__ldg(batch.past + b) + (row - __ldg(batch.row_starts + b));
    return p < 0 || p > 0x7fffffff ? -1 : (int)p;
}

// Page that holds position `pos` of sequence b, or -1 (reported) if the table
// does not reach it or names a page that the cache does not have.
__device__ __forceinline__ int page_of(const CacheMemory& mem, const CacheBatch& batch, int b, int pos, int* flag)
{
    const int entry = pos >> mem.page_shift;
    int page = -1;
    if (pos >= 0 && entry < batch.table_width)
        page = __ldg(batch.page_table + b * batch.table_stride + entry);
    if (page < 0 || page >= mem.pages)
    {
        cache_error(flag, AWA_CACHE_BAD_PAGE);
        return -1;
    }
    return page;
}

// Keys that a row sees: [0, sinks) and [lo, hi), lo <= hi.
struct RowSpan
{
    int lo, hi;
};

// The row at position p of a sequence of `length` positions.
__device__ __forceinline__ RowSpan row_span(int p, int length, int sinks, int window, int frame_tokens)
{
    RowSpan s;
    const bool prefix = p < sinks;
    const int at = prefix ? p : p - sinks;
    const int f = frame_tokens == 1 ? at : at / frame_tokens;  // a division is most of this function
    const int64_t end = (prefix ? 0 : sinks) + ((int64_t)f + 1) * frame_tokens;
    s.hi = (int)min((int64_t)(prefix ? min(sinks, length) : length), end);
    s.lo = !prefix && window > 0 && f >= window ? sinks + (f - window + 1) * frame_tokens : 0;
    return s;
}

// Length of sequence b after this call: past + rows, cut (and reported) at
// what its page table can hold.
__device__ __forceinline__ int sequence_length(const CacheMemory& mem, const CacheBatch& batch, int past, int rows,
                                               int* flag)
{
    const int64_t room = (int64_t)batch.table_width << mem.page_shift;
    const int64_t length = (int64_t)past + rows;
    if (length > room)
    {
        cache_error(flag, AWA_CACHE_BAD_PAGE);
        return (int)room;
    }
    return (int)length;
}

// The key blocks of kb keys (aligned to kb in position) that some row of a
// tile sees: the blocks of the prefix, then those of the window.
struct KeyBlocks
{
    int prefix;  // blocks 0 .. prefix - 1 start at 0
    int shift;   // block i >= prefix is block i + shift of the sequence
    int count;
};

__device__ __forceinline__ KeyBlocks key_blocks(RowSpan first, RowSpan last, int sinks, int kb)
{
    // lo and hi do not fall from row to row, so the first row of a tile has
    // the lowest lo and the last row the highest hi.
    KeyBlocks k;
    const int hi = (last.hi + kb - 1) / kb;
    const int prefix = first.lo > 0 ? min((min(sinks, last.hi) + kb - 1) / kb, hi) : 0;
    const int from = max(first.lo / kb, prefix);
    k.prefix = prefix;
    k.shift = from - prefix;
    k.count = prefix + max(0, hi - from);
    return k;
}

// Rows of sequence b; starts that reach outside the batch's rows get none there.
__device__ __forceinline__ int batch_rows(const CacheBatch& batch, int b)
{
    const int start = __ldg(batch.row_starts + b), end = min(__ldg(batch.row_starts + b + 1), batch.rows);
    return start < 0 ? 0 : max(0, end - start);
}

// A tile of query rows: m rows m0 .. m0 + count - 1 of sequence b, where row m
// is head (m % group) of its group at row m / group of the sequence.
struct QueryTile
{
    int b;      // -1: none
    int m0;
    int count;
    int row0;   // first row of the sequence in the row tensors
    int past;
    int length;
};

// Tile number `index` of the batch, tiles of `tile` m rows counted sequence by
// sequence. Called by one full warp; the result is the same in all lanes.
__device__ __forceinline__ QueryTile find_tile(const CacheMemory& mem, const CacheBatch& batch, int group, int tile,
                                               int index, int* flag)
{
    const int lane = threadIdx.x & 31;
    QueryTile t;
    t.b = -1;
    int before = 0;  // tiles of the sequences before `base`
    for (int base = 0; base < batch.sequences; base += 32)
    {
        const int b = base + lane;
        int start = 0, rows = 0, past = 0;
        if (b < batch.sequences)
        {
            start = __ldg(batch.row_starts + b);
            past = __ldg(batch.past + b);  // in flight with the starts
            rows = batch_rows(batch, b);
        }
        const int tiles = (int)(((int64_t)rows * group + tile - 1) / tile);
        int sum = tiles;
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
            const int first = before + __shfl_sync(0xffffffffu, sum - tiles, src);
            t.b = base + src;
            t.row0 = __shfl_sync(0xffffffffu, start, src);
            const int n = __shfl_sync(0xffffffffu, rows, src);
            t.m0 = (index - first) * tile;
            t.count = min(tile, n * group - t.m0);
            t.past = max(0, __shfl_sync(0xffffffffu, past, src));
            t.length = sequence_length(mem, batch, t.past, n, flag);
            t.past = min(t.past, t.length);  // of a cut sequence: keeps past + rows within 31 bits
            return t;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    return t;
}

}  // namespace awa
