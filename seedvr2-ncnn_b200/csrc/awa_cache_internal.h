// awa_cache_internal.h -- what the host side of the key/value cache
// (awa_cache.cpp) hands to its kernels (awa_cache_*.cu).
#pragma once

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

#include "awa_cache.h"
#include "awa_internal.h"

namespace awa
{

// The cache's memory as the kernels address it. Strides in bytes.
struct CacheMemory
{
    int storage;
    int heads;
    int head_dim;
    int page_shift;  // log2(page_tokens)
    int pages;
    char* k;
    char* v;
    int64_t page_stride, head_stride;
    char* k_params;
    char* v_params;
    int64_t params_page_stride, params_head_stride;
};

struct CacheBatch
{
    int sequences;
    int rows;
    const int* row_starts;
    const int* past;
    const int* page_table;
    int table_width;
    int64_t table_stride;
};

struct CacheAppendArgs
{
    CacheMemory mem;
    CacheBatch batch;
    int q_heads;  // 0: no q
    const char *q, *k, *v;
    int64_t q_stride, k_stride, v_stride;  // elements
    char* q_out;
    int64_t q_out_stride;
    const float2* table;  // NULL: no rotation
    int max_coord, axes, pairs;
    const int* coords;
    int aligned;  // every row can be read and written in 16-byte pieces
    int* error_flag;
};

struct CacheReadArgs
{
    CacheMemory mem;
    CacheBatch batch;
    char *k_out, *v_out;
    int64_t k_stride, v_stride;  // elements
    int aligned;
    int* error_flag;
};

// 4-bit pages that a batch sees -> dense fp16 pages [page][head][slot][head_dim];
// the batch's q rows, bf16 -> dense fp16. The pages take the numbers that they
// have in the cache, or those in which the sequences see them, with a page table
// [sequences][table_width]: whichever needs room for fewer. fp16 keeps 11 bits of
// numbers from 2^-14 to 2^16 only, so all of it is scaled by powers of two: the
// keys and the values of a head's 64 features to below 2^15 (half_shift() of their
// largest, in `ranges`), a row of q to below 2^15 after it has taken the keys'
// powers back. score_scale: what the products of a row's scores are multiplied by,
// `scale` log2(e) and those powers.
struct CacheUnpackArgs
{
    CacheMemory mem;
    CacheBatch batch;
    int sinks, window, frame_tokens;
    char *k_out, *v_out, *q_out;
    int* table;  // NULL: the pages keep their numbers
    const void* q;
    int64_t q_stride;
    int q_row;  // elements of a row
    int most_seen;  // pages of all sequences together, at most
    unsigned* ranges;    // [heads][head_dim / 64][k, v]: bits of the largest magnitude that some row sees
    unsigned* range_parts;  // cache_unpack_range_bytes()
    float* score_scale;  // [rows][q heads]
    float scale;
    int* error_flag;
};

struct CacheAttnArgs
{
    CacheMemory mem;
    CacheBatch batch;
    int group;  // q heads per key/value head
    const void* q;
    int64_t q_stride;  // elements
    void* out;
    int64_t out_stride;
    float scale;
    int sinks, window, frame_tokens;
    const unsigned* ranges;    // of what launch_cache_unpack wrote
    const float* score_scale;
    int* error_flag;
};

int launch_cache_append(const CacheAppendArgs& args, int in_dtype, int q_out_dtype, cudaStream_t stream);
int launch_cache_read(const CacheReadArgs& args, int out_dtype, cudaStream_t stream);
size_t cache_unpack_range_bytes(const CacheMemory& mem, int heads);
int launch_cache_unpack(const CacheUnpackArgs& args, cudaStream_t stream);
// fp32 and bf16 caches of any head_dim, fp32 arithmetic.
int launch_cache_attention_simt(const CacheAttnArgs& args, int max_rows, cudaStream_t stream);
// fp32 caches with head_dim 64 or 128, for many rows per sequence.
int launch_cache_attention_f32(const CacheAttnArgs& args, cudaStream_t stream);
// bf16 and 4-bit caches with head_dim 64 or 128, for few rows per sequence;
// most_keys: no row sees more. The workspace holds the parts of tiles that
// several blocks work on (0 bytes for short caches).
size_t cache_attention_step_workspace(const CacheMemory& mem, int group, int max_rows, int64_t most_keys);
int launch_cache_attention_step(const CacheAttnArgs& args, int max_rows, int64_t most_keys, void* workspace,
                                cudaStream_t stream);
// bf16 caches with head_dim 64 or 128 and at most 128 q heads per key/value
// head, for many rows per sequence.
size_t cache_attention_tile_workspace(int head_dim);
int cache_attention_tile_sequences();  // the most it takes
// half: q, k and v hold fp16 (what launch_cache_unpack writes), out bf16 as ever.
int launch_cache_attention_tile(const CacheAttnArgs& args, bool half, void* workspace, cudaStream_t stream);
// cudaFuncSetAttribute calls of the kernels, once per handle (not allowed to
// fail later, inside a capture).
int prepare_cache_attention_simt();
int prepare_cache_attention_f32();
int prepare_cache_attention_step();
int prepare_cache_attention_tile();

}  // namespace awa
