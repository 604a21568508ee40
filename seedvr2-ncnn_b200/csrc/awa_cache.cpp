// awa_cache.cpp -- host side of the paged key/value cache (include/awa_cache.h):
// the handle, the checks of the arguments and the choice of the kernel.
#include "awa_cache.h"
#include "awa_cache_internal.h"
#include "awa_internal.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <initializer_list>
#include <new>

#include <cuda_runtime.h>

struct awa_cache
{
    awa::CacheMemory mem{};
    int device = -1;
    int* error_flag = nullptr;
};

namespace
{

int fail(int code, const char* fmt, ...)
{
    char buffer[512];
    va_list args;
    va_start(args, fmt);
    std::vsnprintf(buffer, sizeof(buffer), fmt, args);
    va_end(args);
    return awa::report_error(code, buffer);
}

int launch_status(int err, const char* what)
{
    return err == 0 ? AWA_OK
                    : fail(AWA_ERR_CUDA, "%s: %s", what, cudaGetErrorString(static_cast<cudaError_t>(err)));
}

bool float_type(int dtype)
{
    return dtype == AWA_F32 || dtype == AWA_BF16;
}

int type_bytes(int dtype)
{
    return dtype == AWA_F32 ? 4 : 2;
}

bool aligned(const void* p, int64_t stride_bytes, int to)
{
    return reinterpret_cast<uintptr_t>(p) % to == 0 && stride_bytes % to == 0;
}

int check_params(const awa_cache_params& p)
{
    if (p.storage != AWA_F32 && p.storage != AWA_BF16 && p.storage != AWA_INT4)
        return fail(AWA_ERR_INVALID, "awa_cache_create: storage %d is not AWA_F32, AWA_BF16 or AWA_INT4", p.storage);
    if (p.heads <= 0 || p.heads > 65535 || p.pages <= 0)
        return fail(AWA_ERR_INVALID, "awa_cache_create: heads (%d, at most 65535) and pages (%d) must be positive",
                    p.heads, p.pages);
    if (p.head_dim <= 0 || p.head_dim % 8 || p.head_dim > awa::kMaxHeadDim)
        return fail(AWA_ERR_INVALID, "awa_cache_create: head_dim %d must be a multiple of 8 up to %d", p.head_dim,
                    awa::kMaxHeadDim);
    if (p.storage == AWA_INT4 && p.head_dim != 64 && p.head_dim != 128)
        return fail(AWA_ERR_INVALID, "awa_cache_create: a 4-bit cache needs head_dim 64 or 128, not %d", p.head_dim);
    if (p.page_tokens < 16 || p.page_tokens > 256 || (p.page_tokens & (p.page_tokens - 1)))
        return fail(AWA_ERR_INVALID, "awa_cache_create: page_tokens %d must be 16, 32, 64, 128 or 256", p.page_tokens);
    if (!p.k || !p.v || (p.storage == AWA_INT4 && (!p.k_params || !p.v_params)))
        return fail(AWA_ERR_INVALID, "awa_cache_create: NULL memory");
    const int64_t row = p.storage == AWA_INT4 ? p.head_dim / 2 : p.head_dim;
    const int64_t element = p.storage == AWA_INT4 ? 1 : type_bytes(p.storage);
    // what tensor maps take, and far from where products of them pass 64 bits
    const int64_t most = (int64_t)1 << 40;  // bytes
    if (p.head_stride >= most / element || p.page_stride >= most / element ||
        (p.storage == AWA_INT4 && (p.params_head_stride >= most / 2 || p.params_page_stride >= most / 2)))
        return fail(AWA_ERR_INVALID, "awa_cache_create: strides must stay below 2^40 bytes");
    // either order of pages and heads, but no two rows in one place
    const bool fits = p.head_stride >= p.page_tokens * row && p.page_stride >= p.page_tokens * row &&
                      (p.page_stride >= p.heads * p.head_stride || p.head_stride >= p.pages * p.page_stride);
    if (!fits)
        return fail(AWA_ERR_INVALID, "awa_cache_create: strides smaller than the pages they separate");
    if (!aligned(p.k, p.page_stride * element, 16) || !aligned(p.v, p.head_stride * element, 16))
        return fail(AWA_ERR_INVALID, "awa_cache_create: memory and strides must be multiples of 16 bytes");
    if (p.storage == AWA_INT4)
    {
        const int64_t prow = 2 * (p.head_dim / AWA_CACHE_GROUP);
        const bool pfits = p.params_head_stride >= p.page_tokens * prow &&
                           p.params_page_stride >= p.page_tokens * prow &&
                           (p.params_page_stride >= p.heads * p.params_head_stride ||
                            p.params_head_stride >= p.pages * p.params_page_stride);
        if (!pfits || !aligned(p.k_params, p.params_page_stride * 2, 16) ||
            !aligned(p.v_params, p.params_head_stride * 2, 16))
            return fail(AWA_ERR_INVALID,
                        "awa_cache_create: params strides too small, or not multiples of 16 bytes");
    }
    return AWA_OK;
}

// The checks every call makes of its cache and batch, and the batch as the
// kernels take it. *empty: there is nothing to do.
int check_batch(const char* what, const awa_cache* cache, const awa_cache_batch* batch, awa::CacheBatch* out,
                bool* empty)
{
    if (!cache || !batch)
        return fail(AWA_ERR_INVALID, "%s: cache and batch must not be NULL", what);
    if (batch->sequences < 0 || batch->rows < 0 || batch->max_rows < 0 || batch->table_width < 0)
        return fail(AWA_ERR_INVALID, "%s: negative sequences, rows, max_rows or table_width", what);
    // positions and rows add up within 31 bits
    if (((int64_t)batch->table_width << cache->mem.page_shift) > 1 << 30 || batch->rows >= 1 << 30)
        return fail(AWA_ERR_INVALID, "%s: table_width %d and rows %d must stay within 2^30 positions", what,
                    batch->table_width, batch->rows);
    *empty = batch->sequences == 0 || batch->rows == 0;
    if (!*empty)
    {
        if (!batch->row_starts || !batch->past || !batch->page_table)
            return fail(AWA_ERR_INVALID, "%s: NULL row_starts, past or page_table", what);
        if (!aligned(batch->row_starts, 0, 4) || !aligned(batch->past, 0, 4) || !aligned(batch->page_table, 0, 4))
            return fail(AWA_ERR_INVALID, "%s: row_starts, past and page_table must be 4-byte aligned", what);
        if (batch->table_stride < batch->table_width)
            return fail(AWA_ERR_INVALID, "%s: table_stride smaller than table_width", what);
    }
    out->sequences = batch->sequences;
    out->rows = batch->rows;
    out->row_starts = batch->row_starts;
    out->past = batch->past;
    out->page_table = batch->page_table;
    out->table_width = batch->table_width;
    out->table_stride = batch->table_stride;
    return AWA_OK;
}

// The last check of a call, ahead of its launch.
int check_device(const char* what, const awa_cache* cache)
{
    if (cache->device < 0)
        return fail(AWA_ERR_INVALID, "%s: the cache was created without a device (awa_cache_create_host)", what);
    int device = -1;
    if (cudaGetDevice(&device) != cudaSuccess)
        return fail(AWA_ERR_CUDA, "%s: cudaGetDevice failed", what);
    if (device != cache->device)
        return fail(AWA_ERR_INVALID, "%s: the cache lives on device %d but device %d is current", what, cache->device,
                    device);
    return AWA_OK;
}

// The memory of a cache lies where a kernel on `device` reaches it.
int check_memory(const awa_cache_params& p, int device)
{
    const bool four = p.storage == AWA_INT4;
    for (const void* memory : {p.k, p.v, four ? p.k_params : nullptr, four ? p.v_params : nullptr})
    {
        if (!memory)
            continue;
        cudaPointerAttributes at{};
        const cudaError_t err = cudaPointerGetAttributes(&at, memory);
        if (err != cudaSuccess)
        {
            cudaGetLastError();  // not the caller's
            return fail(AWA_ERR_CUDA, "awa_cache_create: %s", cudaGetErrorString(err));
        }
        if (at.type == cudaMemoryTypeUnregistered)
            return fail(AWA_ERR_INVALID, "awa_cache_create: memory that the GPU cannot reach");
        if (at.type == cudaMemoryTypeDevice && at.device != device)
            return fail(AWA_ERR_INVALID, "awa_cache_create: the memory lies on device %d but device %d is current",
                        at.device, device);
    }
    return AWA_OK;
}

int create(const awa_cache_params* params, awa_cache** out, bool on_device)
{
    if (!params || !out)
        return fail(AWA_ERR_INVALID, "awa_cache_create: params and out must not be NULL");
    *out = nullptr;
    const int rc = check_params(*params);
    if (rc)
        return rc;
    awa_cache* cache = new (std::nothrow) awa_cache;
    if (!cache)
        return fail(AWA_ERR_ALLOC, "awa_cache_create: out of host memory");
    awa::CacheMemory& m = cache->mem;
    const int64_t element = params->storage == AWA_INT4 ? 1 : type_bytes(params->storage);
    m.storage = params->storage;
    m.heads = params->heads;
    m.head_dim = params->head_dim;
    for (m.page_shift = 0; (1 << m.page_shift) < params->page_tokens; m.page_shift++)
    {
    }
    m.pages = params->pages;
    m.k = static_cast<char*>(params->k);
    m.v = static_cast<char*>(params->v);
    m.page_stride = params->page_stride * element;
    m.head_stride = params->head_stride * element;
    if (params->storage == AWA_INT4)
    {
        m.k_params = static_cast<char*>(params->k_params);
        m.v_params = static_cast<char*>(params->v_params);
        m.params_page_stride = params->params_page_stride * 2;
        m.params_head_stride = params->params_head_stride * 2;
    }
    if (on_device)
    {
        cudaError_t err = cudaGetDevice(&cache->device);
        if (err == cudaSuccess)
        {
            const int memory_rc = check_memory(*params, cache->device);
            if (memory_rc)
            {
                delete cache;
                return memory_rc;
            }
            err = static_cast<cudaError_t>(awa::prepare_cache_attention_simt());
        }
        if (err == cudaSuccess)
            err = static_cast<cudaError_t>(awa::prepare_cache_attention_f32());
        if (err == cudaSuccess)
            err = static_cast<cudaError_t>(awa::prepare_cache_attention_step());
        if (err == cudaSuccess)
            err = static_cast<cudaError_t>(awa::prepare_cache_attention_tile());
        if (err == cudaSuccess)
            cache->error_flag = awa::device_error_flag();
        if (err != cudaSuccess || !cache->error_flag)
        {
            delete cache;
            return err != cudaSuccess
                       ? fail(AWA_ERR_CUDA, "awa_cache_create: %s", cudaGetErrorString(err))
                       : fail(AWA_ERR_ALLOC, "awa_cache_create: could not allocate the device status flag");
        }
    }
    *out = cache;
    return AWA_OK;
}

}  // namespace

extern "C" {

int awa_cache_create(const awa_cache_params* params, awa_cache** out)
{
    return create(params, out, true);
}

int awa_cache_create_host(const awa_cache_params* params, awa_cache** out)
{
    return create(params, out, false);
}

void awa_cache_destroy(awa_cache* cache)
{
    delete cache;
}

int awa_cache_append(const awa_cache* cache, const awa_cache_batch* batch, int q_heads, int in_dtype, const void* q,
                     int64_t q_token_stride, const void* k, int64_t k_token_stride, const void* v,
                     int64_t v_token_stride, const awa_cache_rope* rope, int q_out_dtype, void* q_out,
                     int64_t q_out_token_stride, awa_stream_t stream)
{
    awa::CacheAppendArgs a{};
    static const char* const kWhat = "awa_cache_append";
    bool empty = false;
    const int rc = check_batch(kWhat, cache, batch, &a.batch, &empty);
    if (rc)
        return rc;
    a.mem = cache->mem;
    const int d = a.mem.head_dim;
    if (!float_type(in_dtype) || (q && !float_type(q_out_dtype)))
        return fail(AWA_ERR_INVALID, "awa_cache_append: rows must be AWA_F32 or AWA_BF16");
    if (rope)
    {
        if (!rope->table || rope->max_coord <= 0 || rope->axes < 1 || rope->axes > 4 || rope->pairs <= 0 ||
            2 * (int64_t)rope->axes * rope->pairs > d || reinterpret_cast<uintptr_t>(rope->table) % 8)
            return fail(AWA_ERR_INVALID,
                        "awa_cache_append: rope needs an 8-byte aligned table, 1 to 4 axes and 2 * axes * pairs <= "
                        "head_dim");
        if (!aligned(rope->coords, 0, 4))
            return fail(AWA_ERR_INVALID, "awa_cache_append: rope's coords must be 4-byte aligned");
        a.table = reinterpret_cast<const float2*>(rope->table);
        a.max_coord = rope->max_coord;
        a.axes = rope->axes;
        a.pairs = rope->pairs;
        a.coords = rope->coords;
    }
    if (empty)
        return check_device(kWhat, cache);
    if (!k || !v || (q && !q_out))
        return fail(AWA_ERR_INVALID, "awa_cache_append: NULL rows");
    if (q && (q_heads <= 0 || (int64_t)q_heads * d > 0x7fffffff || q_token_stride < (int64_t)q_heads * d ||
              q_out_token_stride < (int64_t)q_heads * d))
        return fail(AWA_ERR_INVALID, "awa_cache_append: q_heads must be positive and q's strides hold a row");
    if (k_token_stride < (int64_t)a.mem.heads * d || v_token_stride < (int64_t)a.mem.heads * d)
        return fail(AWA_ERR_INVALID, "awa_cache_append: strides smaller than a row");
    const int e = type_bytes(in_dtype), eo = type_bytes(q_out_dtype);
    if (reinterpret_cast<uintptr_t>(k) % e || reinterpret_cast<uintptr_t>(v) % e ||
        (q && (reinterpret_cast<uintptr_t>(q) % e || reinterpret_cast<uintptr_t>(q_out) % eo)))
        return fail(AWA_ERR_INVALID, "awa_cache_append: rows not aligned to their elements");
    if (q == q_out && q && (in_dtype != q_out_dtype || q_token_stride != q_out_token_stride))
        return fail(AWA_ERR_INVALID, "awa_cache_append: q_out may be q only with the same type and stride");
    const int device_rc = check_device(kWhat, cache);
    if (device_rc)
        return device_rc;
    a.q_heads = q ? q_heads : 0;
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.v = static_cast<const char*>(v);
    a.q_stride = q_token_stride;
    a.k_stride = k_token_stride;
    a.v_stride = v_token_stride;
    a.q_out = static_cast<char*>(q_out);
    a.q_out_stride = q_out_token_stride;
    a.aligned = aligned(k, k_token_stride * e, 16) && aligned(v, v_token_stride * e, 16) &&
                (!q || (aligned(q, q_token_stride * e, 16) && aligned(q_out, q_out_token_stride * eo, 16)));
    a.error_flag = cache->error_flag;
    return launch_status(awa::launch_cache_append(a, in_dtype, q_out_dtype, static_cast<cudaStream_t>(stream)),
                         "awa_cache_append launch");
}

int awa_cache_read(const awa_cache* cache, const awa_cache_batch* batch, int out_dtype, void* k_out,
                   int64_t k_token_stride, void* v_out, int64_t v_token_stride, awa_stream_t stream)
{
    awa::CacheReadArgs a{};
    static const char* const kWhat = "awa_cache_read";
    bool empty = false;
    const int rc = check_batch(kWhat, cache, batch, &a.batch, &empty);
    if (rc)
        return rc;
    a.mem = cache->mem;
    if (!float_type(out_dtype))
        return fail(AWA_ERR_INVALID, "awa_cache_read: rows must be AWA_F32 or AWA_BF16");
    if (empty)
        return check_device(kWhat, cache);
    const int64_t row = (int64_t)a.mem.heads * a.mem.head_dim;
    const int e = type_bytes(out_dtype);
    if (!k_out || !v_out || k_token_stride < row || v_token_stride < row ||
        reinterpret_cast<uintptr_t>(k_out) % e || reinterpret_cast<uintptr_t>(v_out) % e)
        return fail(AWA_ERR_INVALID, "awa_cache_read: NULL or misaligned rows, or strides smaller than a row");
    const int device_rc = check_device(kWhat, cache);
    if (device_rc)
        return device_rc;
    a.k_out = static_cast<char*>(k_out);
    a.v_out = static_cast<char*>(v_out);
    a.k_stride = k_token_stride;
    a.v_stride = v_token_stride;
    a.aligned = aligned(k_out, k_token_stride * e, 16) && aligned(v_out, v_token_stride * e, 16);
    a.error_flag = cache->error_flag;
    return launch_status(awa::launch_cache_read(a, out_dtype, static_cast<cudaStream_t>(stream)),
                         "awa_cache_read launch");
}

static int check_attention(const char* what, const awa_cache* cache, const awa_cache_batch* batch, int q_heads,
                           int sinks, int window, int frame_tokens)
{
    if (q_heads <= 0 || q_heads % cache->mem.heads)
        return fail(AWA_ERR_INVALID, "%s: q_heads %d must be a multiple of the cache's %d heads", what, q_heads,
                    cache->mem.heads);
    if (sinks < 0 || window < 0 || frame_tokens < 1)
        return fail(AWA_ERR_INVALID, "%s: sinks (%d) and window (%d) must be 0 or more, frame_tokens (%d) 1 or more",
                    what, sinks, window, frame_tokens);
    if ((int64_t)batch->rows * q_heads > 0x7fffffff)
        return fail(AWA_ERR_INVALID, "%s: rows * q_heads reaches 2^31", what);
    return AWA_OK;
}

// No max_rows rows of a sequence see more keys than this: the page table's reach,
// and the prefix, a row's window and what the rows after it add, up to the end of a frame.
static int64_t most_seen(const awa::CacheMemory& mem, const awa_cache_batch& batch, int sinks, int window,
                         int frame_tokens)
{
    const int64_t reach = (int64_t)batch.table_width << mem.page_shift;
    const int64_t seen = sinks + (int64_t)window * frame_tokens + batch.max_rows + frame_tokens - 1;
    return window > 0 && seen < reach ? seen : reach;
}

// The kernel that serves a call.
enum Kernel
{
    kStep,        // few rows per head: bf16 and 4 bits
    kTile,        // many rows: bf16
    kUnpackTile,  // many rows of a 4-bit cache: its visible pages become fp16 first
    kF32,         // many rows: fp32
    kSimt         // few rows: fp32; other head sizes
};

// Up to 32 (row, head) pairs per key/value head and sequence the step kernel
// reads the keys once or twice at memory speed and fills its instructions; the
// tile kernel always computes 128 of them.
static Kernel kernel_of(const awa::CacheMemory& mem, const awa_cache_batch& batch, int group)
{
    if (mem.head_dim != 64 && mem.head_dim != 128)
        return kSimt;
    // 17 (row, head) pairs are more than one FMA tile of 16 holds
    if (mem.storage == AWA_F32)
        return (int64_t)batch.max_rows * group <= 16 ? kSimt : kF32;
    if ((int64_t)batch.max_rows * group <= 32 || group > 128 ||
        batch.sequences > awa::cache_attention_tile_sequences())
        return kStep;
    return mem.storage == AWA_INT4 ? kUnpackTile : kTile;
}

// Pages that the rows of a batch can see at most, all sequences together: the
// whole table, or prefix, window and new rows with the pages they only touch.
static int64_t most_pages(const awa::CacheMemory& mem, const awa::CacheBatch& batch, int sinks, int window,
                          int frame_tokens)
{
    const int64_t all = (int64_t)batch.sequences * batch.table_width;
    if (window == 0)
        return all;
    const auto pages = [&](int64_t tokens) { return (tokens + (1 << mem.page_shift) - 1) >> mem.page_shift; };
    // a row's window and its frame, ragged at both ends; then rows - 1 more of them
    int64_t each = pages(sinks) + pages((int64_t)window * frame_tokens) + pages(frame_tokens) + 3;
    each = each < batch.table_width ? each : batch.table_width;
    const int64_t some = batch.sequences * each + pages(batch.rows);
    return some < all ? some : all;
}

// kUnpackTile takes as many of the cache's heads at a time as this holds the unpacked
// pages of, or one. A pass costs some microseconds, and one head a pass leaves the SMs
// uneven shares: 64 sequences of 30000 keys and 9 rows, 8 heads of 128, 3.70 ms in one
// pass of 7.5 GiB, 4.63 ms in four, 5.80 ms in eight.
constexpr size_t kMostUnpacked = (size_t)2 << 30;

// The workspace of kUnpackTile ahead of the tile kernel's: keys, values, page table,
// queries, ranges and the scores' scales, each on 256 bytes.
struct Unpacked
{
    int64_t seen;   // pages of all sequences together, at most
    int64_t pages;  // unpacked ones that there is room for
    bool own_table; // they are numbered as the sequences see them, not as the cache has them
    int heads;      // at a time
    size_t page_bytes, pool_bytes, table_bytes, q_bytes, range_bytes, part_bytes, scale_bytes;
};

static size_t on256(size_t bytes)
{
    return (bytes + 255) / 256 * 256;
}

static Unpacked unpacked_of(const awa::CacheMemory& mem, const awa::CacheBatch& batch, int q_heads, int sinks,
                            int window, int frame_tokens)
{
    Unpacked u;
    u.seen = most_pages(mem, batch, sinks, window, frame_tokens);
    u.own_table = u.seen < mem.pages;
    u.pages = u.own_table ? u.seen : mem.pages;
    const size_t head_bytes = ((size_t)mem.head_dim * 2) << mem.page_shift;
    const size_t at_once = kMostUnpacked / (2 * (u.pages > 0 ? u.pages : 1) * head_bytes);
    const int passes = at_once == 0 ? mem.heads : (int)((mem.heads + at_once - 1) / at_once);
    u.heads = (mem.heads + passes - 1) / passes;
    u.page_bytes = u.heads * head_bytes;
    u.pool_bytes = u.pages * u.page_bytes;
    u.table_bytes = u.own_table ? on256((size_t)batch.sequences * batch.table_width * 4) : 0;
    const size_t rows = (size_t)batch.rows * (q_heads / mem.heads) * u.heads;  // and q heads
    u.q_bytes = on256(rows * mem.head_dim * 2);
    u.range_bytes = on256((size_t)u.heads * (mem.head_dim / AWA_CACHE_GROUP) * 2 * sizeof(unsigned));
    u.part_bytes = on256(awa::cache_unpack_range_bytes(mem, u.heads));
    u.scale_bytes = on256(rows * sizeof(float));
    return u;
}

size_t awa_cache_attention_workspace_bytes(const awa_cache* cache, const awa_cache_batch* batch, int q_heads, int sinks,
                                           int window, int frame_tokens)
{
    awa::CacheBatch b;
    bool empty = false;
    static const char* const kWhat = "awa_cache_attention_workspace_bytes";
    if (check_batch(kWhat, cache, batch, &b, &empty) ||
        check_attention(kWhat, cache, batch, q_heads, sinks, window, frame_tokens) || empty)
        return 0;
    const int group = q_heads / cache->mem.heads;
    const Kernel kernel = kernel_of(cache->mem, *batch, group);
    if (kernel == kStep)
        return awa::cache_attention_step_workspace(cache->mem, group, batch->max_rows,
                                                   most_seen(cache->mem, *batch, sinks, window, frame_tokens));
    if (kernel == kSimt || kernel == kF32)
        return 0;
    const size_t parts = awa::cache_attention_tile_workspace(cache->mem.head_dim);
    if (kernel == kTile)
        return parts;
    const Unpacked u = unpacked_of(cache->mem, b, q_heads, sinks, window, frame_tokens);
    return 2 * u.pool_bytes + u.table_bytes + u.q_bytes + u.range_bytes + u.part_bytes + u.scale_bytes + parts;
}

int awa_cache_attention(const awa_cache* cache, const awa_cache_batch* batch, int q_heads, int dtype, const void* q,
                        int64_t q_token_stride, float scale, int sinks, int window, int frame_tokens, void* out,
                        int64_t out_token_stride, void* workspace, size_t workspace_bytes, awa_stream_t stream)
{
    awa::CacheAttnArgs a{};
    static const char* const kWhat = "awa_cache_attention";
    bool empty = false;
    int rc = check_batch(kWhat, cache, batch, &a.batch, &empty);
    if (rc)
        return rc;
    rc = check_attention("awa_cache_attention", cache, batch, q_heads, sinks, window, frame_tokens);
    if (rc)
        return rc;
    a.mem = cache->mem;
    const int want = a.mem.storage == AWA_F32 ? AWA_F32 : AWA_BF16;
    if (dtype != want)
        return fail(AWA_ERR_INVALID, "awa_cache_attention: this cache takes %s rows",
                    want == AWA_F32 ? "AWA_F32" : "AWA_BF16");
    if (!(scale > 0.f) || std::isinf(scale))
        return fail(AWA_ERR_INVALID, "awa_cache_attention: scale must be positive and finite");
    if (empty)
        return check_device(kWhat, cache);
    const int64_t row = (int64_t)q_heads * a.mem.head_dim;
    const int e = type_bytes(dtype);
    if (!q || !out || q_token_stride < row || out_token_stride < row)
        return fail(AWA_ERR_INVALID, "awa_cache_attention: NULL rows or strides smaller than a row");
    if (!aligned(q, q_token_stride * e, 16) || !aligned(out, out_token_stride * e, 16))
        return fail(AWA_ERR_INVALID, "awa_cache_attention: q and out need 16-byte aligned rows");
    const size_t need = awa_cache_attention_workspace_bytes(cache, batch, q_heads, sinks, window, frame_tokens);
    if (workspace_bytes < need || (need && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256)))
        return fail(AWA_ERR_INVALID, "awa_cache_attention: 256-byte aligned workspace of %zu bytes needed, %zu given",
                    need, workspace_bytes);
    rc = check_device(kWhat, cache);
    if (rc)
        return rc;
    a.group = q_heads / a.mem.heads;
    a.q = q;
    a.q_stride = q_token_stride;
    a.out = out;
    a.out_stride = out_token_stride;
    a.scale = scale;
    a.sinks = sinks;
    a.window = window;
    a.frame_tokens = frame_tokens;
    a.error_flag = cache->error_flag;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    int err = 0;
    switch (kernel_of(a.mem, *batch, a.group))
    {
    case kStep:
        err = awa::launch_cache_attention_step(a, batch->max_rows,
                                               most_seen(a.mem, *batch, sinks, window, frame_tokens), workspace, s);
        break;
    case kTile: err = awa::launch_cache_attention_tile(a, false, workspace, s); break;
    case kSimt: err = awa::launch_cache_attention_simt(a, batch->max_rows, s); break;
    case kF32: err = awa::launch_cache_attention_f32(a, s); break;
    case kUnpackTile:
    {
        const Unpacked u = unpacked_of(a.mem, a.batch, q_heads, sinks, window, frame_tokens);
        if (u.seen > 0x7fffffff)
            return fail(AWA_ERR_INVALID, "awa_cache_attention: the batch reaches too many pages");
        awa::CacheUnpackArgs unpack{};
        unpack.batch = a.batch;
        unpack.sinks = sinks;
        unpack.window = window;
        unpack.frame_tokens = frame_tokens;
        unpack.k_out = static_cast<char*>(workspace);
        unpack.v_out = unpack.k_out + u.pool_bytes;
        char* const table = unpack.v_out + u.pool_bytes;
        unpack.table = u.own_table ? reinterpret_cast<int*>(table) : nullptr;
        unpack.q_out = table + u.table_bytes;
        unpack.q_stride = q_token_stride;
        unpack.most_seen = (int)u.seen;
        unpack.ranges = reinterpret_cast<unsigned*>(unpack.q_out + u.q_bytes);
        unpack.range_parts = reinterpret_cast<unsigned*>(reinterpret_cast<char*>(unpack.ranges) + u.range_bytes);
        unpack.score_scale = reinterpret_cast<float*>(reinterpret_cast<char*>(unpack.range_parts) + u.part_bytes);
        unpack.scale = scale;
        unpack.error_flag = a.error_flag;
        char* const parts = reinterpret_cast<char*>(unpack.score_scale) + u.scale_bytes;
        const awa::CacheMemory mem = a.mem;
        a.mem.storage = AWA_BF16;
        a.mem.pages = (int)u.pages;
        a.mem.k = unpack.k_out;
        a.mem.v = unpack.v_out;
        if (u.own_table)
        {
            a.batch.page_table = unpack.table;
            a.batch.table_stride = a.batch.table_width;
        }
        a.q = unpack.q_out;
        a.ranges = unpack.ranges;
        a.score_scale = unpack.score_scale;
        for (int head = 0; head < mem.heads && !err; head += u.heads)
        {
            const int heads = head + u.heads < mem.heads ? u.heads : mem.heads - head;
            const int64_t first = (int64_t)head * a.group * mem.head_dim;  // of a row
            unpack.mem = mem;
            unpack.mem.heads = heads;
            unpack.mem.k += head * mem.head_stride;
            unpack.mem.v += head * mem.head_stride;
            unpack.mem.k_params += head * mem.params_head_stride;
            unpack.mem.v_params += head * mem.params_head_stride;
            unpack.q = static_cast<const char*>(q) + first * e;
            unpack.q_row = heads * a.group * mem.head_dim;
            err = awa::launch_cache_unpack(unpack, s);
            if (err)
                break;
            a.mem.heads = heads;
            a.mem.head_stride = (int64_t)(u.page_bytes / u.heads);
            a.mem.page_stride = heads * a.mem.head_stride;
            a.q_stride = unpack.q_row;
            a.out = static_cast<char*>(out) + first * e;
            err = awa::launch_cache_attention_tile(a, true, parts, s);
        }
        break;
    }
    }
    return launch_status(err, "awa_cache_attention launch");
}

}  // extern "C"
