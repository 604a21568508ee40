// awa_cache_attn_step.cu -- attention over the paged key/value cache for few
// query rows per head (a generation step): bf16 and 4-bit caches, head_dim 64
// and 128.
//
// With few rows a step reads every visible key and value once and does
// little with them, so memory bounds it: bytes = visible tokens * heads *
// head_dim * 2 (k, v) * (2 for bf16, 0.5625 for 4 bits). The kernel is built to
// keep loads in flight: each warp works alone on its own blocks of keys, fed by
// a ring of cp.async copies in its own shared memory, and only at the end do
// the warps of a block, and the blocks of a cluster, join their parts.
//
// A warp's block of 16 keys: S^T = K Q^T and O^T += V^T P^T with mma.sync
// m16n8k16. Keys (then features) are the 16 rows and up to 8 query rows the 8
// columns, so one row wastes 7/8 of the instruction instead of 15/16. The
// running maximum and sum are those of the warp's keys, base 2, fp32.
//
// 4 bits: a code c stands for scale (c + z), z = minimum / scale. As the bits
// of a bf16 number, the integers 0..255 are the multiples of 2^-133 (the
// subnormals and the binade above them), which mma.sync takes as they are: a
// mask alone turns two codes of a word into an operand, one at bits 0-3 as
// c 2^-133, one at bits 4-7 as 16 c 2^-133, exactly; the other operand carries
// the powers of two that bring the products back. Per 64 features with their own scale,
//   sum q k = scale (sum q c + z sum q)
//   sum p v = sum p' c + sum p' z,  p' = bf16(p scale),
// the sums in fp32, the last one with the same rounded p', so that the one
// rounding acts on p as it does for a bf16 cache.
//
// Measured (B200): 64 streams of 500 to 32000 rows, window 8192, 32 / 8 heads:
// 195 us, 6.0 TB/s, 0.91 of the measured copy rate. The same in 4 bits, 32
// streams up to 32700 rows: 143 us, 4.0 TB/s, 0.60: there the instructions that
// turn codes into operands (320 a 16 keys and warp) bound it, not memory. One
// stream of 700 rows: 8.4 us.
#include "awa_cache_device.cuh"
#include "awa_mma.cuh"
#include "awa_rows.cuh"

#include <cooperative_groups.h>
#include <cuda_bf16.h>

namespace awa
{
namespace
{

namespace cg = cooperative_groups;
using bf16 = __nv_bfloat16;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
constexpr int kStages = 3;  // 2 leave too little in flight (4 bits: 177 us for 142), 4 too few blocks on an SM (163)

// Sizes of one kernel instance.
template <int ST, int D>
struct Step
{
    static constexpr bool kFour = ST == AWA_INT4;
    static constexpr int kGroups = D / AWA_CACHE_GROUP;
    static constexpr int kRowBytes = kFour ? D / 2 : 2 * D;
    // Keys of a stage: 16 or 32 rows of bf16 (8 KB with the values), 32 of
    // codes (less would be mostly overhead)
    static constexpr int kKeys = kFour ? 32 : 2048 / D;
    static constexpr int kParamBytes = kFour ? 4 * kGroups : 0;
    static constexpr int kStageBytes = 2 * kKeys * (kRowBytes + kParamBytes);
    // 4 bits: (scale, z) of the stage's keys, [k, v][key][group]; of the values, scale kProbsUp
    static constexpr int kScaleBytes = kFour ? 2 * kKeys * kGroups * 8 : 0;
    static constexpr int kWarpBytes = kStages * kStageBytes + kScaleBytes;
    static constexpr int kPitch = D + 4;  // floats of a row of partial results
    static constexpr int shared_bytes(int nq)
    {
        const int ring = kWarps * kWarpBytes, parts = (kWarps + 1) * 8 * nq * kPitch * 4;
        return ring > parts ? ring : parts;
    }
};

// 8x8 transpose of one b16 matrix held across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Codes j and j + 4 of a word as the bits of two bf16 numbers: c 2^-133, for odd j 16 c 2^-133.
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int j)
{
    return (word >> (8 * (j >> 1))) & (j & 1 ? 0x00f000f0u : 0x000f000fu);
}

// The other operand's share of the powers of two. q 2^60 leaves q a range of
// 2^67 up; p' 2^90 takes scales from about 2^-80 to 2^29.
constexpr float kQueryUp = 0x1p60f, kScoresUp = 0x1p73f;
constexpr float kProbsUp = 0x1p90f, kProbsDown = 0x1p-90f, kOutUp = 0x1p43f;

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t x, float f)
{
    uint32_t y;
    asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(y) : "r"(x), "r"(pack_bf16x2(f, f)));
    return y;
}

// Where 16-byte piece c of row r of a stage lies. bf16: the 8 rows that one
// ldmatrix reads fall on different banks. 4 bits (64-byte rows of two 32-byte
// groups): the groups of half the rows swap places, so that neither the 8-byte
// reads of keys nor the 4-byte reads of values collide.
// The row is base + r, base a multiple of 8: its share is known when compiling.
template <int ST, int D>
__device__ __forceinline__ int piece_offset(int base, int r, int c)
{
    constexpr int kRowBytes = Step<ST, D>::kRowBytes;
    int at = c;
    if (ST != AWA_INT4)
        at = c ^ (r & 7);
    else if (D == 128)
        at = c ^ ((((r >> 1) ^ (r >> 2)) & 1) << 1);
    return r * kRowBytes + (at << 4) + base * kRowBytes;
}

// The key that row r of a 16-key block holds. 4 bits: rows 2t, 2t + 1 (whose
// values one lane pairs up) are keys t, t + 4 of each eight, so that the lanes'
// reads of values fall on different banks.
template <int ST>
__device__ __forceinline__ int key_of_row(int r)
{
    return ST == AWA_INT4 ? (r & 8) | ((r & 1) << 2) | ((r & 7) >> 1) : r;
}

// (scale, z) of the groups of a key, as the sums use them: with kScoresUp or kProbsUp.
template <typename S>
struct alignas(8 * S::kGroups) Scales
{
    float2 of[S::kGroups];
};

template <int ST, int D, int NQ>
struct WarpState
{
    using S = Step<ST, D>;
    uint32_t q[NQ][D / 16][2];  // Q^T operands
    float q_sum[NQ][S::kGroups][2];  // 4 bits: sum of q over a group over kScoresUp, of columns 2t, 2t + 1
    float o[NQ][D / 16][4];
    float off[NQ][S::kGroups][2];  // 4 bits: sum p' z, times kProbsUp
    float top[NQ][2], sum[NQ][2];
    RowSpan span[NQ][2];
};

// The warp's share of one 16-key block: scores, exponentials, probabilities.
template <int ST, int D, int NQ>
__device__ __forceinline__ void scores(const WarpState<ST, D, NQ>& w, const char* kdata,
                                       const Scales<Step<ST, D>>* kscale, int block,
                                       float (&s)[NQ][4])
{
    using S = Step<ST, D>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (ST != AWA_INT4)
    {
#pragma unroll
        for (int n = 0; n < NQ; n++)
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        const uint32_t base = shared_address(kdata);
#pragma unroll
        for (int i = 0; i < D / 16; i++)
        {
            uint32_t a[4];
            ldmatrix_x4(base + piece_offset<ST, D>(block * 16, lane & 15, 2 * i + (lane >> 4)), a);
#pragma unroll
            for (int n = 0; n < NQ; n++)
                mma(s[n], a[0], a[1], a[2], a[3], w.q[n][i][0], w.q[n][i][1]);
        }
        return;
    }
    const int r = key_of_row<ST>(g);  // and r + 8
    const Scales<S> p0 = kscale[block * 16 + r], p1 = kscale[block * 16 + 8 + r];
#pragma unroll
    for (int gr = 0; gr < S::kGroups; gr++)
    {
        float acc[NQ][4] = {};
        // 16 features of a lane: 8 bytes of each of its two keys
        const uint2 x0 =
            *reinterpret_cast<const uint2*>(kdata + piece_offset<ST, D>(block * 16, r, 2 * gr) + 8 * t);
        const uint2 x1 =
            *reinterpret_cast<const uint2*>(kdata + piece_offset<ST, D>(block * 16 + 8, r, 2 * gr) + 8 * t);
#pragma unroll
        for (int i = 0; i < 4; i++)
        {
            const uint32_t a = i < 2 ? x0.x : x0.y, b = i < 2 ? x1.x : x1.y;
            const int j = 2 * (i & 1);
#pragma unroll
            for (int n = 0; n < NQ; n++)
                mma(acc[n], code_pair(a, j), code_pair(b, j), code_pair(a, j + 1), code_pair(b, j + 1),
                    w.q[n][4 * gr + i][0], w.q[n][4 * gr + i][1]);
        }
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int c = 0; c < 4; c++)
            {
                const float2 p = c < 2 ? p0.of[gr] : p1.of[gr];
                const float part = fmaf(p.y, w.q_sum[n][gr][c & 1], acc[n][c]);
                s[n][c] = gr == 0 ? p.x * part : fmaf(p.x, part, s[n][c]);
            }
    }
}

// O^T += V^T P^T of one 16-key block; p: the exponentials in the layout of the scores.
template <int ST, int D, int NQ>
__device__ __forceinline__ void values(WarpState<ST, D, NQ>& w, const char* vdata,
                                       const Scales<Step<ST, D>>* vscale, int block,
                                       const float (&p)[NQ][4])
{
    using S = Step<ST, D>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (ST != AWA_INT4)
    {
        uint32_t b[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; n++)
        {
            b[n][0] = transpose8x8(pack_bf16x2(p[n][0], p[n][1]));
            b[n][1] = transpose8x8(pack_bf16x2(p[n][2], p[n][3]));
        }
        const uint32_t base = shared_address(vdata);
        const int r = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int i = 0; i < D / 16; i++)
        {
            uint32_t a[4];
            ldmatrix_x4_trans(base + piece_offset<ST, D>(block * 16, r, 2 * i + ((lane >> 3) & 1)), a);
#pragma unroll
            for (int n = 0; n < NQ; n++)
                mma(w.o[n][i], a[0], a[1], a[2], a[3], b[n][0], b[n][1]);
        }
        return;
    }
    const int r = key_of_row<ST>(g);  // and r + 8
    const Scales<S> s0 = vscale[block * 16 + r], s1 = vscale[block * 16 + 8 + r];
#pragma unroll
    for (int gr = 0; gr < S::kGroups; gr++)
    {
        const float2 p0 = s0.of[gr], p1 = s1.of[gr];
        uint32_t b[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; n++)
        {
            const uint32_t lo = pack_bf16x2(p[n][0] * p0.x, p[n][1] * p0.x);
            const uint32_t hi = pack_bf16x2(p[n][2] * p1.x, p[n][3] * p1.x);
            w.off[n][gr][0] = fmaf(__uint_as_float(lo << 16), p0.y,
                                   fmaf(__uint_as_float(hi << 16), p1.y, w.off[n][gr][0]));
            w.off[n][gr][1] = fmaf(__uint_as_float(lo & 0xffff0000u), p0.y,
                                   fmaf(__uint_as_float(hi & 0xffff0000u), p1.y, w.off[n][gr][1]));
            b[n][0] = transpose8x8(lo);
            b[n][1] = transpose8x8(hi);
        }
        // features 8g .. 8g + 7 of the group, of the keys of rows 2t, 2t + 1, 2t + 8, 2t + 9
        uint32_t x[4];
#pragma unroll
        for (int u = 0; u < 4; u++)
            x[u] = *reinterpret_cast<const uint32_t*>(
                vdata + piece_offset<ST, D>(block * 16 + 8 * (u >> 1), t + 4 * (u & 1), 2 * gr + (g >> 2)) + 4 * (g & 3));
        const uint32_t lo01 = __byte_perm(x[0], x[1], 0x5410), hi01 = __byte_perm(x[0], x[1], 0x7632);
        const uint32_t lo23 = __byte_perm(x[2], x[3], 0x5410), hi23 = __byte_perm(x[2], x[3], 0x7632);
        // tile i of the group: rows g = feature 8g + i, rows g + 8 = feature 8g + 4 + i
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int n = 0; n < NQ; n++)
                mma(w.o[n][4 * gr + i], code_pair(lo01, i), code_pair(hi01, i), code_pair(lo23, i), code_pair(hi23, i),
                    b[n][0], b[n][1]);
    }
}

// One piece of work of a block: a tile of query rows of one key/value head and
// some of the key blocks that it sees.
struct Piece
{
    QueryTile tile;
    int kv;
    KeyBlocks blocks;
    RowSpan first, last;  // of the tile's rows
    int begin, end;       // key blocks [begin, end) of `blocks`
};

__device__ __forceinline__ RowSpan tile_span(const CacheAttnArgs& a, const QueryTile& t, int m)
{
    return row_span(t.past + (t.m0 + m) / a.group, t.length, a.sinks, a.window, a.frame_tokens);
}

template <typename S>
__device__ __forceinline__ int block_key(const Piece& p, int i)
{
    return (i < p.blocks.prefix ? i : i + p.blocks.shift) * S::kKeys;
}

// Copies 16 bytes that are all there.
__device__ __forceinline__ void copy16(uint32_t dst, const char* src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// Where the lane's share of the piece's keys comes from.
struct Source
{
    const int* table;
    const char *k, *v;  // of the head, at the lane's 16 bytes of a row run
    const char *k_params, *v_params;
};

template <int ST, int D>
__device__ __forceinline__ Source source_of(const CacheAttnArgs& a, const Piece& p)
{
    const CacheMemory& mem = a.mem;
    const int lane = threadIdx.x & 31;
    Source s;
    s.table = a.batch.page_table + p.tile.b * a.batch.table_stride;
    s.k = mem.k + p.kv * mem.head_stride + 16 * lane;
    s.v = mem.v + p.kv * mem.head_stride + 16 * lane;
    s.k_params = mem.k_params + p.kv * mem.params_head_stride;
    s.v_params = mem.v_params + p.kv * mem.params_head_stride;
    return s;
}

// Page of a position of the piece's sequence; -1, reported, if there is none.
__device__ __forceinline__ int piece_page(const CacheAttnArgs& a, const int* table, int key)
{
    const int page = __ldg(table + (key >> a.mem.page_shift));
    if ((unsigned)page < (unsigned)a.mem.pages)
        return page;
    cache_error(a.error_flag, AWA_CACHE_BAD_PAGE);
    return -1;
}

// Issues the copies of the key block at key0 into a stage of the warp's ring.
template <int ST, int D>
__device__ __forceinline__ void issue_block(const CacheAttnArgs& a, const Piece& p, const Source& src, int key0,
                                            uint32_t dst)
{
    using S = Step<ST, D>;
    const CacheMemory& mem = a.mem;
    const int lane = threadIdx.x & 31;
    const int page_mask = (1 << mem.page_shift) - 1;
    constexpr int kPieces = S::kRowBytes / 16;   // of a row, a power of two: 2, 4, 8 or 16
    constexpr int kRun = 32 / kPieces;           // rows that a warp copies at a time
    constexpr int kValues = S::kKeys * S::kRowBytes;
    int pages[S::kKeys / 16];  // 16 rows, aligned, lie in one page and are contiguous there
    bool whole = key0 + S::kKeys <= p.last.hi && (key0 >= p.first.lo || key0 + S::kKeys <= a.sinks);
    if (whole)
    {
#pragma unroll
        for (int h = 0; h < S::kKeys / 16; h++)
            pages[h] = piece_page(a, src.table, key0 + 16 * h);
#pragma unroll
        for (int h = 0; h < S::kKeys / 16; h++)
            whole = whole && pages[h] >= 0;
    }
    const int c = lane % kPieces;
    if (whole)
    {
#pragma unroll
        for (int h = 0; h < S::kKeys / 16; h++)
        {
            const int64_t at = pages[h] * mem.page_stride + ((key0 + 16 * h) & page_mask) * S::kRowBytes;
#pragma unroll
            for (int j = 0; j < 16 / kRun; j++)
            {
                const int base = 16 * h + j * kRun;  // of 8 rows or more, or within them
                const uint32_t to = dst + piece_offset<ST, D>(base & ~7, (base & 7) + lane / kPieces, c);
                copy16(to, src.k + at + 512 * j);
                copy16(to + kValues, src.v + at + 512 * j);
            }
        }
    }
    else
    {
        // only what some row sees is read: pages outside may be gone
#pragma unroll 1
        for (int base = 0; base < S::kKeys; base += kRun)
        {
            const int r = base + lane / kPieces, key = key0 + r;
            const bool seen = key < p.last.hi && (key >= p.first.lo || key < a.sinks);
            const int page = seen ? piece_page(a, src.table, key) : -1;
            const int64_t at =
                max(page, 0) * mem.page_stride + ((key & page_mask) - lane / kPieces) * (int64_t)S::kRowBytes;
            const uint32_t to = dst + piece_offset<ST, D>(0, r, c);
            copy_async<16>(to, src.k + at, page >= 0);
            copy_async<16>(to + kValues, src.v + at, page >= 0);
        }
    }
    if (S::kFour)
    {
        const int key = key0 + lane;
        int page = -1;
        if (whole)
            page = lane < 16 ? pages[0] : pages[S::kKeys / 16 - 1];
        else if (key < p.last.hi && (key >= p.first.lo || key < a.sinks))
            page = piece_page(a, src.table, key);
        const int64_t at = max(page, 0) * mem.params_page_stride + (key & page_mask) * S::kParamBytes;
        const uint32_t to = dst + 2 * kValues + lane * S::kParamBytes;
        copy_async<S::kFour ? S::kParamBytes : 4>(to, src.k_params + at, page >= 0);
        copy_async<S::kFour ? S::kParamBytes : 4>(to + S::kKeys * S::kParamBytes, src.v_params + at, page >= 0);
    }
}

// The tile's queries as operands, and an empty state.
template <int ST, int D, int NQ>
__device__ __forceinline__ void start(const CacheAttnArgs& a, const Piece& p, WarpState<ST, D, NQ>& w)
{
    using S = Step<ST, D>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const bf16* q = static_cast<const bf16*>(a.q);
#pragma unroll
    for (int n = 0; n < NQ; n++)
    {
        // column g of tile n
        const int m = p.tile.m0 + n * 8 + g;
        const bool mine = n * 8 + g < p.tile.count;
        const bf16* row =
            q + (int64_t)(p.tile.row0 + m / a.group) * a.q_stride + (int64_t)(p.kv * a.group + m % a.group) * D;
        float part[S::kGroups] = {};
        if (ST == AWA_INT4)
#pragma unroll
            for (int gr = 0; gr < S::kGroups; gr++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (mine)
                        x = __ldg(reinterpret_cast<const uint4*>(row + 64 * gr + 16 * t + 8 * h));
                    // pairs of features j, j + 4 as code_pair makes them, odd j with its 16
                    w.q[n][4 * gr + 2 * h][0] = mul_bf16x2(__byte_perm(x.x, x.z, 0x5410), kQueryUp);
                    w.q[n][4 * gr + 2 * h][1] = mul_bf16x2(__byte_perm(x.x, x.z, 0x7632), kQueryUp / 16);
                    w.q[n][4 * gr + 2 * h + 1][0] = mul_bf16x2(__byte_perm(x.y, x.w, 0x5410), kQueryUp);
                    w.q[n][4 * gr + 2 * h + 1][1] = mul_bf16x2(__byte_perm(x.y, x.w, 0x7632), kQueryUp / 16);
                    const uint32_t words[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        part[gr] += __uint_as_float(words[i] << 16) + __uint_as_float(words[i] & 0xffff0000u);
                }
        else
#pragma unroll
            for (int i = 0; i < D / 16; i++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                    w.q[n][i][h] =
                        mine ? __ldg(reinterpret_cast<const uint32_t*>(row + 16 * i + 8 * h + 2 * t)) : 0u;
#pragma unroll
        for (int gr = 0; gr < S::kGroups; gr++)
        {
            if (ST == AWA_INT4)
            {
                part[gr] += __shfl_xor_sync(0xffffffffu, part[gr], 1);
                part[gr] += __shfl_xor_sync(0xffffffffu, part[gr], 2);
            }
#pragma unroll
            for (int c = 0; c < 2; c++)
            {
                w.q_sum[n][gr][c] = ST == AWA_INT4 ? __shfl_sync(0xffffffffu, part[gr], 4 * (2 * t + c)) / kScoresUp : 0.f;
                w.off[n][gr][c] = 0.f;
            }
        }
#pragma unroll
        for (int i = 0; i < D / 16; i++)
            w.o[n][i][0] = w.o[n][i][1] = w.o[n][i][2] = w.o[n][i][3] = 0.f;
#pragma unroll
        for (int c = 0; c < 2; c++)
        {
            w.top[n][c] = -INFINITY;
            w.sum[n][c] = 0.f;
            w.span[n][c] = tile_span(a, p.tile, min(n * 8 + 2 * t + c, p.tile.count - 1));
        }
    }
}

// One key block, arrived in the ring.
template <int ST, int D, int NQ>
__device__ __forceinline__ void consume(const CacheAttnArgs& a, const Piece& p, WarpState<ST, D, NQ>& w, int key0,
                                        const char* kdata,
                                        Scales<Step<ST, D>>* scales)
{
    using S = Step<ST, D>;
    const int lane = threadIdx.x & 31, g = lane >> 2;
    const float to_log2 = a.scale * 1.44269504088896341f;
    const char* vdata = kdata + S::kKeys * S::kRowBytes;
    if (S::kFour)
    {
        // a lane works out (scale, z) of its key. A scale of 0 or next to it
        // (then the value is the minimum) is raised to where z stays finite:
        // that moves the value by at most 15 * 2^-80 of max(1, it)
        struct alignas(4 * S::kGroups) Words
        {
            uint32_t word[S::kGroups];
        };
        const Words* par = reinterpret_cast<const Words*>(vdata + S::kKeys * S::kRowBytes);
#pragma unroll
        for (int x = 0; x < 2; x++)
        {
            const Words words = par[x * S::kKeys + lane];
            Scales<S> out;
#pragma unroll
            for (int gr = 0; gr < S::kGroups; gr++)
            {
                const float low = __uint_as_float(words.word[gr] & 0xffff0000u);
                const float scale = fmaxf(__uint_as_float(words.word[gr] << 16), 0x1p-80f * fmaxf(1.f, fabsf(low)));
                float inverse;  // scale is a normal number: 1 ulp, as a division's
                asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(scale));
                out.of[gr] = make_float2(scale * (x == 0 ? kScoresUp : kProbsUp), low * inverse);
            }
            scales[x * S::kKeys + lane] = out;
        }
        __syncwarp();
    }
    constexpr int kBlocks = S::kKeys / 16;
    float s[kBlocks][NQ][4];
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
        scores<ST, D, NQ>(w, kdata, scales, b, s[b]);
    // rows of the tile see all of these keys: nothing to mask
    const bool all = key0 + S::kKeys <= p.first.hi && (key0 >= p.last.lo || key0 + S::kKeys <= a.sinks);
    if (!all)
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int x = 0; x < NQ; x++)
#pragma unroll
                for (int c = 0; c < 4; c++)
                {
                    const int key = key0 + b * 16 + key_of_row<ST>(g) + (c < 2 ? 0 : 8);
                    const RowSpan& span = w.span[x][c & 1];
                    if (!(key < span.hi && (key >= span.lo || key < a.sinks)))
                        s[b][x][c] = -INFINITY;
                }
    // The exponentials are taken from `top`, the largest score when it was last
    // looked for: until one exceeds it by 8 (log2) they stay below 2^8, and the
    // lanes need not meet.
    float local[NQ][2];
    bool grew = false;
#pragma unroll
    for (int x = 0; x < NQ; x++)
#pragma unroll
        for (int c = 0; c < 2; c++)
        {
            local[x][c] = fmaxf(s[0][x][c], s[0][x][c + 2]);
#pragma unroll
            for (int b = 1; b < kBlocks; b++)
                local[x][c] = fmaxf(local[x][c], fmaxf(s[b][x][c], s[b][x][c + 2]));
            grew |= (local[x][c] - w.top[x][c]) * to_log2 > 8.f;  // from -inf: always; -inf - -inf: never
        }
    if (__any_sync(0xffffffffu, grew))
#pragma unroll
        for (int x = 0; x < NQ; x++)
#pragma unroll
            for (int c = 0; c < 2; c++)
            {
                float top = fmaxf(local[x][c], w.top[x][c]);
#pragma unroll
                for (int off = 4; off < 32; off <<= 1)
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                const float old = w.top[x][c] == top ? 1.f : fast_exp2((w.top[x][c] - top) * to_log2);
                w.top[x][c] = top;
                w.sum[x][c] *= old;
#pragma unroll
                for (int gr = 0; gr < S::kGroups; gr++)
                    w.off[x][gr][c] *= old;
#pragma unroll
                for (int j = 0; j < D / 16; j++)
                {
                    w.o[x][j][c] *= old;
                    w.o[x][j][c + 2] *= old;
                }
            }
#pragma unroll
    for (int x = 0; x < NQ; x++)
#pragma unroll
        for (int c = 0; c < 2; c++)
        {
            // nothing seen yet: all exponentials are 0
            const float from = w.top[x][c] == -INFINITY ? 0.f : w.top[x][c] * to_log2;
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
            {
                s[b][x][c] = fast_exp2(fmaf(s[b][x][c], to_log2, -from));
                s[b][x][c + 2] = fast_exp2(fmaf(s[b][x][c + 2], to_log2, -from));
                w.sum[x][c] += s[b][x][c] + s[b][x][c + 2];
            }
        }
#pragma unroll
    for (int b = 0; b < kBlocks; b++)
        values<ST, D, NQ>(w, vdata, scales + S::kKeys, b, s[b]);
}

// The warp's share of the piece: key blocks begin + turn, + turns, ...
template <int ST, int D, int NQ>
__device__ __forceinline__ void work(const CacheAttnArgs& a, const Piece& p, WarpState<ST, D, NQ>& w, char* ring,
                                     int turn, int turns)
{
    using S = Step<ST, D>;
    Scales<S>* scales = reinterpret_cast<Scales<S>*>(ring + kStages * S::kStageBytes);
    const uint32_t ring_addr = shared_address(ring);
    const Source src = source_of<ST, D>(a, p);
    const auto issue = [&](int i, int stage) {
        if (i < p.end)
            issue_block<ST, D>(a, p, src, block_key<S>(p, i), ring_addr + stage * S::kStageBytes);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    int i = p.begin + turn;
#pragma unroll
    for (int n = 0; n < kStages - 1; n++)
        issue(i + n * turns, n);
    start<ST, D, NQ>(a, p, w);
    int stage = 0;
    for (; i < p.end; i += turns)
    {
        issue(i + (kStages - 1) * turns, stage == 0 ? kStages - 1 : stage - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        consume<ST, D, NQ>(a, p, w, block_key<S>(p, i), ring + stage * S::kStageBytes, scales);
        __syncwarp();  // the stage is free for the copies of the next round
        stage = stage == kStages - 1 ? 0 : stage + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// Joins the parts of `parts` holders of (maximum, sum) and unnormalised
// outputs, in their order: ml(i) and o(i) of this thread's row and two features.
struct Joined
{
    float top, total;
    float2 o;
};

template <typename Ml, typename O>
__device__ __forceinline__ Joined join(int parts, float to_log2, Ml ml, O o)
{
    Joined j;
    j.top = -INFINITY;
    for (int i = 0; i < parts; i++)
        j.top = fmaxf(j.top, ml(i).x);
    const float from = j.top == -INFINITY ? 0.f : j.top;
    j.total = 0.f;
    j.o = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < parts; i++)
    {
        const float2 x = ml(i), y = o(i);
        const float f = fast_exp2((x.x - from) * to_log2);
        j.total = fmaf(x.y, f, j.total);
        j.o.x = fmaf(y.x, f, j.o.x);
        j.o.y = fmaf(y.y, f, j.o.y);
    }
    return j;
}

template <int D>
__device__ __forceinline__ void store_out(const CacheAttnArgs& a, const QueryTile& t, int kv, int r, int f,
                                          const Joined& j)
{
    // a row that sees nothing gets zeros
    const float inv = j.total == 0.f ? 0.f : 1.f / j.total;
    const int m = t.m0 + r;
    *reinterpret_cast<uint32_t*>(static_cast<bf16*>(a.out) + (int64_t)(t.row0 + m / a.group) * a.out_stride +
                                 (int64_t)(kv * a.group + m % a.group) * D + f) =
        pack_bf16x2(j.o.x * inv, j.o.y * inv);
}

// Warp results -> shared memory [warp][row][feature] and ml [warp][row], the
// rings' place; a block barrier before and after.
template <int ST, int D, int NQ>
__device__ __forceinline__ void publish(const WarpState<ST, D, NQ>& w, float* parts, float2 (*ml)[8 * NQ])
{
    using S = Step<ST, D>;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < NQ; x++)
#pragma unroll
        for (int c = 0; c < 2; c++)
        {
            const int r = x * 8 + 2 * t + c;
            float sum = w.sum[x][c];
            float off[S::kGroups];
#pragma unroll
            for (int gr = 0; gr < S::kGroups; gr++)
                off[gr] = w.off[x][gr][c];
#pragma unroll
            for (int o = 4; o < 32; o <<= 1)
            {
                sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (S::kFour)
#pragma unroll
                    for (int gr = 0; gr < S::kGroups; gr++)
                        off[gr] += __shfl_xor_sync(0xffffffffu, off[gr], o);
            }
            if (g == 0)
                ml[warp][r] = make_float2(w.top[x][c], sum);
#pragma unroll
            for (int j = 0; j < D / 16; j++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    const int f = S::kFour ? 64 * (j / 4) + 8 * g + 4 * h + j % 4 : 16 * j + 8 * h + g;
                    float o = w.o[x][j][c + 2 * h];
                    if (S::kFour)
                        o = fmaf(o, j & 1 ? kOutUp / 16 : kOutUp, off[j / 4] * kProbsDown);
                    parts[(warp * 8 * NQ + r) * S::kPitch + f] = o;
                }
        }
    __syncthreads();
}

// Short caches: a cluster of `cluster_size` blocks takes one tile of 8 NQ query
// rows of one key/value head, its warps the key blocks in turn, and the blocks
// join their parts in each other's shared memory: one launch, no workspace.
template <int ST, int D, int NQ>
__global__ void __launch_bounds__(kThreads) cache_attention_step_kernel(CacheAttnArgs a, int cluster_size)
{
    using S = Step<ST, D>;
    constexpr int kRows = 8 * NQ;
    extern __shared__ __align__(128) char shared[];
    __shared__ QueryTile tile_s;
    __shared__ float2 ml_s[kWarps + 1][kRows];  // maximum and sum: of each warp, then of the block
    const int rank = blockIdx.x % cluster_size;
    const int warp = threadIdx.x >> 5;
    if (warp == 0)
    {
        const QueryTile found =
            find_tile(a.mem, a.batch, a.group, kRows, blockIdx.x / cluster_size, rank == 0 ? a.error_flag : nullptr);
        if (threadIdx.x == 0)
            tile_s = found;
    }
    __syncthreads();
    Piece p;
    p.tile = tile_s;
    if (p.tile.b < 0)
        return;  // the whole cluster
    p.kv = blockIdx.y;
    p.first = tile_span(a, p.tile, 0);
    p.last = tile_span(a, p.tile, p.tile.count - 1);
    p.blocks = key_blocks(p.first, p.last, a.sinks, S::kKeys);
    p.begin = 0;
    p.end = p.blocks.count;
    WarpState<ST, D, NQ> w;
    work<ST, D, NQ>(a, p, w, shared + warp * S::kWarpBytes, rank * kWarps + warp, cluster_size * kWarps);
    float* parts_s = reinterpret_cast<float*>(shared);
    publish<ST, D, NQ>(w, parts_s, ml_s);

    const float to_log2 = a.scale * 1.44269504088896341f;
    float* block_s = parts_s + kWarps * kRows * S::kPitch;
    for (int e = threadIdx.x; e < p.tile.count * (D / 2); e += kThreads)
    {
        const int r = e / (D / 2), f = 2 * (e % (D / 2));
        const Joined j = join(
            kWarps, to_log2, [&](int i) { return ml_s[i][r]; },
            [&](int i) { return *reinterpret_cast<const float2*>(parts_s + (i * kRows + r) * S::kPitch + f); });
        if (cluster_size == 1)
            store_out<D>(a, p.tile, p.kv, r, f, j);
        else
        {
            *reinterpret_cast<float2*>(block_s + r * S::kPitch + f) = j.o;
            if (f == 0)
                ml_s[kWarps][r] = make_float2(j.top, j.total);
        }
    }
    if (cluster_size == 1)
        return;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int e = rank * kThreads + threadIdx.x; e < p.tile.count * (D / 2); e += cluster_size * kThreads)
    {
        const int r = e / (D / 2), f = 2 * (e % (D / 2));
        const Joined j = join(
            cluster_size, to_log2, [&](int i) { return *cluster.map_shared_rank(&ml_s[kWarps][r], i); },
            [&](int i) {
                return *reinterpret_cast<const float2*>(cluster.map_shared_rank(block_s, i) + r * S::kPitch + f);
            });
        store_out<D>(a, p.tile, p.kv, r, f, j);
    }
    cluster.sync();  // a block's shared memory stays until every peer has read it
}

// ---------------------------------------------------------------- long caches
// The work of a batch in rounds of kWarps key blocks, counted sequence by
// sequence, head by head, tile by tile. Every tile of a sequence counts the
// rounds of all of its rows, so that a sequence is (tiles * heads) equal parts.
struct Rounds
{
    int tiles;   // of the sequence
    int per;     // rounds of one tile and head
};

template <typename S>
__device__ __forceinline__ Rounds sequence_rounds(const CacheAttnArgs& a, int b, int tile)
{
    Rounds r = {0, 0};
    const int rows = b < a.batch.sequences ? batch_rows(a.batch, b) : 0;
    if (rows > 0)
    {
        const int past = max(0, __ldg(a.batch.past + b));
        const int length = sequence_length(a.mem, a.batch, past, rows, nullptr);
        const int p0 = min(past, length);
        const KeyBlocks k = key_blocks(row_span(p0, length, a.sinks, a.window, a.frame_tokens),
                                       row_span(p0 + rows - 1, length, a.sinks, a.window, a.frame_tokens), a.sinks,
                                       S::kKeys);
        r.tiles = (int)(((int64_t)rows * a.group + tile - 1) / tile);
        r.per = max(1, (k.count + kWarps - 1) / kWarps);
    }
    return r;
}

// Where a round lies: sequence b, whose first round is `before`. Warp-collective.
struct Place
{
    int b;  // -1: past the end
    Rounds r;
    int64_t before;
};

template <typename S>
__device__ __forceinline__ Place find_round(const CacheAttnArgs& a, int tile, int64_t round, int64_t* total)
{
    const int lane = threadIdx.x & 31;
    Place place;
    place.b = -1;
    int64_t before = 0;
    for (int base = 0; base < a.batch.sequences; base += 32)
    {
        const Rounds r = sequence_rounds<S>(a, base + lane, tile);
        const int64_t mine = (int64_t)r.tiles * a.mem.heads * r.per;
        int64_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o)
                sum += up;
        }
        const unsigned holds = __ballot_sync(0xffffffffu, round < before + sum);
        if (!total && holds)
        {
            const int src = __ffs(holds) - 1;
            place.b = base + src;
            place.r.tiles = __shfl_sync(0xffffffffu, r.tiles, src);
            place.r.per = __shfl_sync(0xffffffffu, r.per, src);
            place.before = before + __shfl_sync(0xffffffffu, sum - mine, src);
            return place;
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (total)
        *total = before;
    return place;
}

// The blocks among which `total` rounds are dealt: each gets 4 rounds or more.
__device__ __forceinline__ int dealt(int64_t total, int blocks)
{
    return (int)max((int64_t)1, min((int64_t)blocks, total / 4));
}

// Block c of n has the rounds [first_round(c), first_round(c + 1)).
__device__ __forceinline__ int64_t first_round(int64_t total, int n, int c)
{
    return total * c / n;
}

// Tile number `tile` of sequence b, tiles of `size` (row, head) pairs.
__device__ __forceinline__ QueryTile tile_of(const CacheAttnArgs& a, int b, int tile, int size, int* flag)
{
    QueryTile t;
    t.b = b;
    t.row0 = __ldg(a.batch.row_starts + b);
    const int rows = batch_rows(a.batch, b);
    t.m0 = tile * size;
    t.count = min(size, rows * a.group - t.m0);
    t.past = max(0, __ldg(a.batch.past + b));
    t.length = sequence_length(a.mem, a.batch, t.past, rows, flag);
    t.past = min(t.past, t.length);
    return t;
}

// Long caches: every block takes an equal share of the batch's rounds, however
// the sequences differ in length. A tile that one block has whole is finished
// there; the parts of the others go to the workspace, part 2c (a tile that an
// earlier block began) or 2c + 1 (one that a later block ends) of block c, and
// cache_attention_join_kernel joins them.
template <int ST, int D, int NQ>
__global__ void __launch_bounds__(kThreads, ST == AWA_INT4 && NQ == 1 ? 3 : 2)
    cache_attention_split_kernel(CacheAttnArgs a, float* part_o, float2* part_ml)
{
    using S = Step<ST, D>;
    constexpr int kRows = 8 * NQ;
    extern __shared__ __align__(128) char shared[];
    __shared__ float2 ml_s[kWarps][kRows];
    __shared__ Place place_s;
    __shared__ int64_t total_s;
    const int warp = threadIdx.x >> 5;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 0)
    {
        int64_t total = 0;
        find_round<S>(a, kRows, 0, &total);
        if (threadIdx.x == 0)
            total_s = total;
    }
    __syncthreads();
    const int64_t total = total_s;
    const int n = dealt(total, gridDim.x), c = blockIdx.x;
    if (c >= n)
        return;
    const float to_log2 = a.scale * 1.44269504088896341f;
    const int64_t end = first_round(total, n, c + 1);
    for (int64_t u = first_round(total, n, c); u < end;)
    {
        if (warp == 0)
        {
            const Place found = find_round<S>(a, kRows, u, nullptr);
            if (threadIdx.x == 0)
                place_s = found;
        }
        __syncthreads();
        const Place place = place_s;
        if (place.b < 0)
            break;
        const int64_t within = u - place.before;
        const int which = (int)(within / place.r.per), round0 = (int)(within - (int64_t)which * place.r.per);
        const int rounds = (int)min((int64_t)(place.r.per - round0), end - u);
        Piece p;
        p.kv = which / place.r.tiles;
        p.tile = tile_of(a, place.b, which - p.kv * place.r.tiles, kRows, p.kv == 0 && round0 == 0 ? a.error_flag : nullptr);
        p.first = tile_span(a, p.tile, 0);
        p.last = tile_span(a, p.tile, p.tile.count - 1);
        p.blocks = key_blocks(p.first, p.last, a.sinks, S::kKeys);
        p.begin = round0 * kWarps;
        p.end = min(p.blocks.count, (round0 + rounds) * kWarps);
        WarpState<ST, D, NQ> w;
        work<ST, D, NQ>(a, p, w, shared + warp * S::kWarpBytes, warp, kWarps);
        float* parts_s = reinterpret_cast<float*>(shared);
        publish<ST, D, NQ>(w, parts_s, ml_s);
        const bool whole = rounds == place.r.per;
        const int64_t slot = 2 * c + (round0 == 0 ? 1 : 0);
        for (int e = threadIdx.x; e < p.tile.count * (D / 2); e += kThreads)
        {
            const int r = e / (D / 2), f = 2 * (e % (D / 2));
            const Joined j = join(
                kWarps, to_log2, [&](int i) { return ml_s[i][r]; },
                [&](int i) { return *reinterpret_cast<const float2*>(parts_s + (i * kRows + r) * S::kPitch + f); });
            if (whole)
                store_out<D>(a, p.tile, p.kv, r, f, j);
            else
            {
                *reinterpret_cast<float2*>(part_o + (slot * kRows + r) * D + f) = j.o;
                if (f == 0)
                    part_ml[slot * kRows + r] = make_float2(j.top, j.total);
            }
        }
        __syncthreads();  // the shared memory becomes rings again
        u += rounds;
    }
}

// Joins the parts of the tiles that several blocks of cache_attention_split_kernel
// (`blocks` of them) worked on. Blocks: x = tiles, y = heads, z = rows of a tile.
template <int ST, int D, int NQ>
__global__ void __launch_bounds__(D / 2) cache_attention_join_kernel(CacheAttnArgs a, int blocks, const float* part_o,
                                                                   const float2* part_ml)
{
    using S = Step<ST, D>;
    constexpr int kRows = 8 * NQ;
    __shared__ QueryTile tile_s;
    __shared__ Place place_s;
    __shared__ int64_t total_s;
    if (threadIdx.x < 32)
    {
        int64_t total = 0;
        find_round<S>(a, kRows, 0, &total);
        const QueryTile t = find_tile(a.mem, a.batch, a.group, kRows, blockIdx.x, nullptr);
        // the first round of the sequence: all rounds of the sequences before it
        int64_t before = 0;
        if (t.b >= 0)
            for (int base = 0; base < t.b; base += 32)
            {
                const int b = base + threadIdx.x;
                const Rounds r = b < t.b ? sequence_rounds<S>(a, b, kRows) : Rounds{0, 0};
                before += (int64_t)r.tiles * a.mem.heads * r.per;
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            before += __shfl_xor_sync(0xffffffffu, before, o);
        if (threadIdx.x == 0)
        {
            total_s = total;
            tile_s = t;
            place_s.before = before;
            place_s.r = t.b >= 0 ? sequence_rounds<S>(a, t.b, kRows) : Rounds{0, 0};
        }
    }
    __syncthreads();
    const QueryTile t = tile_s;
    const int r = blockIdx.z, kv = blockIdx.y;
    // every block, before anything else: the grid must not end ahead of the split kernel
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (t.b < 0 || r >= t.count)
        return;
    const int64_t total = total_s;
    const int n = dealt(total, blocks);
    const int per = place_s.r.per;
    const int64_t u = place_s.before + ((int64_t)kv * place_s.r.tiles + t.m0 / kRows) * per;
    // the block that has round v: the largest c with first_round(c) <= v
    const auto block_of = [&](int64_t v) { return (int)(((v + 1) * n - 1) / total); };
    const int c0 = block_of(u), c1 = block_of(u + per - 1);
    if (c0 == c1)
        return;  // finished by one block
    const int f = 2 * threadIdx.x;
    const auto slot = [&](int i) { return 2 * (int64_t)(c0 + i) + (i == 0 ? 1 : 0); };
    const Joined j = join(
        c1 - c0 + 1, a.scale * 1.44269504088896341f, [&](int i) { return part_ml[slot(i) * kRows + r]; },
        [&](int i) { return *reinterpret_cast<const float2*>(part_o + (slot(i) * kRows + r) * D + f); });
    store_out<D>(a, t, kv, r, f, j);
}

// Blocks of the split kernel: as many as shared memory lets run at once on 148
// SMs. Of the 4-bit instances, those with 64 features, or with two tiles, hold
// fewer for their registers, so that some of their blocks run behind the others.
template <int ST, int D, int NQ>
constexpr int split_blocks()
{
    const int by_memory = 232448 / (Step<ST, D>::shared_bytes(NQ) + 2048);
    return 148 * (by_memory < 4 ? by_memory : 4);
}

template <int ST, int D, int NQ>
constexpr size_t part_bytes()
{
    return (size_t)2 * split_blocks<ST, D, NQ>() * 8 * NQ * (D + 2) * 4;
}

template <int ST, int D, int NQ>
int run(const CacheAttnArgs& a, int64_t most_keys, void* workspace, cudaStream_t stream)
{
    using S = Step<ST, D>;
    const int64_t tiles = (int64_t)a.batch.rows * a.group / (8 * NQ) + a.batch.sequences;
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr = {};
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = S::shared_bytes(NQ);
    config.stream = stream;
    if (workspace)
    {
        const int blocks = split_blocks<ST, D, NQ>();
        float* part_o = static_cast<float*>(workspace);
        float2* part_ml = reinterpret_cast<float2*>(part_o + (size_t)2 * blocks * 8 * NQ * D);
        config.gridDim = dim3((unsigned)blocks);
        cudaError_t err = cudaLaunchKernelEx(&config, cache_attention_split_kernel<ST, D, NQ>, a, part_o, part_ml);
        if (err != cudaSuccess)
            return (int)err;
        // starts while the split kernel runs and waits for its end on the device
        attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr.val.programmaticStreamSerializationAllowed = 1;
        config.attrs = &attr;
        config.numAttrs = 1;
        config.gridDim = dim3((unsigned)tiles, (unsigned)a.mem.heads, 8 * NQ);
        config.blockDim = dim3(D / 2);
        config.dynamicSmemBytes = 0;
        return (int)cudaLaunchKernelEx(&config, cache_attention_join_kernel<ST, D, NQ>, a, blocks,
                                       (const float*)part_o, (const float2*)part_ml);
    }
    // Blocks that share a tile's keys, at most 8 (the portable cluster size):
    // enough to fill the GPU, as long as each warp still has a key block or two.
    int cluster = 1;
    while (cluster < 8 && tiles * a.mem.heads * cluster < 148 * 4 && most_keys >= 2 * cluster * kWarps * S::kKeys)
        cluster *= 2;
    if (tiles * cluster > 0x7fffffff)
        return (int)cudaErrorInvalidConfiguration;
    config.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)a.mem.heads);
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&config, cache_attention_step_kernel<ST, D, NQ>, a, cluster);
}

template <int ST, int D, int NQ>
int prepare()
{
    const int bytes = Step<ST, D>::shared_bytes(NQ);
    cudaError_t err = cudaFuncSetAttribute(cache_attention_step_kernel<ST, D, NQ>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute(cache_attention_split_kernel<ST, D, NQ>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return (int)err;
}

// The kernel instance of a cache and a batch: F is called with its parameters.
template <typename F>
auto dispatch(int storage, int head_dim, bool two, F f)
{
    if (storage == AWA_INT4)
        return head_dim == 64 ? (two ? f.template operator()<AWA_INT4, 64, 2>() : f.template operator()<AWA_INT4, 64, 1>())
                              : (two ? f.template operator()<AWA_INT4, 128, 2>() : f.template operator()<AWA_INT4, 128, 1>());
    return head_dim == 64 ? (two ? f.template operator()<AWA_BF16, 64, 2>() : f.template operator()<AWA_BF16, 64, 1>())
                          : (two ? f.template operator()<AWA_BF16, 128, 2>() : f.template operator()<AWA_BF16, 128, 1>());
}

// Up to 8 (row, head) pairs per key/value head and sequence fit one tile of 8
bool two_tiles(int group, int max_rows)
{
    return (int64_t)max_rows * group > 8;
}

struct WorkspaceOf
{
    int64_t most_keys;
    template <int ST, int D, int NQ>
    size_t operator()() const
    {
        // A cluster of 8 blocks gives each warp 4 key blocks of a cache this
        // long: a launch alone is then most of the time
        return most_keys <= 8 * kWarps * 4 * Step<ST, D>::kKeys ? 0 : part_bytes<ST, D, NQ>();
    }
};

struct Run
{
    const CacheAttnArgs& a;
    int64_t most_keys;
    void* workspace;
    cudaStream_t stream;
    template <int ST, int D, int NQ>
    int operator()() const
    {
        return run<ST, D, NQ>(a, most_keys, workspace, stream);
    }
};

struct Prepare
{
    template <int ST, int D, int NQ>
    int operator()() const
    {
        return prepare<ST, D, NQ>();
    }
};

}  // namespace

size_t cache_attention_step_workspace(const CacheMemory& mem, int group, int max_rows, int64_t most_keys)
{
    return dispatch(mem.storage, mem.head_dim, two_tiles(group, max_rows), WorkspaceOf{most_keys});
}

int launch_cache_attention_step(const CacheAttnArgs& a, int max_rows, int64_t most_keys, void* workspace,
                                cudaStream_t stream)
{
    ProfileScope scope("awa_cache_attention_step", stream);
    if (!cache_attention_step_workspace(a.mem, a.group, max_rows, most_keys))
        workspace = nullptr;
    return dispatch(a.mem.storage, a.mem.head_dim, two_tiles(a.group, max_rows),
                    Run{a, most_keys, workspace, stream});
}

int prepare_cache_attention_step()
{
    for (int storage : {AWA_BF16, AWA_INT4})
        for (int head_dim : {64, 128})
            for (bool two : {false, true})
            {
                const int err = dispatch(storage, head_dim, two, Prepare{});
                if (err)
                    return err;
            }
    return 0;
}

}  // namespace awa
