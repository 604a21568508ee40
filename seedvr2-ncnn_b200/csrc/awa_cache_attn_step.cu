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
// 4 bits: a code c stands for scale (c + z), z = minimum / scale. 128 + c is a
// bf16 value whose bits are 0x4300 | c, so codes become operands with a shift
// and a three-input logic operation, exactly. Per 64 features with their own scale,
//   sum q k = scale (sum q (128 + c) + (z - 128) sum q)
//   sum p v = sum p' (128 + c) + sum p' (z - 128),  p' = bf16(p scale),
// the offsets in fp32, the second sum with the same rounded p', so that the
// one rounding acts on p as it does for a bf16 cache.
#include "awa_cache_device.cuh"
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
constexpr int kStages = 3;

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
    // 4 bits: (scale, z - 128) of the stage's keys, [k, v][key][group]
    static constexpr int kScaleBytes = kFour ? 2 * kKeys * kGroups * 8 : 0;
    static constexpr int kWarpBytes = kStages * kStageBytes + kScaleBytes;
    static constexpr int kPitch = D + 4;  // floats of a row of partial results
    static constexpr int shared_bytes(int nq)
    {
        const int ring = kWarps * kWarpBytes, parts = (kWarps + 1) * 8 * nq * kPitch * 4;
        return ring > parts ? ring : parts;
    }
};

__device__ __forceinline__ uint32_t shared_address(const void* p)
{
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// Copies BYTES (4, 8 or 16); none of them is read, and zeros written, if !real.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src, bool real)
{
    const int n = real ? BYTES : 0;
    if (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(n), "n"(BYTES)
                     : "memory");
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t addr, uint32_t (&r)[4])
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// 8x8 transpose of one b16 matrix held across the warp.
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Codes j and j + 4 of a word as the bf16 pair (128 + c_j, 128 + c_(j+4)).
__device__ __forceinline__ uint32_t code_pair(uint32_t word, int j)
{
    return ((word >> (4 * j)) & 0x000f000fu) | 0x43004300u;
}

// Where 16-byte piece c of row r of a stage lies. bf16: the 8 rows that one
// ldmatrix reads fall on different banks. 4 bits (64-byte rows of two 32-byte
// groups): the groups of half the rows swap places, so that neither the 8-byte
// reads of keys nor the 4-byte reads of values collide.
template <int ST, int D>
__device__ __forceinline__ int piece_offset(int r, int c)
{
    if (ST != AWA_INT4)
        return r * 2 * D + ((c ^ (r & 7)) << 4);
    if (D == 64)
        return r * 32 + (c << 4);
    return r * 64 + ((c ^ ((((r >> 1) ^ (r >> 2)) & 1) << 1)) << 4);
}

// The key that row r of a 16-key block holds. 4 bits: rows 2t, 2t + 1 (whose
// values one lane pairs up) are keys t, t + 4 of each eight, so that the lanes'
// reads of values fall on different banks.
template <int ST>
__device__ __forceinline__ int key_of_row(int r)
{
    return ST == AWA_INT4 ? (r & 8) | ((r & 1) << 2) | ((r & 7) >> 1) : r;
}

template <int ST, int D, int NQ>
struct WarpState
{
    using S = Step<ST, D>;
    uint32_t q[NQ][D / 16][2];  // Q^T operands
    float q_sum[NQ][S::kGroups][2];  // 4 bits: sum of q over a group, of columns 2t, 2t + 1
    float o[NQ][D / 16][4];
    float off[NQ][S::kGroups][2];  // 4 bits: sum p' (z - 128)
    float top[NQ][2], sum[NQ][2];
    RowSpan span[NQ][2];
};

// The warp's share of one 16-key block: scores, exponentials, probabilities.
template <int ST, int D, int NQ>
__device__ __forceinline__ void scores(const WarpState<ST, D, NQ>& w, const char* kdata, const float2* kscale, int block,
                                       float (&s)[NQ][4])
{
    using S = Step<ST, D>;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    if (ST != AWA_INT4)
    {
#pragma unroll
        for (int n = 0; n < NQ; n++)
            s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
        const int r = block * 16 + (lane & 15);
        const uint32_t base = shared_address(kdata);
#pragma unroll
        for (int i = 0; i < D / 16; i++)
        {
            uint32_t a[4];
            ldmatrix_x4(base + piece_offset<ST, D>(r, 2 * i + (lane >> 4)), a);
#pragma unroll
            for (int n = 0; n < NQ; n++)
                mma(s[n], a[0], a[1], a[2], a[3], w.q[n][i][0], w.q[n][i][1]);
        }
        return;
    }
    const int r0 = block * 16 + key_of_row<ST>(g), r1 = r0 + 8;
#pragma unroll
    for (int gr = 0; gr < S::kGroups; gr++)
    {
        float acc[NQ][4] = {};
        // 16 features of a lane: 8 bytes of each of its two keys
        const uint2 x0 = *reinterpret_cast<const uint2*>(kdata + piece_offset<ST, D>(r0, 2 * gr) + 8 * t);
        const uint2 x1 = *reinterpret_cast<const uint2*>(kdata + piece_offset<ST, D>(r1, 2 * gr) + 8 * t);
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
        const float2 p0 = kscale[r0 * S::kGroups + gr], p1 = kscale[r1 * S::kGroups + gr];
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
            for (int c = 0; c < 4; c++)
            {
                const float2 p = c < 2 ? p0 : p1;
                const float part = fmaf(p.y, w.q_sum[n][gr][c & 1], acc[n][c]);
                s[n][c] = gr == 0 ? p.x * part : fmaf(p.x, part, s[n][c]);
            }
    }
}

// O^T += V^T P^T of one 16-key block; p: the exponentials in the layout of the scores.
template <int ST, int D, int NQ>
__device__ __forceinline__ void values(WarpState<ST, D, NQ>& w, const char* vdata, const float2* vscale, int block,
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
        const int r = block * 16 + (lane & 7) + ((lane >> 4) << 3);
        const uint32_t base = shared_address(vdata);
#pragma unroll
        for (int i = 0; i < D / 16; i++)
        {
            uint32_t a[4];
            ldmatrix_x4_trans(base + piece_offset<ST, D>(r, 2 * i + ((lane >> 3) & 1)), a);
#pragma unroll
            for (int n = 0; n < NQ; n++)
                mma(w.o[n][i], a[0], a[1], a[2], a[3], b[n][0], b[n][1]);
        }
        return;
    }
    const int r0 = block * 16 + key_of_row<ST>(g), r1 = r0 + 8;
    const int k0 = block * 16 + t;  // keys of rows 2t, 2t + 1, 2t + 8, 2t + 9: k0, + 4, + 8, + 12
#pragma unroll
    for (int gr = 0; gr < S::kGroups; gr++)
    {
        const float2 p0 = vscale[r0 * S::kGroups + gr], p1 = vscale[r1 * S::kGroups + gr];
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
        uint32_t x[4];  // features 8g .. 8g + 7 of the group, of the lane's four keys
#pragma unroll
        for (int u = 0; u < 4; u++)
            x[u] = *reinterpret_cast<const uint32_t*>(vdata + piece_offset<ST, D>(k0 + 4 * u, 2 * gr + (g >> 2)) +
                                                      4 * (g & 3));
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

// A cluster of `cluster_size` blocks takes one tile of 8 NQ query rows of one
// key/value head; its warps take the stages of keys in turn.
template <int ST, int D, int NQ>
__global__ void __launch_bounds__(kThreads) cache_attention_step_kernel(CacheAttnArgs a, int cluster_size)
{
    using S = Step<ST, D>;
    constexpr int kRows = 8 * NQ;
    extern __shared__ __align__(128) char shared[];
    __shared__ QueryTile tile_s;
    __shared__ float2 ml_s[kWarps + 1][kRows];  // maximum and sum: of each warp, then of the block
    const CacheMemory& mem = a.mem;
    const int rank = blockIdx.x % cluster_size;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    if (warp == 0)
    {
        const QueryTile found =
            find_tile(mem, a.batch, a.group, kRows, blockIdx.x / cluster_size, rank == 0 ? a.error_flag : nullptr);
        if (lane == 0)
            tile_s = found;
    }
    __syncthreads();
    const QueryTile tile = tile_s;
    if (tile.b < 0)
        return;  // the whole cluster
    const int kv = blockIdx.y;

    const auto span_of = [&](int m) {
        return row_span(tile.past + (tile.m0 + m) / a.group, tile.length, a.sinks, a.window, a.frame_tokens);
    };
    const RowSpan first = span_of(0), last = span_of(tile.count - 1);
    const KeyBlocks blocks = key_blocks(first, last, a.sinks, S::kKeys);
    const int parts = cluster_size * kWarps;
    char* ring = shared + warp * S::kWarpBytes;
    float2* scales = reinterpret_cast<float2*>(ring + kStages * S::kStageBytes);
    const char* kbase = mem.k + kv * mem.head_stride;
    const char* vbase = mem.v + kv * mem.head_stride;
    const int* table = a.batch.page_table + tile.b * a.batch.table_stride;
    const int page_mask = (1 << mem.page_shift) - 1;

    // Issues the copies of stage n of this warp (n counts from 0) into the ring.
    const auto issue = [&](int n) {
        const int i = rank * kWarps + warp + n * parts;
        if (i < blocks.count)
        {
            const int key0 = (i < blocks.prefix ? i : i + blocks.shift) * S::kKeys;
            const uint32_t dst = shared_address(ring) + (n % kStages) * S::kStageBytes;
            const bool all = key0 + S::kKeys <= last.hi && (key0 >= first.lo || key0 + S::kKeys <= a.sinks);
            constexpr int kPieces = S::kRowBytes / 16;  // a power of two: 2, 4, 8 or 16
#pragma unroll
            for (int j = 0; j < S::kKeys * kPieces / 32; j++)
            {
                const int r = (j * 32 + lane) / kPieces, c = (j * 32 + lane) % kPieces;
                const int key = key0 + r;
                // only what some row sees is read: pages outside may be gone
                bool real = all || (key < last.hi && (key >= first.lo || key < a.sinks));
                int page = real ? __ldg(table + (key >> mem.page_shift)) : 0;
                if ((unsigned)page >= (unsigned)mem.pages)
                {
                    cache_error(a.error_flag, AWA_CACHE_BAD_PAGE);
                    page = 0;
                    real = false;
                }
                const int64_t at = page * mem.page_stride + (int64_t)(key & page_mask) * S::kRowBytes + 16 * c;
                const int to = piece_offset<ST, D>(r, c);
                copy_async<16>(dst + to, kbase + at, real);
                copy_async<16>(dst + S::kKeys * S::kRowBytes + to, vbase + at, real);
            }
            if (S::kFour)
            {
                const int key = key0 + lane;
                bool real = all || (key < last.hi && (key >= first.lo || key < a.sinks));
                int page = real ? __ldg(table + (key >> mem.page_shift)) : 0;
                real = real && (unsigned)page < (unsigned)mem.pages;
                page = real ? page : 0;
                const int64_t at = page * mem.params_page_stride + kv * mem.params_head_stride +
                                   (int64_t)(key & page_mask) * S::kParamBytes;
                const uint32_t to = dst + 2 * S::kKeys * S::kRowBytes + lane * S::kParamBytes;
                copy_async<S::kFour ? S::kParamBytes : 4>(to, mem.k_params + at, real);
                copy_async<S::kFour ? S::kParamBytes : 4>(to + S::kKeys * S::kParamBytes, mem.v_params + at, real);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int n = 0; n < kStages - 1; n++)
        issue(n);

    WarpState<ST, D, NQ> w;
    const bf16* q = static_cast<const bf16*>(a.q);
#pragma unroll
    for (int n = 0; n < NQ; n++)
    {
        // column g of tile n
        const int m = tile.m0 + n * 8 + g;
        const bool mine = n * 8 + g < tile.count;
        const bf16* row = q + (int64_t)(tile.row0 + m / a.group) * a.q_stride + (int64_t)(kv * a.group + m % a.group) * D;
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
                    // pairs of features j, j + 4 as code_pair makes them
                    w.q[n][4 * gr + 2 * h][0] = __byte_perm(x.x, x.z, 0x5410);
                    w.q[n][4 * gr + 2 * h][1] = __byte_perm(x.x, x.z, 0x7632);
                    w.q[n][4 * gr + 2 * h + 1][0] = __byte_perm(x.y, x.w, 0x5410);
                    w.q[n][4 * gr + 2 * h + 1][1] = __byte_perm(x.y, x.w, 0x7632);
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
                w.q_sum[n][gr][c] = ST == AWA_INT4 ? __shfl_sync(0xffffffffu, part[gr], 4 * (2 * t + c)) : 0.f;
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
            w.span[n][c] = span_of(min(n * 8 + 2 * t + c, tile.count - 1));
        }
    }
    const float to_log2 = a.scale * 1.44269504088896341f;

    for (int n = 0;; n++)
    {
        const int i = rank * kWarps + warp + n * parts;
        if (i >= blocks.count)
            break;
        issue(n + kStages - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
        __syncwarp();
        const char* kdata = ring + (n % kStages) * S::kStageBytes;
        const char* vdata = kdata + S::kKeys * S::kRowBytes;
        const int key0 = (i < blocks.prefix ? i : i + blocks.shift) * S::kKeys;
        if (S::kFour)
        {
            // a lane works out (scale, z - 128) of its key. A scale of 0 or next
            // to it (then the value is the minimum) is raised to where z and
            // scale z stay finite: that moves the value by 15 * 2^-100 of it
            const uint32_t* par = reinterpret_cast<const uint32_t*>(vdata + S::kKeys * S::kRowBytes);
#pragma unroll
            for (int x = 0; x < 2; x++)
#pragma unroll
                for (int gr = 0; gr < S::kGroups; gr++)
                {
                    const uint32_t word = par[(x * S::kKeys + lane) * S::kGroups + gr];
                    const float low = __uint_as_float(word & 0xffff0000u);
                    const float scale = fmaxf(__uint_as_float(word << 16), 0x1p-100f * fmaxf(1.f, fabsf(low)));
                    scales[(x * S::kKeys + lane) * S::kGroups + gr] =
                        make_float2(scale, __fdividef(low, scale) - 128.f);
                }
            __syncwarp();
        }
        constexpr int kBlocks = S::kKeys / 16;
        float s[kBlocks][NQ][4];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
            scores<ST, D, NQ>(w, kdata, scales, b, s[b]);
        // rows of the tile see all of these keys: nothing to mask
        const bool all = (key0 >= last.lo && key0 + S::kKeys <= first.hi) ||
                         (key0 + S::kKeys <= a.sinks && key0 + S::kKeys <= first.hi);
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
        float base[NQ][2];
        bool grew = false;
#pragma unroll
        for (int x = 0; x < NQ; x++)
#pragma unroll
            for (int c = 0; c < 2; c++)
            {
                float top = fmaxf(s[0][x][c], s[0][x][c + 2]);
#pragma unroll
                for (int b = 1; b < kBlocks; b++)
                    top = fmaxf(top, fmaxf(s[b][x][c], s[b][x][c + 2]));
#pragma unroll
                for (int off = 4; off < 32; off <<= 1)
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
                base[x][c] = fmaxf(top, w.top[x][c]);
                grew |= top > w.top[x][c];
            }
        if (__any_sync(0xffffffffu, grew))
#pragma unroll
            for (int x = 0; x < NQ; x++)
#pragma unroll
                for (int c = 0; c < 2; c++)
                {
                    const float old = w.top[x][c] == base[x][c] ? 1.f : fast_exp2((w.top[x][c] - base[x][c]) * to_log2);
                    w.top[x][c] = base[x][c];
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
                const float from = base[x][c] == -INFINITY ? 0.f : base[x][c] * to_log2;
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
            values<ST, D, NQ>(w, vdata, scales + S::kKeys * S::kGroups, b, s[b]);
        __syncwarp();  // the stage is free for the copies of the next round
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();  // the rings become the partial results [warp][row][feature]

    float* parts_s = reinterpret_cast<float*>(shared);
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
                ml_s[warp][r] = make_float2(w.top[x][c], sum);
#pragma unroll
            for (int j = 0; j < D / 16; j++)
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    const int f = S::kFour ? 64 * (j / 4) + 8 * g + 4 * h + j % 4 : 16 * j + 8 * h + g;
                    parts_s[(warp * kRows + r) * S::kPitch + f] = w.o[x][j][c + 2 * h] + (S::kFour ? off[j / 4] : 0.f);
                }
        }
    __syncthreads();

    // The block's warps, then the cluster's blocks, joined in a fixed order.
    bf16* out = static_cast<bf16*>(a.out);
    const auto store = [&](int r, int f, float2 v, float total) {
        const float inv = total > 0.f ? 1.f / total : total == 0.f ? 0.f : total;
        const int m = tile.m0 + r;
        *reinterpret_cast<uint32_t*>(out + (int64_t)(tile.row0 + m / a.group) * a.out_stride +
                                     (int64_t)(kv * a.group + m % a.group) * D + f) =
            pack_bf16x2(v.x * inv, v.y * inv);
    };
    float* block_s = parts_s + kWarps * kRows * S::kPitch;
    for (int e = threadIdx.x; e < tile.count * (D / 2); e += kThreads)
    {
        const int r = e / (D / 2), f = 2 * (e % (D / 2));
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kWarps; i++)
            top = fmaxf(top, ml_s[i][r].x);
        const float from = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        float2 v = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < kWarps; i++)
        {
            const float2 ml = ml_s[i][r];
            const float x = fast_exp2((ml.x - from) * to_log2);
            const float2 y = *reinterpret_cast<const float2*>(parts_s + (i * kRows + r) * S::kPitch + f);
            total = fmaf(ml.y, x, total);
            v.x = fmaf(y.x, x, v.x);
            v.y = fmaf(y.y, x, v.y);
        }
        if (cluster_size == 1)
            store(r, f, v, total);
        else
        {
            *reinterpret_cast<float2*>(block_s + r * S::kPitch + f) = v;
            if (f == 0)
                ml_s[kWarps][r] = make_float2(top, total);
        }
    }
    if (cluster_size == 1)
        return;
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int e = rank * kThreads + threadIdx.x; e < tile.count * (D / 2); e += cluster_size * kThreads)
    {
        const int r = e / (D / 2), f = 2 * (e % (D / 2));
        float top = -INFINITY;
        for (int i = 0; i < cluster_size; i++)
            top = fmaxf(top, cluster.map_shared_rank(&ml_s[kWarps][r], i)->x);
        const float from = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        float2 v = make_float2(0.f, 0.f);
        for (int i = 0; i < cluster_size; i++)
        {
            const float2 ml = *cluster.map_shared_rank(&ml_s[kWarps][r], i);
            const float x = fast_exp2((ml.x - from) * to_log2);
            const float2 y = *reinterpret_cast<const float2*>(cluster.map_shared_rank(block_s, i) + r * S::kPitch + f);
            total = fmaf(ml.y, x, total);
            v.x = fmaf(y.x, x, v.x);
            v.y = fmaf(y.y, x, v.y);
        }
        store(r, f, v, total);
    }
    cluster.sync();  // a block's shared memory stays until every peer has read it
}

template <int ST, int D, int NQ>
int run(const CacheAttnArgs& a, int64_t most_keys, cudaStream_t stream)
{
    using S = Step<ST, D>;
    const int64_t tiles = (int64_t)a.batch.rows * a.group / (8 * NQ) + a.batch.sequences;
    // Blocks that share a tile's keys, at most 8 (the portable cluster size):
    // as many as keep every SM busy to the end although sequences differ in
    // length, as long as each warp still has some stages of its own.
    int cluster = 1;
    while (cluster < 8 && tiles * a.mem.heads * cluster < 148 * 8 && most_keys >= 4 * cluster * kWarps * S::kKeys)
        cluster *= 2;
    if (tiles * cluster > 0x7fffffff)
        return (int)cudaErrorInvalidConfiguration;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(tiles * cluster), (unsigned)a.mem.heads);
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = S::shared_bytes(NQ);
    config.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return (int)cudaLaunchKernelEx(&config, cache_attention_step_kernel<ST, D, NQ>, a, cluster);
}

template <int ST, int D>
int run(const CacheAttnArgs& a, int max_rows, int64_t most_keys, cudaStream_t stream)
{
    return (int64_t)max_rows * a.group <= 8 ? run<ST, D, 1>(a, most_keys, stream) : run<ST, D, 2>(a, most_keys, stream);
}

template <int ST, int D>
int prepare()
{
    cudaError_t err = cudaFuncSetAttribute(cache_attention_step_kernel<ST, D, 1>,
                                           cudaFuncAttributeMaxDynamicSharedMemorySize, Step<ST, D>::shared_bytes(1));
    if (err == cudaSuccess)
        err = cudaFuncSetAttribute(cache_attention_step_kernel<ST, D, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   Step<ST, D>::shared_bytes(2));
    return (int)err;
}

}  // namespace

int launch_cache_attention_step(const CacheAttnArgs& a, int max_rows, int64_t most_keys, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_attention_step", stream);
    if (a.mem.storage == AWA_INT4)
        return a.mem.head_dim == 64 ? run<AWA_INT4, 64>(a, max_rows, most_keys, stream)
                                    : run<AWA_INT4, 128>(a, max_rows, most_keys, stream);
    return a.mem.head_dim == 64 ? run<AWA_BF16, 64>(a, max_rows, most_keys, stream)
                                : run<AWA_BF16, 128>(a, max_rows, most_keys, stream);
}

int prepare_cache_attention_step()
{
    for (int (*set)() : {prepare<AWA_BF16, 64>, prepare<AWA_BF16, 128>, prepare<AWA_INT4, 64>, prepare<AWA_INT4, 128>})
    {
        const int err = set();
        if (err)
            return err;
    }
    return 0;
}

}  // namespace awa
