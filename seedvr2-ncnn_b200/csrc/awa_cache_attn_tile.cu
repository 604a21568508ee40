// awa_cache_attn_tile.cu -- attention over the paged key/value cache for many
// query rows, on the sm_100a tensor cores (tcgen05.mma, accumulators in TMEM,
// TMA loads of pages): bf16 caches with head_dim 64 and 128.
//
// out = softmax(scale q K^T) V in one pass: per block of 128 keys, S = Q K^T
// into TMEM, the running maximum and sum of each row (base 2, fp32), P =
// 2^(S - max) as bf16 over S in TMEM, O += P V into TMEM. 4 d flops per visible
// pair of query row and key against 4 d bytes per key and 256 rows: the tensor
// cores and the exponentials bound it, not memory.
//
// A block takes one job: two tiles A and B of up to 128 query rows of one
// key/value head. A tile holds whole rows of the batch with all q heads of
// their group ((row, head) pairs, 128 / group rows), so that grouped heads
// share the keys they read. The blocks of keys that only one of the tiles sees
// (the ends of a causal or sliding window) are computed for that one.
//
//   warps 0-3, 4-7  softmax and epilogue of tile A, B: a thread owns one row
//   warp 8          MMA: S_x(i+1) is issued behind O_x += P_x(i) V(i), for A and
//                   B in turn, so that one tile's products run under the other's
//                   softmax
//   warp 9          TMA: Q once, then K and V blocks of 128 keys through a ring;
//                   a page (or the 128-slot half of a page) of one head is one
//                   box per 64 features
//
// 128 keys a block: S_A, S_B, O_A, O_B fill the 512 TMEM columns at head_dim
// 128, P takes the place of S. Every wait is bounded, as in the window kernel.
#include "awa_cache_device.cuh"
#include "awa_rows.cuh"
#include "tcgen05.cuh"

#include <cuda.h>
#include <cuda_bf16.h>

#include <mutex>

namespace awa
{
namespace
{

using bf16 = __nv_bfloat16;

constexpr int kRows = 128;  // query rows of a tile
constexpr int kKeys = 128;  // keys of a block
constexpr int kMmaWarp = 8;
constexpr int kTmaWarp = 9;
constexpr int kCleanWarp = 10;
constexpr int kThreads = 384;  // 3 warpgroups; the last one gives registers to the softmax (a thread holds 128 scores)
constexpr int kSoftmaxRegs = 208, kOtherRegs = 80;  // 8 * 208 + 4 * 80 <= 12 * 168 per lane
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kColS = 0;    // + 128 * tile
constexpr uint32_t kColO = 256;  // + 128 * tile
constexpr uint64_t kWaitLimitNs = 4000000000ull;  // healthy waits last microseconds
constexpr uint64_t kDrainLimitNs = 200000000ull;

template <int D>
struct Tile
{
    static constexpr int kPanels = D / 64;            // of 64 features (128-byte rows, 128-byte swizzle)
    static constexpr int kPanelBytes = kKeys * 128;   // 16 KB
    static constexpr int kBytes = kPanels * kPanelBytes;
    static constexpr int kStages = D == 128 ? 5 : 10;  // of one K or V block: 160 KB, with Q 224 or 192 KB

    uint8_t q[2][kBytes];
    uint8_t ring[kStages][kBytes];
    static constexpr int kLanded = 8;  // at least the V copies in the ring

    uint64_t q_full, full[kStages], empty[kStages], landed[kLanded], s_full[2], p_full[2][2], o_full[2], mma_done;
    uint32_t tmem_base;
    int abort;
    QueryTile job;
};

struct Maps
{
    CUtensorMap q, k, v;
};

// ---------------------------------------------------------------- waits and copies
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* abort, int* error_flag,
                                         int code)
{
    if (tc::mbar_try_wait(bar, parity))
        return true;
    const uint64_t start = tc::global_ns();
    for (;;)
    {
        if (tc::mbar_try_wait_sleep(bar, parity, 20000))
            return true;
        if (*abort)
            return false;
        if (tc::global_ns() - start > kWaitLimitNs)
        {
            *abort = 1;
            cache_error(error_flag, code);
            return false;
        }
    }
}

__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, int* error_flag,
                                          int code)
{
    return __all_sync(0xffffffffu, wait_bar(bar, parity, abort, error_flag, code));
}

// On the way out: copies and MMAs in flight end whatever the abort flag says.
__device__ __forceinline__ void drain_bar(uint64_t* bar, uint32_t parity, int* error_flag, int code)
{
    const uint64_t start = tc::global_ns();
    while (!tc::mbar_try_wait_sleep(bar, parity, 20000))
        if (tc::global_ns() - start > kDrainLimitNs)
        {
            cache_error(error_flag, code);
            return;
        }
}

__device__ __forceinline__ void mbar_arrive(uint64_t* bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(tc::smem_addr(bar)) : "memory");
}

__device__ __forceinline__ void mbar_expect(uint64_t* bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::smem_addr(bar)), "r"(bytes)
                 : "memory");
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(tc::smem_addr(bar))
        : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(tc::smem_addr(bar))
        : "memory");
}

// ---------------------------------------------------------------- the job
// What a job's rows see, and which blocks of keys each tile takes part in.
struct Job
{
    QueryTile t;
    int kv;
    int rows_per_tile;  // batch rows of a tile
    bool has_b;
    RowSpan first[2], last[2];  // of tile A, B
    KeyBlocks blocks;           // of both
    // tile x takes part in the key blocks b < hi[x] with b >= lo[x] or b < sinks
    int lo[2], hi[2], sinks;
};

__device__ __forceinline__ Job make_job(const CacheAttnArgs& a, const QueryTile& t)
{
    Job job;
    job.t = t;
    job.kv = blockIdx.y;
    job.rows_per_tile = kRows / a.group;
    const int m_tile = job.rows_per_tile * a.group;
    job.has_b = t.count > m_tile;
    const int p0 = t.past + t.m0 / a.group;
    const auto span = [&](int p) { return row_span(p, t.length, a.sinks, a.window, a.frame_tokens); };
    job.first[0] = span(p0);
    job.last[0] = span(p0 + (min(t.count, m_tile) - 1) / a.group);
    job.first[1] = job.has_b ? span(p0 + job.rows_per_tile) : job.first[0];
    job.last[1] = job.has_b ? span(p0 + (t.count - 1) / a.group) : job.last[0];
    job.blocks = key_blocks(job.first[0], job.last[1], a.sinks, kKeys);
#pragma unroll
    for (int x = 0; x < 2; x++)
    {
        job.lo[x] = job.first[x].lo / kKeys;
        job.hi[x] = x == 1 && !job.has_b ? 0 : (job.last[x].hi + kKeys - 1) / kKeys;
    }
    job.sinks = (a.sinks + kKeys - 1) / kKeys;
    return job;
}

// Block i of the job's is block number ... of the sequence.
__device__ __forceinline__ int block_of(const Job& job, int i)
{
    return i < job.blocks.prefix ? i : i + job.blocks.shift;
}

// Whether some row of tile x sees a key of block b of the sequence.
__device__ __forceinline__ bool takes_part(const Job& job, int x, int b)
{
    return b < job.hi[x] && (b >= job.lo[x] || b < job.sinks);
}

// Whether some row of the job sees the key.
__device__ __forceinline__ bool seen(const CacheAttnArgs& a, const Job& job, int key)
{
    return key < job.last[1].hi && (key >= job.first[0].lo || key < a.sinks);
}

// Whether every key of block b of the sequence is seen by some row. The others,
// at the ends of the prefix and the window, have slots that may hold anything.
__device__ __forceinline__ bool all_seen(const CacheAttnArgs& a, const Job& job, int b)
{
    const int key0 = b * kKeys;
    return key0 + kKeys <= job.last[1].hi && (key0 >= job.first[0].lo || key0 + kKeys <= a.sinks);
}

// ---------------------------------------------------------------- TMA warp
template <int D>
__device__ void tma_role(const CacheAttnArgs& a, const Maps& maps, Tile<D>& sh, const Job& job)
{
    using T = Tile<D>;
    const int lane = threadIdx.x & 31;
    volatile int* abort = &sh.abort;
    const int m_tile = job.rows_per_tile * a.group;
    if (lane == 0)
        mbar_expect(&sh.q_full, (uint32_t)((job.has_b ? 2 : 1) * T::kPanels * m_tile * 128));
    __syncwarp();
    if (lane < (job.has_b ? 2 : 1) * T::kPanels)
    {
        const int x = lane / T::kPanels, panel = lane % T::kPanels;
        tma_load_3d(tc::smem_addr(sh.q[x] + panel * T::kPanelBytes), &maps.q, 64 * panel, job.kv * a.group,
                    job.t.row0 + job.t.m0 / a.group + x * job.rows_per_tile, &sh.q_full);
    }
    // lanes = (piece of a page, panel) of a block
    const int piece = min(kKeys, 1 << a.mem.page_shift);
    const int pieces = kKeys / piece;
    const int mine = lane / T::kPanels, panel = lane % T::kPanels;
    const int* table = a.batch.page_table + job.t.b * a.batch.table_stride;
    const auto lookup = [&](int i) {
        int page = a.mem.pages;  // past the last: the load brings zeros
        const int key = block_of(job, i) * kKeys + mine * piece;
        if (i < job.blocks.count && mine < pieces && key < job.last[1].hi &&
            (key + piece > job.first[0].lo || key < a.sinks))
        {
            page = __ldg(table + (key >> a.mem.page_shift));
            if ((unsigned)page >= (unsigned)a.mem.pages)
            {
                cache_error(a.error_flag, AWA_CACHE_BAD_PAGE);
                page = a.mem.pages;
            }
        }
        return page;
    };
    int next = lookup(0);
    int n = 0;       // copies issued
    int ragged = 0;  // of them through the clean-up warp
    for (int i = 0; i < job.blocks.count; i++)
    {
        const int page = next;
        next = lookup(i + 1);
        const int block = block_of(job, i);
        const int slot = (block * kKeys + mine * piece) & ((1 << a.mem.page_shift) - 1);
        bool ok = true;
#pragma unroll
        for (int v = 0; v < 2; v++, n++)
        {
            const int stage = n % T::kStages;
            if (!warp_wait(&sh.empty[stage], ((n / T::kStages) & 1) ^ 1, abort, a.error_flag, 73))
            {
                ok = false;
                break;
            }
            // values with unseen slots reach the MMA through the clean-up warp
            uint64_t* bar = &sh.full[stage];
            if (v && !all_seen(a, job, block))
                bar = &sh.landed[ragged++ % T::kLanded];
            if (lane == 0)
                mbar_expect(bar, T::kBytes);
            __syncwarp();
            if (mine < pieces)
                tma_load_4d(tc::smem_addr(sh.ring[stage] + panel * T::kPanelBytes + mine * piece * 128),
                            v ? &maps.v : &maps.k, 64 * panel, slot, job.kv, page, bar);
        }
        if (!ok)
            break;
    }
    drain_bar(&sh.q_full, 0, a.error_flag, 74);
    for (int k = 0; k < T::kLanded && k < ragged; k++)
        drain_bar(&sh.landed[(ragged - 1 - k) % T::kLanded], ((ragged - 1 - k) / T::kLanded) & 1, a.error_flag, 75);
    // (the full barrier of such a copy completes once the clean-up warp is through)
    for (int k = 0; k < T::kStages && k < n; k++)
        drain_bar(&sh.full[(n - 1 - k) % T::kStages], ((n - 1 - k) / T::kStages) & 1, a.error_flag, 75);
}

// ---------------------------------------------------------------- clean-up warp
// Values in slots that no row sees become zeros: their probabilities are 0,
// but 0 * NaN is NaN.
template <int D>
__device__ void clean_role(const CacheAttnArgs& a, Tile<D>& sh, const Job& job)
{
    using T = Tile<D>;
    const int lane = threadIdx.x & 31;
    volatile int* abort = &sh.abort;
    int ragged = 0;
    for (int i = 0; i < job.blocks.count; i++)
    {
        const int block = block_of(job, i);
        if (all_seen(a, job, block))
            continue;
        const bool ok = warp_wait(&sh.landed[ragged % T::kLanded], (ragged / T::kLanded) & 1, abort, a.error_flag, 76);
        ragged++;
        const int stage = (2 * i + 1) % T::kStages;
        if (ok)
            for (int r = lane; r < kKeys; r += 32)
                if (!seen(a, job, block * kKeys + r))
#pragma unroll
                    for (int c = 0; c < 8 * T::kPanels; c++)
                        reinterpret_cast<uint4*>(sh.ring[stage] + (c >> 3) * T::kPanelBytes + r * 128)[c & 7] =
                            make_uint4(0, 0, 0, 0);
        tc::fence_async_smem();
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&sh.full[stage]);
        if (!ok)
            return;
    }
}

// ---------------------------------------------------------------- MMA warp
// S[128 x 128] = Q K^T, both K-major in panels of 64 features.
template <int D>
__device__ __forceinline__ void issue_qk(uint32_t tmem_s, uint32_t q_addr, uint32_t k_addr)
{
    const uint32_t idesc = tc::idesc_bf16_f32(128, kKeys, false);
    const uint64_t q = tc::smem_desc_sw128(q_addr, 16, 1024), k = tc::smem_desc_sw128(k_addr, 16, 1024);
#pragma unroll
    for (int s = 0; s < D / 16; s++)
    {
        const uint64_t step = (uint64_t)((s >> 2) * (Tile<D>::kPanelBytes >> 4) + (s & 3) * 2);
        tc::mma_ss(tmem_s, q + step, k + step, idesc, s > 0 ? 1u : 0u);
    }
}

// O[128 x D] (+)= P[128 x 128] V[128 x D], P in TMEM, V MN-major: 8-key groups
// 1024 bytes apart, panels of 64 features kPanelBytes apart.
template <int D>
__device__ __forceinline__ void issue_pv(uint32_t tmem_o, uint32_t tmem_p, uint32_t v_addr, bool accumulate, int half)
{
    const uint32_t idesc = tc::idesc_bf16_f32(128, D, true);
    const uint64_t v = tc::smem_desc_sw128(v_addr, Tile<D>::kPanelBytes, 1024);
#pragma unroll
    for (int s = half * kKeys / 32; s < (half + 1) * kKeys / 32; s++)
        tc::mma_ts(tmem_o, tmem_p + (uint32_t)(s * 8), v + (uint64_t)(s * (2048 >> 4)), idesc,
                   (accumulate || s > 0) ? 1u : 0u);
}

// One thread: between the MMAs of one tile and the other's there is nothing but
// waits that are mostly over, so the tensor cores do not run dry.
template <int D>
__device__ void mma_issue(const CacheAttnArgs& a, Tile<D>& sh, const Job& job, uint32_t tmem)
{
    using T = Tile<D>;
    volatile int* abort = &sh.abort;
    const int count = job.blocks.count;
    uint32_t p_phase = 0;   // bit x: of tile x
    uint32_t started = 0;
    if (count > 0 && !wait_bar(&sh.q_full, 0, abort, a.error_flag, 81))
        return;
    // copy 2i is K of block i, copy 2i + 1 its V
    int k_stage = 0, v_stage = T::kStages - 1;
    uint32_t k_phase = 0, v_phase = 1;
    bool now[2] = {false, false};  // the tile takes part in block i
    // step i: O += P V of block i, S of block i + 1
    for (int i = -1; i < count; i++)
    {
        const bool more = i + 1 < count;
        const int next = more ? block_of(job, i + 1) : 0;
        const bool then[2] = {more && takes_part(job, 0, next), more && takes_part(job, 1, next)};
        if (i >= 0 && !wait_bar(&sh.full[v_stage], v_phase, abort, a.error_flag, 82))
            return;
        const uint32_t v_addr = tc::smem_addr(sh.ring[v_stage]), k_addr = tc::smem_addr(sh.ring[k_stage]);
        bool k_here = !more;
#pragma unroll
        for (int x = 0; x < 2; x++)
        {
            const uint32_t t_s = tmem + kColS + 128 * x, t_o = tmem + kColO + 128 * x;
            if (now[x])
            {
                // the first half of the keys while the softmax works on the second
#pragma unroll
                for (int h = 0; h < 2; h++)
                {
                    if (!wait_bar(&sh.p_full[x][h], (p_phase >> x) & 1, abort, a.error_flag, 84))
                        return;
                    tc::fence_after_sync();
                    issue_pv<D>(t_o, t_s, v_addr, (started >> x) & 1, h);
                }
                p_phase ^= 1u << x;
                started |= 1u << x;
            }
            if (!k_here)
            {
                if (!wait_bar(&sh.full[k_stage], k_phase, abort, a.error_flag, 83))
                    return;
                k_here = true;
            }
            // S of the next block overwrites P of this one: the MMAs of one
            // thread execute in issue order. The commit covers the P V before
            // it too: the softmax may scale O once the scores are in.
            if (then[x])
            {
                issue_qk<D>(t_s, tc::smem_addr(sh.q[x]), k_addr);
                tc::mma_commit(&sh.s_full[x]);
            }
            now[x] = then[x];
        }
        if (i >= 0)
            tc::mma_commit(&sh.empty[v_stage]);
        if (more)
            tc::mma_commit(&sh.empty[k_stage]);
        const auto advance = [](int& stage, uint32_t& phase) {  // two copies on
            stage += 2;
            if (stage >= T::kStages)
            {
                stage -= T::kStages;
                phase ^= 1;
            }
        };
        advance(k_stage, k_phase);
        advance(v_stage, v_phase);
    }
    tc::mma_commit(&sh.o_full[0]);
    tc::mma_commit(&sh.o_full[1]);
}

template <int D>
__device__ void mma_role(const CacheAttnArgs& a, Tile<D>& sh, const Job& job, uint32_t tmem)
{
    if ((threadIdx.x & 31) == 0)
    {
        mma_issue<D>(a, sh, job, tmem);
        tc::mma_commit(&sh.mma_done);
    }
    __syncwarp();
    drain_bar(&sh.mma_done, 0, a.error_flag, 85);  // complete before TMEM is released
}

// ---------------------------------------------------------------- softmax
// Two fp32 lanes per instruction (.f32x2); each rounds as the scalar one does.
__device__ __forceinline__ void fma_x2(float& d0, float& d1, float a0, float a1, float b, float c)
{
    asm("{\n\t.reg .b64 ra, rb, rc, rd;\n\t"
        "mov.b64 ra, {%2, %3};\n\t"
        "mov.b64 rb, {%4, %4};\n\t"
        "mov.b64 rc, {%5, %5};\n\t"
        "fma.rn.f32x2 rd, ra, rb, rc;\n\t"
        "mov.b64 {%0, %1}, rd;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b), "f"(c));
}

__device__ __forceinline__ void add_x2(float& acc0, float& acc1, float a0, float a1)
{
    asm("{\n\t.reg .b64 ra, rb;\n\t"
        "mov.b64 ra, {%0, %1};\n\t"
        "mov.b64 rb, {%2, %3};\n\t"
        "add.rn.f32x2 ra, ra, rb;\n\t"
        "mov.b64 {%0, %1}, ra;\n\t}"
        : "+f"(acc0), "+f"(acc1)
        : "f"(a0), "f"(a1));
}

__device__ __forceinline__ void mul_x2(float& d0, float& d1, float a0, float a1, float b)
{
    asm("{\n\t.reg .b64 ra, rb;\n\t"
        "mov.b64 ra, {%2, %3};\n\t"
        "mov.b64 rb, {%4, %4};\n\t"
        "mul.rn.f32x2 ra, ra, rb;\n\t"
        "mov.b64 {%0, %1}, ra;\n\t}"
        : "=f"(d0), "=f"(d1)
        : "f"(a0), "f"(a1), "f"(b));
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Bits i with lo <= i < hi of 0..31.
__device__ __forceinline__ uint32_t bit_range(int lo, int hi)
{
    const uint32_t below_hi = hi >= 32 ? ~0u : hi <= 0 ? 0u : (1u << hi) - 1u;
    const uint32_t below_lo = lo >= 32 ? ~0u : lo <= 0 ? 0u : (1u << lo) - 1u;
    return below_hi & ~below_lo;
}

template <int D>
__device__ void softmax_role(const CacheAttnArgs& a, Tile<D>& sh, const Job& job, uint32_t tmem)
{
    const int warp = threadIdx.x >> 5;
    const int x = warp >> 2;
    if (x == 1 && !job.has_b)
        return;
    const int r = threadIdx.x & 127;  // row of the tile = TMEM lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + kColS + 128 * x + lane_base;
    const uint32_t t_o = tmem + kColO + 128 * x + lane_base;
    const float scale_log2 = a.scale * 1.4426950408889634f;
    volatile int* abort = &sh.abort;
    const int m_tile = job.rows_per_tile * a.group;
    const int m = job.t.m0 + x * m_tile + min(r, m_tile - 1);
    const bool mine = r < m_tile && x * m_tile + r < job.t.count;
    const RowSpan span =
        row_span(job.t.past + m / a.group, job.t.length, a.sinks, a.window, a.frame_tokens);
    float m_run = -INFINITY;  // running maximum, in log2 units of the scaled scores
    float l_run = 0.f;
    uint32_t phase = 0;
    bool any = false;
    for (int i = 0; i < job.blocks.count; i++)
    {
        const int block = block_of(job, i), key0 = block * kKeys;
        if (!takes_part(job, x, block))
            continue;
        if (!warp_wait(&sh.s_full[x], phase, abort, a.error_flag, 91))
            return;
        phase ^= 1;
        tc::fence_after_sync();
        uint32_t v[kKeys];
#pragma unroll
        for (int c = 0; c < 4; c++)
            tc::tmem_ld32(t_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&v[32 * c]));
        tc::tmem_wait_ld();
        // the rows of the tile all see all of these keys: nothing to mask
        const bool whole = key0 + kKeys <= job.first[x].hi && (key0 >= job.last[x].lo || key0 + kKeys <= a.sinks);
        if (!whole)
        {
            const int hi = span.hi - key0, lo = span.lo - key0, sinks = min(a.sinks, span.hi) - key0;
#pragma unroll
            for (int c = 0; c < 4; c++)
            {
                const uint32_t bits = bit_range(lo - 32 * c, hi - 32 * c) | bit_range(0, sinks - 32 * c);
#pragma unroll
                for (int j = 0; j < 32; j++)
                    if (!((bits >> j) & 1u))
                        v[32 * c + j] = 0xff800000u;  // -inf: p = 0
            }
        }
        float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < kKeys / 2; j++)
            top[j & 3] = max3(top[j & 3], __uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
        const float m_blk = max3(max3(top[0], top[1], top[2]), top[3], -INFINITY) * scale_log2;
        // O is scaled only when the maximum has grown by more than 2^8: until
        // then the larger exponentials stay well inside fp32 and bf16
        float alpha = 1.f;
        bool rescale = false;
        if (!any)
            m_run = m_blk;
        else if (m_blk > m_run + 8.f)
        {
            alpha = fast_exp2(m_run - m_blk);  // 0 while no key has been seen (m_run = -inf)
            m_run = m_blk;
            rescale = true;
        }
        if (__any_sync(0xffffffffu, rescale))
        {
#pragma unroll 1
            for (int c = 0; c < D / 16; c++)
            {
                uint32_t o[16];
                tc::tmem_ld16(t_o + c * 16, o);
                tc::tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; j += 2)
                {
                    float o0, o1;
                    mul_x2(o0, o1, __uint_as_float(o[j]), __uint_as_float(o[j + 1]), alpha);
                    o[j] = __float_as_uint(o0);
                    o[j + 1] = __float_as_uint(o1);
                }
                tc::tmem_st16(t_o + c * 16, o);
            }
        }
        any = true;
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < 4; c++)
        {
            uint32_t pk[16];
#pragma unroll
            for (int j = 0; j < 16; j++)
            {
                const int k = 32 * c + 2 * j;
                float x0, x1;
                fma_x2(x0, x1, __uint_as_float(v[k]), __uint_as_float(v[k + 1]), scale_log2, neg_m);
                const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
                add_x2(sums[2 * (j & 1)], sums[2 * (j & 1) + 1], p0, p1);
                pk[j] = pack_bf16x2(p0, p1);  // the operand type of P V; the sums keep fp32
            }
            tc::tmem_st16(t_s + 16 * c, pk);
            if (c & 1)  // half of the keys
            {
                tc::tmem_wait_st();
                tc::fence_before_sync();
                mbar_arrive(&sh.p_full[x][c >> 1]);
            }
        }
        l_run = l_run * alpha + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
    }
    if (!warp_wait(&sh.o_full[x], 0, abort, a.error_flag, 92))
        return;
    tc::fence_after_sync();
    // a row that sees nothing (l = 0) gets zeros; O was never written if no block was taken
    const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
    bf16* row = static_cast<bf16*>(a.out) + (int64_t)(job.t.row0 + m / a.group) * a.out_stride +
                (int64_t)(job.kv * a.group + m % a.group) * D;
#pragma unroll
    for (int h = 0; h < D / 32; h++)
    {
        uint32_t o[32];
#pragma unroll
        for (int j = 0; j < 32; j++)
            o[j] = 0;
        if (any)
        {
            tc::tmem_ld32(t_o + 32 * h, o);
            tc::tmem_wait_ld();
        }
        uint32_t pk[16];
#pragma unroll
        for (int j = 0; j < 16; j++)
        {
            float o0, o1;
            mul_x2(o0, o1, __uint_as_float(o[2 * j]), __uint_as_float(o[2 * j + 1]), inv);
            pk[j] = pack_bf16x2(o0, o1);
        }
        if (mine)
#pragma unroll
            for (int j = 0; j < 4; j++)
                reinterpret_cast<uint4*>(row + 32 * h)[j] =
                    make_uint4(pk[4 * j], pk[4 * j + 1], pk[4 * j + 2], pk[4 * j + 3]);
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    cache_attention_tile_kernel(const CacheAttnArgs a, const __grid_constant__ Maps maps)
{
    extern __shared__ uint8_t smem_raw[];
    // 1024-byte alignment for the 128-byte swizzle atoms
    const uint32_t raw_addr = tc::smem_addr(smem_raw);
    Tile<D>& sh = *reinterpret_cast<Tile<D>*>(smem_raw + ((1024 - (raw_addr & 1023)) & 1023));
    const int warp = threadIdx.x >> 5;
    if (warp == 0)
    {
        // the last tiles of a sequence see the most keys of a causal mask: they come first
        const QueryTile t = find_tile(a.mem, a.batch, a.group, 2 * (kRows / a.group) * a.group,
                                      gridDim.x - 1 - blockIdx.x, blockIdx.y == 0 ? a.error_flag : nullptr);
        if (threadIdx.x == 0)
            sh.job = t;
    }
    if (threadIdx.x == 32)
    {
        tc::mbar_init(&sh.q_full, 1);
        for (int s = 0; s < Tile<D>::kStages; s++)
        {
            tc::mbar_init(&sh.full[s], 1);
            tc::mbar_init(&sh.empty[s], 1);
        }
        for (int s = 0; s < Tile<D>::kLanded; s++)
            tc::mbar_init(&sh.landed[s], 1);
        for (int x = 0; x < 2; x++)
        {
            tc::mbar_init(&sh.s_full[x], 1);
            tc::mbar_init(&sh.p_full[x][0], kRows);
            tc::mbar_init(&sh.p_full[x][1], kRows);
            tc::mbar_init(&sh.o_full[x], 1);
        }
        tc::mbar_init(&sh.mma_done, 1);
        tc::mbar_fence_init();
        sh.abort = 0;
    }
    __syncthreads();
    if (sh.job.b < 0)
        return;
    const Job job = make_job(a, sh.job);
    if (warp == kMmaWarp)
    {
        tc::tmem_alloc(&sh.tmem_base, kTmemColumns);
        tc::tmem_relinquish();
    }
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sh.tmem_base;

    if (warp < kMmaWarp)
    {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        softmax_role<D>(a, sh, job, tmem);
    }
    else
    {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kMmaWarp)
            mma_role<D>(a, sh, job, tmem);
        else if (warp == kTmaWarp)
            tma_role<D>(a, maps, sh, job);
        else if (warp == kCleanWarp)
            clean_role<D>(a, sh, job);
    }

    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp)
    {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemColumns);
    }
}

// ---------------------------------------------------------------- tensor maps (host)
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled()
{
    static std::once_flag once;
    static EncodeTiledFn fn = nullptr;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult status;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &status) == cudaSuccess &&
            status == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
    });
    return fn;
}

// A bf16 map with 128-byte swizzle, zeros outside. strides in bytes, of dims 1..
bool encode(CUtensorMap* map, const void* base, int rank, const int64_t* dims, const int64_t* strides, const int* box)
{
    const EncodeTiledFn fn = encode_tiled();
    if (!fn)
        return false;
    cuuint64_t d[4], s[3];
    cuuint32_t b[4], e[4];
    for (int i = 0; i < rank; i++)
    {
        d[i] = (cuuint64_t)dims[i];
        b[i] = (cuuint32_t)box[i];
        e[i] = 1;
        if (i > 0)
            s[i - 1] = (cuuint64_t)strides[i - 1];
    }
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<void*>(base), d, s, b, e,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D>
int run(const CacheAttnArgs& a, cudaStream_t stream)
{
    Maps maps;
    const int page = 1 << a.mem.page_shift, rows_per_tile = kRows / a.group;
    const int64_t dims[4] = {D, page, a.mem.heads, a.mem.pages};
    const int64_t strides[3] = {2 * D, a.mem.head_stride, a.mem.page_stride};
    const int box[4] = {64, page < kKeys ? page : kKeys, 1, 1};
    const int64_t q_dims[3] = {D, (int64_t)a.mem.heads * a.group, a.batch.rows};
    const int64_t q_strides[2] = {2 * D, a.q_stride * 2};
    const int q_box[3] = {64, a.group, rows_per_tile};
    if (!encode(&maps.k, a.mem.k, 4, dims, strides, box) || !encode(&maps.v, a.mem.v, 4, dims, strides, box) ||
        !encode(&maps.q, a.q, 3, q_dims, q_strides, q_box))
        return (int)cudaErrorInvalidValue;
    const int64_t jobs = (int64_t)a.batch.rows / (2 * rows_per_tile) + a.batch.sequences;
    cache_attention_tile_kernel<D><<<dim3((unsigned)jobs, (unsigned)a.mem.heads), kThreads,
                                     sizeof(Tile<D>) + 1024, stream>>>(a, maps);
    return (int)cudaGetLastError();
}

template <int D>
cudaError_t prepare()
{
    return cudaFuncSetAttribute(cache_attention_tile_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(Tile<D>) + 1024);
}

}  // namespace

int launch_cache_attention_tile(const CacheAttnArgs& a, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_attention_tile", stream);
    return a.mem.head_dim == 64 ? run<64>(a, stream) : run<128>(a, stream);
}

int prepare_cache_attention_tile()
{
    const cudaError_t err = prepare<64>();
    return (int)(err != cudaSuccess ? err : prepare<128>());
}

}  // namespace awa
