// awa_cache_attn_tile.cu -- attention over the paged key/value cache for many
// query rows, on the sm_100a tensor cores (tcgen05.mma, accumulators in TMEM,
// TMA loads of pages): bf16 caches with head_dim 64 and 128, and what was
// unpacked to fp16 from 4-bit ones.
//
// out = softmax(scale q K^T) V in one pass: per block of 128 keys, S = Q K^T
// into TMEM, the running maximum and sum of each row (base 2, fp32), P =
// 2^(S - max) in 16 bits over S in TMEM, O += P V into TMEM. fp16 operands come
// scaled by powers of two, which the scores and O take back. 4 d flops per visible
// pair of query row and key against 4 d bytes per key and 256 rows: the tensor
// cores and the exponentials bound it, not memory.
//
// A job is two tiles A and B of up to 128 query rows of one key/value head. A
// tile holds whole rows of the batch with all q heads of their group ((row,
// head) pairs, 128 / group rows), so that grouped heads share the keys they
// read. The blocks of keys that only one of the tiles sees (the ends of a
// causal or sliding window) are computed for that one.
//
// One thread block per SM, each with an equal share of the batch's work in its
// order, however sequences and masks differ: work is counted in key blocks, a job
// costing kJobCost more for its start and its end. A share is the end of one
// job, some whole ones and the beginning of another; its bounds move to the
// edges of jobs that are small beside it. What a block does not finish alone
// goes to the workspace as fp32 sums, and cache_attention_tile_join_kernel joins
// the parts in order.
//
//   warps 0-3, 4-7  softmax and epilogue of tile A, B: a thread owns one row
//   warp 8          MMA: S_x(i+1) is issued behind O_x += P_x(i) V(i), for A and
//                   B in turn, so that one tile's products run under the other's
//                   softmax
//   warp 9          TMA: Q of a job, then K and V blocks of 128 keys through a
//                   ring; a page (or the 128-slot half of a page) of one head is
//                   one box per 64 features
//   warp 10         clean-up: zeros for the values that no row sees
//   warp 11         works out the next job while the others work on this one
//
// 128 keys a block: S_A, S_B, O_A, O_B fill the 512 TMEM columns at head_dim
// 128, P takes the place of S. Every wait is bounded, as in the window kernel.
//
// Measured (B200): 8192 rows of 20 heads over 20538 keys 1.89 ms, 911 TFLOP/s,
// under the power limit (1.61 ms, 1070 TFLOP/s, with pauses between the calls);
// 1024 rows over 9274 keys of 4 bits 0.163 ms, 597 TFLOP/s with the unpacking. A key block
// of both tiles takes about 3300 clocks where the MMAs alone need 2048 and the
// exponentials 2048: the softmax of a tile (2100-2300 clocks, half of it
// exponentials) and the MMAs behind it (1050) follow one another, and only two
// tiles fit TMEM to overlap them. Tried and slower: a quarter of the exponentials
// as polynomials on the FMA pipe, exponentials from the old maximum while the
// new one is looked for, half a row a thread on 16 warps, an epilogue of its own
// on 4 more warps.
#include "awa_cache_device.cuh"
#include "awa_rows.cuh"
#include "tcgen05.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <mutex>

namespace awa
{
namespace
{

using bf16 = __nv_bfloat16;

constexpr int kRows = 128;  // query rows of a tile
constexpr int kKeys = 128;  // keys of a block
constexpr int kSoftmaxWarps = 8;
constexpr int kMmaWarp = 8, kTmaWarp = 9, kCleanWarp = 10, kJobWarp = 11;
constexpr int kThreads = 384;  // 3 warpgroups; the last one gives registers to the softmax (a thread holds 128 scores)
constexpr int kSoftmaxRegs = 192, kOtherRegs = 120;  // 8 * 192 + 4 * 120 = 12 * 168 per lane
constexpr uint32_t kTmemColumns = 512;
constexpr uint32_t kColS = 0;    // + 128 * tile
constexpr uint32_t kColO = 256;  // + 128 * tile
constexpr uint64_t kWaitLimitNs = 4000000000ull;  // healthy waits last microseconds
constexpr uint64_t kDrainLimitNs = 200000000ull;
constexpr int kMostSequences = 16384;  // their sums lie in the ring before it is used

// What a job's rows see, which blocks of keys each tile takes part in, and the
// share of them that this thread block has.
struct Job
{
    QueryTile t;  // b = -1: no more jobs
    int kv;
    int rows_per_tile;  // batch rows of a tile
    bool has_b;
    RowSpan first[2], last[2];  // of tile A, B
    KeyBlocks blocks;           // of both
    int lo[2], hi[2], sinks;    // the Part of tile x
    int from, to;  // blocks [from, to) of `blocks`
    int slot;      // where the sums go; -1: the job is whole and goes to `out`
};

template <int D>
struct Tile
{
    static constexpr int kPanels = D / 64;            // of 64 features (128-byte rows, 128-byte swizzle)
    static constexpr int kPanelBytes = kKeys * 128;   // 16 KB
    static constexpr int kBytes = kPanels * kPanelBytes;
    static constexpr int kStages = D == 128 ? 5 : 10;  // of one K or V block: 160 KB, with Q 224 or 192 KB
    static constexpr int kLanded = 8;  // at least the V copies in the ring

    uint8_t q[2][kBytes];
    uint8_t ring[kStages][kBytes];
    uint64_t q_full, q_empty, full[kStages], empty[kStages], landed[kLanded];
    uint64_t s_full[2], p_full[2][2], o_full[2], o_empty[2], job_full[2], job_empty[2], mma_done;
    Job job[2];
    int64_t from, to;  // this block's share
    int64_t total;
    int dealt;  // blocks that have a share
    uint32_t tmem_base;
    int abort;
};

struct Maps
{
    CUtensorMap q, k, v;
};

// ---------------------------------------------------------------- waits and copies
// Codes of the waits: 70 and 73 to 92. 71 and 72 are AWA_CACHE_BAD_PAGE and AWA_CACHE_BAD_COORD.
static_assert(AWA_CACHE_BAD_PAGE == 71 && AWA_CACHE_BAD_COORD == 72, "the waits' codes stay clear of these");
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

// ---------------------------------------------------------------- the jobs
// The rows of sequence b.
struct Sequence
{
    int row0, rows, past, length;
};

__device__ __forceinline__ Sequence sequence_of(const CacheAttnArgs& a, int b, int* flag)
{
    Sequence s;
    s.row0 = __ldg(a.batch.row_starts + b);
    s.rows = batch_rows(a.batch, b);
    s.past = max(0, __ldg(a.batch.past + b));
    s.length = sequence_length(a.mem, a.batch, s.past, s.rows, flag);
    s.past = min(s.past, s.length);
    return s;
}

// Job t of a sequence has the rows [t * step, ...) of it; the key blocks they
// see, at least one (a job without any still writes its zeros).
__device__ __forceinline__ int job_blocks(const CacheAttnArgs& a, const Sequence& s, int t, int step)
{
    const int r0 = t * step, r1 = min(r0 + step, s.rows) - 1;
    const KeyBlocks k =
        key_blocks(row_span(s.past + r0, s.length, a.sinks, a.window, a.frame_tokens),
                   row_span(s.past + r1, s.length, a.sinks, a.window, a.frame_tokens), a.sinks, kKeys);
    return max(1, k.count);
}

constexpr int kJobCost = 3;  // 2: ragged prompts of 10 blocks a job 156 us for 152, long jobs 1% less

// The cost of all jobs of one head of a sequence. By one warp.
__device__ __forceinline__ int64_t sequence_cost(const CacheAttnArgs& a, const Sequence& s, int step)
{
    int64_t sum = 0;
    for (int t = threadIdx.x & 31; t * step < s.rows; t += 32)
        sum += job_blocks(a, s, t, step) + kJobCost;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum;
}

__device__ __forceinline__ Job make_job(const CacheAttnArgs& a, const Sequence& s, int b, int kv, int t, int step)
{
    Job job;
    job.kv = kv;
    job.rows_per_tile = step / 2;
    job.t.b = b;
    job.t.m0 = t * step * a.group;
    job.t.count = min(step, s.rows - t * step) * a.group;
    job.t.row0 = s.row0;
    job.t.past = s.past;
    job.t.length = s.length;
    const int m_tile = job.rows_per_tile * a.group;
    job.has_b = job.t.count > m_tile;
    const int p0 = s.past + t * step, rows = job.t.count / a.group;
    const auto span = [&](int p) { return row_span(p, s.length, a.sinks, a.window, a.frame_tokens); };
    job.first[0] = span(p0);
    job.last[0] = span(p0 + min(rows, job.rows_per_tile) - 1);
    job.first[1] = job.has_b ? span(p0 + job.rows_per_tile) : job.first[0];
    job.last[1] = job.has_b ? span(p0 + rows - 1) : job.last[0];
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

// The split of a cost of `total` over n thread blocks: c has [first_of(c), first_of(c + 1)).
__device__ __forceinline__ int64_t first_of(int64_t total, int n, int c)
{
    return total * c / n;
}

// A bound of a share as it falls on a job with the costs [first, first + cost):
// one inside the job goes to its nearer edge, if the job is at most an eighth of
// a share (parts and their join would cost more than the uneven shares).
__device__ __forceinline__ int64_t bound_on_job(int64_t bound, int64_t first, int cost, int64_t share)
{
    if (bound <= first || bound >= first + cost)
        return bound <= first ? first : first + cost;
    if (cost * 8 > share)
        return bound;
    return 2 * (bound - first) < cost ? first : first + cost;
}

// Parts of a job that several thread blocks work on, for the join: written by
// the one that begins it.
struct Joint
{
    QueryTile t;
    int kv;
    int parts;  // 0: nothing to join
};

// ---------------------------------------------------------------- job warp
// Walks over the thread block's share and hands the jobs to the other warps,
// two ahead at most. It begins at sequence b, before which there are costs of
// `before` and whose jobs cost `head` a head.
template <int D>
__device__ void job_role(const CacheAttnArgs& a, Tile<D>& sh, int b, int64_t before, int64_t head, Joint* joint)
{
    const int lane = threadIdx.x & 31;
    volatile int* abort = &sh.abort;
    const int step = 2 * (kRows / a.group);
    const int64_t from = sh.from, to = sh.to, share = sh.total / sh.dealt;
    Joint begun;
    begun.parts = 0;
    int n = 0;
    const auto hand_out = [&](const Job& job) {
        const bool ok = warp_wait(&sh.job_empty[n & 1], ((n >> 1) & 1) ^ 1, abort, a.error_flag, 77);
        if (lane == 0)
        {
            if (ok)
                sh.job[n & 1] = job;
            else
                sh.job[n & 1].t.b = -1;
            mbar_arrive(&sh.job_full[n & 1]);  // releases the writes
        }
        n++;
        return ok;
    };
    bool ok = true;
    for (; before < to && b < a.batch.sequences && ok; b++, head = 0)
    {
        const Sequence s = sequence_of(a, b, a.error_flag);
        if (s.rows == 0)
            continue;
        if (head == 0)
            head = sequence_cost(a, s, step);
        for (int kv = before < from ? (int)((from - before) / head) : 0; kv < a.mem.heads && ok; kv++)
        {
            int64_t at = before + kv * head;  // the cost ahead of the head's job t0
            if (at >= to)
                break;
            // a lane looks at one job of 32 at a time
            for (int t0 = 0; t0 * step < s.rows && at < to && ok; t0 += 32)
            {
                const int blocks = (t0 + lane) * step < s.rows ? job_blocks(a, s, t0 + lane, step) : 0;
                const int cost = blocks ? blocks + kJobCost : 0;
                int sum = cost;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1)
                {
                    const int up = __shfl_up_sync(0xffffffffu, sum, o);
                    if (lane >= o)
                        sum += up;
                }
                const int64_t first = at + sum - cost;
                // the job's blocks that are ours: [lo, hi)
                const int lo =
                    (int)max((int64_t)0, min((int64_t)blocks, bound_on_job(from, first, cost, share) - first - kJobCost));
                const int hi =
                    (int)max((int64_t)0, min((int64_t)blocks, bound_on_job(to, first, cost, share) - first - kJobCost));
                unsigned ours = __ballot_sync(0xffffffffu, lo < hi);
                for (; ours && ok; ours &= ours - 1)
                {
                    const int which = __ffs(ours) - 1;
                    const int all = __shfl_sync(0xffffffffu, blocks, which);
                    const int begin = __shfl_sync(0xffffffffu, lo, which), end = __shfl_sync(0xffffffffu, hi, which);
                    Job job = make_job(a, s, b, kv, t0 + which, step);
                    job.from = begin;
                    job.to = min(end, job.blocks.count);
                    job.slot = begin == 0 && end == all ? -1 : 2 * (int)blockIdx.x + (begin == 0 ? 1 : 0);
                    if (job.slot >= 0 && begin == 0)
                    {
                        begun.t = job.t;
                        begun.kv = kv;
                        // the thread block that has the job's last block: the largest c with first_of(c) <= it
                        const int64_t behind = __shfl_sync(0xffffffffu, first, which) + kJobCost + all;
                        begun.parts = (int)((behind * sh.dealt - 1) / sh.total) - (int)blockIdx.x + 1;
                    }
                    ok = hand_out(job);
                }
                at += __shfl_sync(0xffffffffu, sum, 31);
            }
        }
        before += head * a.mem.heads;
    }
    Job none;
    none.t.b = -1;
    if (ok)
        hand_out(none);
    if (lane == 0)
        joint[blockIdx.x] = begun;
}

// Block i of the job's is block number ... of the sequence.
__device__ __forceinline__ int block_of(const KeyBlocks& blocks, int i)
{
    return i < blocks.prefix ? i : i + blocks.shift;
}

// The blocks b of the sequence of which some row of a tile sees a key.
struct Part
{
    int lo, hi, sinks;
    __device__ __forceinline__ bool takes(int b) const
    {
        return b < hi && (b >= lo || b < sinks);
    }
};

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
__device__ void tma_role(const CacheAttnArgs& a, const Maps& maps, Tile<D>& sh)
{
    using T = Tile<D>;
    const int lane = threadIdx.x & 31;
    volatile int* abort = &sh.abort;
    // lanes = (piece of a page, panel) of a block
    const int piece = min(kKeys, 1 << a.mem.page_shift);
    const int pieces = kKeys / piece;
    const int mine = lane / T::kPanels, panel = lane % T::kPanels;
    int n = 0;       // copies issued
    int ragged = 0;  // of them through the clean-up warp
    int q_issued = 0;
    bool ok = true;
    for (int jobs = 0;; jobs++)
    {
        if (!warp_wait(&sh.job_full[jobs & 1], (jobs >> 1) & 1, abort, a.error_flag, 70))
            break;
        const Job& job = sh.job[jobs & 1];
        if (job.t.b < 0)
            break;
        const int tiles = job.has_b ? 2 : 1;
        const auto load_q = [&]() {
            if (!warp_wait(&sh.q_empty, (jobs & 1) ^ 1, abort, a.error_flag, 73))
                return false;
            if (lane == 0)
                mbar_expect(&sh.q_full, (uint32_t)(tiles * T::kPanels * job.rows_per_tile * a.group * 128));
            __syncwarp();
            if (lane < tiles * T::kPanels)
            {
                const int x = lane / T::kPanels;
                tma_load_3d(tc::smem_addr(sh.q[x] + panel * T::kPanelBytes), &maps.q, 64 * panel, job.kv * a.group,
                            job.t.row0 + job.t.m0 / a.group + x * job.rows_per_tile, &sh.q_full);
            }
            q_issued++;
            return true;
        };
        if (job.from >= job.to)
            ok = load_q();
        const int* table = a.batch.page_table + job.t.b * a.batch.table_stride;
        const auto lookup = [&](int i) {
            int page = a.mem.pages;  // past the last: the load brings zeros
            const int key = block_of(job.blocks, i) * kKeys + mine * piece;
            if (i < job.to && mine < pieces && key < job.last[1].hi && (key + piece > job.first[0].lo || key < a.sinks))
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
        int next = lookup(job.from);
        for (int i = job.from; i < job.to && ok; i++)
        {
            const int page = next;
            next = lookup(i + 1);
            const int block = block_of(job.blocks, i);
            const int slot = (block * kKeys + mine * piece) & ((1 << a.mem.page_shift) - 1);
#pragma unroll
            for (int v = 0; v < 2; v++, n++)
            {
                const int stage = n % T::kStages;
                ok = warp_wait(&sh.empty[stage], ((n / T::kStages) & 1) ^ 1, abort, a.error_flag, 73);
                if (!ok)
                    break;
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
                // Q behind the first keys: its place may still be in use by the job before
                if (v == 0 && i == job.from && !load_q())
                {
                    ok = false;
                    n++;
                    break;
                }
            }
        }
        if (!ok)
            break;
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&sh.job_empty[jobs & 1]);
    }
    // The copies in flight: the last use of each barrier.
    if (q_issued > 0)
        drain_bar(&sh.q_full, (q_issued - 1) & 1, a.error_flag, 74);
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
__device__ void clean_role(const CacheAttnArgs& a, Tile<D>& sh)
{
    using T = Tile<D>;
    const int lane = threadIdx.x & 31;
    volatile int* abort = &sh.abort;
    int n = 0;  // key blocks of the jobs before
    int ragged = 0;
    for (int jobs = 0;; jobs++)
    {
        if (!warp_wait(&sh.job_full[jobs & 1], (jobs >> 1) & 1, abort, a.error_flag, 79))
            return;
        const Job& job = sh.job[jobs & 1];
        if (job.t.b < 0)
            return;
        for (int i = job.from; i < job.to; i++, n++)
        {
            const int block = block_of(job.blocks, i);
            if (all_seen(a, job, block))
                continue;
            const bool ok =
                warp_wait(&sh.landed[ragged % T::kLanded], (ragged / T::kLanded) & 1, abort, a.error_flag, 76);
            ragged++;
            const int stage = (2 * n + 1) % T::kStages;
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
        __syncwarp();
        if (lane == 0)
            mbar_arrive(&sh.job_empty[jobs & 1]);
    }
}

// ---------------------------------------------------------------- MMA warp
// The warp runs the role together and one lane issues: what the instructions
// take (descriptors, addresses) is then uniform and stays in uniform registers.
// With a single thread in the role each MMA took some 80 cycles to issue, longer
// than the 64 it runs.
__device__ __forceinline__ uint32_t elect_one()
{
    uint32_t leader;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(leader));
    return leader;
}

template <bool ACCUMULATE>
__device__ __forceinline__ void mma_ss(uint32_t leader, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc)
{
    asm volatile(
        "{\n\t.reg .pred p, l;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 l, %5, 0;\n\t"
        "@l tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "n"(ACCUMULATE ? 1 : 0), "r"(leader)
        : "memory");
}

__device__ __forceinline__ void mma_ts(uint32_t leader, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                       uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p, l;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "setp.ne.b32 l, %5, 0;\n\t"
        "@l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader)
        : "memory");
}

__device__ __forceinline__ void commit(uint32_t leader, uint64_t* bar)
{
    asm volatile(
        "{\n\t.reg .pred l;\n\t"
        "setp.ne.b32 l, %1, 0;\n\t"
        "@l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(tc::smem_addr(bar)),
        "r"(leader)
        : "memory");
}

// Instruction descriptor: bf16 operands, or fp16 (Q, K, P and V alike) for what
// was unpacked from 4 bits.
template <bool HALF>
__device__ __forceinline__ uint32_t operands(int n, bool b_mn_major)
{
    return tc::idesc_bf16_f32(128, n, b_mn_major) & (HALF ? ~((1u << 7) | (1u << 10)) : ~0u);
}

// S[128 x 128] = Q K^T, both K-major in panels of 64 features.
template <int D, bool HALF>
__device__ __forceinline__ void issue_qk(uint32_t leader, uint32_t tmem_s, uint32_t q_addr, uint32_t k_addr)
{
    const uint32_t idesc = operands<HALF>(kKeys, false);
    const uint64_t q = tc::smem_desc_sw128(q_addr, 16, 1024), k = tc::smem_desc_sw128(k_addr, 16, 1024);
#pragma unroll
    for (int s = 0; s < D / 16; s++)
    {
        const uint64_t step = (uint64_t)((s >> 2) * (Tile<D>::kPanelBytes >> 4) + (s & 3) * 2);
        if (s == 0)
            mma_ss<false>(leader, tmem_s, q, k, idesc);
        else
            mma_ss<true>(leader, tmem_s, q + step, k + step, idesc);
    }
}

// O[128 x D] (+)= P[128 x 128] V[128 x D], P in TMEM, V MN-major: 8-key groups
// 1024 bytes apart, panels of 64 features kPanelBytes apart. One half of the keys.
template <int D, bool HALF>
__device__ __forceinline__ void issue_pv(uint32_t leader, uint32_t tmem_o, uint32_t tmem_p, uint32_t v_addr,
                                         uint32_t accumulate, int half)
{
    const uint32_t idesc = operands<HALF>(D, true);
    const uint64_t v = tc::smem_desc_sw128(v_addr, Tile<D>::kPanelBytes, 1024);
#pragma unroll
    for (int s = half * kKeys / 32; s < (half + 1) * kKeys / 32; s++)
        mma_ts(leader, tmem_o, tmem_p + (uint32_t)(s * 8), v + (uint64_t)(s * (2048 >> 4)), idesc,
               s > 0 ? 1u : accumulate);
}

// A value that all lanes hold, in a form that the compiler knows to be uniform.
__device__ __forceinline__ int uniform(int x)
{
    return __shfl_sync(0xffffffffu, x, 0);
}

template <int D, bool HALF>
__device__ void mma_issue(const CacheAttnArgs& a, Tile<D>& sh, uint32_t tmem_any)
{
    using T = Tile<D>;
    volatile int* abort = &sh.abort;
    const uint32_t leader = elect_one();
    const uint32_t tmem = (uint32_t)uniform((int)tmem_any);
    uint32_t p_phase = 0;  // bit x: of tile x
    // copy 2n is K of the n-th key block, copy 2n + 1 its V
    int k_stage = 0, v_stage = T::kStages - 1;
    uint32_t k_phase = 0, v_phase = 1;
    const auto advance = [](int& stage, uint32_t& phase) {  // two copies on
        stage += 2;
        if (stage >= T::kStages)
        {
            stage -= T::kStages;
            phase ^= 1;
        }
    };
    const auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
        return warp_wait(bar, parity, abort, a.error_flag, code);
    };
    const uint32_t q0 = tc::smem_addr(sh.q[0]), ring = tc::smem_addr(sh.ring[0]);
    // What the role needs of a job; b = -1: there is none, -2: a wait gave up.
    struct Share
    {
        int b, from, to;
        KeyBlocks blocks;
        Part part[2];
    };
    const auto fetch = [&](int jobs) {
        Share s;
        s.b = -2;
        if (!wait(&sh.job_full[jobs & 1], (jobs >> 1) & 1, 80))
            return s;
        const Job& job = sh.job[jobs & 1];
        s.b = uniform(job.t.b);
        if (s.b < 0)
            return s;
        s.from = uniform(job.from);
        s.to = uniform(job.to);
        s.blocks.prefix = uniform(job.blocks.prefix);
        s.blocks.shift = uniform(job.blocks.shift);
        const int sinks = uniform(job.sinks);
#pragma unroll
        for (int x = 0; x < 2; x++)
            s.part[x] = {uniform(job.lo[x]), uniform(job.hi[x]), sinks};
        return s;
    };
    bool now[2] = {false, false};   // the tile takes part in the block whose P is next
    bool then[2] = {false, false};  // ... in the one whose S is next
    // S of the next block for tile x. The first call for a block waits for its
    // keys (and the first of a job, job_parity >= 0, for its queries).
    const auto scores = [&](int job_parity, int x, bool& here) {
        if (!here)
        {
            if (job_parity >= 0 && !wait(&sh.q_full, job_parity, 81))
                return false;
            if (!wait(&sh.full[k_stage], k_phase, 83))
                return false;
            here = true;
        }
        // S overwrites P of the block before: the MMAs of one thread execute in
        // issue order. The commit covers the P V before it too: the softmax may
        // scale O once the scores are in.
        if (then[x])
        {
            issue_qk<D, HALF>(leader, tmem + kColS + 128 * x, q0 + x * T::kBytes, ring + k_stage * T::kBytes);
            commit(leader, &sh.s_full[x]);
        }
        now[x] = then[x];
        return true;
    };
    const auto scores_done = [&](bool last_of_job) {
        commit(leader, &sh.empty[k_stage]);
        advance(k_stage, k_phase);
        if (last_of_job)
            commit(leader, &sh.q_empty);
    };
    Share job = fetch(0);
    bool primed = false;  // the scores of the job's first block have been issued
    for (int jobs = 0; job.b >= 0; jobs++)
    {
        Share next = job;
        if (job.from >= job.to)  // no keys at all
        {
#pragma unroll
            for (int x = 0; x < 2; x++)
            {
                if (!wait(&sh.o_empty[x], (jobs & 1) ^ 1, 86))
                    return;
                commit(leader, &sh.o_full[x]);
            }
            if (!wait(&sh.q_full, jobs & 1, 81))
                return;
            commit(leader, &sh.q_empty);
            next = fetch(jobs + 1);
        }
        else if (!primed)
        {
            bool here = false;
#pragma unroll
            for (int x = 0; x < 2; x++)
            {
                then[x] = job.part[x].takes(block_of(job.blocks, job.from));
                if (!scores(jobs & 1, x, here))
                    return;
            }
            scores_done(job.from + 1 == job.to);
        }
        primed = false;
        uint32_t started = 0;
        // step i: O += P V of block i, S of the block after it -- behind the last
        // one that of the next job
        for (int i = job.from; i < job.to; i++)
        {
            const bool last = i + 1 == job.to;
            bool more = true, last_scores = i + 2 == job.to;
            int job_parity = -1;
            if (last)
            {
                next = fetch(jobs + 1);
                more = primed = next.b >= 0 && next.from < next.to;
                last_scores = next.from + 1 == next.to;
                job_parity = (jobs + 1) & 1;
#pragma unroll
                for (int x = 0; x < 2; x++)
                    then[x] = more && next.part[x].takes(block_of(next.blocks, next.from));
            }
            else
#pragma unroll
                for (int x = 0; x < 2; x++)
                    then[x] = job.part[x].takes(block_of(job.blocks, i + 1));
            advance(v_stage, v_phase);
            if (!wait(&sh.full[v_stage], v_phase, 82))
                return;
            const uint32_t v_addr = ring + v_stage * T::kBytes;
            bool here = false;
#pragma unroll
            for (int x = 0; x < 2; x++)
            {
                // the epilogue of the job before has read O (waited for once a job, whoever takes part)
                if (i == job.from && !wait(&sh.o_empty[x], (jobs & 1) ^ 1, 86))
                    return;
                if (now[x])
                {
#pragma unroll
                    for (int h = 0; h < 2; h++)
                    {
                        if (!wait(&sh.p_full[x][h], (p_phase >> x) & 1, 84))
                            return;
                        tc::fence_after_sync();
                        issue_pv<D, HALF>(leader, tmem + kColO + 128 * x, tmem + kColS + 128 * x, v_addr, (started >> x) & 1,
                                    h);
                    }
                    p_phase ^= 1u << x;
                    started |= 1u << x;
                }
                if (last)
                    commit(leader, &sh.o_full[x]);
                if (more && !scores(job_parity, x, here))
                    return;
            }
            commit(leader, &sh.empty[v_stage]);
            if (more)
                scores_done(last_scores);
        }
        if (leader)
            mbar_arrive(&sh.job_empty[jobs & 1]);
        __syncwarp();
        job = next;
    }
}

template <int D, bool HALF>
__device__ void mma_role(const CacheAttnArgs& a, Tile<D>& sh, uint32_t tmem)
{
    mma_issue<D, HALF>(a, sh, tmem);
    commit(elect_one(), &sh.mma_done);
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

// 32-byte global store (sm_100): eight 32-bit words at a 32-byte aligned address.
__device__ __forceinline__ void st_global_v8(void* p, const uint32_t (&r)[8])
{
    asm volatile("st.global.L1::no_allocate.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]),
                 "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

template <bool HALF>
__device__ __forceinline__ uint32_t operand_pair(float lo, float hi)
{
    if (!HALF)
        return pack_bf16x2(lo, hi);
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// part_o, part_ml: the sums of unfinished jobs, [slot][tile][row] of D features
// and (maximum, sum).
template <int D, bool HALF>
__device__ void softmax_role(const CacheAttnArgs& a, Tile<D>& sh, uint32_t tmem, float* part_o, float2* part_ml)
{
    const int warp = threadIdx.x >> 5;
    const int x = warp >> 2;
    const int r = threadIdx.x & 127;  // row of the tile = TMEM lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + kColS + 128 * x + lane_base;
    const uint32_t t_o = tmem + kColO + 128 * x + lane_base;
    float scale_log2 = a.scale * 1.4426950408889634f;
    volatile int* abort = &sh.abort;
    // whole sectors at a time, where the rows are aligned to them
    const bool v8 = ((reinterpret_cast<uintptr_t>(a.out) | (uintptr_t)(a.out_stride * sizeof(bf16))) & 31) == 0;
    // fp16 ends at 2^-24: with the largest p at 2^7 to 2^15, what is below 2^-32 of
    // it is dropped instead of 2^-25 (bf16 has fp32's exponents)
    constexpr float kHeadroom = HALF ? 7.f : 0.f;
    uint32_t phase = 0;
    for (int jobs = 0;; jobs++)
    {
        if (!warp_wait(&sh.job_full[jobs & 1], (jobs >> 1) & 1, abort, a.error_flag, 90))
            return;
        const Job& job = sh.job[jobs & 1];
        if (job.t.b < 0)
            return;
        const int m_tile = job.rows_per_tile * a.group;
        const int m = job.t.m0 + x * m_tile + min(r, m_tile - 1);
        const bool mine = r < m_tile && x * m_tile + r < job.t.count;
        if (HALF)
            scale_log2 = mine ? __ldg(a.score_scale + (int64_t)(job.t.row0 + m / a.group) * (a.group * a.mem.heads) +
                                      job.kv * a.group + m % a.group)
                              : 1.f;
        const RowSpan span =
            row_span(job.t.past + m / a.group, job.t.length, a.sinks, a.window, a.frame_tokens);
        float m_run = -INFINITY;  // running maximum, in log2 units of the scaled scores, less kHeadroom
        float l_run = 0.f;
        bool any = false;
        const KeyBlocks blocks = job.blocks;
        const Part part = {job.lo[x], job.hi[x], job.sinks};
        const RowSpan first = job.first[x], last = job.last[x];
        const int to = job.to;
        for (int i = job.from; i < to; i++)
        {
            const int block = block_of(blocks, i), key0 = block * kKeys;
            if (!part.takes(block))
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
            const bool whole = key0 + kKeys <= first.hi && (key0 >= last.lo || key0 + kKeys <= a.sinks);
            if (!whole)
            {
                const int hi = span.hi - key0, lo = span.lo - key0, sinks = min(a.sinks, span.hi) - key0;
#pragma unroll
                for (int c = 0; c < 4; c++)
                {
                    const uint32_t bits = bit_range(lo - 32 * c, hi - 32 * c) | bit_range(0, sinks - 32 * c);
                    if (__all_sync(0xffffffffu, bits == ~0u))
                        continue;
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
            const float m_blk = max3(max3(top[0], top[1], top[2]), top[3], -INFINITY) * scale_log2 - kHeadroom;
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
                    pk[j] = operand_pair<HALF>(p0, p1);  // the operand type of P V; the sums keep fp32
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
        // Epilogue: O divided by the sums as bf16 or, of a job that other thread
        // blocks share, as it is.
        const int slot = job.slot, kv = job.kv;
        if (slot >= 0 && mine)
            part_ml[((int64_t)slot * 2 + x) * kRows + r] = make_float2(m_run, l_run);
        // a row that sees nothing (l = 0) gets zeros
        const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
        char* const row =
            reinterpret_cast<char*>(static_cast<bf16*>(a.out) + (int64_t)(job.t.row0 + m / a.group) * a.out_stride +
                                    (int64_t)(kv * a.group + m % a.group) * D);
        float* const sum = part_o + (((int64_t)slot * 2 + x) * kRows + r) * D;
        __syncwarp();
        if ((threadIdx.x & 31) == 0)
            mbar_arrive(&sh.job_empty[jobs & 1]);
        if (!warp_wait(&sh.o_full[x], jobs & 1, abort, a.error_flag, 92))
            return;
        tc::fence_after_sync();
        uint32_t o[D];
        if (any)
        {
#pragma unroll
            for (int c = 0; c < D / 32; c++)
                tc::tmem_ld32(t_o + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(&o[32 * c]));
            tc::tmem_wait_ld();
        }
        else  // O was never written
        {
#pragma unroll
            for (int j = 0; j < D; j++)
                o[j] = 0;
        }
        tc::fence_before_sync();
        mbar_arrive(&sh.o_empty[x]);
        if (!mine)
            continue;
        if (HALF)  // the power of two of the unpacked values
#pragma unroll
            for (int c = 0; c < D / 64; c++)
            {
                const float down = power_of_two(-half_shift(__ldg(a.ranges + (kv * (D / 64) + c) * 2 + 1)));
#pragma unroll
                for (int j = 64 * c; j < 64 * c + 64; j++)
                    o[j] = __float_as_uint(__uint_as_float(o[j]) * down);
            }
        if (slot >= 0)
        {
#pragma unroll
            for (int c = 0; c < D / 8; c++)
                st_global_v8(sum + 8 * c, *reinterpret_cast<uint32_t(*)[8]>(&o[8 * c]));
            continue;
        }
#pragma unroll
        for (int c = 0; c < D / 16; c++)
        {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; j++)
            {
                float o0, o1;
                mul_x2(o0, o1, __uint_as_float(o[16 * c + 2 * j]), __uint_as_float(o[16 * c + 2 * j + 1]), inv);
                w[j] = pack_bf16x2(o0, o1);
            }
            if (v8)
                st_global_v8(row + 32 * c, w);
            else
            {
                reinterpret_cast<uint4*>(row + 32 * c)[0] = make_uint4(w[0], w[1], w[2], w[3]);
                reinterpret_cast<uint4*>(row + 32 * c)[1] = make_uint4(w[4], w[5], w[6], w[7]);
            }
        }
    }
}

template <int D, bool HALF>
__global__ void __launch_bounds__(kThreads, 1)
    cache_attention_tile_kernel(const CacheAttnArgs a, const __grid_constant__ Maps maps, float* part_o,
                                float2* part_ml, Joint* joint)
{
    using T = Tile<D>;
    // 1024-byte alignment for the 128-byte swizzle atoms; there is no room to align
    // by hand, and without static shared memory the array starts at a multiple of it
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    T& sh = *reinterpret_cast<T*>(smem_raw);
    if (tc::smem_addr(smem_raw) & 1023)
    {
        if (threadIdx.x == 0)
            cache_error(a.error_flag, 78);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 32)
        for (const CUtensorMap* map : {&maps.q, &maps.k, &maps.v})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
    if (threadIdx.x == 0)
    {
        tc::mbar_init(&sh.q_full, 1);
        tc::mbar_init(&sh.q_empty, 1);
        for (int s = 0; s < T::kStages; s++)
        {
            tc::mbar_init(&sh.full[s], 1);
            tc::mbar_init(&sh.empty[s], 1);
        }
        for (int s = 0; s < T::kLanded; s++)
            tc::mbar_init(&sh.landed[s], 1);
        for (int x = 0; x < 2; x++)
        {
            tc::mbar_init(&sh.s_full[x], 1);
            tc::mbar_init(&sh.p_full[x][0], kRows);
            tc::mbar_init(&sh.p_full[x][1], kRows);
            tc::mbar_init(&sh.o_full[x], 1);
            tc::mbar_init(&sh.o_empty[x], kRows);
            tc::mbar_init(&sh.job_full[x], 1);
            tc::mbar_init(&sh.job_empty[x], kSoftmaxWarps + 3);  // all but the job warp's own
        }
        tc::mbar_init(&sh.mma_done, 1);
        tc::mbar_fence_init();
        sh.abort = 0;
    }
    // the work of every sequence: a warp each, the sums in the ring's place
    int64_t* sums = reinterpret_cast<int64_t*>(sh.ring);
    const int step = 2 * (kRows / a.group);
    for (int b = warp; b < a.batch.sequences; b += kThreads / 32)
    {
        const int64_t sum = sequence_cost(a, sequence_of(a, b, nullptr), step) * a.mem.heads;
        if (lane == 0)
            sums[b] = sum;
    }
    if (warp == kMmaWarp)
    {
        tc::tmem_alloc(&sh.tmem_base, kTmemColumns);
        tc::tmem_relinquish();
    }
    __syncthreads();
    // the job warp finds the block's share: it begins in sequence b0, behind costs of `before`
    int b0 = 0, searched = 0;
    int64_t before = 0, head = 0;
    if (warp == kJobWarp)
    {
        int64_t total = 0;
        for (int b = lane; b < a.batch.sequences; b += 32)
            total += sums[b];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            total += __shfl_xor_sync(0xffffffffu, total, o);
        // a job and 4 key blocks or more each: less would be spent on the parts
        const int dealt = (int)max((int64_t)1, min((int64_t)gridDim.x, total / (4 + kJobCost)));
        const int c = blockIdx.x;
        const int64_t from = c < dealt ? first_of(total, dealt, c) : 0, to = c < dealt ? first_of(total, dealt, c + 1) : 0;
        for (b0 = a.batch.sequences; b0 == a.batch.sequences && searched < a.batch.sequences; searched += 32)
        {
            int64_t sum = searched + lane < a.batch.sequences ? sums[searched + lane] : 0;
            const int64_t mine = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1)
            {
                const int64_t up = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o)
                    sum += up;
            }
            const unsigned holds = __ballot_sync(0xffffffffu, from < before + sum);
            const int64_t all = __shfl_sync(0xffffffffu, sum, 31);
            if (holds)
            {
                b0 = searched + __ffs(holds) - 1;
                head = sums[b0] / a.mem.heads;
                before += __shfl_sync(0xffffffffu, sum - mine, __ffs(holds) - 1);
            }
            else
                before += all;
        }
        if (lane == 0)
        {
            sh.from = from;
            sh.to = to;
            sh.total = total;
            sh.dealt = dealt;
        }
    }
    tc::fence_async_smem();  // the sums' reads come before the ring's first copies
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = sh.tmem_base;

    if (warp < kSoftmaxWarps)
    {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        softmax_role<D, HALF>(a, sh, tmem, part_o, part_ml);
    }
    else
    {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        if (warp == kMmaWarp)
            mma_role<D, HALF>(a, sh, tmem);
        else if (warp == kTmaWarp)
            tma_role<D>(a, maps, sh);
        else if (warp == kCleanWarp)
            clean_role<D>(a, sh);
        else
            job_role<D>(a, sh, b0, before, head, joint);
    }

    tc::fence_before_sync();
    __syncthreads();
    if (warp == kMmaWarp)
    {
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemColumns);
    }
}

// Joins the parts of the jobs that several thread blocks worked on: block x
// began one (or none), y takes kJoinRows of its rows.
constexpr int kJoinRows = 16, kJoinThreads = 256;

template <int D>
__global__ void __launch_bounds__(kJoinThreads)
    cache_attention_tile_join_kernel(const CacheAttnArgs a, const float* part_o, const float2* part_ml,
                                     const Joint* joint)
{
    // every block, before anything else: the grid must not end ahead of the tile kernel
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Joint j = joint[blockIdx.x];
    const int m_tile = kRows / a.group * a.group;
    const int f = 4 * (threadIdx.x % (D / 4));
    for (int i = threadIdx.x / (D / 4); j.parts > 0 && i < kJoinRows; i += kJoinThreads / (D / 4))
    {
        const int row = blockIdx.y * kJoinRows + i;
        if (row >= j.t.count)
            return;
        const int x = row / m_tile, r = row - x * m_tile;
        const auto part = [&](int k) {
            const int64_t slot = 2 * ((int64_t)blockIdx.x + k) + (k == 0 ? 1 : 0);
            return (slot * 2 + x) * kRows + r;
        };
        float top = -INFINITY;
        for (int k = 0; k < j.parts; k++)
            top = fmaxf(top, part_ml[part(k)].x);
        const float from = top == -INFINITY ? 0.f : top;
        float total = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int k = 0; k < j.parts; k++)
        {
            const float2 ml = part_ml[part(k)];
            const float4 y = *reinterpret_cast<const float4*>(part_o + part(k) * D + f);
            const float w = fast_exp2(ml.x - from);
            total = fmaf(ml.y, w, total);
            o.x = fmaf(y.x, w, o.x);
            o.y = fmaf(y.y, w, o.y);
            o.z = fmaf(y.z, w, o.z);
            o.w = fmaf(y.w, w, o.w);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        const int m = j.t.m0 + row;
        *reinterpret_cast<uint2*>(static_cast<bf16*>(a.out) + (int64_t)(j.t.row0 + m / a.group) * a.out_stride +
                                  (int64_t)(j.kv * a.group + m % a.group) * D + f) =
            make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv));
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

constexpr int kBlocks = 148;  // one per SM; more or fewer SMs change the time, not the result

// The workspace: sums, (maximum, sum)s, joints.
template <int D>
constexpr size_t workspace_bytes()
{
    return (size_t)2 * kBlocks * 2 * kRows * (D * sizeof(float) + sizeof(float2)) + kBlocks * sizeof(Joint);
}

static_assert(sizeof(Tile<128>) <= 232448 && sizeof(Tile<64>) <= 232448, "shared memory of a block");

template <int D, bool HALF>
int run(const CacheAttnArgs& a, void* workspace, cudaStream_t stream)
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
    float* part_o = static_cast<float*>(workspace);
    float2* part_ml = reinterpret_cast<float2*>(part_o + (size_t)2 * kBlocks * 2 * kRows * D);
    Joint* joint = reinterpret_cast<Joint*>(part_ml + (size_t)2 * kBlocks * 2 * kRows);
    cache_attention_tile_kernel<D, HALF>
        <<<kBlocks, kThreads, sizeof(Tile<D>), stream>>>(a, maps, part_o, part_ml, joint);
    const cudaError_t err = cudaGetLastError();
    if (err != cudaSuccess)
        return (int)err;
    // starts while the tile kernel runs and waits for its end on the device
    cudaLaunchConfig_t config = {};
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    config.stream = stream;
    config.gridDim = dim3(kBlocks, 2 * kRows / kJoinRows);
    config.blockDim = dim3(kJoinThreads);
    return (int)cudaLaunchKernelEx(&config, cache_attention_tile_join_kernel<D>, a, (const float*)part_o,
                                   (const float2*)part_ml, (const Joint*)joint);
}

template <int D, bool HALF>
cudaError_t prepare()
{
    return cudaFuncSetAttribute(cache_attention_tile_kernel<D, HALF>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                (int)sizeof(Tile<D>));
}

}  // namespace

size_t cache_attention_tile_workspace(int head_dim)
{
    return head_dim == 64 ? workspace_bytes<64>() : workspace_bytes<128>();
}

int cache_attention_tile_sequences()
{
    return kMostSequences;
}

int launch_cache_attention_tile(const CacheAttnArgs& a, bool half, void* workspace, cudaStream_t stream)
{
    ProfileScope scope("awa_cache_attention_tile", stream);
    if (a.mem.head_dim == 64)
        return half ? run<64, true>(a, workspace, stream) : run<64, false>(a, workspace, stream);
    return half ? run<128, true>(a, workspace, stream) : run<128, false>(a, workspace, stream);
}

int prepare_cache_attention_tile()
{
    for (cudaError_t (*set)() : {prepare<64, false>, prepare<64, true>, prepare<128, false>, prepare<128, true>})
    {
        const cudaError_t err = set();
        if (err != cudaSuccess)
            return (int)err;
    }
    return 0;
}

}  // namespace awa
