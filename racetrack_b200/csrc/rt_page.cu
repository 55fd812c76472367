// Upkeep of a paged cache: which pages a sequence holds, and the copies that follow from it.
//
// A cache is a set of page buffers [n_pages, page_size, row bytes] (latent rows, rope keys, index
// keys, ...) under ONE block table: table[s, m] is the page that holds positions [m * page_size, (m + 1)
// * page_size) of sequence s (-1: none), lens[s] its length, refs[p] the number of table entries that
// name page p (0: free). Full pages may be shared by several sequences; a partial last page has one
// owner, so rows are only ever written into pages that one sequence holds.
//
// All of it lives and changes on the device: no call reads anything back, so a decode step with its
// growth of the cache is one CUDA graph. What needs an order (which entry gets which page) is done by
// one block, with prefix sums over the list, so the result does not depend on timing: pages are handed
// out lowest number first, in the order of the list. Counts change by integer atomics, whose order
// does not show. These plans are chains of dependent loads and block barriers; the copies behind them run at
// memory speed. Measured on one B200 (rows of 1152 bytes, pages of 64): extension by 64 tokens 6 us, by 8192 12
// (their rows 5); fork of 512 sequences with tails plan 5, copies 7, commit 3; compaction of 16384 pages plan 12, the
// 428 MB of its moves 69 us, 6.15 TB/s.
//
// No counterpart in racetrack, whose caches are [batch, max_len, dim] tensors
// (racetrack/models/deepseek.py:735-736).
#include "rt_common.cuh"

namespace rt {
namespace page {

constexpr int kPlanThreads = 1024;
constexpr int kMaxSeqs = 32768;             // owners of a list's entries are resolved in shared memory
constexpr int kCopyThreads = 256;

struct Buffer {
    uint8_t* base;
    int64_t page_stride;                    // bytes
    int64_t page_bytes;                     // page_size * row_bytes
    int64_t row_bytes;
};
// Buffers travel as kernel arguments. A layer's cache has two to four of them; all layers' at once
// (RT_PAGE_MAX_BUFFERS) are 4 KB of arguments, which only the calls that need them pass on.
constexpr int kFewBuffers = 8;
template <int CAP>
struct Buffers {
    Buffer b[CAP];
    int n;
};
template <int CAP>
struct Rows {
    const uint8_t* base[CAP];
    int64_t stride[CAP];                    // bytes
};
using AllBuffers = Buffers<RT_PAGE_MAX_BUFFERS>;
using AllRows = Rows<RT_PAGE_MAX_BUFFERS>;

static Rows<kFewBuffers> few(const AllRows& all) {
    Rows<kFewBuffers> f;
    for (int i = 0; i < kFewBuffers; ++i) {
        f.base[i] = all.base[i];
        f.stride[i] = all.stride[i];
    }
    return f;
}
static Buffers<kFewBuffers> few(const AllBuffers& all) {
    Buffers<kFewBuffers> f;
    f.n = all.n;
    for (int i = 0; i < kFewBuffers; ++i) f.b[i] = all.b[i];
    return f;
}

// Exclusive prefix sum over the block (kPlanThreads threads); `total` is the sum of all.
__device__ __forceinline__ int block_exclusive(int v, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int w = warp_sums[lane];                // 32 warps
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const int before = warp > 0 ? __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0) : 0;
    __syncthreads();                        // warp_sums may be written again
    return before + x - v;
}

// found[r] = the r-th lowest page with refs == 0, r < want; returns how many of them there are.
__device__ int find_free(const int32_t* refs, int pages, int want, int32_t* found, int* warp_sums) {
    int have = 0;
    for (int p0 = 0; p0 < pages && have < want; p0 += 4 * kPlanThreads) {
        const int p = p0 + 4 * static_cast<int>(threadIdx.x);
        int free4 = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (p + i < pages && refs[p + i] == 0) free4 |= 1 << i;
        int total;
        int r = have + block_exclusive(__popc(free4), warp_sums, total);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (free4 >> i & 1) {
                if (r < want) found[r] = p + i;
                ++r;
            }
        have += total;
    }
    __syncthreads();
    return min(have, want);
}

// The largest i in [0, n) with a[i] <= x, or -1 (a ascending).
__device__ __forceinline__ int last_not_above(const int32_t* a, int n, int x) {
    int lo = -1, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }

struct ExtendArgs {
    int32_t* table;
    int64_t table_stride;
    int32_t* lens;
    int32_t* refs;
    int32_t* status;
    const int32_t* seqs;        // [n] or null: entry i is sequence i
    const int32_t* offsets;     // [n + 1] or null: one token an entry
    int32_t* slots;             // [tokens]
    int32_t* work;              // need prefix [n] | old length [n] | found pages
    int n_seqs, width, pages, page, n, tokens;
};

// Sequence, first token and tokens of entry i.
__device__ __forceinline__ void extend_entry(const ExtendArgs& a, int i, int& s, int& first, int& count) {
    s = a.seqs ? a.seqs[i] : i;
    first = a.offsets ? min(max(a.offsets[i], 0), a.tokens) : i;
    count = (a.offsets ? min(max(a.offsets[i + 1], first), a.tokens) : i + 1) - first;
}

// Row t of buffer k's rows into slot `slot`, by one warp.
template <int CAP>
__device__ __forceinline__ void write_row(const Buffers<CAP>& bufs, const Rows<CAP>& rows, int k, int64_t t, int slot,
                                          int page) {
    const int lane = threadIdx.x & 31;
    const Buffer& b = bufs.b[k];
    const uint8_t* src = rows.base[k] + t * rows.stride[k];
    uint8_t* dst = b.base + (slot / page) * b.page_stride + (slot % page) * b.row_bytes;
    if (b.row_bytes % 16 == 0 && rows.stride[k] % 16 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
        for (int64_t o = lane * 16; o < b.row_bytes; o += 512)
            *reinterpret_cast<uint4*>(dst + o) = ld_once16(src + o);
    } else {
        for (int64_t o = lane * 4; o < b.row_bytes; o += 128)
            *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(src + o);
    }
}

__device__ void extend(const ExtendArgs& a) {
    extern __shared__ int32_t owner[];       // [n_seqs]: the first entry that names the sequence
    __shared__ int warp_sums[32];
    int32_t* const cum = a.work;
    int32_t* const old_len = a.work + a.n;
    int32_t* const found = a.work + 2 * a.n;
    for (int s = threadIdx.x; s < a.n_seqs; s += kPlanThreads) owner[s] = 0x7fffffff;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
        const int s = a.seqs ? a.seqs[i] : i;
        if (s >= 0 && s < a.n_seqs) atomicMin(&owner[s], i);
    }
    __syncthreads();
    // pages that each entry needs, and where they begin among the pages found
    int total = 0, refused = 0;
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
        const int i = i0 + static_cast<int>(threadIdx.x);
        int need = 0, old = -1;
        if (i < a.n) {
            int s, first, count;
            extend_entry(a, i, s, first, count);
            if (s >= 0) {
                if (s < a.n_seqs && owner[s] == i) {
                    old = a.lens[s];
                    // in 64 bits: a length near the int's end plus the new tokens
                    if (old < 0 || static_cast<int64_t>(old) + count > static_cast<int64_t>(a.width) * a.page) old = -1;
                }
                if (old < 0) ++refused;
                else need = ceil_div(old + count, a.page) - ceil_div(old, a.page);
            }
        }
        int sum;
        const int before = total + block_exclusive(need, warp_sums, sum);
        if (i < a.n) {
            cum[i] = before;
            old_len[i] = old;
        }
        total += sum;
    }
    // (an entry needs no more pages than it has tokens; offsets that overlap could ask for more than
    // the workspace holds)
    const int got = total > 0 ? find_free(a.refs, a.pages, min(total, a.tokens), found, warp_sums) : 0;
    __syncthreads();
    // every entry whose pages were all found grows
    int lacking = 0;
    for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
        const int old = old_len[i];
        if (old < 0) continue;
        int s, first, count;
        extend_entry(a, i, s, first, count);
        const int have = ceil_div(old, a.page), need = ceil_div(old + count, a.page) - have;
        if (need > 0 && cum[i] + need > got) {
            old_len[i] = -1;
            ++refused;
            lacking += need;
        } else {
            a.lens[s] = old + count;
        }
    }
    __syncthreads();
    for (int r = threadIdx.x; r < got; r += kPlanThreads) {
        const int i = last_not_above(cum, a.n, r), old = old_len[i];
        if (old < 0) continue;
        int s, first, count;
        extend_entry(a, i, s, first, count);
        // (offsets that overlap can take the prefix sums past 31 bits: no entry takes more pages than it needs)
        const int have = ceil_div(old, a.page), k = r - cum[i];
        if (static_cast<unsigned>(k) >= static_cast<unsigned>(ceil_div(old + count, a.page) - have)) continue;
        a.table[s * a.table_stride + have + k] = found[r];
        a.refs[found[r]] = 1;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < a.tokens; t += kPlanThreads) {
        const int i = a.offsets ? last_not_above(a.offsets, a.n, t) : t;
        int slot = -1;
        if (i >= 0 && i < a.n && old_len[i] >= 0) {
            int s, first, count;
            extend_entry(a, i, s, first, count);
            const int pos = old_len[i] + (t - first);
            if (t >= first && t < first + count) {
                const int p = a.table[s * a.table_stride + pos / a.page];
                if (p >= 0 && p < a.pages) slot = p * a.page + pos % a.page;
            }
        }
        a.slots[t] = slot;
    }
    if (refused) atomicAdd(a.status, refused);
    if (lacking) atomicAdd(a.status + 1, lacking);
}

__global__ void __launch_bounds__(kPlanThreads) page_extend_kernel(const ExtendArgs a) { extend(a); }

// The same, and the rows of a decode step behind it: for few tokens a launch costs more than the blocks that it
// brings save (rows of 1152 bytes, calls in a row: 16 tokens 10.5 us in two launches, 7.4 in one; 64 10.9 and 10.2;
// 128 12.1 and 15.6).
constexpr int kAppendTokens = 64;
constexpr int64_t kAppendBytes = 80 << 10;
__global__ void __launch_bounds__(kPlanThreads) page_append_kernel(const ExtendArgs a,
                                                                   const __grid_constant__ Buffers<kFewBuffers> bufs,
                                                                   const __grid_constant__ Rows<kFewBuffers> rows) {
    extend(a);
    __syncthreads();
    for (int w = threadIdx.x >> 5; w < a.tokens * bufs.n; w += kPlanThreads / 32) {
        const int t = w / bufs.n, slot = a.slots[t];
        if (slot >= 0) write_row(bufs, rows, w - t * bufs.n, t, slot, a.page);
    }
}

// rows[b][t] -> row slots[t] of buffer b: one warp a row and buffer.
template <int CAP>
__global__ void __launch_bounds__(kCopyThreads) page_write_kernel(const __grid_constant__ Buffers<CAP> bufs,
                                                                  const __grid_constant__ Rows<CAP> rows,
                                                                  const int32_t* __restrict__ slots, int64_t tokens,
                                                                  int64_t pages, int page) {
    const int64_t warps = static_cast<int64_t>(gridDim.x) * (kCopyThreads / 32);
    for (int64_t w = blockIdx.x * static_cast<int64_t>(kCopyThreads / 32) + (threadIdx.x >> 5); w < tokens * bufs.n; w += warps) {
        const int64_t t = w / bufs.n;
        const int slot = __ldg(slots + t);
        if (slot >= 0 && slot < pages * page) write_row(bufs, rows, static_cast<int>(w - t * bufs.n), t, slot, page);
    }
}

__global__ void __launch_bounds__(kCopyThreads) page_free_kernel(int32_t* table, int64_t table_stride, int32_t* lens,
                                                                 int32_t* refs, const int32_t* seqs, int n_seqs,
                                                                 int width, int pages) {
    const int s = seqs[blockIdx.x];
    if (s < 0 || s >= n_seqs) return;
    // an entry is taken by exchange, so a sequence that is named twice gives its pages back once
    for (int m = blockIdx.y * kCopyThreads + threadIdx.x; m < width; m += gridDim.y * kCopyThreads) {
        int32_t* const e = table + s * table_stride + m;
        if (*e < 0) continue;
        const int p = atomicExch(e, -1);
        if (p >= 0 && p < pages) atomicSub(refs + p, 1);
    }
    if (blockIdx.y == 0 && threadIdx.x == 0) lens[s] = 0;
}

// ---- fork -------------------------------------------------------------------------------------
// dst[i] becomes a second holder of src[i]'s full pages and gets a copy of the used rows of its
// partial last page. All entries take effect at once (a sequence may be source of some and
// destination of one, as when the beams of a search change places), in three steps: the plan,
// which hands out the pages of the partial copies; the new rows of the table, staged, with the
// references they add and the copies; then the old rows' references go and the new rows come. Pages
// are therefore handed out before the destinations' old ones return, and no page that is still read is
// handed out.
struct ForkPlan {
    int32_t src, len, fresh, last;           // src -1: the entry does nothing
};
struct ForkArgs {
    int32_t* table;
    int64_t table_stride;
    int32_t* lens;
    int32_t* refs;
    int32_t* status;
    const int32_t* src;
    const int32_t* dst;
    ForkPlan* plan;              // [n]
    int32_t* staged;             // [n, width]
    int32_t* found;              // [n]
    int n_seqs, width, pages, page, n;
};

__device__ void fork_plan(const ForkArgs& a) {
    extern __shared__ int32_t owner[];
    __shared__ int warp_sums[32];
    for (int s = threadIdx.x; s < a.n_seqs; s += kPlanThreads) owner[s] = 0x7fffffff;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
        const int d = a.dst[i];
        if (d >= 0 && d < a.n_seqs && a.src[i] >= 0 && a.src[i] < a.n_seqs) atomicMin(&owner[d], i);
    }
    __syncthreads();
    int total = 0, refused = 0, lacking = 0;
    for (int i0 = 0; i0 < a.n; i0 += kPlanThreads) {
        const int i = i0 + static_cast<int>(threadIdx.x);
        ForkPlan p{-1, 0, -1, -1};
        int need = 0;
        if (i < a.n) {
            const int s = a.src[i], d = a.dst[i];
            if (s >= 0 && d >= 0) {
                const bool known = s < a.n_seqs && d < a.n_seqs;
                const int len = known ? a.lens[s] : -1;
                if (!known || owner[d] != i || len < 0 || len > static_cast<int64_t>(a.width) * a.page) {
                    ++refused;
                } else if (s != d) {
                    p.src = s;
                    p.len = len;
                    if (len % a.page) {
                        p.last = a.table[s * a.table_stride + len / a.page];
                        need = 1;
                    }
                }
            }
        }
        int sum;
        const int before = total + block_exclusive(need, warp_sums, sum);
        if (need) p.fresh = before;          // its rank among the pages found, for now
        if (i < a.n) a.plan[i] = p;
        total += sum;
    }
    const int got = total > 0 ? find_free(a.refs, a.pages, total, a.found, warp_sums) : 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.n; i += kPlanThreads) {
        const int rank = a.plan[i].fresh;
        if (rank < 0) continue;
        if (rank < got) {
            a.plan[i].fresh = a.found[rank];
            a.refs[a.found[rank]] = 1;
        } else {
            a.plan[i].src = -1;
            ++refused;
            ++lacking;
        }
    }
    if (refused) atomicAdd(a.status, refused);
    if (lacking) atomicAdd(a.status + 1, lacking);
}

// Entry i's new row of the table, the references it adds, and its copies: thread t0 of `step`.
template <int CAP>
__device__ __forceinline__ void fork_stage(const ForkArgs& a, const Buffers<CAP>& bufs, int i, int t0, int step) {
    const ForkPlan p = a.plan[i];
    if (p.src < 0) return;
    const int full = p.len / a.page, tail = p.len % a.page;
    for (int m = t0; m < a.width; m += step) {
        int e = -1;
        if (m < full) {
            e = a.table[p.src * a.table_stride + m];
            if (e >= 0 && e < a.pages) atomicAdd(a.refs + e, 1);
        } else if (m == full && tail) {
            e = p.fresh;
        }
        a.staged[static_cast<int64_t>(i) * a.width + m] = e;
    }
    if (tail == 0 || p.last < 0 || p.last >= a.pages) return;
    for (int k = 0; k < bufs.n; ++k) {
        const Buffer& b = bufs.b[k];
        const uint8_t* src = b.base + p.last * b.page_stride;
        uint8_t* dst = b.base + p.fresh * b.page_stride;
        const int64_t bytes = tail * b.row_bytes, whole = bytes / 16 * 16;
        for (int64_t o = t0 * 16ll; o < whole; o += step * 64ll) {       // four loads under way (512 forks: 7.0 us, one 7.9)
            uint4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (o + i * step * 16ll < whole) v[i] = ld_once16(src + o + i * step * 16ll);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (o + i * step * 16ll < whole) *reinterpret_cast<uint4*>(dst + o + i * step * 16ll) = v[i];
        }
        for (int64_t o = whole + t0 * 4ll; o < bytes; o += step * 4ll)
            *reinterpret_cast<uint32_t*>(dst + o) = *reinterpret_cast<const uint32_t*>(src + o);
    }
}

// The old row's references go, the new one comes.
__device__ __forceinline__ void fork_commit(const ForkArgs& a, int i, int t0, int step) {
    const ForkPlan p = a.plan[i];
    if (p.src < 0) return;
    const int d = a.dst[i];
    for (int m = t0; m < a.width; m += step) {
        int32_t* const e = a.table + d * a.table_stride + m;
        const int old = *e;
        if (old >= 0 && old < a.pages) atomicSub(a.refs + old, 1);
        *e = a.staged[static_cast<int64_t>(i) * a.width + m];
    }
    if (t0 == 0) a.lens[d] = p.len;
}

__global__ void __launch_bounds__(kPlanThreads) page_fork_plan_kernel(const ForkArgs a) { fork_plan(a); }

// blockIdx.x: entry; blockIdx.y: part of its row of the table, and of its copies.
template <int CAP>
__global__ void __launch_bounds__(kCopyThreads) page_fork_stage_kernel(const ForkArgs a,
                                                                       const __grid_constant__ Buffers<CAP> bufs) {
    fork_stage(a, bufs, blockIdx.x, blockIdx.y * kCopyThreads + threadIdx.x, gridDim.y * kCopyThreads);
}
__global__ void __launch_bounds__(kCopyThreads) page_fork_commit_kernel(const ForkArgs a) {
    fork_commit(a, blockIdx.x, blockIdx.y * kCopyThreads + threadIdx.x, gridDim.y * kCopyThreads);
}

// All three in one block, for few entries and small pages (pages of 64 rows of 1152 bytes, calls in a row: 14.4 us in
// three launches whatever the tail; in one 8.2 for one entry, 10.3 to 13.6 for 4 with tails of 28 and 63 rows, 12.7 to
// 19.0 for 8).
constexpr int kForkEntries = 4;
constexpr int64_t kForkBytes = 320 << 10;
__global__ void __launch_bounds__(kPlanThreads) page_fork_kernel(const ForkArgs a,
                                                                 const __grid_constant__ Buffers<kFewBuffers> bufs) {
    fork_plan(a);
    __syncthreads();
    const int share = kPlanThreads / a.n, i = threadIdx.x / share, t0 = threadIdx.x % share;
    if (i < a.n) fork_stage(a, bufs, i, t0, share);
    __syncthreads();
    if (i < a.n) fork_commit(a, i, t0, share);
}

// ---- compact and copy ---------------------------------------------------------------------------
// The live pages come to lie in [0, live): the k-th lowest live page outside that range moves into the
// k-th lowest free one inside it. moves[k] = {from, to}; rank[p] = k for page p >= live (-1: not in
// use); head = {live, number of moves}.
__global__ void __launch_bounds__(kPlanThreads) page_compact_plan_kernel(const int32_t* refs, int pages, int32_t* head,
                                                                         int2* moves, int32_t* rank) {
    __shared__ int warp_sums[32];
    // a warp takes consecutive pages, a lane one of 32, so ranks come from ballots and neighbours write to
    // neighbouring places
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int share = ((pages + kPlanThreads - 1) / kPlanThreads) * 32;
    const int p0 = min(warp * share, pages), p1 = min(p0 + share, pages);
    auto used32 = [&](int p) { return __ballot_sync(0xffffffffu, p + lane < p1 && refs[p + lane] > 0); };
    int mine = 0, live;
#pragma unroll 8
    for (int p = p0; p < p1; p += 32) mine += __popc(used32(p));
    block_exclusive(lane == 0 ? mine : 0, warp_sums, live);
    // live pages outside the range, free pages inside it
    auto below = [&](int p) { return p >= live ? 0u : live - p >= 32 ? ~0u : (1u << (live - p)) - 1; };
    auto there = [&](int p) { return p1 - p >= 32 ? ~0u : (1u << (p1 - p)) - 1; };
    int outs = 0, ins = 0;
#pragma unroll 8
    for (int p = p0; p < p1; p += 32) {
        const uint32_t used = used32(p);
        outs += __popc(used & ~below(p));
        ins += __popc(~used & below(p) & there(p));
    }
    int out, in;
    int ko = block_exclusive(lane == 0 ? outs : 0, warp_sums, out), ki = block_exclusive(lane == 0 ? ins : 0, warp_sums, in);
    ko = __shfl_sync(0xffffffffu, ko, 0);
    ki = __shfl_sync(0xffffffffu, ki, 0);
    const uint32_t before = (1u << lane) - 1;
#pragma unroll 4
    for (int p = p0; p < p1; p += 32) {
        const uint32_t used = used32(p), o = used & ~below(p), h = ~used & below(p) & there(p);
        if (o >> lane & 1) moves[ko + __popc(o & before)].x = p + lane;
        if (h >> lane & 1) moves[ki + __popc(h & before)].y = p + lane;
        if (p + lane >= live && p + lane < p1) rank[p + lane] = (o >> lane & 1) ? ko + __popc(o & before) : -1;
        ko += __popc(o);
        ki += __popc(h);
    }
    if (threadIdx.x == 0) {
        head[0] = live;
        head[1] = out;
    }
}

// Copies page from[k] to page to[k] of every buffer, in pieces of kPiece bytes: with `moves` the pairs
// of a compaction (their number on the device), else the lists of a copy. A compaction's table entries
// and counts are rewritten on the way. What bounds it is memory: four 16-byte loads in flight a
// thread, eight blocks an SM.
constexpr int kPiece = kCopyThreads * 16 * 4;
struct MoveArgs {
    const int2* moves;
    const int32_t* head;
    const int32_t* from;
    const int32_t* to;
    int n;
    int32_t* table;              // compaction only
    int64_t table_stride;
    int32_t* refs;
    const int32_t* rank;
    int n_seqs, width, pages;
    int64_t pieces;              // of one page over all buffers
};

template <int CAP>
__global__ void __launch_bounds__(kCopyThreads) page_move_kernel(const MoveArgs a, const __grid_constant__ Buffers<CAP> bufs) {
    const int n = a.moves ? a.head[1] : a.n;
    if (a.moves) {
        const int64_t step = static_cast<int64_t>(gridDim.x) * kCopyThreads;
        const int64_t t0 = blockIdx.x * static_cast<int64_t>(kCopyThreads) + threadIdx.x;
        const int live = a.head[0];
        if (n > 0)
            for (int64_t j = t0; j < static_cast<int64_t>(a.n_seqs) * a.width; j += step) {
                int32_t* const e = a.table + (j / a.width) * a.table_stride + j % a.width;
                const int p = *e;
                if (p >= live && p < a.pages) {
                    const int k = a.rank[p];
                    if (k >= 0) *e = a.moves[k].y;
                }
            }
        for (int64_t k = t0; k < n; k += step) {
            const int2 m = a.moves[k];
            a.refs[m.y] = a.refs[m.x];
            a.refs[m.x] = 0;
        }
    }
    for (int64_t u = blockIdx.x; u < n * a.pieces; u += gridDim.x) {
        const int64_t k = u / a.pieces;
        int64_t piece = u - k * a.pieces;
        const int from = a.moves ? a.moves[k].x : a.from[k], to = a.moves ? a.moves[k].y : a.to[k];
        if (from < 0 || from >= a.pages || to < 0 || to >= a.pages || from == to) continue;
        int b = 0;
        for (; b < bufs.n; ++b) {
            const int64_t mine = (bufs.b[b].page_bytes + kPiece - 1) / kPiece;
            if (piece < mine) break;
            piece -= mine;
        }
        const Buffer& f = bufs.b[b];
        const uint8_t* src = f.base + from * f.page_stride;
        uint8_t* dst = f.base + to * f.page_stride;
        const int64_t o = piece * kPiece + threadIdx.x * 16;
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i * (kCopyThreads * 16) < f.page_bytes) v[i] = ld_once16(src + o + i * (kCopyThreads * 16));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (o + i * (kCopyThreads * 16) < f.page_bytes) st_stream16(dst + o + i * (kCopyThreads * 16), v[i]);
    }
}

static int sms() {
    int dev = 0, n = 148;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) {
        cudaGetLastError();
        n = 148;
    }
    return n;
}

static int check_table(const char* who, const void* table, const void* lens, const void* refs, int64_t table_stride,
                       int64_t n_seqs, int64_t width, int64_t pages, int64_t page) {
    RT_REQUIRE(n_seqs >= 0 && width >= 0 && pages >= 0 && page > 0, RT_ERR_BAD_ARG, "%s: bad shape", who);
    RT_REQUIRE(n_seqs <= kMaxSeqs, RT_ERR_UNSUPPORTED, "%s: at most %d sequences", who, kMaxSeqs);
    RT_REQUIRE(pages * page < (1ll << 31) && width * page < (1ll << 31) && width < (1ll << 24), RT_ERR_UNSUPPORTED,
               "%s: positions of the pool and of a sequence must fit 31 bits", who);
    RT_REQUIRE(table_stride >= width, RT_ERR_BAD_ARG, "%s: table rows overlap", who);
    RT_REQUIRE((n_seqs * width == 0 || table) && (n_seqs == 0 || lens) && (pages == 0 || refs), RT_ERR_BAD_ARG,
               "%s: null pointer", who);
    return RT_OK;
}

static int fill_buffers(const char* who, AllBuffers* out, void* const* bases, const int64_t* page_strides,
                        const int64_t* row_bytes, int64_t n, int64_t page) {
    RT_REQUIRE(n >= 0 && n <= RT_PAGE_MAX_BUFFERS, RT_ERR_UNSUPPORTED, "%s: at most %d page buffers", who, RT_PAGE_MAX_BUFFERS);
    RT_REQUIRE(n == 0 || (bases && page_strides && row_bytes), RT_ERR_BAD_ARG, "%s: null pointer", who);
    out->n = static_cast<int>(n);
    for (int64_t i = 0; i < n; ++i) {
        Buffer& b = out->b[i];
        b.base = static_cast<uint8_t*>(bases[i]);
        b.page_stride = page_strides[i];
        b.row_bytes = row_bytes[i];
        b.page_bytes = row_bytes[i] * page;
        RT_REQUIRE(b.base && aligned16(b.base), RT_ERR_BAD_ARG, "%s: page buffers must be 16-byte aligned", who);
        RT_REQUIRE(b.row_bytes > 0 && b.row_bytes % 4 == 0 && b.page_bytes % 16 == 0 && b.page_stride % 16 == 0 &&
                       b.page_stride >= b.page_bytes,
                   RT_ERR_BAD_ARG, "%s: rows must be multiples of 4 bytes, pages and their stride multiples of 16", who);
    }
    return RT_OK;
}

static int fill_rows(const char* who, AllRows* out, const void* const* rows, const int64_t* row_strides, int64_t n) {
    RT_REQUIRE(rows && row_strides, RT_ERR_BAD_ARG, "%s: null pointer", who);
    for (int64_t i = 0; i < n; ++i) {
        RT_REQUIRE(rows[i] && (reinterpret_cast<uintptr_t>(rows[i]) & 3) == 0 && row_strides[i] % 4 == 0 && row_strides[i] >= 0,
                   RT_ERR_BAD_ARG, "%s: rows must be 4-byte aligned", who);
        out->base[i] = static_cast<const uint8_t*>(rows[i]);
        out->stride[i] = row_strides[i];
    }
    return RT_OK;
}

}  // namespace page
}  // namespace rt

using namespace rt;

extern "C" int64_t rt_page_extend_workspace_ints(int64_t n, int64_t tokens) { return 2 * n + tokens; }

// The arguments of an extension, checked.
static int extend_args(const char* who, page::ExtendArgs* a, int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int32_t* status,
                       const int32_t* seqs, const int32_t* offsets, int32_t* slots, int32_t* workspace, int64_t n_seqs,
                       int64_t width, int64_t pages, int64_t page_size, int64_t n, int64_t tokens) {
    if (int rc = page::check_table(who, table, lens, refs, table_stride, n_seqs, width, pages, page_size))
        return rc;
    RT_REQUIRE(n >= 0 && tokens >= 0 && n < (1ll << 30) && tokens < (1ll << 30), RT_ERR_BAD_ARG, "%s: bad list", who);
    RT_REQUIRE(offsets || tokens == n, RT_ERR_BAD_ARG, "%s: without offsets every entry brings one token", who);
    RT_REQUIRE(seqs || n <= n_seqs, RT_ERR_BAD_ARG, "%s: more entries than sequences", who);
    RT_REQUIRE((n == 0 && tokens == 0) || (status && workspace && (tokens == 0 || slots)), RT_ERR_BAD_ARG, "%s: null pointer", who);
    *a = page::ExtendArgs{table, table_stride, lens, refs, status, seqs, offsets, slots, workspace,
                          static_cast<int>(n_seqs), static_cast<int>(width), static_cast<int>(pages),
                          static_cast<int>(page_size), static_cast<int>(n), static_cast<int>(tokens)};
    return RT_OK;
}

extern "C" int rt_page_extend(int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int32_t* status,
                              const int32_t* seqs, const int32_t* offsets, int32_t* slots, int32_t* workspace,
                              int64_t n_seqs, int64_t width, int64_t pages, int64_t page_size, int64_t n, int64_t tokens,
                              void* stream) {
    page::ExtendArgs a;
    if (int rc = extend_args("rt_page_extend", &a, table, table_stride, lens, refs, status, seqs, offsets, slots, workspace,
                             n_seqs, width, pages, page_size, n, tokens))
        return rc;
    if (n == 0 && tokens == 0) return RT_OK;
    const int smem = static_cast<int>(n_seqs * 4);
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&page::page_extend_kernel), smem, "rt_page_extend"))
        return rc;
    page::page_extend_kernel<<<1, page::kPlanThreads, smem, as_stream(stream)>>>(a);
    count_launch();
    return check_launch("page_extend_kernel");
}

extern "C" int rt_page_write(void* const* bases, const int64_t* page_strides, const int64_t* row_bytes,
                             const void* const* rows, const int64_t* row_strides, int64_t n_buffers,
                             const int32_t* slots, int64_t tokens, int64_t pages, int64_t page_size, void* stream) {
    RT_REQUIRE(tokens >= 0 && pages >= 0 && page_size > 0 && pages * page_size < (1ll << 31), RT_ERR_BAD_ARG,
               "rt_page_write: bad shape");
    page::AllBuffers bufs{};
    page::AllRows r{};
    if (tokens == 0 || pages == 0 || n_buffers == 0) return RT_OK;
    if (int rc = page::fill_buffers("rt_page_write", &bufs, bases, page_strides, row_bytes, n_buffers, page_size)) return rc;
    RT_REQUIRE(slots, RT_ERR_BAD_ARG, "rt_page_write: null pointer");
    if (int rc = page::fill_rows("rt_page_write", &r, rows, row_strides, n_buffers)) return rc;
    const int64_t blocks = (tokens * n_buffers + page::kCopyThreads / 32 - 1) / (page::kCopyThreads / 32);
    const int64_t most = 8ll * page::sms();
    const unsigned grid = static_cast<unsigned>(blocks < most ? blocks : most);
    if (n_buffers <= page::kFewBuffers) {
        page::page_write_kernel<<<grid, page::kCopyThreads, 0, as_stream(stream)>>>(
            page::few(bufs), page::few(r), slots, tokens, pages, static_cast<int>(page_size));
    } else {
        page::page_write_kernel<<<grid, page::kCopyThreads, 0, as_stream(stream)>>>(bufs, r, slots, tokens, pages,
                                                                                    static_cast<int>(page_size));
    }
    count_launch();
    return check_launch("page_write_kernel");
}

extern "C" int rt_page_append(void* const* bases, const int64_t* page_strides, const int64_t* row_bytes,
                              const void* const* rows, const int64_t* row_strides, int64_t n_buffers, int32_t* table,
                              int64_t table_stride, int32_t* lens, int32_t* refs, int32_t* status, const int32_t* seqs,
                              const int32_t* offsets, int32_t* slots, int32_t* workspace, int64_t n_seqs, int64_t width,
                              int64_t pages, int64_t page_size, int64_t n, int64_t tokens, void* stream) {
    page::ExtendArgs a;
    page::AllBuffers bufs{};
    page::AllRows r{};
    if (int rc = extend_args("rt_page_append", &a, table, table_stride, lens, refs, status, seqs, offsets, slots, workspace,
                             n_seqs, width, pages, page_size, n, tokens))
        return rc;
    const bool writes = tokens > 0 && pages > 0 && n_buffers != 0;
    int64_t row_total = 0;
    if (writes) {
        if (int rc = page::fill_buffers("rt_page_append", &bufs, bases, page_strides, row_bytes, n_buffers, page_size)) return rc;
        if (int rc = page::fill_rows("rt_page_append", &r, rows, row_strides, n_buffers)) return rc;
        for (int i = 0; i < bufs.n; ++i) row_total += bufs.b[i].row_bytes;
    }
    if (!writes || tokens > page::kAppendTokens || tokens * row_total > page::kAppendBytes || bufs.n > page::kFewBuffers) {
        if (int rc = rt_page_extend(table, table_stride, lens, refs, status, seqs, offsets, slots, workspace, n_seqs, width,
                                    pages, page_size, n, tokens, stream))
            return rc;
        return writes ? rt_page_write(bases, page_strides, row_bytes, rows, row_strides, n_buffers, slots, tokens, pages,
                                      page_size, stream) : RT_OK;
    }
    const int smem = static_cast<int>(n_seqs * 4);
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&page::page_append_kernel), smem, "rt_page_append"))
        return rc;
    page::page_append_kernel<<<1, page::kPlanThreads, smem, as_stream(stream)>>>(a, page::few(bufs), page::few(r));
    count_launch();
    return check_launch("page_append_kernel");
}

extern "C" int rt_page_free(int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, const int32_t* seqs,
                            int64_t n_seqs, int64_t width, int64_t pages, int64_t n, void* stream) {
    if (int rc = page::check_table("rt_page_free", table, lens, refs, table_stride, n_seqs, width, pages, 1)) return rc;
    RT_REQUIRE(n >= 0 && n < (1ll << 31), RT_ERR_BAD_ARG, "rt_page_free: bad list");
    if (n == 0 || n_seqs == 0) return RT_OK;
    RT_REQUIRE(seqs, RT_ERR_BAD_ARG, "rt_page_free: null pointer");
    const int64_t parts = (width + page::kCopyThreads * 4 - 1) / (page::kCopyThreads * 4);
    dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(parts < 1 ? 1 : parts < 64 ? parts : 64));
    page::page_free_kernel<<<grid, page::kCopyThreads, 0, as_stream(stream)>>>(
        table, table_stride, lens, refs, seqs, static_cast<int>(n_seqs), static_cast<int>(width), static_cast<int>(pages));
    count_launch();
    return check_launch("page_free_kernel");
}

extern "C" int64_t rt_page_fork_workspace_ints(int64_t n, int64_t width) { return n * (4 + width + 1); }

extern "C" int rt_page_fork(void* const* bases, const int64_t* page_strides, const int64_t* row_bytes, int64_t n_buffers,
                            int32_t* table, int64_t table_stride, int32_t* lens, int32_t* refs, int32_t* status,
                            const int32_t* src, const int32_t* dst, int32_t* workspace, int64_t n_seqs, int64_t width,
                            int64_t pages, int64_t page_size, int64_t n, void* stream) {
    if (int rc = page::check_table("rt_page_fork", table, lens, refs, table_stride, n_seqs, width, pages, page_size))
        return rc;
    RT_REQUIRE(n >= 0 && n < (1ll << 31), RT_ERR_BAD_ARG, "rt_page_fork: bad list");
    page::AllBuffers bufs{};
    if (int rc = page::fill_buffers("rt_page_fork", &bufs, bases, page_strides, row_bytes, n_buffers, page_size)) return rc;
    if (n == 0 || n_seqs == 0) return RT_OK;
    RT_REQUIRE(src && dst && status && workspace && aligned16(workspace), RT_ERR_BAD_ARG, "rt_page_fork: null or unaligned pointer");
    const int smem = static_cast<int>(n_seqs * 4);
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&page::page_fork_plan_kernel), smem, "rt_page_fork"))
        return rc;
    page::ForkArgs a;
    a.table = table; a.table_stride = table_stride; a.lens = lens; a.refs = refs; a.status = status;
    a.src = src; a.dst = dst;
    a.plan = reinterpret_cast<page::ForkPlan*>(workspace);
    a.staged = workspace + 4 * n;
    a.found = a.staged + n * width;
    a.n_seqs = static_cast<int>(n_seqs); a.width = static_cast<int>(width); a.pages = static_cast<int>(pages);
    a.page = static_cast<int>(page_size); a.n = static_cast<int>(n);
    cudaStream_t st = as_stream(stream);
    int64_t page_bytes = 0;
    for (int i = 0; i < bufs.n; ++i) page_bytes += bufs.b[i].page_bytes;
    if (n <= page::kForkEntries && bufs.n <= page::kFewBuffers && n * page_bytes <= page::kForkBytes &&
        n * width <= 4 * page::kPlanThreads) {
        if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(&page::page_fork_kernel), smem, "rt_page_fork"))
            return rc;
        page::page_fork_kernel<<<1, page::kPlanThreads, smem, st>>>(a, page::few(bufs));
        count_launch();
        return check_launch("page_fork_kernel");
    }
    page::page_fork_plan_kernel<<<1, page::kPlanThreads, smem, st>>>(a);
    count_launch();
    if (int rc = check_launch("page_fork_plan_kernel")) return rc;
    int64_t parts = (2 * page::sms() + n - 1) / n;
    if (parts > 16) parts = 16;
    dim3 grid(static_cast<unsigned>(n), static_cast<unsigned>(parts));
    if (bufs.n <= page::kFewBuffers)
        page::page_fork_stage_kernel<<<grid, page::kCopyThreads, 0, st>>>(a, page::few(bufs));
    else
        page::page_fork_stage_kernel<<<grid, page::kCopyThreads, 0, st>>>(a, bufs);
    count_launch();
    if (int rc = check_launch("page_fork_stage_kernel")) return rc;
    page::page_fork_commit_kernel<<<grid, page::kCopyThreads, 0, st>>>(a);
    count_launch();
    return check_launch("page_fork_commit_kernel");
}

static int page_move(const char* who, page::MoveArgs& a, const page::AllBuffers& bufs, int64_t most_moves, void* stream) {
    a.pieces = 0;
    for (int i = 0; i < bufs.n; ++i) a.pieces += (bufs.b[i].page_bytes + page::kPiece - 1) / page::kPiece;
    int64_t blocks = most_moves * a.pieces;
    const int64_t rows = a.moves ? (static_cast<int64_t>(a.n_seqs) * a.width + page::kCopyThreads - 1) / page::kCopyThreads : 0;
    if (blocks < rows) blocks = rows;
    const int64_t most = 8ll * page::sms();
    if (blocks > most) blocks = most;
    if (blocks < 1) blocks = 1;
    if (bufs.n <= page::kFewBuffers)
        page::page_move_kernel<<<static_cast<unsigned>(blocks), page::kCopyThreads, 0, as_stream(stream)>>>(a, page::few(bufs));
    else
        page::page_move_kernel<<<static_cast<unsigned>(blocks), page::kCopyThreads, 0, as_stream(stream)>>>(a, bufs);
    count_launch();
    return check_launch(who);
}

extern "C" int64_t rt_page_compact_workspace_ints(int64_t pages) { return 4 + 3 * pages; }

extern "C" int rt_page_compact(void* const* bases, const int64_t* page_strides, const int64_t* row_bytes,
                               int64_t n_buffers, int32_t* table, int64_t table_stride, int32_t* refs,
                               int32_t* workspace, int64_t n_seqs, int64_t width, int64_t pages, int64_t page_size,
                               void* stream) {
    if (int rc = page::check_table("rt_page_compact", table, refs, refs, table_stride, n_seqs, width, pages, page_size))
        return rc;
    page::AllBuffers bufs{};
    if (int rc = page::fill_buffers("rt_page_compact", &bufs, bases, page_strides, row_bytes, n_buffers, page_size))
        return rc;
    RT_REQUIRE(workspace && aligned16(workspace), RT_ERR_BAD_ARG, "rt_page_compact: null or unaligned workspace");
    page::page_compact_plan_kernel<<<1, page::kPlanThreads, 0, as_stream(stream)>>>(
        refs, static_cast<int>(pages), workspace, reinterpret_cast<int2*>(workspace + 4), workspace + 4 + 2 * pages);
    count_launch();
    if (int rc = check_launch("page_compact_plan_kernel")) return rc;
    page::MoveArgs a{};
    a.moves = reinterpret_cast<const int2*>(workspace + 4);
    a.head = workspace;
    a.table = table; a.table_stride = table_stride; a.refs = refs;
    a.rank = workspace + 4 + 2 * pages;
    a.n_seqs = static_cast<int>(n_seqs); a.width = static_cast<int>(width); a.pages = static_cast<int>(pages);
    return page_move("page_move_kernel", a, bufs, pages, stream);
}

extern "C" int rt_page_copy(void* const* bases, const int64_t* page_strides, const int64_t* row_bytes, int64_t n_buffers,
                            const int32_t* from, const int32_t* to, int64_t n, int64_t pages, int64_t page_size,
                            void* stream) {
    RT_REQUIRE(n >= 0 && n < (1ll << 31) && pages >= 0 && pages < (1ll << 31) && page_size > 0, RT_ERR_BAD_ARG,
               "rt_page_copy: bad shape");
    page::AllBuffers bufs{};
    if (int rc = page::fill_buffers("rt_page_copy", &bufs, bases, page_strides, row_bytes, n_buffers, page_size)) return rc;
    if (n == 0 || n_buffers == 0) return RT_OK;
    RT_REQUIRE(from && to, RT_ERR_BAD_ARG, "rt_page_copy: null pointer");
    page::MoveArgs a{};
    a.from = from; a.to = to;
    a.n = static_cast<int>(n);
    a.pages = static_cast<int>(pages);
    return page_move("page_move_kernel", a, bufs, n, stream);
}
