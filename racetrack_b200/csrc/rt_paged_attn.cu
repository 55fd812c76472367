// Attention of one new token a sequence over a paged latent cache (the MLA decode step):
//
//   out[b, h, :] = sum_j p_j kv[j, :],   p = softmax_j( scale * (q_abs[b, h, :] . kv[j, :] + q_pe[b, h, :] . pe[j, :]) )
//
// over the positions j of sequence b that its newest token (position L - 1) sees: all j < L, or under a
// window of W positions with s sinks those with j >= L - W or j < s. kv [pages, page, 512] and pe [pages,
// page, 64] hold the rows, block_table their pages. The dense counterpart of mla_sparse_decode_kernel
// (racetrack/models/deepseek.py:793-810 without the indexer's mask).
//
// A row of 1152 bytes serves 2 * 1088 flops for each head, 242 flop/B at 128 heads: with few heads the
// kernel is bound by reading the cache once, with all of them memory and tensor cores take about the same.
// Measured on one B200, kernels and join, short runs of calls in a row on inputs of three sets (copy rate 6546 GB/s); in
// brackets the whole call in long runs among other work, host and power cap included:
//   16 heads, 48 sequences of up to 32768 (0.56 GB)  96 us, 5800 GB/s (98-105); 64 of 4096 (0.30 GB) 58 us
//   32 heads, 128 under a window of 1024 (0.11 GB)   38 us (39-40); 64 of 4096 65 us
//   128 heads, 64 of 4096                            92 us, 790 TFLOP/s (106-112); 64 heads 69.5 us
//   one sequence of 17 positions, 16 heads           8.7 us (10); of 131072 37 us
// Two kernels share the walk over the tiles and the join. mla_paged_kernel serves up to 32 heads,
// mla_paged_wide_kernel more of them in groups of 64; each served all groups once, with an earlier join: the first
// took 124 us for 64 x 4096 at 128 heads where the second took 97 (80 and 75 at 64), the second 44 for the
// window's case and 99 for the ragged one where the first took 40 and 97.
#include "rt_tc.cuh"

namespace rt {
namespace tc {

constexpr int kPTile = 64;                          // positions per tile
constexpr int kPHalf = kPTile / 2;                  // positions that are loaded and given back together
constexpr uint32_t kPLatBytes = kPTile * 1024;      // latent part of a tile
constexpr uint32_t kPTileBytes = kPTile * 1152;
constexpr int kPMaxBatch = 65535;

// ---- which CTA walks which tiles --------------------------------------------------------------
// The visible positions of row b are the tiles {0 .. na - 1} (sinks) and {b0 .. b0 + nb - 1} of 64
// positions. All rows' tiles in one line are cut into as many equal ranges as there are CTAs, so
// ragged lengths keep every SM busy alike; a row that crosses from one range into the next is finished by
// the join kernel. The host knows no length: each CTA sums them itself.
struct PagedArgs {
    const int32_t* table;         // [slots, width]
    const int32_t* lens;          // [slots]
    const int32_t* seqs;          // [batch] or null: row b is slot b
    __nv_bfloat16* out;           // [batch, heads, 512]
    int4* ranges;                 // [ranges]: row, tile within it, its tiles, tiles per range
    float* part_ml;               // [2 ranges, heads, 2]: running maximum, denominator
    float* part_o;                // [2 ranges, heads, 512], not normalised
    int64_t table_stride;
    int batch, heads, slots, width, pages;
    int page_log;                 // log2(page size)
    int window, sinks;            // window 0: none
    int n_ranges;
    float scale_log2;
};

struct RowTiles {
    int len, na, b0, n;           // length, sink tiles, first window tile, all tiles
};

__device__ __forceinline__ int row_slot(const PagedArgs& a, int b) {
    const int s = a.seqs ? __ldg(a.seqs + b) : b;
    return s >= 0 && s < a.slots ? s : -1;
}

__device__ __forceinline__ RowTiles slot_tiles(const PagedArgs& a, int s) {
    const int most = a.width << a.page_log;
    RowTiles t;
    t.len = s < 0 ? 0 : min(max(__ldg(a.lens + s), 0), most);
    const int all = (t.len + kPTile - 1) / kPTile;
    if (a.window == 0 || a.window >= t.len) {
        t.na = 0;
        t.b0 = 0;
        t.n = all;
    } else {
        t.na = (min(a.sinks, t.len) + kPTile - 1) / kPTile;
        t.b0 = max(t.na, (t.len - a.window) / kPTile);
        t.n = t.na + max(0, all - t.b0);
    }
    return t;
}
__device__ __forceinline__ RowTiles row_tiles(const PagedArgs& a, int b) { return slot_tiles(a, row_slot(a, b)); }

__device__ __forceinline__ int tile_of(const RowTiles& t, int j) { return j < t.na ? j : t.b0 + (j - t.na); }

// Bit i: position 64 * tile + i is visible (by its position alone).
__device__ __forceinline__ uint64_t tile_mask(const PagedArgs& a, const RowTiles& t, int tile) {
    const int p0 = tile * kPTile;
    auto below = [&](int x) {                        // positions p0 .. x - 1
        const int n = x - p0;
        return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
    };
    uint64_t m = below(t.len);
    if (a.window != 0 && a.window < t.len) m &= ~below(t.len - a.window) | below(a.sinks);
    return m;
}

// The range of this CTA: its first row and tile, and how many tiles it walks. All threads call it; every
// thread sums the rows of one slice of the batch. `scratch`: THREADS / 32 + 4 ints of shared memory.
struct RangeStart {
    int row, tile, count, slot;      // (the row's slot: a load less in front of the first tile)
};
template <int THREADS>
__device__ RangeStart find_range(const PagedArgs& a, int range, volatile int* scratch) {
    volatile int* found = scratch + THREADS / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int per = (a.batch + THREADS - 1) / THREADS;
    const int b0 = min(static_cast<int>(threadIdx.x) * per, a.batch), b1 = min(b0 + per, a.batch);
    int mine = 0;
    for (int b = b0; b < b1; ++b) mine += row_tiles(a, b).n;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) scratch[warp] = x;
    if (threadIdx.x == 0) {
        found[0] = -1;
        found[1] = found[2] = found[3] = 0;
    }
    __syncthreads();
    int before = x - mine, total = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        const int v = scratch[w];
        if (w < warp) before += v;
        total += v;
    }
    const int per_range = (total + a.n_ranges - 1) / a.n_ranges;
    const int first = range * per_range;             // below 2^31: the host bounds batch * tiles
    if (first >= before && first < before + mine) {
        int at = before, b = b0;
        RowTiles t = row_tiles(a, b);
        while (at + t.n <= first) {
            at += t.n;
            t = row_tiles(a, ++b);
        }
        found[0] = b;
        found[1] = first - at;
        found[2] = t.n;
        found[3] = row_slot(a, b);
    }
    __syncthreads();
    RangeStart r{found[0], found[1], 0, found[3]};
    if (r.row >= 0) r.count = min(per_range, total - first);
    if (threadIdx.x == 0) a.ranges[range] = make_int4(r.row, r.tile, found[2], per_range);
    return r;
}

// ---- up to 32 heads ---------------------------------------------------------------------------
// Work of a CTA: its range of tiles for all heads, padded to G = 16 or 32. Positions and dims are the rows of the
// products, heads the columns: with few heads what the tensor core reads from shared memory is then little more than the tile
// itself. (Heads as rows, padded to 128, took 2300 + 1400 cycles a tile for 16 heads: 4 KB of mostly empty
// query rows for each instruction. This form takes about half.) Per tile of 64 positions:
//   producer  one TMA box a page (32 positions at most, which are also given back together) brings the latent
//             rows as [8-row groups][8 blocks of 64 dims][8 rows][128 B] (128-byte swizzle), one the rope keys: a
//             page of any size lands in the same layout, of which both products read their operand (the group
//             stride is a field of the descriptor), so the rows are staged once. Two tiles are staged (144 KB);
//             the one behind them is asked into L2 (when it came the ragged batch above took 99 us with it, 104
//             without, 101 two tiles ahead, 105 three). Boxes of half or a quarter of the dims instead of the positions: 64 x 4096 x 128
//             heads, when this kernel served them, 134 and 142 us instead of 125;
//   S = K Q^T 36 tcgen05.mma (M = 64 positions, N = G heads, K = 16 dims), both K-major;
//   softmax   warps 4-7. An M = 64 product lies in lanes 0-15 of each quarter of tensor memory; read in 16 x 256
//             bit blocks a thread holds two positions of G / 4 heads, so all lanes work. The maxima change only
//             when a score exceeds one by 2^8: all warps vote on that, and only then (and at a row's first tile)
//             look for new maxima, across lanes and warps. P = 2^(s - m) goes as bf16 into shared memory, one
//             128-byte line of heads a position; a thread sums its own probabilities in fp32, and the sums meet
//             at the row's end;
//   O^T += V^T P^T  tcgen05.mma (M = 128 of the 512 dims, N = G, K = 16 positions): the tile again, as the
//             MN-major operand, P MN-major too. Only steps that hold a visible position are multiplied;
//   output    warps 8-11 read a finished row from tensor memory while the next one's first tile is under way.
// O is 4 blocks of G columns in tensor memory, the two score buffers 2 G behind it. All sums, maxima and O
// are fp32; P is rounded to bf16 because the tensor core multiplies it with bf16 rows (2^-8 of a
// probability at most, no more than the rounding of the rows). Positions that are not visible weigh
// exactly nothing whatever memory holds there: their scores are not looked at, their rows are zeroed in
// shared memory between the two products (0 * NaN). A page number outside the pool reads as zeros (the
// TMA unit's bounds) and its positions are not visible.
constexpr uint32_t kPQRow = 9 * 128;                 // bytes of a staged head
constexpr uint32_t kPQBytes = 2 * 32 * kPQRow;       // two rows' queries
constexpr uint32_t kPKOff = kPQBytes;
constexpr uint32_t kPPOff = kPKOff + 2 * kPTileBytes;        // P: [64 positions][64 heads] bf16
constexpr uint32_t kPBarOff = kPPOff + kPTile * 128;
constexpr int kPBars = 18;      // qfull[2] qfree[2] kfull[2] kfree[2][2] sfull[2] vote pfull pfree efull odone ofree
constexpr uint32_t kPInfoOff = kPBarOff + kPBars * 8 + 16;   // (tensor memory slot, abort flag before it)
constexpr uint32_t kPVoteOff = kPInfoOff + 2 * 16;           // [2][4] ints, then the finished row, its part and tiles
constexpr uint32_t kPMaxOff = kPVoteOff + 12 * 4;            // m or 0 [64], per quarter [4][64], factors [64]
constexpr uint32_t kPSmemBytes = kPMaxOff + 6 * 64 * 4 + 1024;
static_assert(kPKOff % 1024 == 0 && kPPOff % 1024 == 0 && kPInfoOff % 16 == 0 && kPMaxOff % 16 == 0, "alignment");
static_assert(kPSmemBytes <= 232448, "shared memory budget");

struct TileInfo {
    uint64_t mask;
    int32_t row;
    int32_t flags;                // 1: first tile of the row in this range, 2: last one, 4: the row's first, 8: its last
};

// Descriptor with a stride between 8-row groups of its own (K-major: rows of one 64-dim block; MN-major: K
// indices, `lbo` between 64-element blocks).
__device__ __forceinline__ uint64_t smem_desc_groups(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (static_cast<uint64_t>(lbo >> 4) << 16) |
           (static_cast<uint64_t>(sbo >> 4) << 32) | (1ull << 46) | (2ull << 61);
}

// A descriptor whose halves are known apart: start address and leading offset (in 16 bytes), group stride and mode.
__device__ __forceinline__ uint64_t smem_desc_at(uint32_t low, uint32_t sbo) {
    return static_cast<uint64_t>(low) | (static_cast<uint64_t>((sbo >> 4) | (1u << 14) | (2u << 29)) << 32);
}

__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* m, int c0, int c1, int c2, int c3,
                                            int c4, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(dst),
        "l"(m), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
        : "memory");
}

// The box of a load into L2.
__device__ __forceinline__ void tma_prefetch_5d(const CUtensorMap* m, int c0, int c1, int c2, int c3, int c4) {
    asm volatile("cp.async.bulk.prefetch.tensor.5d.L2.global [%0, {%1, %2, %3, %4, %5}];" ::"l"(m), "r"(c0), "r"(c1), "r"(c2),
                 "r"(c3), "r"(c4)
                 : "memory");
}
__device__ __forceinline__ void tma_prefetch_3d(const CUtensorMap* m, int c0, int c1, int c2) {
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(m), "r"(c0), "r"(c1), "r"(c2)
                 : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// mbar_wait of a whole warp: all lanes go on or none does (a lane whose cycle budget runs out while another
// still sees the phase complete must not leave the warp's shuffles behind).
__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort, int code) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, code));
}

// 16 or 32 consecutive columns of the warp's lanes, complete on return.
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[32]) {
    tmem_ld_32x32(taddr, r);
    tmem_ld_wait(r);
}
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&r)[16]) {
    uint32_t lo[8], hi[8];
    tmem_ld_32x8(taddr, lo);
    tmem_ld_32x8(taddr + 8, hi);
    tmem_ld_wait(lo);
    tmem_ld_wait(hi);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        r[i] = lo[i];
        r[8 + i] = hi[i];
    }
}
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[32]) { tmem_st_32x32(taddr, r); }
__device__ __forceinline__ void tmem_st_cols(uint32_t taddr, const uint32_t (&r)[16]) { tmem_st_32x16(taddr, r); }

// Lanes 0-15 of the warp's quarter, 8 columns a register quadruple: lane t gets rows t / 4 (r[4 u], r[4 u + 1])
// and t / 4 + 8 (r[4 u + 2], r[4 u + 3]) of columns 8 u + 2 (t % 4) and the next. Complete on return.
__device__ __forceinline__ void tmem_ld_16x256b(uint32_t taddr, float (&x)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256b(uint32_t taddr, float (&x)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]),
                   "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_16x256b(uint32_t taddr, float (&x)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
                 "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
                 "tcgen05.wait::ld.sync.aligned;"
                 : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3]), "=f"(x[4]), "=f"(x[5]), "=f"(x[6]), "=f"(x[7]),
                   "=f"(x[8]), "=f"(x[9]), "=f"(x[10]), "=f"(x[11]), "=f"(x[12]), "=f"(x[13]), "=f"(x[14]), "=f"(x[15]),
                   "=f"(x[16]), "=f"(x[17]), "=f"(x[18]), "=f"(x[19]), "=f"(x[20]), "=f"(x[21]), "=f"(x[22]), "=f"(x[23]),
                   "=f"(x[24]), "=f"(x[25]), "=f"(x[26]), "=f"(x[27]), "=f"(x[28]), "=f"(x[29]), "=f"(x[30]), "=f"(x[31])
                 : "r"(taddr)
                 : "memory");
}
// Four 8 x 8 blocks of bf16 pairs held like the rows above into shared memory; lane t gives the address of row
// t % 8 of block t / 8.
__device__ __forceinline__ void stmatrix_x4(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r0), "r"(r1), "r"(r2),
                 "r"(r3)
                 : "memory");
}

// Where the result of a row's tiles in a range goes: the row's own output if they are all of its tiles, else
// the range's slot for a row that began in an earlier range (2 r) or ends in a later one (2 r + 1).
__device__ __forceinline__ int part_slot(int flags, int range) {
    return (flags & 12) == 12 ? -1 : 2 * range + ((flags & 4) ? 1 : 0);
}

// O (the same quarter) times a factor a head.
template <int G>
__device__ __forceinline__ void rescale(uint32_t o_at, const float* w) {
    constexpr int kCols = G < 32 ? G : 32;
#pragma unroll 1
    for (int c = 0; c < 4 * G; c += kCols) {
        uint32_t o[kCols];
        tmem_ld_cols(o_at + c, o);
#pragma unroll
        for (int i = 0; i < kCols; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * w[(c & (G - 1)) + i]);
        tmem_st_cols(o_at + c, o);
    }
    tmem_st_wait();
}

// A finished row's O (warp: a quarter of each block of 128 dims, all G heads) times f, to its output or its part.
template <int G>
__device__ __forceinline__ void write_row(const PagedArgs& a, int part, int row, int head0, uint32_t o_at, const float* f) {
    constexpr int kCols = G < 32 ? G : 32;
    const int d0 = threadIdx.x & 127;
#pragma unroll 1
    for (int c = 0; c < 4 * G; c += kCols) {
        uint32_t o[kCols];
        tmem_ld_cols(o_at + c, o);
        const int h = c & (G - 1), d = (c / G) * 128 + d0;
        const int64_t at = (static_cast<int64_t>(part < 0 ? row : part) * a.heads + head0 + h) * 512 + d;
        const int live = a.heads - head0 - h;
        // (factors before stores, and no branch a head: with both a head took 37 cycles, now 20)
        float v[kCols];
#pragma unroll
        for (int i = 0; i < kCols; i += 4) *reinterpret_cast<float4*>(v + i) = *reinterpret_cast<const float4*>(f + h + i);
#pragma unroll
        for (int i = 0; i < kCols; ++i) v[i] = v[i] == 0.f ? 0.f : __uint_as_float(o[i]) * v[i];
        auto each = [&](auto put) {
            if (live >= kCols) {
#pragma unroll
                for (int i = 0; i < kCols; ++i) put(i);
            } else {
#pragma unroll
                for (int i = 0; i < kCols; ++i)
                    if (i < live) put(i);
            }
        };
        if (part < 0) each([&](int i) { a.out[at + i * 512] = __float2bfloat16_rn(v[i]); });
        else each([&](int i) { a.part_o[at + i * 512] = v[i]; });
    }
}

// Rows without a visible tile are nobody's: zeros, shared out over the ranges (128 threads).
__device__ __forceinline__ void clear_empty_rows(const PagedArgs& a, int range) {
    for (int b = range; b < a.batch; b += a.n_ranges)
        if (row_tiles(a, b).n == 0)
            for (int c = threadIdx.x & 127; c < a.heads * 64; c += 128)
                reinterpret_cast<uint4*>(a.out + static_cast<int64_t>(b) * a.heads * 512)[c] = make_uint4(0u, 0u, 0u, 0u);
}

// Where the tile walk of a range stands.
struct TileWalk {
    int b, j, slot, row_at;                          // row, tile within it, its slot, the row that `t` is of
    RowTiles t;
    int32_t fetched = -1;                            // lane: page number of entry fetched0 + lane of row fetched_row
    int fetched0 = -1, fetched_row = -1;
    int tile, flags, id[4];                          // of this step: tile, TileInfo flags, the page of each box
    uint64_t mask;

    __device__ __forceinline__ TileWalk(const PagedArgs& a, const RangeStart& start)
        : b(start.row), j(start.tile), slot(start.slot), row_at(start.row),
          t(start.count > 0 ? slot_tiles(a, start.slot) : RowTiles{}) {}

    // The range's tile g (whole warp: the lanes fetch page numbers). rows: positions of a box.
    __device__ __forceinline__ void step(const PagedArgs& a, int g, int n_tiles, int rows) {
        const int lane = threadIdx.x & 31, page = 1 << a.page_log, boxes = kPTile / rows;
        if (row_at != b) {
            t = slot_tiles(a, slot = row_slot(a, b));
            while (t.n == 0) t = slot_tiles(a, slot = row_slot(a, ++b));     // rows without a tile
            row_at = b;
        }
        flags = (g == 0 || j == 0 ? 1 : 0) | (g == n_tiles - 1 || j == t.n - 1 ? 2 : 0) | (j == 0 ? 4 : 0) |
                (j == t.n - 1 ? 8 : 0);
        tile = tile_of(t, j);
        const int m0 = (tile * kPTile) >> a.page_log, m1 = (tile * kPTile + kPTile - rows) >> a.page_log;
        if (fetched_row != b || m0 < fetched0 || m1 >= fetched0 + 32) {
            fetched0 = m0;
            fetched_row = b;
            const int m = m0 + lane;
            fetched = m < a.width ? __ldg(a.table + slot * a.table_stride + m) : -1;
        }
        mask = tile_mask(a, t, tile);
        const int used = (t.len + page - 1) >> a.page_log;      // entries behind the sequence's end are not read
        const uint64_t row_bits = rows < 64 ? (1ull << rows) - 1 : ~0ull;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            id[i] = -1;
            if (i < boxes) {
                const int m = (tile * kPTile + i * rows) >> a.page_log;
                id[i] = __shfl_sync(0xffffffffu, fetched, m - fetched0);
                if (m >= used || id[i] < 0 || id[i] >= a.pages) mask &= ~(row_bits << (i * rows));
                if ((mask >> (i * rows) & row_bits) == 0) id[i] = -1;     // nothing visible: not read
            }
        }
    }
    __device__ __forceinline__ void advance() {
        if (++j == t.n) {
            ++b;
            j = 0;
        }
    }
};

constexpr int kPThreads = 384;      // warps: 0 MMA, 1 producer, 4-7 softmax, 8-11 finished rows

template <int G>
__global__ void __launch_bounds__(kPThreads, 1) mla_paged_kernel(const __grid_constant__ CUtensorMap tm_qa,
                                                                 const __grid_constant__ CUtensorMap tm_qp,
                                                                 const __grid_constant__ CUtensorMap tm_kv,
                                                                 const __grid_constant__ CUtensorMap tm_pe,
                                                                 const PagedArgs a) {
    static_assert(G <= 32, "heads");
    constexpr uint32_t kTmemS = 4 * G, kTmemCols = 8 * G;
    // fp32 accumulate, bf16 x bf16; S: both K-major, M = 64; O: both MN-major, M = 128
    constexpr uint32_t kSIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(G >> 3) << 17) | (4u << 24);
    constexpr uint32_t kOIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (1u << 16) |
                                 (static_cast<uint32_t>(G >> 3) << 17) | (8u << 24);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + kPBarOff;
    auto qfull = [&](int s) { return bars + 8u * s; };
    auto qfree = [&](int s) { return bars + 8u * (2 + s); };
    auto sfull = [&](int s) { return bars + 8u * (4 + s); };
    const uint32_t vote = bars + 8u * 6, pfull = bars + 8u * 7, pfree = bars + 8u * 8, efull = bars + 8u * 9,
                   odone = bars + 8u * 10, ofree = bars + 8u * 11;
    auto kfull = [&](int s) { return bars + 8u * (12 + s); };
    auto kfree = [&](int s, int half) { return bars + 8u * (14 + 2 * s + half); };
    const uint32_t slot = bars + 8u * kPBars;
    volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(base_ptr + kPBarOff + 8 * kPBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(slot_ptr + 1);
    volatile TileInfo* info_s = reinterpret_cast<volatile TileInfo*>(base_ptr + kPInfoOff);
    volatile int* vote_s = reinterpret_cast<volatile int*>(base_ptr + kPVoteOff);
    volatile int* done_s = vote_s + 8;                                       // finished row, its part, its tiles
    float* const mu_s = reinterpret_cast<float*>(base_ptr + kPMaxOff);       // running maxima, 0 for -infinity
    float* const w_s = mu_s + 64;                                            // [4][64]
    float* const f_s = w_s + 256;                                            // what a finished row's O is multiplied with

    const int warp = uniform_warp_id(), lane = threadIdx.x & 31;
    const int range = blockIdx.x;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < 2; ++s) {
            mbar_init(qfull(s), 1);
            mbar_init(qfree(s), 1);
            mbar_init(kfull(s), 1);
            mbar_init(kfree(s, 0), 1);
            mbar_init(kfree(s, 1), 1);
            mbar_init(sfull(s), 1);
        }
        mbar_init(vote, 4);
        mbar_init(pfull, 4);
        mbar_init(pfree, 1);
        mbar_init(efull, 4);
        mbar_init(odone, 1);
        mbar_init(ofree, 4);
        fence_mbar_init();
        tma_prefetch_desc(&tm_qa);
        tma_prefetch_desc(&tm_qp);
        tma_prefetch_desc(&tm_kv);
        tma_prefetch_desc(&tm_pe);
    }
    if (warp == 0) {
        tmem_alloc(slot, kTmemCols);
        tmem_relinquish();
    }
    const RangeStart start = find_range<kPThreads>(a, range, reinterpret_cast<volatile int*>(w_s));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *slot_ptr;
    const int n_tiles = start.count;

    if (warp == 0) {
        if (n_tiles > 0 && elect_one()) {
            bool ok = true;
            int q = 0, v = 0, q_seg = 0, v_seg = 0;            // tiles scored and accumulated, and their rows
            bool q_open = false, v_open = false;               // the current row's first tile has been taken
            long long t0 = 0;
            uint32_t spins = 0, acc = 0;
            // scores of the next landed tile or P V of the tile whose probabilities are written, whichever
            // is ready first
            while (ok && v < n_tiles) {
                bool progressed = false;
                if (q < n_tiles && q - v < 2 && mbar_try_wait(kfull(q & 1), (q >> 1) & 1)) {
                    const int flags = info_s[q & 1].flags;
                    const int qb = q_seg & 1;
                    if (q_open || mbar_try_wait(qfull(qb), (q_seg >> 1) & 1)) {
                        tc_fence_after();
                        const uint32_t kb = base + kPKOff + (q & 1) * kPTileBytes;
                        const uint32_t qa = base + qb * (G * kPQRow);
                        const uint32_t d = tmem_base + kTmemS + static_cast<uint32_t>(q & 1) * G;
#pragma unroll
                        for (int c = 0; c < 9; ++c) {
                            const uint64_t adesc = c < 8 ? smem_desc_groups(kb + c * 1024, 16, 8192)
                                                         : smem_desc_sw128(kb + kPLatBytes);
                            const uint64_t bdesc = smem_desc_sw128(qa + c * G * 128);
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                mma_f16(d, adesc + 2u * j, bdesc + 2u * j, kSIdesc, (c | j) != 0 ? 1u : 0u);
                        }
                        mma_commit(sfull(q & 1));
                        q_open = true;
                        if (flags & 2) {
                            mma_commit(qfree(qb));
                            ++q_seg;
                            q_open = false;
                        }
                        ++q;
                        progressed = true;
                    }
                }
                if (v < q && mbar_try_wait(pfull, v & 1) &&
                    (v_open || v_seg == 0 || mbar_try_wait(ofree, (v_seg - 1) & 1))) {
                    tc_fence_after();
                    const uint64_t mask = info_s[v & 1].mask;
                    const int flags = info_s[v & 1].flags;
                    if (!v_open) acc = 0;
                    const uint32_t kb = base + kPKOff + (v & 1) * kPTileBytes;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if ((mask >> (16 * j) & 0xffffu) != 0) {
                            const uint64_t bdesc = smem_desc_groups(base + kPPOff + j * 2048, 16, 1024);
#pragma unroll
                            for (int f = 0; f < 4; ++f)
                                mma_f16(tmem_base + f * G, smem_desc_groups(kb + j * 16384 + f * 2048, 1024, 8192), bdesc,
                                        kOIdesc, acc);
                            acc = 1;
                        }
                        if (j & 1) mma_commit(kfree(v & 1, j >> 1));       // its positions are done with
                    }
                    mma_commit(pfree);
                    v_open = true;
                    if (flags & 2) {
                        mma_commit(odone);
                        ++v_seg;
                        v_open = false;
                    }
                    ++v;
                    progressed = true;
                }
                if (progressed) {
                    spins = 0;
                } else if ((++spins & 63u) == 0) {
                    if (spins == 64) t0 = clock64();
                    if (*abort_flag) ok = false;
                    else if (clock64() - t0 > kWaitCycles) {
                        *abort_flag = 81;
                        atomicCAS(&g_tc_error, 0, 81);
                        ok = false;
                    }
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        // the whole warp walks the range, one thread issues the loads
        TileWalk w(a, start);
        const int page = 1 << a.page_log, rows = min(page, kPHalf), boxes = kPTile / rows;    // rows of a box, boxes of a tile
        int seg = 0;
        if (n_tiles > 0) w.step(a, 0, n_tiles, rows);
        for (int g = 0; g < n_tiles; ++g) {
            const int st = g & 1, qb = seg & 1;
            const uint32_t free_par = ((g >> 1) & 1) ^ 1u;
            const uint32_t dst = base + kPKOff + st * kPTileBytes;
            bool ok = true;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (!(ok = mbar_wait_warp(kfree(st, half), free_par, abort_flag, 82))) break;
                if (half == 0 && (w.flags & 1) &&
                    !(ok = mbar_wait_warp(qfree(qb), ((seg >> 1) & 1) ^ 1u, abort_flag, 83)))
                    break;
                if (elect_one()) {
                    if (half == 0) {
                        if (w.flags & 1) {
                            const uint32_t qd = base + qb * (G * kPQRow);
                            mbar_arrive_expect_tx(qfull(qb), G * kPQRow);
                            tma_load_4d(qd, &tm_qa, 0, 0, 0, w.b, qfull(qb));
                            tma_load_3d(qd + G * 1024, &tm_qp, 0, 0, w.b, qfull(qb));
                        }
                        info_s[st].mask = w.mask;
                        info_s[st].row = w.b;
                        info_s[st].flags = w.flags;
                        mbar_arrive_expect_tx(kfull(st), kPTileBytes);     // both halves
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < boxes && i * rows / kPHalf == half) {
                            const int row = (w.tile * kPTile + i * rows) & (page - 1);
                            tma_load_5d(dst + i * rows * 1024, &tm_kv, 0, 0, 0, row >> 3, w.id[i], kfull(st));
                            tma_load_3d(dst + kPLatBytes + i * rows * 128, &tm_pe, 0, row, w.id[i], kfull(st));
                        }
                }
                __syncwarp();
            }
            if (!ok) break;
            if (w.flags & 2) ++seg;
            w.advance();
            if (g + 1 < n_tiles) {
                // the next tile, whose place in shared memory is still taken, on its way into L2
                w.step(a, g + 1, n_tiles, rows);
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < boxes && w.id[i] >= 0) {
                            const int row = (w.tile * kPTile + i * rows) & (page - 1);
                            tma_prefetch_5d(&tm_kv, 0, 0, 0, row >> 3, w.id[i]);
                            tma_prefetch_3d(&tm_pe, 0, row, w.id[i]);
                        }
                }
                __syncwarp();
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const int quad = warp & 3, tid = threadIdx.x - 128;
        const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
        const int h0 = 2 * (lane & 3);                         // this thread's heads: 8 u + h0 and the next
        const int key = 16 * quad + (lane >> 2);               // its positions within the tile: key and key + 8
        const float ninf = __int_as_float(0xff800000);
        uint32_t votes = 0;                                    // phases of `vote` taken
        auto meet = [&](int code) {                            // all softmax warps have come this far
            __syncwarp();
            if (lane == 0) mbar_arrive(vote);
            return mbar_wait_warp(vote, votes++ & 1, abort_flag, code);
        };
        // combines v of the thread's two positions' lanes 8 u + h0 .. over the warp's positions
        auto over_lanes = [&](float v, auto f) {
            v = f(v, __shfl_xor_sync(0xffffffffu, v, 4));
            v = f(v, __shfl_xor_sync(0xffffffffu, v, 8));
            return f(v, __shfl_xor_sync(0xffffffffu, v, 16));
        };
        auto larger = [](float u, float w) { return fmaxf(u, w); };
        auto plus = [](float u, float w) { return u + w; };
        // lane t: row t % 8 of block t / 8; blocks: positions 0-7 and 8-15 of eight heads, then of the next eight
        const int st_key = 16 * quad + (lane & 15);
        const uint32_t st_line = base + kPPOff + st_key * 128;
        float l[G / 4];
        int flags4 = 0, seg = 0, seg_first = 0;
        bool open = false;                                     // every head has a maximum
        float m_own = ninf;                                    // that of head tid
        for (int g = 0; g < n_tiles; ++g) {
            const int st = g & 1;
            if (!mbar_wait_warp(kfull(st), (g >> 1) & 1, abort_flag, 84)) break;
            const uint64_t mask = info_s[st].mask;
            const int flags = info_s[st].flags, b = info_s[st].row;
            const bool first = flags & 1, last = flags & 2;
            flags4 = (first ? 0 : flags4) | (flags & 12);
            const bool seen0 = mask >> key & 1, seen1 = mask >> (key + 8) & 1;
            if (first) {
                open = false;
                seg_first = g;
#pragma unroll
                for (int i = 0; i < G / 4; ++i) l[i] = 0.f;
            }
            if (!mbar_wait_warp(sfull(st), (g >> 1) & 1, abort_flag, 85)) break;
            tc_fence_after();
            float x[G / 2];                                    // [8 heads][position, position + 8][2 heads]
            // P against the maxima so far, and whether a score exceeds one of them by more than 2^8; what the
            // other warps found comes in while the exponentials are evaluated
            auto scores = [&] { tmem_ld_16x256b(tmem_base + lane_base + kTmemS + static_cast<uint32_t>(st) * G, x); };
            float top0 = ninf, top1 = ninf;
            auto against = [&] {
#pragma unroll
                for (int u = 0; u < G / 8; ++u) {
                    const float2 mu = *reinterpret_cast<const float2*>(mu_s + 8 * u + h0);
                    x[4 * u] = fmaf(x[4 * u], a.scale_log2, -mu.x);
                    x[4 * u + 1] = fmaf(x[4 * u + 1], a.scale_log2, -mu.y);
                    x[4 * u + 2] = fmaf(x[4 * u + 2], a.scale_log2, -mu.x);
                    x[4 * u + 3] = fmaf(x[4 * u + 3], a.scale_log2, -mu.y);
                    top0 = fmaxf(top0, fmaxf(x[4 * u], x[4 * u + 1]));
                    top1 = fmaxf(top1, fmaxf(x[4 * u + 2], x[4 * u + 3]));
                }
            };
            auto exponentials = [&] {
#pragma unroll
                for (int i = 0; i < G / 2; ++i) x[i] = ((i & 2) ? seen1 : seen0) ? exp2_fast(x[i]) : 0.f;
            };
            scores();
            bool over = !open;
            if (open) {
                against();
                over = (seen0 && top0 > 8.f) || (seen1 && top1 > 8.f);
            }
            over = __any_sync(0xffffffffu, over);
            if (lane == 0) {
                vote_s[st * 4 + quad] = over ? 1 : 0;
                mbar_arrive(vote);
            }
            if (open) exponentials();
            if (!mbar_wait_warp(vote, votes++ & 1, abort_flag, 86)) break;
#pragma unroll
            for (int w = 0; w < 4; ++w) over |= vote_s[st * 4 + w] != 0;
            if (over) {
                if (open) scores();
#pragma unroll
                for (int i = 0; i < G / 4; ++i) {
                    const float y0 = seen0 ? x[(i >> 1) * 4 + (i & 1)] * a.scale_log2 : ninf;
                    const float y1 = seen1 ? x[(i >> 1) * 4 + 2 + (i & 1)] * a.scale_log2 : ninf;
                    const float most = over_lanes(fmaxf(y0, y1), larger);
                    if (lane < 4) w_s[quad * 64 + 8 * (i >> 1) + h0 + (i & 1)] = most;
                }
                if (!meet(89)) break;
                bool blank = false;
                if (tid < G) {
                    const float mt = fmaxf(fmaxf(w_s[tid], w_s[64 + tid]), fmaxf(w_s[128 + tid], w_s[192 + tid]));
                    const float old = first ? ninf : m_own;
                    const bool grow = mt > old + 8.f;          // false while mt is -infinity
                    m_own = grow ? mt : old;
                    blank = m_own == ninf;
                    mu_s[tid] = blank ? 0.f : m_own;
                    w_s[tid] = grow ? exp2_fast(old - m_own) : 1.f;
                }
                blank = __any_sync(0xffffffffu, blank);
                if (lane == 0) vote_s[st * 4 + quad] = blank ? 1 : 0;      // (the votes have been read)
                if (!meet(90)) break;
#pragma unroll
                for (int i = 0; i < G / 4; ++i) l[i] *= w_s[8 * (i >> 1) + h0 + (i & 1)];
                open = (vote_s[st * 4] | vote_s[st * 4 + 1] | vote_s[st * 4 + 2] | vote_s[st * 4 + 3]) == 0;
                against();
                exponentials();
            }
#pragma unroll
            for (int i = 0; i < G / 4; ++i) l[i] += x[(i >> 1) * 4 + (i & 1)] + x[(i >> 1) * 4 + 2 + (i & 1)];
            // rows of a step that is multiplied, but not visible: zeros
            const uint32_t step = static_cast<uint32_t>(mask >> (16 * quad)) & 0xffffu;
            if (step != 0 && step != 0xffffu) {
                uint8_t* kt = base_ptr + kPKOff + st * kPTileBytes + quad * 16384;
                for (uint32_t z = ~step & 0xffffu; z; z &= z - 1) {
                    const int row = __ffs(static_cast<int>(z)) - 1;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        *reinterpret_cast<uint4*>(kt + (row >> 3) * 8192 + ((lane >> 3) + 4 * i) * 1024 + (row & 7) * 128 +
                                                  (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            if (g > 0) {
                // O += P V of the tile before has retired: P may be overwritten, O is at rest
                if (!mbar_wait_warp(pfree, (g - 1) & 1, abort_flag, 87)) break;
                tc_fence_after();
                if (over && !first) rescale<G>(tmem_base + lane_base, w_s);
            }
#pragma unroll
            for (int u = 0; u < G / 8; u += 2)
                stmatrix_x4(st_line + (((u + (lane >> 4)) ^ (st_key & 7)) << 4), pack_bf16x2(x[4 * u], x[4 * u + 1]),
                            pack_bf16x2(x[4 * u + 2], x[4 * u + 3]), pack_bf16x2(x[4 * u + 4], x[4 * u + 5]),
                            pack_bf16x2(x[4 * u + 6], x[4 * u + 7]));
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull);
            if (last) {
                // the sums of a head over the positions: lanes, then quarters (in order)
                if (!meet(91)) break;                          // w_s has been read
#pragma unroll
                for (int i = 0; i < G / 4; ++i) {
                    const float sum = over_lanes(l[i], plus);
                    if (lane < 4) w_s[quad * 64 + 8 * (i >> 1) + h0 + (i & 1)] = sum;
                }
                if (!meet(92)) break;
                // the row before has been written, so its factors may go
                if (seg > 0 && !mbar_wait_warp(ofree, (seg - 1) & 1, abort_flag, 93)) break;
                const int part = part_slot(flags4, range);
                // one thread a head: the denominator, and what O is multiplied with (0 for a head of no weight at
                // all, every page out of the pool or every score -infinity: it is zero)
                if (tid < G) {
                    const float den = (w_s[tid] + w_s[64 + tid]) + (w_s[128 + tid] + w_s[192 + tid]);
                    if (part >= 0 && tid < a.heads)
                        *reinterpret_cast<float2*>(a.part_ml + (static_cast<int64_t>(part) * a.heads + tid) * 2) =
                            make_float2(den == 0.f ? ninf : m_own, den);
                    f_s[tid] = den == 0.f ? 0.f : part < 0 ? 1.f / den : 1.f;
                }
                if (tid == 0) {
                    done_s[0] = b;
                    done_s[1] = part;
                    done_s[2] = g - seg_first + 1;
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(efull);
                ++seg;
            }
        }
    } else if (warp >= 8) {
        // finished rows out of tensor memory, while the next row's first tile is on its way
        const int quad = warp & 3;
        const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
        clear_empty_rows(a, range);
        for (int seg = 0, left = n_tiles; left > 0; ++seg) {
            if (!mbar_wait_warp(efull, seg & 1, abort_flag, 94)) break;
            const int b = done_s[0], part = done_s[1], tiles = done_s[2];
            if (!mbar_wait_warp(odone, seg & 1, abort_flag, 88)) break;
            tc_fence_after();
            left -= tiles;
            write_row<G>(a, part, b, 0, tmem_base + lane_base, f_s);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ofree);
        }
    }
    tc_fence_before();
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // the join kernel may be set up
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// ---- 33 heads and more ------------------------------------------------------------------------
// Groups of 64 heads, whose CTAs run side by side and share the tiles in L2; the same mathematics. With 64 query rows in shared memory only two tiles fit beside them,
// and a tile's way (load 2000 cycles, scores 1400, softmax 1400, P V 1100) took 3100 cycles over two places. Here
// the queries lie in tensor memory, as the A operand of the scores: 64 heads are its rows, dims 0-287 of the
// rows 16 i .. 16 i + 15 in lanes 32 i .. of 144 columns, dims 288-575 in lanes 32 i + 16 .. of the same columns,
// each half with a product of its own (18 tcgen05.mma, M = 64, N = 64 positions), and the softmax adds
// the two. O^T (256 columns), the scores (64) and the queries (144) fill the 512 columns, and the ring in
// shared memory has three places. A row's queries travel through one of them (TMA, swizzled) before its
// first tile; warps 8-11 bring them into tensor memory and give the place back.
//   scores    warp 0, P V warp 2: issued by one warp in turn, with a question to every barrier between them, the
//             tensor core stood still for 650 of 2650 cycles a tile;
//   softmax   warps 4-7, a thread has 16 positions of two heads: a head's maximum and sum are found in four
//             lanes. All warps still vote whether any head's maximum grew, since a warp that scales O holds all
//             heads of its dims;
//   P         K-major [head][position] in shared memory, the B operand of O^T += V^T P^T.
// 2100 to 2400 cycles a tile at 128 heads, kernel alone 83 to 90 us for 64 x 4096 where the first form took 117. The
// tensor core is busy for 66 % of them; the rest is the way of the scores (36 instructions of 29 cycles, about half
// the rate of M = 128 ones; 450 until they are seen, 265 to read them, 250 until the next may begin: with all
// 576 dims of the queries in tensor memory it holds one buffer of scores) and loads behind it (without asking the next tile into L2: 4 us more). Measured and not kept: the scores'
// halves as buffers of their own (4 us more), eight softmax warps (4 us more, with both 18), the halves' instructions
// in turn (no difference), queries read from global memory by the warps (1 x 4096: 1 us more).
constexpr int kWideG = 64;
constexpr int kWideStages = 3;
constexpr uint32_t kWidePOff = kWideStages * kPTileBytes;    // P: [64 heads][64 positions] bf16
constexpr uint32_t kWideBarOff = kWidePOff + kWideG * 128;
constexpr int kWideBars = 14 + 3 * kWideStages;
constexpr uint32_t kWideInfoOff = kWideBarOff + kWideBars * 8 + 8;     // (tensor memory slot and abort flag before it)
constexpr uint32_t kWideVoteOff = kWideInfoOff + kWideStages * 16;     // [2][4] ints
constexpr uint32_t kWideMaxOff = kWideVoteOff + 8 * 4;       // factors of O [64], of a finished row [64]
constexpr uint32_t kWideSmemBytes = kWideMaxOff + 2 * kWideG * 4 + 1024;
static_assert(kWidePOff % 1024 == 0 && kWideInfoOff % 16 == 0 && kWideMaxOff % 16 == 0, "alignment");
static_assert(kWideSmemBytes <= 232448, "shared memory budget");
constexpr uint32_t kWideQCols = 18 * 8;      // columns of half a query row in tensor memory

__global__ void __launch_bounds__(kPThreads, 1) mla_paged_wide_kernel(const __grid_constant__ CUtensorMap tm_qa,
                                                                      const __grid_constant__ CUtensorMap tm_qp,
                                                                      const __grid_constant__ CUtensorMap tm_kv,
                                                                      const __grid_constant__ CUtensorMap tm_pe,
                                                                      const PagedArgs a) {
    constexpr int G = kWideG;
    constexpr uint32_t kTmemS = 4 * G, kTmemQ = kTmemS + kPTile, kTmemCols = 512;
    static_assert(kTmemQ + kWideQCols <= kTmemCols, "tensor memory");
    // fp32 accumulate, bf16 x bf16; S: M = 64, N = 64, both K-major; O: V^T MN-major, P K-major, M = 128
    constexpr uint32_t kSIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(kPTile >> 3) << 17) | (4u << 24);
    constexpr uint32_t kOIdesc = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 15) | (static_cast<uint32_t>(G >> 3) << 17) |
                                 (8u << 24);
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base_ptr = smem_raw + (base - smem_u32(smem_raw));
    const uint32_t bars = base + kWideBarOff;
    const uint32_t vote = bars, pfull = bars + 8u, pfree = bars + 8u * 2, efull = bars + 8u * 3, odone = bars + 8u * 4,
                   ofree = bars + 8u * 5, sfull = bars + 8u * 6, sfree = bars + 8u * 7, qfull = bars + 8u * 8, qfree = bars + 8u * 9;
    auto qland = [&](int s) { return bars + 8u * (10 + s); };      // (two rows' queries may be in the ring)
    auto qread = [&](int s) { return bars + 8u * (12 + s); };
    auto kfull = [&](int s) { return bars + 8u * (14 + s); };
    auto kfree = [&](int s, int half) { return bars + 8u * (14 + kWideStages + 2 * s + half); };
    // A row of the batch takes one place of the ring for its queries, then one a tile.
    struct Place {
        int at = 0;
        uint32_t parity = 0;
        __device__ __forceinline__ void next() {
            if (++at == kWideStages) {
                at = 0;
                parity ^= 1u;
            }
        }
    };
    const uint32_t slot = bars + 8u * kWideBars;
    volatile uint32_t* slot_ptr = reinterpret_cast<volatile uint32_t*>(base_ptr + kWideBarOff + 8 * kWideBars);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(slot_ptr + 1);
    volatile TileInfo* info_s = reinterpret_cast<volatile TileInfo*>(base_ptr + kWideInfoOff);
    volatile int* vote_s = reinterpret_cast<volatile int*>(base_ptr + kWideVoteOff);
    float* const w_s = reinterpret_cast<float*>(base_ptr + kWideMaxOff);        // what O is multiplied with when maxima grow
    float* const f_s = w_s + 64;                                             // what a finished row's O is multiplied with

    const int warp = uniform_warp_id(), lane = threadIdx.x & 31;
    const int groups = (a.heads + G - 1) / G;
    const int hg = blockIdx.x % groups, range = blockIdx.x / groups;

    if (threadIdx.x == 0) {
        *abort_flag = 0;
        for (int s = 0; s < kWideStages; ++s) {
            mbar_init(kfull(s), 1);
            mbar_init(kfree(s, 0), 1);
            mbar_init(kfree(s, 1), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(qland(s), 1);
            mbar_init(qread(s), 4);
        }
        mbar_init(qfull, 4);
        mbar_init(qfree, 1);
        mbar_init(sfull, 1);
        mbar_init(sfree, 4);
        mbar_init(vote, 4);
        mbar_init(pfull, 4);
        mbar_init(pfree, 1);
        mbar_init(efull, 4);
        mbar_init(odone, 1);
        mbar_init(ofree, 4);
        fence_mbar_init();
        tma_prefetch_desc(&tm_qa);
        tma_prefetch_desc(&tm_qp);
        tma_prefetch_desc(&tm_kv);
        tma_prefetch_desc(&tm_pe);
    }
    if (warp == 0) {
        tmem_alloc(slot, kTmemCols);
        tmem_relinquish();
    }
    const RangeStart start = find_range<kPThreads>(a, range, reinterpret_cast<volatile int*>(w_s));
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *slot_ptr;
    const int n_tiles = start.count;

    if (warp == 0) {
        // scores
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem_base, 0);
        Place p;
        p.next();
        int seg = 0;
        bool open = false;                                     // the current row's queries have been waited for
        for (int g = 0; g < n_tiles; ++g) {
            if (!open && !mbar_wait_warp(qfull, seg & 1, abort_flag, 76)) break;
            if (!mbar_wait_warp(kfull(p.at), p.parity, abort_flag, 81)) break;
            const bool last = info_s[p.at].flags & 2;
            const uint32_t k0 = __shfl_sync(0xffffffffu, ((base + p.at * kPTileBytes) >> 4) | (1u << 16), 0);
            if (g > 0 && !mbar_wait_warp(sfree, (g - 1) & 1, abort_flag, 80)) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int i = 0; i < 36; ++i) {
                    const uint32_t lanes = i >= 18 ? 16u << 16 : 0u;
                    const uint64_t k = i < 32 ? smem_desc_at(k0 + 64 * (i >> 2) + 2 * (i & 3), 8192)
                                              : smem_desc_at(k0 + (kPLatBytes >> 4) + 2 * (i & 3), 1024);
                    mma_f16_ts(tm + kTmemS + lanes, tm + kTmemQ + lanes + 8u * (i % 18), k, kSIdesc, i % 18 != 0 ? 1u : 0u);
                }
                mma_commit(sfull);
                if (last) mma_commit(qfree);
            }
            __syncwarp();
            open = !last;
            if (last) {
                ++seg;
                p.next();
            }
            p.next();
        }
    } else if (warp == 2) {
        // O += P V
        const uint32_t tm = __shfl_sync(0xffffffffu, tmem_base, 0);
        const uint32_t p0 = ((base + kWidePOff) >> 4) | (1u << 16);
        Place p;
        p.next();
        int seg = 0;
        bool open = false;                                     // the row before is out of tensor memory
        uint32_t acc = 0;
        for (int g = 0; g < n_tiles; ++g) {
            if (!mbar_wait_warp(kfull(p.at), p.parity, abort_flag, 79)) break;
            const uint64_t mask = info_s[p.at].mask;
            const bool last = info_s[p.at].flags & 2;
            const uint32_t v0 = __shfl_sync(0xffffffffu, ((base + p.at * kPTileBytes) >> 4) | (64u << 16), 0);
            if (!open) {
                if (seg > 0 && !mbar_wait_warp(ofree, (seg - 1) & 1, abort_flag, 78)) break;
                acc = 0;
            }
            if (!mbar_wait_warp(pfull, g & 1, abort_flag, 77)) break;
            tc_fence_after();
            if (elect_one()) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if ((mask >> (16 * j) & 0xffffu) != 0) {
#pragma unroll
                        for (int f = 0; f < 4; ++f)
                            mma_f16(tm + f * G, smem_desc_at(v0 + j * 1024u + f * 128u, 8192),
                                    smem_desc_at(p0 + 2u * j, 1024), kOIdesc, acc);
                        acc = 1;
                    }
                    if (j & 1) mma_commit(kfree(p.at, j >> 1));            // its positions are done with
                }
                mma_commit(pfree);
                if (last) mma_commit(odone);
            }
            __syncwarp();
            if (mask != 0) acc = 1;
            open = !last;
            if (last) {
                ++seg;
                p.next();
            }
            p.next();
        }
    } else if (warp == 1) {
        // the whole warp walks the range, one thread issues the loads
        TileWalk w(a, start);
        const int page = 1 << a.page_log, rows = min(page, kPHalf), boxes = kPTile / rows;    // rows of a box, boxes of a tile
        if (n_tiles > 0) w.step(a, 0, n_tiles, rows);
        Place p;
        p.parity = 1;                                          // (the ring begins free)
        int segs = 0;
        for (int g = 0; g < n_tiles; ++g) {
            bool ok = true;
            if (w.flags & 1) {
                const uint32_t dst = base + p.at * kPTileBytes;
                if (!mbar_wait_warp(kfree(p.at, 0), p.parity, abort_flag, 95)) break;
                if (!mbar_wait_warp(kfree(p.at, 1), p.parity, abort_flag, 96)) break;
                if (elect_one()) {
                    mbar_arrive_expect_tx(qland(segs & 1), G * 1152);
                    tma_load_4d(dst, &tm_qa, 0, hg * G, 0, w.b, qland(segs & 1));
                    tma_load_3d(dst + G * 1024, &tm_qp, 0, hg * G, w.b, qland(segs & 1));
                    mbar_arrive(kfull(p.at));                  // (its phases count all uses of the place)
                }
                __syncwarp();
                ++segs;
                p.next();
            }
            const int st = p.at;
            const uint32_t dst = base + st * kPTileBytes;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                if (!(ok = mbar_wait_warp(kfree(st, half), p.parity, abort_flag, 82))) break;
                if (elect_one()) {
                    if (half == 0) {
                        info_s[st].mask = w.mask;
                        info_s[st].flags = w.flags;
                        mbar_arrive_expect_tx(kfull(st), kPTileBytes);     // both halves
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < boxes && i * rows / kPHalf == half) {
                            const int row = (w.tile * kPTile + i * rows) & (page - 1);
                            tma_load_5d(dst + i * rows * 1024, &tm_kv, 0, 0, 0, row >> 3, w.id[i], kfull(st));
                            tma_load_3d(dst + kPLatBytes + i * rows * 128, &tm_pe, 0, row, w.id[i], kfull(st));
                        }
                }
                __syncwarp();
            }
            if (!ok) break;
            p.next();
            w.advance();
            if (g + 1 < n_tiles) {
                // the next tile, whose place in shared memory is still taken, on its way into L2
                w.step(a, g + 1, n_tiles, rows);
                if (elect_one()) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i < boxes && w.id[i] >= 0) {
                            const int row = (w.tile * kPTile + i * rows) & (page - 1);
                            tma_prefetch_5d(&tm_kv, 0, 0, 0, row >> 3, w.id[i]);
                            tma_prefetch_3d(&tm_pe, 0, row, w.id[i]);
                        }
                }
                __syncwarp();
            }
        }
    } else if (warp >= 4 && warp < 8) {
        const int quad = warp & 3;
        const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
        const int p0 = 2 * (lane & 3);                         // this thread's positions: 8 u + p0 and the next
        const int h0 = 16 * quad + (lane >> 2);                // its heads within the group: h0 and h0 + 8
        const float ninf = __int_as_float(0xff800000);
        uint32_t votes = 0;                                    // phases of `vote` taken
        // over the four lanes that hold a head's positions
        auto over_lanes = [&](float v, auto f) {
            v = f(v, __shfl_xor_sync(0xffffffffu, v, 1));
            return f(v, __shfl_xor_sync(0xffffffffu, v, 2));
        };
        auto larger = [](float u, float w) { return fmaxf(u, w); };
        auto plus = [](float u, float w) { return u + w; };
        // lane t: row t % 8 of block t / 8; blocks: heads 0-7 and 8-15 of eight positions, then of the next eight
        const int st_head = 16 * quad + (lane & 15);
        const uint32_t st_line = base + kWidePOff + st_head * 128;
        float l[2], m[2];                                      // denominators (the thread's share), maxima
        int flags4 = 0, seg = 0;
        Place p;
        p.next();
        for (int g = 0; g < n_tiles; ++g) {
            const int st = p.at;
            if (!mbar_wait_warp(kfull(st), p.parity, abort_flag, 84)) break;
            const uint64_t mask = info_s[st].mask;
            const int flags = info_s[st].flags;
            const bool first = flags & 1, last = flags & 2;
            flags4 = (first ? 0 : flags4) | (flags & 12);
            if (first) {
                l[0] = l[1] = 0.f;
                m[0] = m[1] = ninf;
            }
            float x[32], y[32];                                // [8 positions][head, head + 8][2 positions]
            if (!mbar_wait_warp(sfull, g & 1, abort_flag, 85)) break;
            tc_fence_after();
            tmem_ld_16x256b(tmem_base + lane_base + kTmemS, x);
            tmem_ld_16x256b(tmem_base + lane_base + (16u << 16) + kTmemS, y);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(sfree);                 // the next tile's may come
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = (x[i] + y[i]) * a.scale_log2;
            if (mask != ~0ull) {
#pragma unroll
                for (int i = 0; i < 32; ++i)
                    if (!(mask >> (8 * (i >> 2) + p0 + (i & 1)) & 1)) x[i] = ninf;
            }
            float top[2] = {ninf, ninf};
#pragma unroll
            for (int i = 0; i < 32; ++i) top[i >> 1 & 1] = fmaxf(top[i >> 1 & 1], x[i]);
            // (false while a top is -infinity)
            bool over = top[0] > m[0] + 8.f || top[1] > m[1] + 8.f;
            over = __any_sync(0xffffffffu, over);
            if (!first) {
                // does any head's maximum grow: what the others found comes in while new maxima are found
                if (lane == 0) {
                    vote_s[(g & 1) * 4 + quad] = over ? 1 : 0;
                    mbar_arrive(vote);
                }
            }
            float w[2] = {1.f, 1.f};
            if (over) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float mt = over_lanes(top[r], larger);
                    if (mt > m[r] + 8.f) {
                        w[r] = exp2_fast(m[r] - mt);
                        m[r] = mt;
                        l[r] *= w[r];
                    }
                }
            }
            const float mu0 = m[0] == ninf ? 0.f : m[0], mu1 = m[1] == ninf ? 0.f : m[1];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                x[i] = exp2_fast(x[i] - ((i & 2) ? mu1 : mu0));
                l[i >> 1 & 1] += x[i];
            }
            bool grown = false;
            if (!first) {
                if (!mbar_wait_warp(vote, votes++ & 1, abort_flag, 86)) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) grown |= vote_s[(g & 1) * 4 + i] != 0;
                // (all warps vote on this tile, so none reads the factors of one before)
                if (grown && (lane & 3) == 0) {
                    w_s[h0] = w[0];
                    w_s[h0 + 8] = w[1];
                }
            }
            // rows of a step that is multiplied, but not visible: zeros
            const uint32_t step = static_cast<uint32_t>(mask >> (16 * quad)) & 0xffffu;
            if (step != 0 && step != 0xffffu) {
                uint8_t* kt = base_ptr + st * kPTileBytes + quad * 16384;
                for (uint32_t z = ~step & 0xffffu; z; z &= z - 1) {
                    const int row = __ffs(static_cast<int>(z)) - 1;
#pragma unroll
                    for (int i = 0; i < 2; ++i)
                        *reinterpret_cast<uint4*>(kt + (row >> 3) * 8192 + ((lane >> 3) + 4 * i) * 1024 + (row & 7) * 128 +
                                                  (lane & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
                }
            }
            if (g > 0) {
                // O += P V of the tile before has retired: P may be overwritten, O is at rest
                if (!mbar_wait_warp(pfree, (g - 1) & 1, abort_flag, 87)) break;
                tc_fence_after();
            }
            if (grown) {
                __syncwarp();
                if (lane == 0) mbar_arrive(vote);              // the factors are written
                if (!mbar_wait_warp(vote, votes++ & 1, abort_flag, 90)) break;
                rescale<G>(tmem_base + lane_base, w_s);
            }
#pragma unroll
            for (int u = 0; u < 8; u += 2)
                stmatrix_x4(st_line + (((u + (lane >> 4)) ^ (st_head & 7)) << 4), pack_bf16x2(x[4 * u], x[4 * u + 1]),
                            pack_bf16x2(x[4 * u + 2], x[4 * u + 3]), pack_bf16x2(x[4 * u + 4], x[4 * u + 5]),
                            pack_bf16x2(x[4 * u + 6], x[4 * u + 7]));
            fence_proxy_async();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(pfull);
            if (last) {
                // the row before has been written, so its factors may go
                if (seg > 0 && !mbar_wait_warp(ofree, (seg - 1) & 1, abort_flag, 93)) break;
                const int part = part_slot(flags4, range);
                // a head's denominator, and what O is multiplied with (0 for a head of no weight at all, every page
                // out of the pool or every score -infinity: it is zero)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float den = over_lanes(l[r], plus);
                    const int h = h0 + 8 * r;
                    if ((lane & 3) == 0) {
                        if (part >= 0 && hg * G + h < a.heads)
                            *reinterpret_cast<float2*>(a.part_ml + (static_cast<int64_t>(part) * a.heads + hg * G + h) * 2) =
                                make_float2(den == 0.f ? ninf : m[r], den);
                        f_s[h] = den == 0.f ? 0.f : part < 0 ? 1.f / den : 1.f;
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(efull);
                ++seg;
                p.next();
            }
            p.next();
        }
    } else if (warp >= 8) {
        // queries into tensor memory, and finished rows out of it while the next row's first tile is on its way
        const int quad = warp & 3;
        const uint32_t lane_base = static_cast<uint32_t>(quad * 32) << 16;
        int b = start.row, j = start.tile, segs = 0;
        RowTiles t = n_tiles > 0 ? slot_tiles(a, start.slot) : RowTiles{};
        Place p;
        // lanes 0-15: dims 0-287 of 16 heads, lanes 16-31: dims 288-511 and the rope's
        auto load_queries = [&] {
            if (!mbar_wait_warp(qland(segs & 1), segs >> 1 & 1, abort_flag, 97)) return false;
            const uint32_t head = 16 * quad + (lane & 15);
            const uint8_t* line = base_ptr + p.at * kPTileBytes + head * 128;      // of the first block of 64 dims
            const uint32_t first = lane < 16 ? 0 : 36;
            if (segs > 0 && !mbar_wait_warp(qfree, (segs - 1) & 1, abort_flag, 83)) return false;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < 36; c += 4) {
                uint32_t r[16];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t piece = first + c + i;
                    const uint4 v = *reinterpret_cast<const uint4*>(line + (piece >> 3) * (G * 128) + (((piece ^ head) & 7) << 4));
                    r[4 * i] = v.x;
                    r[4 * i + 1] = v.y;
                    r[4 * i + 2] = v.z;
                    r[4 * i + 3] = v.w;
                }
                tmem_st_32x16(tmem_base + lane_base + kTmemQ + 4 * c, r);
            }
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(qread(segs & 1));
                mbar_arrive(qfull);
            }
            if (warp == 8) {                                   // the place is free for a tile
                if (!mbar_wait_warp(qread(segs & 1), segs >> 1 & 1, abort_flag, 98)) return false;
                if (lane == 0) {
                    mbar_arrive(kfree(p.at, 0));
                    mbar_arrive(kfree(p.at, 1));
                }
            }
            p.next();
            ++segs;
            return true;
        };
        bool ok = n_tiles == 0 || load_queries();
        if (hg == 0) clear_empty_rows(a, range);
        for (int seg = 0, left = n_tiles; ok && left > 0; ++seg) {
            const int row = b, tiles = min(t.n - j, left);
            const int part = part_slot((j == 0 ? 4 : 0) | (j + tiles == t.n ? 8 : 0), range);
            left -= tiles;
            j = 0;
            if (left > 0) {
                do t = row_tiles(a, ++b);
                while (t.n == 0);
                for (int i = 0; i < tiles; ++i) p.next();
                if (!(ok = load_queries())) break;
            }
            if (!(ok = mbar_wait_warp(efull, seg & 1, abort_flag, 94))) break;
            if (!(ok = mbar_wait_warp(odone, seg & 1, abort_flag, 88))) break;
            tc_fence_after();
            write_row<G>(a, part, row, hg * G, tmem_base + lane_base, f_s);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(ofree);
        }
    }
    tc_fence_before();
    __syncthreads();
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");     // the join kernel may be set up
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

// Joins the parts of every row that crosses ranges: out = sum_s o_s 2^(m_s - M) / sum_s l_s 2^(m_s - M). A row
// of P parts crosses P - 1 range borders, and blockIdx.x + 1 is a range, so the row has P - 1 blocks: the first S of
// them (the largest power of two, at most 64) take 512 / S dims each. A warp has one head: its lanes cover the
// dims with one, two or four pieces of four, and beyond S = 4 they are S / 4 groups that sum every S / 4-th part.
// So a lane has at most eight pieces of parts to read (P up to 128), all under way at once, whether a row is
// cut once or 127 times; the groups' sums are added in order, so the result does not depend on timing.
// Measured with the kernel before it: 64 x 4096 at 64 heads 69.5 us, at 128 92; 1 x 4096 at 128 heads 17.9, at 16 11.4;
// 1 x 131072 37.4. Blocks of one head and slice that met twice at a barrier took 75.6, 97, 20.5, 10.8 and 40.6; blocks that
// walk several heads 78.8 and 98. The kernel before lets this one's blocks in when a CTA of it has finished: let
// in from the start they fill the first SMs that come free and work there side by side (1 x 131072 40.7 us).
constexpr int kJoinThreads = 128;
constexpr int kJoinMaxParts = 160;
__global__ void __launch_bounds__(kJoinThreads) mla_paged_join_kernel(const PagedArgs a) {
    asm volatile("griddepcontrol.wait;" ::: "memory");        // the parts are complete
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = blockIdx.x + 1, head = blockIdx.y * (kJoinThreads / 32) + warp;
    const int4 rg = a.ranges[r];
    if (rg.x < 0 || rg.y == 0 || head >= a.heads) return;
    const int per = rg.w, t0 = r * per - rg.y, r0 = t0 / per, r1 = (t0 + rg.z - 1) / per, parts = r1 - r0 + 1;
    const int log_s = min(6, 31 - __clz(parts - 1)), slice = r - r0 - 1;
    if (slice >> log_s) return;
    __shared__ float w_all[kJoinThreads / 32][kJoinMaxParts];
    float* const w_s = w_all[warp];
    const float ninf = __int_as_float(0xff800000);
    auto row_of = [&](int s) { return static_cast<int64_t>(s == 0 ? 2 * r0 + 1 : 2 * (r0 + s)) * a.heads + head; };
    // pieces of a lane and lanes of a group; the lane's first piece and its group
    const int log_p = max(0, 2 - log_s), log_w = min(5, 7 - log_s), groups = 32 >> log_w;
    const int c = (slice << (7 - log_s)) + (lane & ((1 << log_w) - 1)), q = lane >> log_w;
    auto part_of = [&](int i, int s0) {                        // load i: piece i % pieces of part s0 + (i / pieces) * groups
        const int s = min(s0 + (i >> log_p) * groups, parts - 1);
        return *(reinterpret_cast<const float4*>(a.part_o + row_of(s) * 512) + c + ((i & ((1 << log_p) - 1)) << 5));
    };
    float4 o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = part_of(i, q);
    float2 ml[kJoinMaxParts / 32];
    float m = ninf;
#pragma unroll
    for (int i = 0; i < kJoinMaxParts / 32; ++i) {
        const int s = lane + 32 * i;
        ml[i] = s < parts ? *reinterpret_cast<const float2*>(a.part_ml + row_of(s) * 2) : make_float2(ninf, 0.f);
        m = fmaxf(m, ml[i].x);
    }
    m = warp_max(m);
    float den = 0.f;
#pragma unroll
    for (int i = 0; i < kJoinMaxParts / 32; ++i) {
        // a part without a maximum has no weight, or (NaN scores alone) NaN
        const float w = ml[i].x == ninf ? (ml[i].y != 0.f ? ml[i].y : 0.f) : exp2f(ml[i].x - m);
        if (lane + 32 * i < parts) w_s[lane + 32 * i] = w;
        den += ml[i].y * w;
    }
    den = warp_sum(den);
    __syncwarp();
    float4 acc[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    const int step = groups << (3 - log_p);                    // parts of a round
    for (int s0 = q; s0 < parts; s0 += step) {
        if (s0 != q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] = part_of(i, s0);
        }
        auto add = [&](float4& to, int i) {
            const int s = s0 + (i >> log_p) * groups;
            if (s < parts) {
                const float w = w_s[s];
                to.x += o[i].x * w; to.y += o[i].y * w; to.z += o[i].z * w; to.w += o[i].w * w;
            }
        };
        if (log_p == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) add(acc[0], i);
        } else if (log_p == 1) {
#pragma unroll
            for (int i = 0; i < 8; ++i) add(acc[i & 1], i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) add(acc[i & 3], i);
        }
    }
    for (int b = 1 << log_w; b < 32; b <<= 1) {
        acc[0].x += __shfl_xor_sync(0xffffffffu, acc[0].x, b);
        acc[0].y += __shfl_xor_sync(0xffffffffu, acc[0].y, b);
        acc[0].z += __shfl_xor_sync(0xffffffffu, acc[0].z, b);
        acc[0].w += __shfl_xor_sync(0xffffffffu, acc[0].w, b);
    }
    if (q != 0) return;
    const float inv = 1.f / den;
    uint2* const to = reinterpret_cast<uint2*>(a.out + (static_cast<int64_t>(rg.x) * a.heads + head) * 512) + c;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (k >> log_p == 0)
            to[32 * k] = den == 0.f ? make_uint2(0u, 0u) : make_uint2(pack_bf16x2(acc[k].x * inv, acc[k].y * inv),
                                                                    pack_bf16x2(acc[k].z * inv, acc[k].w * inv));
}

int sm_count();                                      // rt_gemm.cu
int make_tmap_bf16(CUtensorMap* map, const void* ptr, int rank, const uint64_t* dims, const uint64_t* strides,
                   const uint32_t* box);

int paged_attn_error_take() {
    int v = 0;
    if (cudaMemcpyFromSymbol(&v, g_tc_error, sizeof(int)) != cudaSuccess) {
        cudaGetLastError();
        return -1;
    }
    if (v != 0) {
        const int zero = 0;
        cudaMemcpyToSymbol(g_tc_error, &zero, sizeof(int));
    }
    return v;
}

// Heads of a CTA (the fewest groups, then the narrowest that holds its share: below 64 there is one group), and the
// ranges that the tiles are cut into.
static int paged_group(int64_t heads) {
    const int64_t groups = (heads + kWideG - 1) / kWideG, share = (heads + groups - 1) / groups;
    return share <= 16 ? 16 : share <= 32 ? 32 : 64;
}
static int paged_ranges(int64_t heads) {
    const int64_t groups = (heads + paged_group(heads) - 1) / paged_group(heads);
    const int64_t r = sm_count() / groups;
    return static_cast<int>(r < 1 ? 1 : r < kJoinMaxParts ? r : kJoinMaxParts);
}

static int launch_paged(int group, const CUtensorMap& tm_qa, const CUtensorMap& tm_qp, const CUtensorMap& tm_kv,
                        const CUtensorMap& tm_pe, const PagedArgs& a, cudaStream_t s) {
    auto* kernel = group == 16 ? &mla_paged_kernel<16> : group == 32 ? &mla_paged_kernel<32> : &mla_paged_wide_kernel;
    const int smem = static_cast<int>(group == kWideG ? kWideSmemBytes : kPSmemBytes);
    if (int rc = ensure_dynamic_smem(reinterpret_cast<const void*>(kernel), smem, "rt_mla_paged_decode")) return rc;
    const int groups = (a.heads + group - 1) / group;          // one below groups of 64
    kernel<<<static_cast<unsigned>(a.n_ranges * groups), kPThreads, smem, s>>>(tm_qa, tm_qp, tm_kv, tm_pe, a);
    count_launch();
    return check_launch("mla_paged_kernel");
}

}  // namespace tc
}  // namespace rt

using namespace rt;

extern "C" int64_t rt_mla_paged_decode_workspace_bytes(int64_t heads) {
    if (heads < 1) return 0;
    const int64_t r = tc::paged_ranges(heads);
    return r * 16 + 2 * r * heads * (2 + 512) * 4;
}

extern "C" int rt_mla_paged_decode(const void* q_abs, const void* q_pe, const void* kv, const void* pe,
                                   const int32_t* table, const int32_t* lens, const int32_t* seqs, void* out,
                                   void* workspace, int64_t batch, int64_t heads, int64_t slots, int64_t width,
                                   int64_t pages, int64_t page_size, int64_t qa_batch_stride, int64_t qa_head_stride,
                                   int64_t qp_batch_stride, int64_t qp_head_stride, int64_t kv_page_stride,
                                   int64_t kv_row_stride, int64_t pe_page_stride, int64_t pe_row_stride,
                                   int64_t table_stride, int64_t window, int64_t sinks, float softmax_scale, void* stream) {
    RT_REQUIRE(batch >= 0 && heads > 0 && slots >= 0 && width >= 0 && pages >= 0, RT_ERR_BAD_ARG, "rt_mla_paged_decode: bad shape");
    if (batch == 0) return RT_OK;
    RT_REQUIRE(page_size >= 16 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0, RT_ERR_UNSUPPORTED,
               "rt_mla_paged_decode: page_size must be a power of two, 16 or more");
    RT_REQUIRE(q_abs && q_pe && kv && pe && out && workspace && (table || slots * width == 0) && (lens || slots == 0),
               RT_ERR_BAD_ARG, "rt_mla_paged_decode: null pointer");
    RT_REQUIRE(aligned16(q_abs) && aligned16(q_pe) && aligned16(kv) && aligned16(pe) && aligned16(out) && aligned16(workspace),
               RT_ERR_BAD_ARG, "rt_mla_paged_decode: pointers must be 16-byte aligned");
    const int64_t strides[] = {qa_batch_stride, qa_head_stride, qp_batch_stride, qp_head_stride, kv_page_stride,
                               kv_row_stride, pe_page_stride, pe_row_stride};
    for (int64_t s : strides)
        RT_REQUIRE(s >= 0 && s % 8 == 0 && s < (1ll << 38), RT_ERR_BAD_ARG,
                   "rt_mla_paged_decode: strides must be non-negative multiples of 8 elements");
    // (a tensor map's strides are those of rows that lie apart; one of a dimension of 1 is not looked at)
    RT_REQUIRE(kv_row_stride >= 512 && pe_row_stride >= 64 && (pages <= 1 || (kv_page_stride >= 512 && pe_page_stride >= 64)) &&
                   (heads == 1 || (qa_head_stride >= 512 && qp_head_stride >= 64)) &&
                   (batch == 1 || (qa_batch_stride >= 512 && qp_batch_stride >= 64)),
               RT_ERR_BAD_ARG, "rt_mla_paged_decode: rows must not overlap");
    RT_REQUIRE(window >= 0 && sinks >= 0, RT_ERR_BAD_ARG, "rt_mla_paged_decode: window and sinks must not be negative");
    RT_REQUIRE(pages > 0, RT_ERR_BAD_ARG, "rt_mla_paged_decode: the pool has no page");
    const int64_t tiles = (width * page_size + tc::kPTile - 1) / tc::kPTile;
    RT_REQUIRE(batch <= tc::kPMaxBatch && heads <= 1024 && pages < (1ll << 31) && slots < (1ll << 31) &&
                   width * page_size < (1ll << 31) - 64 && batch * tiles < (1ll << 31) - 65536,
               RT_ERR_UNSUPPORTED, "rt_mla_paged_decode: dimension too large");
    tc::PagedArgs a;
    a.table = table; a.lens = lens; a.seqs = seqs;
    a.out = static_cast<__nv_bfloat16*>(out);
    a.table_stride = table_stride;
    a.batch = static_cast<int>(batch); a.heads = static_cast<int>(heads); a.slots = static_cast<int>(slots);
    a.width = static_cast<int>(width); a.pages = static_cast<int>(pages);
    a.page_log = 0;
    while ((1ll << a.page_log) < page_size) ++a.page_log;
    const int64_t longest = width * page_size;
    a.window = static_cast<int>(window > longest ? 0 : window);
    a.sinks = static_cast<int>(sinks > longest ? longest : sinks);
    a.scale_log2 = softmax_scale * 1.4426950408889634f;
    const int group = tc::paged_group(heads);
    a.n_ranges = tc::paged_ranges(heads);
    // (the host knows no length, but what the table holds at most: fewer tiles than CTAs leave the join less to look
    // at, one tile nothing; 1 x 4096 in a table of 64 pages 11.5 -> 11.0 us at 16 heads)
    if (a.n_ranges > batch * tiles) a.n_ranges = batch * tiles > 0 ? static_cast<int>(batch * tiles) : 1;
    a.ranges = static_cast<int4*>(workspace);
    a.part_ml = reinterpret_cast<float*>(a.ranges + a.n_ranges);
    a.part_o = a.part_ml + 2ll * a.n_ranges * heads * 2;

    // one row of dims as eight blocks of 64: {dims, heads, blocks, rows} and {dims, 8 rows, blocks, groups of
    // rows, pages}
    CUtensorMap tm_qa, tm_qp, tm_kv, tm_pe;
    const uint32_t box_rows = static_cast<uint32_t>(page_size < tc::kPHalf ? page_size : tc::kPHalf);
    const int64_t u = 2;
    {
        const uint64_t dims[] = {64, static_cast<uint64_t>(heads), 8, static_cast<uint64_t>(batch)};
        const uint64_t st[] = {static_cast<uint64_t>(u * qa_head_stride), 128, static_cast<uint64_t>(u * qa_batch_stride)};
        const uint32_t box[] = {64, static_cast<uint32_t>(group), 8, 1};
        if (int rc = tc::make_tmap_bf16(&tm_qa, q_abs, 4, dims, st, box)) return rc;
    }
    {
        const uint64_t dims[] = {64, static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
        const uint64_t st[] = {static_cast<uint64_t>(u * qp_head_stride), static_cast<uint64_t>(u * qp_batch_stride)};
        const uint32_t box[] = {64, static_cast<uint32_t>(group), 1};
        if (int rc = tc::make_tmap_bf16(&tm_qp, q_pe, 3, dims, st, box)) return rc;
    }
    {
        const uint64_t dims[] = {64, 8, 8, static_cast<uint64_t>(page_size / 8), static_cast<uint64_t>(pages)};
        const uint64_t st[] = {static_cast<uint64_t>(u * kv_row_stride), 128, static_cast<uint64_t>(8 * u * kv_row_stride), static_cast<uint64_t>(u * kv_page_stride)};
        const uint32_t box[] = {64, 8, 8, box_rows / 8, 1};
        if (int rc = tc::make_tmap_bf16(&tm_kv, kv, 5, dims, st, box)) return rc;
    }
    {
        const uint64_t dims[] = {64, static_cast<uint64_t>(page_size), static_cast<uint64_t>(pages)};
        const uint64_t st[] = {static_cast<uint64_t>(u * pe_row_stride), static_cast<uint64_t>(u * pe_page_stride)};
        const uint32_t box[] = {64, box_rows, 1};
        if (int rc = tc::make_tmap_bf16(&tm_pe, pe, 3, dims, st, box)) return rc;
    }
    cudaStream_t s = as_stream(stream);
    if (int rc = tc::launch_paged(group, tm_qa, tm_qp, tm_kv, tm_pe, a, s)) return rc;
    if (a.n_ranges == 1) return RT_OK;
    dim3 grid(static_cast<unsigned>(a.n_ranges - 1), static_cast<unsigned>((heads + 3) / 4));
    // launched while the last CTAs of the kernel before still run; it waits for their parts itself
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(tc::kJoinThreads);
    cfg.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, tc::mla_paged_join_kernel, a);
    count_launch();
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(RT_ERR_CUDA, "mla_paged_join_kernel: %s", cudaGetErrorString(e));
    }
    return RT_OK;
}
